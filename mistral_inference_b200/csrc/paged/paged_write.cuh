// Keys and values of new tokens into pages of e4m3 numbers.
//
//   scale = 2^e, e the smallest with max |x| <= 448 * 2^e over the page's new tokens of a head, and no smaller than the page's scale where it holds earlier
//   tokens already; code = x / scale to nearest even.  Where the scale grows, the codes of the earlier tokens are rounded again (exact above e4m3's subnormal numbers).
//   Numbers that are not finite are stored as NaN and do not count for the scale.
//
// Memory: 2 bytes read and 1 written per number.  A page of a head and kind is written by one group of threads alone: a CTA, whose up to 64 rows stay in
// registers between the maximum and the conversion so that each byte moves once, or, for few tokens a request, a warp.
// Eight CTAs an SM, 128 KB of rows on their way: 34.7 us for 32000 tokens of 8 heads, 5.7 TB/s; 39.6 us at the five that the compiler's own choice of registers
// leaves; eight spill 60 bytes a thread, ten more: 44 us.  11.5 us for three prompts of 6900 tokens together, 6.6 of them for the bytes; the rest is the launch and a chain of loads
// (request, place, slot, scale) ahead of the only rows that a CTA has.
#pragma once
#include "paged_common.cuh"

namespace mb200 {

constexpr int PW_THREADS = 128, PW_WARPS = PW_THREADS / 32;
// Up to this many tokens a request on average, a warp writes a page: a CTA for each would have most of its threads without a row, and most of the items of a
// decode step have no page at all (one token each: 3.0 us and 4.2 by CTAs for 32 requests, 33 us and 134 for 2000; 18 each: 5.5 and 5.5 for 32, 12.4 and 27.7 for
// 300).  Beyond it a warp would read its rows twice (45 each: 8.8 us, 5.7 by CTAs for 32; a prompt of 8000: 17.0 and 9.1).
constexpr int PW_FEW = 32;

struct PagedWriteParams {
  const bf16 *k, *v;        // [T, KV * 128], rows ldk / ldv elements apart
  int64_t ldk, ldv;
  uint8_t* kv;
  float* scale;
  const int32_t *slots, *q_start, *seqpos;
  int B, T, KV, n_pages;
};

// GROUP threads (a warp, or the CTA) write one page; 16 threads a row.  A CTA holds a page's rows at once, a warp 16 of them at a time (read again where there
// are more: they are a request's last tokens or its first, and hit L1).
template <int GROUP>
__global__ void __launch_bounds__(PW_THREADS, 8) page_write_kernel(PagedWriteParams p) {
  constexpr int ROWS = GROUP / 16, PASSES = 8, HOLD = ROWS * PASSES;
  static_assert(GROUP == 32 || HOLD == PG_TOKENS, "a CTA holds a page");
  __shared__ float part[PW_WARPS];
  pdl_trigger();
  pdl_wait();
  const int in = threadIdx.x % GROUP, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int across = GROUP == 32 ? (2 * p.KV + PW_WARPS - 1) / PW_WARPS : 2 * p.KV, item = blockIdx.x / across, at = blockIdx.x % across;
  const int gk = GROUP == 32 ? at * PW_WARPS + warp : at, g = gk >> 1, kind = gk & 1;
  if (g >= p.KV) return;
  // Item i belongs to the last request b with q_start[b] / 64 + 2 b <= i: n tokens touch at most n / 64 + 2 pages, so its items are enough.
  const int b = warp_last_not_above(p.B, item, [&](int j) { return p.q_start[j] / PG_TOKENS + 2 * j; });
  const int t0 = p.q_start[b], n = p.q_start[b + 1] - t0, pos0 = p.seqpos[b];
  const int page_at = pos0 / PG_TOKENS + item - (t0 / PG_TOKENS + 2 * b);
  const int lo = max(pos0, page_at * PG_TOKENS), hi = min(pos0 + n, (page_at + 1) * PG_TOKENS);  // positions
  if (n <= 0 || t0 < 0 || pos0 < 0 || t0 + n > p.T || lo >= hi) return;
  const int slot = p.slots[t0 + lo - pos0];
  const int64_t ld = kind ? p.ldv : p.ldk;
  const bf16* x = (kind ? p.v : p.k) + (int64_t)(t0 + lo - pos0) * ld + g * kHeadDim;
  const int row = in >> 4, col = in & 15;

  uint4 v[PASSES];
  auto load = [&](int first, int rows) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = first + i * ROWS + row;
      v[i] = make_uint4(0, 0, 0, 0);
      if (r < rows) v[i] = *reinterpret_cast<const uint4*>(x + (int64_t)r * ld + col * 8);
    }
  };
  auto largest = [&](float most) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) most = fmaxf(most, fmaxf(finite_abs(bf16lo(u[j])), finite_abs(bf16hi(u[j]))));
    }
    return most;
  };
  load(0, hi - lo);  // on its way together with the slot (hi - lo rows are there whatever the slot says)
  if (slot < 0 || slot / PG_TOKENS >= p.n_pages) return;
  const int off = slot % PG_TOKENS, m = hi - lo;
  if (m > PG_TOKENS - off) return;  // (slots that are not this request's)
  const int64_t block = ((int64_t)(slot / PG_TOKENS) * p.KV + g) * 2 + kind;
  uint8_t* page = p.kv + block * PG_BYTES;
  const float held = off > 0 ? p.scale[block] : 0.f;

  float most = largest(0.f);
  if constexpr (GROUP == 32) {
    for (int first = HOLD; first < m; first += HOLD) {
      load(first, m);
      most = largest(most);
    }
    most = warp_max(most);
  } else {
    most = warp_max(most);
    if (lane == 0) part[warp] = most;
    __syncthreads();  // (and the scale has been read)
    most = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  }
  int e = e4m3_exponent(most);
  if (off > 0) {
    const int old = min(max(exponent_of(held), PG_LOWEST_EXP), 120);
    if (e > old) {  // the earlier tokens' codes at the new scale
      const float shrink = pow2i(max(old - e, -126));
      for (int c = in; c < off * (kHeadDim / 16); c += GROUP) {
        uint4 w = *reinterpret_cast<uint4*>(page + c * 16);
        uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 a = from_e4m3x2(u[j] & 0xffff), z = from_e4m3x2(u[j] >> 16);
          u[j] = to_e4m3x2(a.x * shrink, a.y * shrink) | to_e4m3x2(z.x * shrink, z.y * shrink) << 16;
        }
        *reinterpret_cast<uint4*>(page + c * 16) = w;
      }
    }
    e = max(e, old);
  }
  if (GROUP == 32) __syncwarp();  // the scale has been read
  const float inv = pow2i(-e);
  for (int first = 0; first < m; first += HOLD) {
    if (GROUP == 32 && m > HOLD) load(first, m);
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = first + i * ROWS + row;
      if (r < m) {
        const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        uint32_t c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = to_e4m3x2(scaled(bf16lo(u[j]), inv), scaled(bf16hi(u[j]), inv));
        *reinterpret_cast<uint2*>(page + (off + r) * kHeadDim + col * 8) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
      }
    }
  }
  if (in == 0) p.scale[block] = pow2i(e);
}

}  // namespace mb200
