// Keys and values of new tokens into pages of e4m3 numbers.
//
//   scale = 2^e, e the smallest with max |x| <= 448 * 2^e over the page's new tokens of a head, and no smaller than the page's scale where it holds earlier
//   tokens already; code = x / scale to nearest even.  Where the scale grows, the codes of the earlier tokens are rounded again (exact above e4m3's subnormal numbers).
//   Numbers that are not finite are stored as NaN and do not count for the scale.
//
// Memory: 2 bytes read and 1 written per number.  A CTA is one (page, head, kind): its up to 64 rows stay in registers between the maximum and the
// conversion, so each byte moves once, and a page is written by one CTA alone.
#pragma once
#include "paged_common.cuh"

namespace mb200 {

constexpr int PW_THREADS = 128, PW_PASSES = PG_TOKENS * 16 / PW_THREADS;  // 16 threads a row, 8 rows a pass

struct PagedWriteParams {
  const bf16 *k, *v;        // [T, KV * 128], rows ldk / ldv elements apart
  int64_t ldk, ldv;
  uint8_t* kv;
  float* scale;
  const int32_t *slots, *q_start, *seqpos;
  int B, T, KV, n_pages;
};

__global__ void __launch_bounds__(PW_THREADS) page_write_kernel(PagedWriteParams p) {
  __shared__ float part[PW_THREADS / 32];
  pdl_trigger();
  pdl_wait();
  // Item i belongs to the last request b with q_start[b] / 64 + 2 b <= i: n tokens touch at most n / 64 + 2 pages, so its items are enough.
  const int item = blockIdx.x;
  const int b = last_not_above(p.B, item, [&](int j) { return p.q_start[j] / PG_TOKENS + 2 * j; });
  const int t0 = p.q_start[b], n = p.q_start[b + 1] - t0, pos0 = p.seqpos[b];
  const int page_at = pos0 / PG_TOKENS + item - (t0 / PG_TOKENS + 2 * b);
  const int lo = max(pos0, page_at * PG_TOKENS), hi = min(pos0 + n, (page_at + 1) * PG_TOKENS);  // positions
  if (n <= 0 || t0 < 0 || pos0 < 0 || t0 + n > p.T || lo >= hi) return;
  const int slot = p.slots[t0 + lo - pos0];
  if (slot < 0 || slot / PG_TOKENS >= p.n_pages) return;
  const int off = slot % PG_TOKENS, m = min(hi - lo, PG_TOKENS - off), g = blockIdx.y, kind = blockIdx.z;
  const int64_t block = ((int64_t)(slot / PG_TOKENS) * p.KV + g) * 2 + kind;
  const int64_t ld = kind ? p.ldv : p.ldk;
  const bf16* x = (kind ? p.v : p.k) + (int64_t)(t0 + lo - pos0) * ld + g * kHeadDim;
  uint8_t* page = p.kv + block * PG_BYTES;
  const int row = threadIdx.x >> 4, col = threadIdx.x & 15, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  uint4 v[PW_PASSES];
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < PW_PASSES; ++i) {
    v[i] = make_uint4(0, 0, 0, 0);
    if (i * 8 + row < m) v[i] = *reinterpret_cast<const uint4*>(x + (int64_t)(i * 8 + row) * ld + col * 8);
  }
#pragma unroll
  for (int i = 0; i < PW_PASSES; ++i) {
    const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) most = fmaxf(most, fmaxf(finite_abs(bf16lo(u[j])), finite_abs(bf16hi(u[j]))));
  }
  most = warp_max(most);
  if (lane == 0) part[warp] = most;
  __syncthreads();
  int e = e4m3_exponent(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
  if (off > 0) {
    const int old = min(max(exponent_of(p.scale[block]), PG_LOWEST_EXP), 120);
    if (e > old) {  // the earlier tokens' codes at the new scale
      const float shrink = pow2i(max(old - e, -126));
      for (int c = threadIdx.x; c < off * (kHeadDim / 16); c += PW_THREADS) {
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
    __syncthreads();  // the scale has been read
  }
  const float inv = pow2i(-e);
#pragma unroll
  for (int i = 0; i < PW_PASSES; ++i)
    if (i * 8 + row < m) {
      const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      uint32_t c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = to_e4m3x2(scaled(bf16lo(u[j]), inv), scaled(bf16hi(u[j]), inv));
      *reinterpret_cast<uint2*>(page + (off + i * 8 + row) * kHeadDim + col * 8) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
    }
  if (threadIdx.x == 0) p.scale[block] = pow2i(e);
}

}  // namespace mb200
