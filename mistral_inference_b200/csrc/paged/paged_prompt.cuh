// Portions of prompts over pages: the pages that a portion sees go into 16-bit rings, and the prompt kernel (attn_prompt_tcgen05.cuh) attends over those.
//
// From some tokens on the tensor pipe bounds attention, not the pages' bytes: the 128 x 128 tiles of the prompt kernel use it four times as well as the few query columns of
// paged_attn.cuh, and a page is converted once instead of once a tile of queries.  A number is code * scale, a power of two: exact in bf16.  Converting is memory-bound: 1 byte
// read and 2 written a number, and read once more by the attention.  Three portions of ~650 tokens behind ~2000, 32 heads over 8: 133 us, 597 TFLOP/s, of which converting takes 11.6
// (4.4 TB/s).  The rest is 336 CTAs of the prompt kernel on 148 SMs, a third round of which is a quarter full.
#pragma once
#include "../attn_prompt_tcgen05.cuh"
#include "paged_common.cuh"

namespace mb200 {

constexpr int PR_THREADS = 256;

struct PagedRingParams {
  const uint8_t* kv;
  const float* scale;
  const int32_t *table, *rows, *q_start, *seqpos;
  bf16 *ring_k, *ring_v;  // [B, W, KV, 128], position p in row p % W
  int32_t* status;
  bf16* out;
  int T, R, P, n_pages, H, KV, window, W, longest;
};

// CTA = (page of a request, key/value head, request): 64 rows of keys and of values
__global__ void __launch_bounds__(PR_THREADS) paged_ring_kernel(PagedRingParams p) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.z, g = blockIdx.y, t0 = p.q_start[b], n = p.q_start[b + 1] - t0, past = p.seqpos[b], row = p.rows[b];
  if (t0 < 0 || n <= 0 || n > p.T - t0 || past < 0) return;
  const int lo = p.window > 0 ? max(0, past + 1 - p.window) : 0, end = past + n;
  const int page_at = lo / PG_TOKENS + blockIdx.x, from = max(lo, page_at * PG_TOKENS), to = min(end, (page_at + 1) * PG_TOKENS);
  const bool fits = end - lo <= p.W && n <= p.longest;
  if (!fits && blockIdx.x == 0) {
    if (g == 0 && threadIdx.x == 0 && p.status) atomicOr(p.status, PG_TOO_LONG);
    no_numbers(p.out + (int64_t)t0 * p.H * kHeadDim + g * (p.H / p.KV) * kHeadDim, (p.longest + FA_BM - 1) / FA_BM * FA_BM, n, p.H, p.H / p.KV);
  }
  if (from >= to) return;
  int page = row >= 0 && row < p.R && page_at < p.P ? p.table[(int64_t)row * p.P + page_at] : -1;
  const bool is = page >= 0 && page < p.n_pages && fits;  // (else nothing is read out of bounds, and what is attended to is no number)
  if (!is) page = 0;
  const int64_t block = ((int64_t)page * p.KV + g) * 2;
  const float scale[2] = {is ? p.scale[block] : __int_as_float(0x7fffffff), is ? p.scale[block + 1] : __int_as_float(0x7fffffff)};
  const uint8_t* src = p.kv + block * PG_BYTES;
  constexpr int STEPS = 2 * PG_BYTES / 16 / PR_THREADS;  // 16 codes a thread and step, all fetched before the first is used
  uint4 v[STEPS];
  auto pos_of = [&](int at) { return page_at * PG_TOKENS + at % (PG_BYTES / 16) / (kHeadDim / 16); };
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int at = i * PR_THREADS + threadIdx.x, pos = pos_of(at);
    v[i] = make_uint4(0, 0, 0, 0);
    if (pos >= from && pos < to) v[i] = *reinterpret_cast<const uint4*>(src + (int64_t)at * 16);
  }
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int at = i * PR_THREADS + threadIdx.x, kind = at / (PG_BYTES / 16), col = at % (kHeadDim / 16) * 16, pos = pos_of(at);
    if (pos < from || pos >= to) continue;
    const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
    uint32_t out[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = from_e4m3x2(u[j] & 0xffff), z = from_e4m3x2(u[j] >> 16);
      out[2 * j] = pack_bf16x2(a.x * scale[kind], a.y * scale[kind]);
      out[2 * j + 1] = pack_bf16x2(z.x * scale[kind], z.y * scale[kind]);
    }
    bf16* dst = (kind ? p.ring_v : p.ring_k) + (((int64_t)b * p.W + pos % p.W) * p.KV + g) * kHeadDim + col;
    *reinterpret_cast<uint4*>(dst) = make_uint4(out[0], out[1], out[2], out[3]);
    *reinterpret_cast<uint4*>(dst + 8) = make_uint4(out[4], out[5], out[6], out[7]);
  }
}

// Rows of a request's rings: what its longest portion sees
inline int64_t paged_ring_rows(int64_t longest, int64_t most, int64_t window) {
  const int64_t rows = window > 0 && window + longest < most ? window + longest : most;
  return (rows + 127) / 128 * 128;
}

inline int make_query_map(CUtensorMap* map, const void* q, int64_t T, int64_t cols, int64_t ld) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (enc == nullptr) return fail(MB200_E_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)T};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, 128};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MB200_E_CUDA, "cuTensorMapEncodeTiled (queries) failed (%d)", (int)r);
  return MB200_OK;
}

// p: the whole call's; requests b0 .. b0 + B - 1 of it through rings of W rows at `scratch`
inline int launch_paged_prompt(PagedRingParams p, const void* q, int64_t ldq, bf16* out, int64_t b0, int64_t B, int64_t longest, int H, float scale_log2, void* scratch, cudaStream_t st) {
  p.out = out;
  p.H = H;
  p.longest = (int)longest;
  p.rows += b0;
  p.q_start += b0;
  p.seqpos += b0;
  p.ring_k = (bf16*)scratch;
  p.ring_v = p.ring_k + B * p.W * p.KV * kHeadDim;
  const dim3 grid((unsigned)(p.W / PG_TOKENS + 1), (unsigned)p.KV, (unsigned)B);
  MB_CHECK_CUDA(launch_pdl(paged_ring_kernel, grid, dim3(PR_THREADS), 0, st, p));
  CUtensorMap mq, rk, rv;
  int rc = make_query_map(&mq, q, p.T, (int64_t)H * kHeadDim, ldq);
  if (rc == 0) rc = make_tensor_map_rows(&rk, p.ring_k, p.W, (int64_t)p.KV * kHeadDim, B);
  if (rc == 0) rc = make_tensor_map_rows(&rv, p.ring_v, p.W, (int64_t)p.KV * kHeadDim, B);
  if (rc) return rc;
  FaParams f;
  f.q_start = p.q_start;
  f.seqpos = p.seqpos;
  f.slots = nullptr;
  f.bias = nullptr;
  f.out = out;
  f.B = (int)B;
  f.W = p.W;
  f.window = p.window > 0 ? p.window : 0x3fffffff;
  f.H = H;
  f.KV = p.KV;
  f.own = 0;
  f.n_tab = 0;
  f.scale_log2 = scale_log2;
  f.T = p.T;
  // Two heads a CTA share every key and value tile, unless single ones all run at once.  (257 tokens of 32 heads behind 2000: 53 us, 58 by two; 3 x 700: 163 and 115.)
  const bool two = (H / p.KV) % 2 == 0 && H * B * ceil_div(longest, FA_BM) > device_info::sm_count();
  const dim3 fgrid((unsigned)(H / (two ? 2 : 1)), (unsigned)ceil_div(longest, FA_BM), (unsigned)B);
  if (two) {
    MB_CHECK_CUDA((device_info::allow_shared<attn_prompt_tcgen05_kernel<2, false>>(FA_SMEM_BASE)));
    attn_prompt_tcgen05_kernel<2, false><<<fgrid, FA_THREADS, FA_SMEM_BASE, st>>>(mq, rk, rv, rk, rv, f);
  } else {
    MB_CHECK_CUDA((device_info::allow_shared<attn_prompt_tcgen05_kernel<1, false>>(FA_SMEM_BASE)));
    attn_prompt_tcgen05_kernel<1, false><<<fgrid, FA_THREADS, FA_SMEM_BASE, st>>>(mq, rk, rv, rk, rv, f);
  }
  MB_CHECK_LAUNCH("attn_prompt_tcgen05_kernel (pages)");
  return MB200_OK;
}

}  // namespace mb200
