// Rows of 16- or 32-bit numbers to rows of 8-bit ones, by themselves or behind a root-mean-square norm.
//
//   quantise  c = e4m3(x 2^-e), e the smallest with max |x| <= 448 2^e over a block of 128 (at least -100)
//   norm      h = x + add, rounded to the stream's type; y = h rsqrt(mean h^2 + eps) w; quantise(y)
//
// Memory bounds both: an entry is read once and its code written once.  A warp takes 512 entries of a row, 16 next to one another a lane: a block is 8 lanes (three shuffles give
// its largest magnitude), a lane's codes are one 16-byte store, and the warp's four scales are one word of the scales' tile.  y is not rounded to 16 bits on its way.
#pragma once
#include "rows8_common.cuh"

namespace mb200 {

constexpr int R8_CHUNK = 4 * R8_BLOCK;  // entries of a warp's step
constexpr int RQ_WARPS = 8;

// 16 entries of a row, K of them in all from `row` on; zeros behind the end.  ALIGNED: the row starts on 16 bytes.
template <typename ST, bool ALIGNED>
__device__ __forceinline__ void r8_load16(const ST* row, int64_t k, int64_t K, float (&v)[16]) {
  constexpr int PER = 16 / sizeof(ST);  // entries of 16 bytes
  if (ALIGNED && k + 16 <= K) {
    const uint4* src = reinterpret_cast<const uint4*>(row + k);
#pragma unroll
    for (int i = 0; i < 16 / PER; ++i) {
      const uint4 u = src[i];
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(ST) == 2) v[8 * i + 2 * j] = bf16lo(w[j]), v[8 * i + 2 * j + 1] = bf16hi(w[j]);
        else v[4 * i + j] = __uint_as_float(w[j]);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = k + i < K ? (float)row[k + i] : 0.f;
}
// The codes and scales of a warp's 512 entries of row r, quad q
__device__ __forceinline__ void r8_store_chunk(uint8_t* codes, uint8_t* scales, int64_t r, int64_t R, int q, int quads, int64_t width, const float (&v)[16]) {
  const int lane = threadIdx.x & 31;
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) amax = max(amax, r8_bits(v[i]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const uint32_t byte = r8_byte(amax);
  const int64_t k = (int64_t)q * R8_CHUNK + lane * 16;
  if (k < width) *reinterpret_cast<uint4*>(codes + r * width + k) = r8_codes16(v, amax, r8_inverse(byte));
  uint32_t word = k < width ? byte << (lane & 24) : 127u << (lane & 24);  // a block's byte is its lanes' eighth
  word |= __shfl_xor_sync(0xffffffffu, word, 8);
  word |= __shfl_xor_sync(0xffffffffu, word, 16);
  if (lane == 0) *reinterpret_cast<uint32_t*>(scales + r8_scale_at(r, q, quads)) = word;
  if (r == R - 1)  // the places of the last tile that have no row
    for (int64_t i = R + lane; i < ((R + 127) & ~(int64_t)127); i += 32) *reinterpret_cast<uint32_t*>(scales + r8_scale_at(i, q, quads)) = R8_ONES;
}

struct QuantiseParams {
  const void* x;
  uint8_t *codes, *scales;
  int64_t T, K, ld, width;
  int quads;
};
template <typename ST, bool ALIGNED>
__global__ void __launch_bounds__(32 * RQ_WARPS) rows8_quantise_kernel(const QuantiseParams p) {
  pdl_trigger();
  pdl_wait();
  const int64_t at = (int64_t)blockIdx.x * RQ_WARPS + (threadIdx.x >> 5);
  if (at >= p.T * p.quads) return;
  const int64_t r = at / p.quads;
  const int q = (int)(at % p.quads);
  float v[16];
  r8_load16<ST, ALIGNED>(reinterpret_cast<const ST*>(p.x) + r * p.ld, (int64_t)q * R8_CHUNK + (threadIdx.x & 31) * 16, p.K, v);
  r8_store_chunk(p.codes, p.scales, r, p.T, q, p.quads, p.width, v);
}

struct NormParams {
  const void *x, *add, *w;
  void* stream;  // x + add; null without `add`
  uint8_t *codes, *scales;
  int64_t T, K, ld, ld_add, width;
  int quads;
  float eps;
};
constexpr int RN8_MAX_CHUNKS = 4;                                     // a warp's steps of a row, which stay in registers
constexpr int64_t RN8_MAX_K = (int64_t)32 * RN8_MAX_CHUNKS * R8_CHUNK;  // entries of a row
// A CTA a row: its entries are read once and stay in registers behind the sum of their squares.
template <typename ST, bool ALIGNED, bool ADD, int CHUNKS>
__global__ void __launch_bounds__(1024) rows8_norm_kernel(const NormParams p) {
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int64_t r = blockIdx.x;
  __shared__ float part[32];
  pdl_wait();
  float v[CHUNKS][16];
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int64_t k = ((int64_t)c * warps + warp) * R8_CHUNK + lane * 16;
    r8_load16<ST, ALIGNED>(reinterpret_cast<const ST*>(p.x) + r * p.ld, k, p.K, v[c]);
    if constexpr (ADD) {
      float a[16];
      r8_load16<ST, ALIGNED>(reinterpret_cast<const ST*>(p.add) + r * p.ld_add, k, p.K, a);
      ST* out = reinterpret_cast<ST*>(p.stream) + r * p.K;
#pragma unroll
      for (int i = 0; i < 16; ++i) v[c][i] = sizeof(ST) == 2 ? round_bf16(v[c][i] + a[i]) : v[c][i] + a[i];
      if (ALIGNED && k + 16 <= p.K) {
        uint4* to = reinterpret_cast<uint4*>(out + k);
        if constexpr (sizeof(ST) == 2) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            to[i] = make_uint4(pack_bf16x2(v[c][8 * i], v[c][8 * i + 1]), pack_bf16x2(v[c][8 * i + 2], v[c][8 * i + 3]), pack_bf16x2(v[c][8 * i + 4], v[c][8 * i + 5]),
                               pack_bf16x2(v[c][8 * i + 6], v[c][8 * i + 7]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) to[i] = make_uint4(__float_as_uint(v[c][4 * i]), __float_as_uint(v[c][4 * i + 1]), __float_as_uint(v[c][4 * i + 2]), __float_as_uint(v[c][4 * i + 3]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k + i < p.K) out[k + i] = (ST)v[c][i];
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sum = fmaf(v[c][i], v[c][i], sum);
  }
  sum = warp_sum(sum);
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  sum = warp_sum(lane < warps ? part[lane] : 0.f);
  const float scale = ref_rsqrt(sum / (float)p.K + p.eps);
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int q = c * warps + warp;
    if (q >= p.quads) continue;
    float w[16];
    r8_load16<ST, ALIGNED>(reinterpret_cast<const ST*>(p.w), (int64_t)q * R8_CHUNK + lane * 16, p.K, w);
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] *= v[c][i] * scale;
    r8_store_chunk(p.codes, p.scales, r, p.T, q, p.quads, p.width, w);
  }
}

// ---- host ----
template <typename ST>
int launch_rows8_quantise(const QuantiseParams& p, cudaStream_t st) {
  const int64_t ctas = (p.T * p.quads + RQ_WARPS - 1) / RQ_WARPS;
  const bool aligned = (uintptr_t)p.x % 16 == 0 && (p.T == 1 || p.ld * sizeof(ST) % 16 == 0);
  if (aligned) MB_CHECK_CUDA(launch_pdl(rows8_quantise_kernel<ST, true>, dim3((unsigned)ctas), dim3(32 * RQ_WARPS), 0, st, p));
  else MB_CHECK_CUDA(launch_pdl(rows8_quantise_kernel<ST, false>, dim3((unsigned)ctas), dim3(32 * RQ_WARPS), 0, st, p));
  return MB200_OK;
}
template <typename ST, bool ALIGNED, bool ADD>
int launch_rows8_norm(const NormParams& p, cudaStream_t st) {
  const int chunks = (p.quads + 31) / 32 == 1 ? 1 : (p.quads + 31) / 32 == 2 ? 2 : RN8_MAX_CHUNKS, warps = (p.quads + chunks - 1) / chunks;
  const dim3 grid((unsigned)p.T), block(32 * (unsigned)warps);
  if (chunks == 1) MB_CHECK_CUDA(launch_pdl(rows8_norm_kernel<ST, ALIGNED, ADD, 1>, grid, block, 0, st, p));
  else if (chunks == 2) MB_CHECK_CUDA(launch_pdl(rows8_norm_kernel<ST, ALIGNED, ADD, 2>, grid, block, 0, st, p));
  else MB_CHECK_CUDA(launch_pdl(rows8_norm_kernel<ST, ALIGNED, ADD, RN8_MAX_CHUNKS>, grid, block, 0, st, p));
  return MB200_OK;
}
template <typename ST>
int launch_rows8_norm(const NormParams& p, cudaStream_t st) {
  auto apart = [&](const void* at, int64_t ld) { return (uintptr_t)at % 16 == 0 && (p.T == 1 || ld * sizeof(ST) % 16 == 0); };
  const bool aligned = apart(p.x, p.ld) && (uintptr_t)p.w % 16 == 0 && (p.add == nullptr || (apart(p.add, p.ld_add) && apart(p.stream, p.K)));
  if (p.add == nullptr) return aligned ? launch_rows8_norm<ST, true, false>(p, st) : launch_rows8_norm<ST, false, false>(p, st);
  return aligned ? launch_rows8_norm<ST, true, true>(p, st) : launch_rows8_norm<ST, false, true>(p, st);
}

}  // namespace mb200
