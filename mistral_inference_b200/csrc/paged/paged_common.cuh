// Pages of 8-bit keys and values, shared by the kernels of libmb200_paged.so.
//
// Pool: kv [pages, KV, 2 (keys, values), 64 tokens, 128] e4m3, scale [pages, KV, 2] fp32; a number is its code times the scale of its (page, head, kind).
// Scales are powers of two: an e4m3 code is a floating-point number, so a scale between two powers would gain no precision inside a page, only its
// range matters; and a page's scale can grow by a power of two without changing any code but the few that fall below e4m3's normal numbers.
#pragma once
#include "../../../include/mistral_b200_paged.h"
#include "../gemm_tcgen05.cuh"

namespace mb200 {

constexpr int PG_TOKENS = 64;                       // tokens of a page
constexpr int PG_BYTES = PG_TOKENS * kHeadDim;      // one head's keys (or values) of a page: 8 KB, contiguous
constexpr int PG_LOWEST_EXP = -100;                 // the scale of a page of zeros is 2^-100

__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127
// the smallest e with amax <= 448 * 2^e (448 = 1.75 * 2^8 is e4m3's largest number); amax finite
__device__ __forceinline__ int e4m3_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  return max((int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0), PG_LOWEST_EXP);
}
__device__ __forceinline__ int exponent_of(float scale) { return (int)(__float_as_uint(scale) >> 23) - 127; }
__device__ __forceinline__ float finite_abs(float x) {  // |x|, 0 where x is no number or infinite
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}
// two numbers to two codes (lo in the low byte), to nearest even; |x| <= 448 or NaN
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t codes) {  // exact: every e4m3 number is an fp16 number
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes));
  float2 f;
  asm("{.reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.f32.f16 %0, l;\n cvt.f32.f16 %1, h;\n}" : "=f"(f.x), "=f"(f.y) : "r"(h));
  return f;
}
// x times a power of two; not a number where x is infinite (e4m3 has no infinity, and the largest code would pass for a number)
__device__ __forceinline__ float scaled(float x, float inv) { return fmaf(x, inv, x - x); }

__device__ __forceinline__ float warp_max_f32(float v) {  // (NaN does not count)
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// two fp32 numbers in one instruction
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Allows launches of Kernel in clusters of up to 16 on the current device
template <auto Kernel>
inline cudaError_t allow_wide_clusters() {
  static std::atomic<uint64_t> done{0};
  const int dev = device_info::current();
  const uint64_t bit = dev >= 0 && dev < device_info::MAX_DEVICES ? (uint64_t)1 << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

constexpr uint32_t PG_SPINS = 1u << 22;  // polls of a wait before it gives up (seconds)
// false: the wait ran out, or another thread's has
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
  for (uint32_t i = 0; i < PG_SPINS; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63u) == 63u && *gave_up) return false;
  }
  *gave_up = 1;
  return false;
}

enum { PG_TOO_LONG = 32 };  // status of attention: a request has more tokens than the call was told
// Rows first .. n - 1 of a request's results (its first row at `out`, H heads a row), which no tile of queries is there for: no numbers, for `heads` heads.  By a CTA.
__device__ __forceinline__ void no_numbers(bf16* out, int first, int n, int H, int heads) {
  for (int64_t i = (int64_t)first * heads * kHeadDim + threadIdx.x; i < (int64_t)n * heads * kHeadDim; i += blockDim.x) {
    const int64_t t = i / (heads * kHeadDim), c = i % (heads * kHeadDim);
    out[t * H * kHeadDim + c] = __ushort_as_bfloat16((unsigned short)0x7fff);
  }
}
// largest i in [0, n) with start[i] <= x, start ascending, start[0] <= x
template <typename F>
__device__ __forceinline__ int last_not_above(int n, int x, F start) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start(mid) <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// the same by a whole warp, 32 places looked at in one trip to memory
template <typename F>
__device__ __forceinline__ int warp_last_not_above(int n, int x, F start) {
  int lo = 0, len = n;  // the answer is in [lo, lo + len)
  while (len > 1) {
    const int step = (len + 31) / 32, at = lo + (int)(threadIdx.x & 31) * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < lo + len && start(at < lo + len ? at : lo) <= x);
    const int last = below ? 31 - __clz(below) : 0;
    len = min(step, lo + len - (lo + last * step));
    lo += last * step;
  }
  return lo;
}

}  // namespace mb200
