// Rows of 16- or 32-bit numbers to rows of 8-bit ones, by themselves or behind a root-mean-square norm.
//
//   quantise  c = e4m3(x 2^-e), e the smallest with max |x| <= 448 2^e over a block of 128 (at least -100)
//   norm      h = x + add, rounded to the stream's type; y = h rsqrt(mean h^2 + eps) w; quantise(y)
//
// Memory bounds both: an entry is read once and its code written once.  A warp's step is 512 entries of a row, 16 next to one another a lane: a block is 8 lanes (three shuffles give
// its largest magnitude), a lane's codes are one 16-byte store, and the step's four scales are one word of the scales' tile.  All of a warp's steps are requested before the first is
// worked on.  y is not rounded to 16 bits on its way.  Instructions count: with one number at a time and a division to find a warp's place, 440 a step of the norm and 220 of the
// other, issue slots were half to two thirds full and 8000 x 5120 took 65 us.
#pragma once
#include "rows8_common.cuh"

namespace mb200 {

constexpr int R8_CHUNK = 4 * R8_BLOCK;  // entries of a warp's step
constexpr int RQ_WARPS = 8;

// 16 entries of a row as they lie in memory, 32 or 64 bytes
template <typename ST>
struct Entries {
  static constexpr int WORDS = 4 * sizeof(ST), VECTORS = WORDS / 4, PER = 16 / sizeof(ST) /* entries of 16 bytes */;
  uint32_t w[WORDS];
  // word i of what begins `bytes` bytes (even) into x, i + bytes / 4 + 1 <= N - 1 or bytes a multiple of four
  template <int SKIP, int N>
  static __device__ __forceinline__ uint32_t shifted(const uint32_t (&x)[N], int i, int bytes) {
    if constexpr (sizeof(ST) == 4) return x[i + SKIP];
    else return __funnelshift_r(x[i + SKIP], x[i + SKIP + 1 < N ? i + SKIP + 1 : N - 1], (bytes & 2) * 8);
  }
  template <int N, int M>
  static __device__ __forceinline__ void shift(uint32_t (&to)[M], const uint32_t (&x)[N], int first, int bytes) {  // M words from word `first` on
    switch (bytes >> 2) {
#define R8_SHIFT(SKIP)          \
  case SKIP:                    \
    _Pragma("unroll") for (int i = 0; i < M; ++i) to[i] = shifted<SKIP>(x, first + i, bytes); \
    break;
      R8_SHIFT(0)
      R8_SHIFT(1)
      R8_SHIFT(2)
      R8_SHIFT(3)
#undef R8_SHIFT
    }
  }
  // Of `row`, K entries in all, from k on; zeros behind the end.  ALIGNED: the row starts on 16 bytes.  Else what lies between two multiples of 16 bytes is loaded as a whole where the
  // row has all of it, and shifted.
  template <bool ALIGNED>
  __device__ __forceinline__ void load(const ST* row, int k, int K) {
    if (ALIGNED && k + 16 <= K) {
#pragma unroll
      for (int i = 0; i < VECTORS; ++i) {
        const uint4 u = reinterpret_cast<const uint4*>(row + k)[i];
        w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
      }
      return;
    }
    if constexpr (!ALIGNED) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(row + k), base = at & ~(uintptr_t)15;
      if (base >= reinterpret_cast<uintptr_t>(row) && base + (VECTORS + 1) * 16 <= reinterpret_cast<uintptr_t>(row + K)) {
        uint32_t x[WORDS + 4];
#pragma unroll
        for (int i = 0; i <= VECTORS; ++i) {
          const uint4 u = reinterpret_cast<const uint4*>(base)[i];
          x[4 * i] = u.x, x[4 * i + 1] = u.y, x[4 * i + 2] = u.z, x[4 * i + 3] = u.w;
        }
        shift(w, x, 0, (int)(at & 15));
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const bool there = k + i < K;
      if constexpr (sizeof(ST) == 2) {
        const uint32_t x = there ? (uint32_t) reinterpret_cast<const uint16_t*>(row)[k + i] : 0u;
        w[i / 2] = i % 2 == 0 ? x : w[i / 2] | x << 16;
      } else {
        w[i] = there ? reinterpret_cast<const uint32_t*>(row)[k + i] : 0u;
      }
    }
  }
  // The same places of `row`, by a whole warp whose lanes have 16 entries next to one another.  Not aligned: a lane takes the first entries of the next one and writes from its first multiple of 16
  // bytes on; what lies before that in lane 0 and behind it in lane 31, or at the row's end, goes entry by entry.
  template <bool ALIGNED>
  __device__ __forceinline__ void store(ST* row, int k, int K) const {
    if constexpr (ALIGNED) {
      if (k + 16 <= K) {
#pragma unroll
        for (int i = 0; i < VECTORS; ++i) reinterpret_cast<uint4*>(row + k)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k + i < K) put(row + k + i, w, i);
      }
    } else {
      const int lane = threadIdx.x & 31, skip = (int)(-reinterpret_cast<intptr_t>(row + k) & 15);  // bytes to the next multiple of 16 (the same in all lanes)
      uint32_t x[WORDS + 4];
#pragma unroll
      for (int i = 0; i < WORDS; ++i) x[i] = w[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[WORDS + i] = __shfl_down_sync(0xffffffffu, w[i], 1);
      const int limit = min(lane < 31 ? 16 + PER : 16, K - k), first = skip / (int)sizeof(ST);  // entries that this lane may write; its first one in a vector
      if (lane == 0) {
#pragma unroll
        for (int i = 0; i < PER - 1; ++i)
          if (i < first && i < limit) put(row + k + i, w, i);
      }
#pragma unroll
      for (int v = 0; v < VECTORS; ++v) {
        uint32_t y[4];
        shift(y, x, 4 * v, skip);
        const int from = first + v * PER;
        if (from + PER <= limit) {
          *reinterpret_cast<uint4*>(row + k + from) = make_uint4(y[0], y[1], y[2], y[3]);
        } else {
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (from + i < limit) put(row + k + from + i, y, i);
        }
      }
    }
  }
  template <int N>
  static __device__ __forceinline__ void put(ST* to, const uint32_t (&x)[N], int i) {
    if constexpr (sizeof(ST) == 2) *reinterpret_cast<uint16_t*>(to) = (uint16_t)(x[i / 2] >> (i % 2 * 16));
    else *reinterpret_cast<uint32_t*>(to) = x[i];
  }
  // entries 2 i and 2 i + 1
  __device__ __forceinline__ uint64_t two(int i) const {
    if constexpr (sizeof(ST) == 2) return pair(bf16lo(w[i]), bf16hi(w[i]));
    else return pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  }
  __device__ __forceinline__ void add(const Entries& a) {  // rounded to the type
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if constexpr (sizeof(ST) == 2) asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(w[i]) : "r"(a.w[i]));
      else w[i] = __float_as_uint(__uint_as_float(w[i]) + __uint_as_float(a.w[i]));
    }
  }
};
// The codes and scales of a warp's 512 entries of row r, quad q
__device__ __forceinline__ void r8_store_chunk(uint8_t* codes, uint8_t* scales, int r, int R, int q, int quads, int width, const uint64_t (&v)[8]) {
  const int lane = threadIdx.x & 31, k = q * R8_CHUNK + lane * 16;
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 x = unpair(v[i]);
    most = r8_larger(most, x.x, x.y);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) most = r8_larger(most, __shfl_xor_sync(0xffffffffu, most, o), 0.f);
  const uint32_t amax = __float_as_uint(most);
  if (k < width) *reinterpret_cast<uint4*>(codes + (int64_t)r * width + k) = r8_codes16(v, amax);
  uint32_t word = (k < width ? r8_byte(amax) : 127u) << (lane & 24);  // a block's byte is its lanes' eighth
  word |= __shfl_xor_sync(0xffffffffu, word, 8);
  word |= __shfl_xor_sync(0xffffffffu, word, 16);
  if (lane == 0) *reinterpret_cast<uint32_t*>(scales + r8_scale_at(r, q, quads)) = word;
  if (r == R - 1)  // the places of the last tile that have no row
    for (int i = R + lane; i < ((R + 127) & ~127); i += 32) *reinterpret_cast<uint32_t*>(scales + r8_scale_at(i, q, quads)) = R8_ONES;
}

struct QuantiseParams {
  const void* x;
  uint8_t *codes, *scales;
  int64_t ld;
  int T, K, width, quads;
};
// A warp a row and STEPS steps of it
template <typename ST, bool ALIGNED, int STEPS>
__global__ void __launch_bounds__(32 * RQ_WARPS) rows8_quantise_kernel(const QuantiseParams p) {
  pdl_trigger();
  const int r = (int)(blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)), q0 = (int)blockIdx.y * STEPS, lane = threadIdx.x & 31;
  pdl_wait();
  if (r >= p.T) return;
  const ST* row = reinterpret_cast<const ST*>(p.x) + r * p.ld;
  Entries<ST> x[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) x[i].template load<ALIGNED>(row, (q0 + i) * R8_CHUNK + lane * 16, p.K);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    if (q0 + i >= p.quads) break;
    uint64_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = x[i].two(j);
    r8_store_chunk(p.codes, p.scales, r, p.T, q0 + i, p.quads, p.width, v);
  }
}

struct NormParams {
  const void *x, *add, *w;
  void* stream;  // x + add; null without `add`
  uint8_t *codes, *scales;
  int64_t ld, ld_add;
  int T, K, width, quads;
  float eps;
};
constexpr int RN8_MAX_STEPS = 4;                          // a warp's steps of a row, which stay in registers
constexpr int RN8_MAX_K = 32 * RN8_MAX_STEPS * R8_CHUNK;  // entries of a row
// A CTA a row: its entries are read once and stay in registers behind the sum of their squares.  ALIGNED: rows start on 16 bytes; W_ALIGNED: the weights do.
template <typename ST, bool ALIGNED, bool W_ALIGNED, bool ADD, int STEPS, int THREADS>
__global__ void __launch_bounds__(THREADS) rows8_norm_kernel(const NormParams p) {
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, r = (int)blockIdx.x;
  __shared__ float part[32];
  auto place = [&](int i) { return (i * warps + warp) * R8_CHUNK + lane * 16; };
  pdl_wait();
  Entries<ST> h[STEPS];
  {
    Entries<ST> add[ADD ? STEPS : 1];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) h[i].template load<ALIGNED>(reinterpret_cast<const ST*>(p.x) + r * p.ld, place(i), p.K);
    if constexpr (ADD) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) add[i].template load<ALIGNED>(reinterpret_cast<const ST*>(p.add) + r * p.ld_add, place(i), p.K);
    }
    if constexpr (ADD) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        h[i].add(add[i]);
        h[i].template store<ALIGNED>(reinterpret_cast<ST*>(p.stream) + (int64_t)r * p.K, place(i), p.K);
      }
    }
  }
  uint64_t sums = pair(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) sums = fma_pair(h[i].two(j), h[i].two(j), sums);
  const float2 two = unpair(sums);
  float sum = warp_sum(two.x + two.y);
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  sum = warp_sum(lane < warps ? part[lane] : 0.f);
  const float inverse = ref_rsqrt(sum / (float)p.K + p.eps);
  const uint64_t scale = pair(inverse, inverse);
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int q = i * warps + warp;
    if (q >= p.quads) break;
    Entries<ST> w;
    w.template load<W_ALIGNED>(reinterpret_cast<const ST*>(p.w), place(i), p.K);
    uint64_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = mul_pair(mul_pair(h[i].two(j), scale), w.two(j));
    r8_store_chunk(p.codes, p.scales, r, p.T, q, p.quads, p.width, v);
  }
}

// ---- host ----
template <typename ST, bool ALIGNED>
int launch_rows8_quantise(const QuantiseParams& p, cudaStream_t st) {
  // a warp takes four steps where that leaves warps enough (28672 x 4096 56 us; one step a warp, with a division for its place, 69)
  const int warps = p.T < RQ_WARPS ? p.T : RQ_WARPS, steps = (int64_t)p.T * p.quads >= 32 * 1024 ? 4 : 1;
  const dim3 grid((unsigned)((p.T + warps - 1) / warps), (unsigned)((p.quads + steps - 1) / steps)), block(32 * (unsigned)warps);
  if (steps == 4) MB_CHECK_CUDA(launch_pdl(rows8_quantise_kernel<ST, ALIGNED, 4>, grid, block, 0, st, p));
  else MB_CHECK_CUDA(launch_pdl(rows8_quantise_kernel<ST, ALIGNED, 1>, grid, block, 0, st, p));
  return MB200_OK;
}
template <typename ST>
int launch_rows8_quantise(const QuantiseParams& p, cudaStream_t st) {
  return (uintptr_t)p.x % 16 == 0 && (p.T == 1 || p.ld * sizeof(ST) % 16 == 0) ? launch_rows8_quantise<ST, true>(p, st) : launch_rows8_quantise<ST, false>(p, st);
}
template <typename ST, bool ALIGNED, bool W_ALIGNED, bool ADD>
int launch_rows8_norm(const NormParams& p, cudaStream_t st) {
  // As many warps as a CTA has, a step each, while a row is no longer than that.  What counts is how many rows are on their way: with more steps a warp, or the weights requested ahead of the sum, fewer
  // CTAs share an SM (16000 x 5000 bf16, us, with addition and without: a step a warp 91, 56; two 96, 64; four 120, 92; weights ahead 106, 66).
  const int steps = p.quads <= 32 ? 1 : RN8_MAX_STEPS, warps = (p.quads + steps - 1) / steps;
  const dim3 grid((unsigned)p.T), block(32 * (unsigned)warps);
  if (steps == 1) MB_CHECK_CUDA((launch_pdl(rows8_norm_kernel<ST, ALIGNED, W_ALIGNED, ADD, 1, 1024>, grid, block, 0, st, p)));
  else if (warps <= 16) MB_CHECK_CUDA((launch_pdl(rows8_norm_kernel<ST, ALIGNED, W_ALIGNED, ADD, RN8_MAX_STEPS, 512>, grid, block, 0, st, p)));
  else MB_CHECK_CUDA((launch_pdl(rows8_norm_kernel<ST, ALIGNED, W_ALIGNED, ADD, RN8_MAX_STEPS, 1024>, grid, block, 0, st, p)));
  return MB200_OK;
}
template <typename ST, bool ADD>
int launch_rows8_norm(const NormParams& p, cudaStream_t st) {
  auto apart = [&](const void* at, int64_t ld) { return (uintptr_t)at % 16 == 0 && (p.T == 1 || ld * sizeof(ST) % 16 == 0); };
  const bool aligned = apart(p.x, p.ld) && (!ADD || (apart(p.add, p.ld_add) && apart(p.stream, p.K))), w_aligned = (uintptr_t)p.w % 16 == 0;
  if (aligned && w_aligned) return launch_rows8_norm<ST, true, true, ADD>(p, st);
  return w_aligned ? launch_rows8_norm<ST, false, true, ADD>(p, st) : launch_rows8_norm<ST, false, false, ADD>(p, st);
}
template <typename ST>
int launch_rows8_norm(const NormParams& p, cudaStream_t st) {
  return p.add == nullptr ? launch_rows8_norm<ST, false>(p, st) : launch_rows8_norm<ST, true>(p, st);
}

}  // namespace mb200
