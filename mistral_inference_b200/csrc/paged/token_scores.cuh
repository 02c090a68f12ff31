// Scores of tokens: the log-probability of a given token, the entropy of the distribution it was drawn from, and the most likely tokens.
//
//   m = max x, d_i = x_i - m, S = sum of e^d over all but one largest, W = sum d e^d:   ln sum e^x = m + log1p(S), entropy = log1p(S) - W / (1 + S)
// Leaving the largest entry's 1 out of the sum keeps a peaked distribution's small entropy and log-probabilities exact.
// Tokens are ranked by (value, lowest index first) in one 64-bit key; -0 and 0 are equal, NaN ranks first.  An entry of -infinity weighs nothing.  A row that holds
// NaN or +infinity, or nothing but -infinity, has no distribution: its scores are NaN.
//
// Memory: the logits once.  A row is cut into slices of TS_SLICE entries that stay in registers between the maximum, the sums and the ranking; a second kernel
// joins the slices' results.
#pragma once
#include <cfloat>

#include "paged_common.cuh"

namespace mb200 {

constexpr int TS_THREADS = 512, TS_EACH = 16, TS_SLICE = TS_THREADS * TS_EACH, TS_MAX_TOP = 64;
constexpr int TS_JOIN_ROWS = 4;

struct TokenScoresParams {
  const void* logits;  // [T, V], rows ld elements apart
  int64_t ld;
  const int64_t* target;  // [T] or null
  float* sums;            // [T, slices, 3]: maximum, S, W
  unsigned long long* best;  // [T, slices, top]
  float *logprob, *entropy;  // [T] or null
  int64_t* top_ids;          // [T, top]
  float* top_logprobs;
  int T, V, slices, top;
};

__device__ __forceinline__ unsigned long long ts_key(float v, uint32_t i) {
  uint32_t u = __float_as_uint(v + 0.f);
  u = v != v ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (unsigned long long)u << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float ts_value(unsigned long long key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return u == 0xffffffffu ? __int_as_float(0x7fffffff) : __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ uint32_t ts_index(unsigned long long key) { return ~(uint32_t)key; }
__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  return k;
}
// the block's largest key, to every thread
template <int THREADS>
__device__ __forceinline__ unsigned long long block_max_key(unsigned long long k, unsigned long long* sm) {
  k = warp_max_key(k);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = k;
  __syncthreads();
  k = sm[threadIdx.x & (THREADS / 32 - 1)];
  return warp_max_key(k);
}
__device__ __forceinline__ float ts_load(const float* p) { return *p; }
__device__ __forceinline__ float ts_load(const bf16* p) { return __bfloat162float(*p); }

template <typename ST>
__global__ void __launch_bounds__(TS_THREADS) token_scores_slice_kernel(TokenScoresParams p) {
  __shared__ unsigned long long keys[32];
  __shared__ float part[2][32];
  pdl_trigger();
  pdl_wait();
  const int slice = blockIdx.x, t = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const ST* row = static_cast<const ST*>(p.logits) + (int64_t)t * p.ld;
  const int i0 = slice * TS_SLICE, count = min(TS_SLICE, p.V - i0);
  float x[TS_EACH];
#pragma unroll
  for (int j = 0; j < TS_EACH; ++j) {
    const int i = j * TS_THREADS + tid;
    x[j] = i < count ? ts_load(row + i0 + i) : -INFINITY;
  }
  // a place behind the row has a key below every entry's
  auto key_of = [&](int j) { return j * TS_THREADS + tid < count ? ts_key(x[j], i0 + j * TS_THREADS + tid) : 0ull; };
  unsigned long long mine = 0ull;
#pragma unroll
  for (int j = 0; j < TS_EACH; ++j) mine = max(mine, key_of(j));
  unsigned long long top = block_max_key<TS_THREADS>(mine, keys);
  const unsigned long long first = top;
  const float m = ts_value(top);
  float s = 0.f, w = 0.f;
#pragma unroll
  for (int j = 0; j < TS_EACH; ++j) {
    const float d = x[j] - m, e = key_of(j) == first || j * TS_THREADS + tid >= count ? 0.f : __expf(d);
    s += e;
    w = fmaf(e, fmaxf(d, -FLT_MAX), w);
  }
  s = warp_sum(s);
  w = warp_sum(w);
  if (lane == 0) {
    part[0][warp] = s;
    part[1][warp] = w;
  }
  for (int k = 0; k < p.top; ++k) {  // the largest, over and over
    if (tid == 0) p.best[((int64_t)t * p.slices + slice) * p.top + k] = top;
    if (k + 1 == p.top) break;
    if (mine == top && top != 0ull) {  // this thread's next
      mine = 0ull;
#pragma unroll
      for (int j = 0; j < TS_EACH; ++j) {
        const unsigned long long key = key_of(j);
        if (key < top) mine = max(mine, key);
      }
    }
    top = block_max_key<TS_THREADS>(mine, keys);
  }
  __syncthreads();
  if (warp == 0) {
    s = warp_sum(lane < TS_THREADS / 32 ? part[0][lane] : 0.f);
    w = warp_sum(lane < TS_THREADS / 32 ? part[1][lane] : 0.f);
    if (lane == 0) {
      float* out = p.sums + ((int64_t)t * p.slices + slice) * 3;
      out[0] = m;
      out[1] = s;
      out[2] = w;
    }
  }
}

// A warp per row joins its slices.
template <typename ST>
__global__ void __launch_bounds__(TS_JOIN_ROWS * 32) token_scores_join_kernel(TokenScoresParams p) {
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x * TS_JOIN_ROWS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= p.T) return;
  const float* sums = p.sums + (int64_t)t * p.slices * 3;
  float M = -INFINITY;
  bool bad = false;
  for (int i = lane; i < p.slices; i += 32) {
    M = fmaxf(M, sums[i * 3]);
    bad |= sums[i * 3] != sums[i * 3];
  }
  M = warp_max(M);
  bad = __any_sync(0xffffffffu, bad) || !(fabsf(M) <= FLT_MAX);
  int owner = 0x7fffffff;  // of the slices that hold the maximum, the one that leaves its 1 out
  for (int i = lane; i < p.slices; i += 32)
    if (sums[i * 3] == M) owner = min(owner, i);
  owner = __reduce_min_sync(0xffffffffu, owner);
  float S = 0.f, W = 0.f;
  for (int i = lane; i < p.slices; i += 32) {
    const float m = sums[i * 3];
    if (m == -INFINITY) continue;
    const float d = m - M, f = expf(d), s = sums[i * 3 + 1];
    S = fmaf(f, i == owner ? s : 1.f + s, S);
    W = fmaf(f, fmaf(d, 1.f + s, sums[i * 3 + 2]), W);
  }
  S = warp_sum(S);
  W = warp_sum(W);
  const float none = __int_as_float(0x7fffffff), z = log1pf(S);
  if (lane == 0) {
    if (p.entropy) p.entropy[t] = bad ? none : z - W / (1.f + S);
    if (p.logprob && p.target[t] >= 0) {
      const int64_t i = p.target[t];
      p.logprob[t] = bad || i >= p.V ? none : (ts_load(static_cast<const ST*>(p.logits) + (int64_t)t * p.ld + i) - M) - z;
    }
  }
  // the slices' lists are sorted: the largest of their heads, over and over.  Lane i has the lists of slices i, i + 32, ...
  const unsigned long long* best = p.best + (int64_t)t * p.slices * p.top;
  unsigned long long below = ~0ull;  // the last one taken: keys differ
  for (int k = 0; k < p.top; ++k) {
    unsigned long long head = 0ull;
    for (int i = lane; i < p.slices; i += 32)
      for (int j = 0; j < p.top; ++j) {
        const unsigned long long key = best[(int64_t)i * p.top + j];
        if (key < below) {
          head = max(head, key);
          break;
        }
      }
    below = warp_max_key(head);
    if (lane == 0) {
      p.top_ids[(int64_t)t * p.top + k] = ts_index(below);
      p.top_logprobs[(int64_t)t * p.top + k] = bad ? none : (ts_value(below) - M) - z;
    }
  }
}

}  // namespace mb200
