// Scores of tokens: the log-probability of a given token, the entropy of the distribution it was drawn from, and the most likely tokens.
//
//   m = max x, d_i = x_i - m, S = sum of e^d over all but one largest, W = sum d e^d:   ln sum e^x = m + log1p(S), entropy = log1p(S) - W / (1 + S)
// Leaving the largest entry's 1 out of the sum keeps a peaked distribution's small entropy and log-probabilities exact.
// Tokens are ranked by (value, lowest index first) in one 64-bit key; -0 and 0 are equal, NaN ranks first.  An entry of -infinity weighs nothing.  A row that holds
// NaN or +infinity, or nothing but -infinity, has no distribution: its scores are NaN.
//
// Memory bounds it: the logits once, at 23 bytes a clock and SM.  A CTA takes segments of rows, up to 64 KB, into shared memory and walks over them twice: maximum; then sums relative to
// the segment's maximum, in pairs (3.5 instructions an entry).  Every 16-byte piece is fetched, read and replaced by the next segment's by the same thread, so copies are in flight from
// the middle of one segment to the beginning of the next and need no barrier.  The best are not sorted: a warp's r-th largest thread maximum, the least of them
// over the warps, is a value that at least r * warps >= top entries reach, and few more; the threads that have some pick them out, and they are ranked by counting.  Two block
// barriers a segment.  A warp a row joins the segments, in a second kernel or, where few rows leave room, behind a cluster's barrier.
// 1000 x 131072 fp32, 8 alternatives: 104 us, 5.0 TB/s (20 of them 118; bf16 79, whose entries take more of the bound by instructions).  Before: the largest taken off over and
// over 1540 us; entries in registers, a CTA for 8192 of them 141; longer walks with a list kept up to date 205 (a barrier a slice, and more code than the instruction
// cache holds); whole segments by one bulk copy each, fetched behind the second barrier 107.  32 rows, 20 alternatives: 14.4 us (15.7 where L2 does not hold them), 2.6 for the bytes, the rest two launches and
// two segments' latency; 1 x 32000: 7.6.
#pragma once
#include <cfloat>

#include "paged_common.cuh"

namespace mb200 {

constexpr int TS_THREADS = 256, TS_WARPS = TS_THREADS / 32, TS_MAX_TOP = 64;
constexpr int TS_CTAS = 3;              // of an SM
constexpr int TS_BYTES = 64 * 1024;     // of a segment, at most
constexpr int TS_PIECES = TS_BYTES / 16 / TS_THREADS;  // of 16 bytes, of a thread
constexpr int TS_ROOM = 512;            // entries that are ranked by counting
constexpr int TS_JOIN_SEGMENTS = 32;    // lists that a warp joins from shared memory, one a lane

struct TokenScoresParams {
  const void* logits;  // [T, V], rows ld elements apart
  int64_t ld;
  const int64_t* target;  // [T] or null
  float* sums;            // [T, segments, 3]: maximum, S, W
  unsigned long long* best;  // [T, segments, top], largest first
  float *logprob, *entropy;  // [T] or null
  int64_t* top_ids;          // [T, top]
  float* top_logprobs;
  int T, V, segments, length, top;  // length: entries of a segment, a multiple of 16 bytes a thread
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
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return (unsigned long long)hi << 32 | lo;
}
// the block's largest key, to every thread
__device__ __forceinline__ unsigned long long block_max_key(unsigned long long k, unsigned long long* sm) {
  k = warp_max_key(k);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = k;
  __syncthreads();
  return warp_max_key(sm[threadIdx.x & (TS_WARPS - 1)]);
}
__device__ __forceinline__ float max_nan(float x, float y) {  // NaN if one is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
template <typename ST> __device__ __forceinline__ ST ts_lowest();
template <> __device__ __forceinline__ float ts_lowest<float>() { return -INFINITY; }
template <> __device__ __forceinline__ bf16 ts_lowest<bf16>() { return __ushort_as_bfloat16((unsigned short)0xff80u); }
__device__ __forceinline__ float ts_load(const float* p) { return *p; }
__device__ __forceinline__ float ts_load(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void ts_load16(const float* p, float* x) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ __forceinline__ void ts_load16(const bf16* p, float* x) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = bf16lo(u[i]), x[2 * i + 1] = bf16hi(u[i]);
}

__device__ __forceinline__ void ts_load16(const float* p, uint64_t* x) {
  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p);
  x[0] = v.x, x[1] = v.y;
}
__device__ __forceinline__ void ts_load16(const bf16* p, uint64_t* x) {
  float y[8];
  ts_load16(p, y);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = pair(y[2 * i], y[2 * i + 1]);
}

// A warp joins the segments of row t.  lists: [segments][top] of shared memory, up to TS_JOIN_SEGMENTS
template <typename ST>
__device__ __forceinline__ void token_scores_join(const TokenScoresParams& p, int t, unsigned long long* lists) {
  const int lane = threadIdx.x & 31;
  const float* sums = p.sums + (int64_t)t * p.segments * 3;
  const unsigned long long* best = p.best + (int64_t)t * p.segments * p.top;
  const bool staged = p.segments <= TS_JOIN_SEGMENTS;
  if (staged) {
#pragma unroll 8
    for (int i = lane; i < p.segments * p.top; i += 32) lists[i] = best[i];
  }
  const int64_t target = p.logprob ? p.target[t] : -1;
  const float x = target >= 0 && target < p.V ? ts_load(static_cast<const ST*>(p.logits) + (int64_t)t * p.ld + target) : 0.f;
  float M = -INFINITY;
  bool bad = false;
  for (int i = lane; i < p.segments; i += 32) {
    M = fmaxf(M, sums[i * 3]);
    bad |= sums[i * 3 + 2] != sums[i * 3 + 2];
  }
  M = warp_max_f32(M);
  bad = __any_sync(0xffffffffu, bad) || !(fabsf(M) <= FLT_MAX);
  int owner = 0x7fffffff;  // of the segments that hold the maximum, the one that leaves its 1 out
  for (int i = lane; i < p.segments; i += 32)
    if (sums[i * 3] == M) owner = min(owner, i);
  owner = __reduce_min_sync(0xffffffffu, owner);
  float S = 0.f, W = 0.f;
  for (int i = lane; i < p.segments; i += 32) {
    const float m = sums[i * 3];
    if (m == -INFINITY) continue;
    const float d = m - M, f = expf(d), s = sums[i * 3 + 1];
    if (f == 0.f) continue;
    S = fmaf(f, i == owner ? s : 1.f + s, S);
    W = fmaf(f, fmaf(d, 1.f + s, sums[i * 3 + 2]), W);
  }
  S = warp_sum(S);
  W = warp_sum(W);
  const float none = __int_as_float(0x7fffffff), z = log1pf(S);
  if (lane == 0) {
    if (p.entropy) p.entropy[t] = bad ? none : z - W / (1.f + S);
    if (p.logprob) p.logprob[t] = target < 0 ? 0.f : bad || target >= p.V ? none : (x - M) - z;
  }
  auto put = [&](int k, unsigned long long key) {
    p.top_ids[(int64_t)t * p.top + k] = ts_index(key);
    p.top_logprobs[(int64_t)t * p.top + k] = bad ? none : (ts_value(key) - M) - z;
  };
  if (staged) {  // lane i walks down the list of segment i: the largest of the heads, over and over
    __syncwarp();
    int at = 0;
    unsigned long long head = lane < p.segments && p.top > 0 ? lists[lane * p.top] : 0ull, mine = 0ull;
    for (int k = 0; k < p.top; ++k) {
      const unsigned long long top = warp_max_key(head);
      if (head == top) {
        ++at;
        head = lane < p.segments && at < p.top ? lists[lane * p.top + at] : 0ull;
      }
      if ((k & 31) == lane) mine = top;
      if ((k & 31) == 31 || k + 1 == p.top)  // 32 results at a time
        if ((k & ~31) + lane <= k) put((k & ~31) + lane, mine);
    }
    return;
  }
  unsigned long long below = ~0ull;  // lane i has the lists of segments i, i + 32, ...; keys differ
  for (int k = 0; k < p.top; ++k) {
    unsigned long long head = 0ull;
    for (int i = lane; i < p.segments; i += 32)
      for (int j = 0; j < p.top; ++j) {
        const unsigned long long key = best[(int64_t)i * p.top + j];
        if (key < below) {
          head = max(head, key);
          break;
        }
      }
    below = warp_max_key(head);
    if (lane == 0) put(k, below);
  }
}

// BYTES: of a copy: 16, or 4 where rows begin on 4-byte boundaries only, or 0 (rows of 16-bit numbers that begin on odd ones are loaded entry by entry).  Entries go to the
// same places in all three, so that a row's results do not depend on where it lies.  251 rows of 50257 fp32: 33.7 us loaded entry by entry, 28.0 by 4-byte copies.
// JOINS: the segments of a row are a cluster, a CTA each, whose first CTA joins them: one launch, for so few rows that all segments run at once.
template <typename ST, int BYTES, bool JOINS>
__global__ void __launch_bounds__(TS_THREADS, TS_CTAS) token_scores_segment_kernel(TokenScoresParams p) {
  constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
  constexpr bool COPIED = BYTES > 0;
  constexpr int VEC = 16 / (int)sizeof(ST), ROW = TS_THREADS * VEC;  // entries of a piece, of all threads' pieces
  extern __shared__ __align__(128) uint8_t ts_data[];
  ST* const data = reinterpret_cast<ST*>(ts_data);
  __shared__ unsigned long long list[TS_ROOM], keys[TS_WARPS];
  __shared__ float part[4][TS_WARPS];  // maximum, what enough entries reach; sums
  __shared__ int part_n[TS_WARPS], n_list[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, top = p.top, items = p.T * p.segments;
  if (tid == 0) n_list[0] = n_list[1] = 0;
  pdl_wait();
  auto row_of = [&](int t, int i0) { return static_cast<const ST*>(p.logits) + (int64_t)t * p.ld + i0; };
  auto count_of = [&](int t, int i0) { return t < p.T ? min(p.length, p.V - i0) : 0; };
  const int step_t = gridDim.x / p.segments, step_i = gridDim.x % p.segments * p.length, wrap = p.segments * p.length;
  int t_here = blockIdx.x / p.segments, i_here = blockIdx.x % p.segments * p.length;  // row and first entry of the segment
  ST* const mine = data + tid * VEC;
  const uint32_t mine_at = smem_u32(mine);
  auto whole_of = [&](int count) { return (count - tid * VEC - VEC + ROW) / ROW; };  // pieces that are all there
  // piece j of a segment whose first one is at `src`; `after`: a value that was read from the place before
  auto fetch = [&](const ST* src, int j, uint64_t after) {
    if constexpr (BYTES == 16) {
      asm volatile("{.reg .b64 x; mov.b64 x, %2; cp.async.cg.shared.global [%0], [%1], 16;}" ::"r"(mine_at + j * ROW * (int)sizeof(ST)), "l"(src + j * ROW), "l"(after) : "memory");
    } else {
#pragma unroll
      for (int c = 0; c < 16; c += 4)
        asm volatile("{.reg .b64 x; mov.b64 x, %2; cp.async.ca.shared.global [%0], [%1], 4;}" ::"r"(mine_at + j * ROW * (int)sizeof(ST) + c),
                     "l"(reinterpret_cast<const uint8_t*>(src + j * ROW) + c), "l"(after) : "memory");
    }
  };
  if (COPIED)
    for (int j = 0; j < whole_of(count_of(t_here, i_here)); ++j) fetch(row_of(t_here, i_here) + tid * VEC, j, 0);
  for (int item = blockIdx.x, turn = 0; item < items; item += gridDim.x, turn ^= 1) {
    const int t = t_here, i0 = i_here;
    const int count = count_of(t, i0), t_next = t + step_t + (i0 + step_i >= wrap), i_next = i0 + step_i >= wrap ? i0 + step_i - wrap : i0 + step_i;
    const int whole_next = COPIED ? whole_of(count_of(t_next, i_next)) : 0;
    t_here = t_next;
    i_here = i_next;
    const ST* row = row_of(t, i0);
    const ST* next = row_of(t_next, i_next) + tid * VEC;
    const int pieces = (count + ROW - 1) / ROW;  // of this thread: at (j * TS_THREADS + tid) * VEC, j < pieces
    // A dependent grid may come once this CTA's work is nearly done: its CTAs, waiting, would take the place of this grid's own.  (107 us; from the start on 137.)
    if (item + (int)gridDim.x >= items) pdl_trigger();
    if (COPIED) asm volatile("cp.async.wait_all;" ::: "memory");
    // what no copy brings: entries behind the last whole piece, -infinity behind the row
    if (!COPIED || count < pieces * ROW)
#pragma unroll 4
      for (int j = 0; j < pieces; ++j)
        if (!COPIED || j * ROW + tid * VEC + VEC > count)
#pragma unroll
          for (int c = 0; c < VEC; ++c) mine[j * ROW + c] = j * ROW + tid * VEC + c < count ? row[j * ROW + tid * VEC + c] : ts_lowest<ST>();
    float piece_most[TS_PIECES], most = -INFINITY;  // (NaN does not count)
#pragma unroll
    for (int j = 0; j < TS_PIECES; ++j) {
      piece_most[j] = -INFINITY;
      if (j < pieces) {
        float x[VEC];
        ts_load16(mine + j * ROW, x);
#pragma unroll
        for (int c = 0; c < VEC; ++c) piece_most[j] = fmaxf(piece_most[j], x[c]);
      }
      most = fmaxf(most, piece_most[j]);
    }
    float v = most, reach = warp_max_f32(v);
    const float warp_most = reach;
    const int warps = max(1, min(TS_WARPS, (count + 32 * VEC - 1) / (32 * VEC)));  // those that have entries
    for (int k = warps; k < top; k += warps) {  // the warp's next largest thread maximum
      if (lane == __ffs(__ballot_sync(0xffffffffu, v == reach)) - 1) v = -INFINITY;
      reach = warp_max_f32(v);
    }
    if (lane == 0) {
      part[0][warp] = warp_most;
      part[1][warp] = warp < warps ? reach : INFINITY;
    }
    __syncthreads();
    const float M = warp_max_f32(part[0][lane & (TS_WARPS - 1)]);
    reach = -warp_max_f32(-part[1][lane & (TS_WARPS - 1)]);
    // The entries that reach the limit go into the list, and those that equal the maximum out of the data (and are counted): the sums below are those of the others
    auto take = [&](float x, int i) {
      const int place = atomicAdd(&n_list[turn], 1);  // (in any order: they are ranked)
      if (place < TS_ROOM) list[place] = ts_key(x, i0 + i);
    };
    const float limit = top > 0 ? fmaxf(reach, -FLT_MAX) : M;
    int n = 0;
    if (most >= limit && most > -INFINITY) {
      uint32_t some = 0;  // pieces that have some (one copy of the code below for all: unrolled, the kernel outgrew the instruction cache)
#pragma unroll
      for (int j = 0; j < TS_PIECES; ++j) some |= piece_most[j] >= limit ? 1u << j : 0u;
#pragma unroll 1
      for (; some; some &= some - 1) {
        const int i = (__ffs(some) - 1) * ROW + tid * VEC;
        float x[VEC];
        ts_load16(data + i, x);
#pragma unroll
        for (int c = 0; c < VEC; ++c)
          if (x[c] >= limit) {
            if (top > 0) take(x[c], i + c);
            if (x[c] == M) {
              ++n;
              data[i + c] = ts_lowest<ST>();
            }
          }
      }
    }
    // t = log2(e) x - R, R = log2(e) M rounded: e^(x - M) = 2^t * 2^(R - log2(e) M), the second factor put right below
    // R is off by half a step at most: 64 up to |M| = 2^30 (masks of -1e9 among them), where 2^64 times the sums is still far inside fp32.  Beyond, the difference comes first.
    // (M is a segment's maximum: that of one whose entries are all masked by a finite number is the mask's.)
    const bool none = M == -INFINITY, huge = fabsf(M) > 1073741824.f && !none;
    const float R = huge || none ? 0.f : M * LOG2E;
    float s = 0.f, w = 0.f;
    int j = 0;
    if (!huge) {
      uint64_t s2[2] = {0, 0}, w2[2] = {0, 0};
      const uint64_t scale2 = pair(LOG2E, LOG2E), R2 = pair(-R, -R);
#pragma unroll 4
      for (; j < pieces; ++j) {
        uint64_t x[VEC / 2];
        ts_load16(mine + j * ROW, x);
#pragma unroll
        for (int c = 0; c < VEC / 2; ++c) {
          const float2 t = unpair(fma_pair(x[c], scale2, R2));
          // masked entries weigh 0, not 0 * infinity; what is no number stays so
          const float t0 = max_nan(t.x, -1000.f), t1 = max_nan(t.y, -1000.f);
          const uint64_t e2 = pair(exp2_ftz(t0), exp2_ftz(t1));
          s2[c & 1] = add_pair(s2[c & 1], e2);
          w2[c & 1] = fma_pair(e2, pair(t0, t1), w2[c & 1]);
        }
        if (j < whole_next) fetch(next, j, x[0]);
      }
      const float2 s0 = unpair(add_pair(s2[0], s2[1])), w0 = unpair(add_pair(w2[0], w2[1]));
      s = s0.x + s0.y;
      w = w0.x + w0.y;
    } else {
#pragma unroll 1
      for (int i = 0; i < pieces * VEC; ++i) {
        const float t = max_nan((ts_load(mine + i / VEC * ROW + i % VEC) - M) * LOG2E, -1000.f), e = exp2_ftz(t);
        s += e;
        w = fmaf(e, t, w);
      }
    }
    for (; j < whole_next; ++j) fetch(next, j, 0);
    if (top > 0 && reach == -INFINITY)  // a warp has fewer entries above -infinity than it should: masked ones, lowest index first, as many as could be short
      for (int i = tid; i < min(2 * top, count); i += TS_THREADS)
        if (ts_load(row + i) == -INFINITY) take(-INFINITY, i);
    s = warp_sum(s);
    w = warp_sum(w);
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) {
      part[2][warp] = s;
      part[3][warp] = w;
      part_n[warp] = n;
    }
    const bool odd = __syncthreads_or(w != w);
    if (tid == 0) n_list[turn ^ 1] = 0;
    if (warp == 0) {
      const bool one = lane < TS_WARPS;
      s = warp_sum(one ? part[2][lane] : 0.f);
      w = warp_sum(one ? part[3][lane] : 0.f);
      n = __reduce_add_sync(0xffffffffu, one ? part_n[lane] : 0) - 1;
      if (lane == 0) {
        const float off = huge || none ? 0.f : fmaf(M, LOG2E, -R), f = exp2_ftz(-off);
        float* out = p.sums + (int64_t)item * 3;
        out[0] = M;
        out[1] = fmaf(f, s, (float)n);
        out[2] = LN2 * f * fmaf(-off, s, w);
      }
    }
    if (top == 0) continue;
    unsigned long long* best = p.best + (int64_t)item * top;
    const int have = n_list[turn];
    if (have <= TS_ROOM && !odd) {
      // 2^g threads an entry.  (32 alternatives of 1500 x 32768: 56.6 us; a warp an entry up to 64 of them and one thread beyond 60.8)
      const int g = have <= 32 ? 3 : have <= 64 ? 2 : have <= 128 ? 1 : 0;
      for (int first = 0; first < have; first += TS_THREADS >> g) {
        const int i = first + (tid >> g);
        const unsigned long long key = i < have ? list[i] : ~0ull;
        int rank = 0;
#pragma unroll 4
        for (int k = tid & ((1 << g) - 1); k < have; k += 1 << g) rank += list[k] > key;
        for (int o = 1; o < 1 << g; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
        if (i < have && (tid & ((1 << g) - 1)) == 0 && rank < top) best[rank] = key;
      }
      for (int i = have + tid; i < top; i += TS_THREADS) best[i] = 0ull;  // (a segment of fewer entries)
      continue;
    }
    // Entries that are no numbers, or more that reach the value than are ranked (equal ones, sorted ones): the largest, over and over
    unsigned long long below = ~0ull;
    for (int k = 0; k < top; ++k) {
      unsigned long long largest = 0ull;
      for (int i = tid; i < count; i += TS_THREADS) {
        const unsigned long long key = ts_key(ts_load(row + i), i0 + i);
        if (key < below) largest = max(largest, key);
      }
      below = block_max_key(largest, keys);
      if (tid == 0) best[k] = below;
      if (below == 0ull) below = 1ull;  // (none is left: the rest stays 0)
    }
  }
  if (JOINS) {
    cluster_sync_all();  // (what the other CTAs have written is seen behind it)
    if (cluster_ctarank() == 0 && warp == 0) token_scores_join<ST>(p, blockIdx.x / p.segments, reinterpret_cast<unsigned long long*>(ts_data));
  }
}

template <typename ST>
__global__ void __launch_bounds__(32) token_scores_join_kernel(TokenScoresParams p) {
  extern __shared__ unsigned long long lists[];
  pdl_trigger();
  pdl_wait();
  token_scores_join<ST>(p, blockIdx.x, lists);
}


// Short rows: a warp each, entries in registers, nothing to join.  (4000 x 1003 fp32, 20 alternatives: 12.9 us, 2.5 of them for the
// bytes; as segments, a CTA and two barriers a row, 47.3.  64 x 2000: 7.0 and 9.8.)  With one alternative 8.7: the other 19 are steps of one ballot and one maximum each, one after the
// other, and places in a list; 0.2 us each, 26.1 us for 64.
// The best: the maxima of four parts of each lane's entries; the top-th largest of those 128 is a value that at least `top` entries reach, and few more, which are ranked
// by counting.  (One maximum a lane: 32 alternatives 89 us, where the least of them lets hundreds pass.)
constexpr int TS_SHORT = 2048, TS_SHORT_WARPS = 4, TS_SHORT_LIST = 128;

template <typename ST, int NV>  // NV entries a lane
__global__ void __launch_bounds__(TS_SHORT_WARPS * 32) token_scores_short_kernel(TokenScoresParams p) {
  constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
  __shared__ unsigned long long lists[TS_SHORT_WARPS][TS_SHORT_LIST];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, top = p.top, t = blockIdx.x * TS_SHORT_WARPS + warp;
  if (t >= p.T) return;
  const ST* row = static_cast<const ST*>(p.logits) + (int64_t)t * p.ld;
  float x[NV], part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < NV; ++i) x[i] = i * 32 + lane < p.V ? ts_load(row + i * 32 + lane) : -INFINITY;
  const int64_t target = p.logprob ? p.target[t] : -1;
  const float given = target >= 0 && target < p.V ? ts_load(row + target) : 0.f;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    odd |= x[i] != x[i];
    part[i % 4] = fmaxf(part[i % 4], x[i]);
  }
  odd = __any_sync(0xffffffffu, odd);
  const float M = warp_max_f32(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
  const bool bad = odd || !(fabsf(M) <= FLT_MAX);
  int n = 0;
  float s = 0.f, w = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const bool largest = x[i] == M;
    const float d = fmaxf((x[i] - M) * LOG2E, -1000.f), e = largest ? 0.f : exp2_ftz(d);
    n += largest;
    s += e;
    w = fmaf(e, d, w);
  }
  n = __reduce_add_sync(0xffffffffu, n);
  s = warp_sum(s);
  w = warp_sum(w);
  const float S = s + (float)(n - 1), none = __int_as_float(0x7fffffff), z = log1pf(S);
  if (lane == 0) {
    if (p.entropy) p.entropy[t] = bad ? none : z - LN2 * w / (1.f + S);
    if (p.logprob) p.logprob[t] = target < 0 ? 0.f : bad || target >= p.V ? none : (given - M) - z;
  }
  if (top == 0) return;
  auto put = [&](int k, unsigned long long key) {
    p.top_ids[(int64_t)t * top + k] = ts_index(key);
    p.top_logprobs[(int64_t)t * top + k] = bad ? none : (ts_value(key) - M) - z;
  };
  if (!odd) {
    auto order = [&](int i, int j) {
      const float hi = fmaxf(part[i], part[j]), lo = fminf(part[i], part[j]);
      part[i] = hi;
      part[j] = lo;
    };
    order(0, 1), order(2, 3), order(0, 2), order(1, 3), order(1, 2);
    float limit = M;
    for (int k = 1; k < top; ++k) {  // the next largest of them
      if (lane == __ffs(__ballot_sync(0xffffffffu, part[0] == limit)) - 1) part[0] = part[1], part[1] = part[2], part[2] = part[3], part[3] = -INFINITY;
      limit = warp_max_f32(part[0]);
    }
    unsigned long long* list = lists[warp];
    int have = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool hit = i * 32 + lane < p.V && x[i] >= limit;
      const uint32_t with = __ballot_sync(0xffffffffu, hit);
      if (with == 0) continue;
      const int place = have + __popc(with & ((1u << lane) - 1));
      if (hit && place < TS_SHORT_LIST) list[place] = ts_key(x[i], i * 32 + lane);
      have += __popc(with);
    }
    __syncwarp();
    if (have <= TS_SHORT_LIST) {
      for (int i = lane; i < have; i += 32) {
        const unsigned long long key = list[i];
        int rank = 0;
        for (int j = 0; j < have; ++j) rank += list[j] > key;
        if (rank < top) put(rank, key);
      }
      return;
    }
  }
  unsigned long long below = ~0ull;  // no numbers, or many equal ones: the largest, over and over
  for (int k = 0; k < top; ++k) {
    unsigned long long best = 0ull;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const unsigned long long key = ts_key(x[i], i * 32 + lane);
      if (i * 32 + lane < p.V && key < below) best = max(best, key);
    }
    below = warp_max_key(best);
    if (lane == 0) put(k, below);
  }
}

}  // namespace mb200
