// Causal attention of new tokens over pages of e4m3 keys and values, head size 128: decode steps, drafts of a few tokens, short portions.
//
//   o = softmax(scale * q K^T + mask) V with K, V = codes * page scales; a query at position p sees the positions (p - window, p] of its own request.
//
// The codes never leave 8 bits on their way to the tensor cores.  tcgen05 multiplies e4m3 by e4m3, so it is the QUERIES and the WEIGHTS that are given in
// e4m3, each as two numbers: hi + lo / 16, hi = e4m3(x), lo = e4m3(16 (x - hi)).  The 8 significant bits of a bf16 query are held exactly that way (a row is
// first scaled by a power of two to at most 448; entries below 2^-14 of the row's largest keep fewer bits, never worse than 2^-23 of that largest), a weight
// to 2^-8 of itself, as bf16 weights are, or to 2^-22 of the weight 1 where that is more.  That lets many small weights beside a large one vanish (30000 of 2^-22
// are 0.7 % of it), so the score that has weight 1 is not the running maximum for good: it goes up with the maximum, and, after a CTA's first 2048 keys, down
// to a tile's own maximum where that lies more than 8 binary places below.  A tile's weights are then off by 128 * 2^-22 * 2^8 = 2^-7 of its largest in all, those of the
// first 2048 keys by 2^-11 of theirs.  Scores, maxima and sums, and the values' sums stay in fp32; the pages' scales multiply in fp32, the keys' on the scores, the values' on
// each page's own accumulator.
//
// Keys are the MMA's 128 rows (S^T = K Q^T) and so are the values' dimensions (O^T = V^T P^T, V as it lies in the page: MN-major), the hi and lo parts of up to NQ
// query columns (tokens x heads of one key/value head) its columns.  Memory bounds it: 256 bytes a key and key/value head, where converting them to 16 bits on the way to
// mma.sync fragments would take more issue slots than the bytes take time.  CTA = (a range of pages, key/value head and tile of queries, request); the ranges of one
// request's head are a cluster and are merged through distributed shared memory: one launch, no scratch, the same order every time.
//   softmax   groups of four warps, a part of the query columns each, a thread per key: scores -> maximum (over the group) -> weights -> shared memory; then, a thread
//             per dimension, the values' sums of the tile before
//   producer  TMA: tiles of two pages (8 KB of keys and of values each) into a ring of PA_STAGES x 32 KB
//   issuer    MMAs: S(0) S(1) | PV(t) S(t + 2) ...
// What it measured, on inputs that L2 does not hold: single tokens of 4 requests with 32500 tokens each, 32 heads over 8: 42.8 us, 5.65 TB/s; of 32 with ~1000 each: 16.2 us, of which
// the bytes take 10 and launch, the first loads and the merge 6.  A tile of a token's few columns takes 1700 clocks, the last 600 to 1000 of them waiting for the bytes.  (Four warps
// with eight columns each, half of them empty for groups of four heads: 3200 clocks, 21.0 us.)  A tile of 32 columns takes 3600: scores and maximum 1050, weights 620, sums 470 by 16
// warps.  Latency bounds those: 1.8 of 4 instructions a clock, one CTA an SM whose warps all wait for a tile's scores, the group's barrier and the sums of the tile before; 96 registers
// a thread leave 48 bytes of it spilled.  Drafts of 5 tokens x 6 heads for 8 requests behind 2100: 22.4 us for 4.9 of bytes.  The score of weight 1 that goes down costs drafts
// behind 8400 tokens 56.9 us for 55.5, the four long requests 42.4 for 42.0.  Keys and values in slots of their own, keys' freed after S(t): no faster (44.8 us for 42.3 with the four
// long requests): what lies in flight is enough.
#pragma once
#include <type_traits>

#include "paged_common.cuh"

namespace mb200 {

constexpr int PA_STAGES = 3, PA_KEYS = 2 * PG_TOKENS, PA_STAGE_BYTES = 4 * PG_BYTES;
constexpr int PA_MAX_SPLITS = 16;
constexpr int PA_ROW = kHeadDim + 4;     // numbers of a split's result for one query: the score of weight 1, sum, -, -, the values' sums
constexpr float PA_NOTHING = -1.0e30f;   // the maximum of no score
constexpr int PA_NEAR_TILES = 16;        // tiles whose weights are held against the running maximum only
constexpr float PA_FAR = 8.f, PA_DOWN = 16.f;  // log2 units: how far below a tile's maximum may lie, and how far weight 1 may at most (2^16 times the sums is far inside fp32)
enum { PA_GAVE_UP = 16 };                // status: a wait ran out; the call's results are NaN

struct PagedAttnParams {
  const bf16* q;
  int64_t ldq;  // elements between tokens
  const float* scale;
  const int32_t *table, *rows, *q_start, *seqpos;
  bf16* out;  // [T, H * 128]
  int32_t* status;
  int T, B, R, P, n_pages, H, KV, window, tokens;  // tokens: of a query tile
  float scale_log2;
};

// NQ query columns, Q of them a group of softmax warps; column c of the MMA: group i has hi parts at i * 2 Q, lo parts at i * 2 Q + Q
template <int NQ>
struct PaCfg {
  static constexpr int G = NQ >= 32 ? 4 : 2, Q = NQ / G;   // (32 columns: two groups 31.1 us for drafts of 8 requests behind 2100, four 25.5; now 21.2)
  static constexpr int kSoftWarps = 4 * G, kThreads = 32 * (kSoftWarps + 2), kResident = NQ >= 32 ? 1 : 2;
  static constexpr int N = 2 * NQ < 16 ? 16 : 2 * NQ;      // (16 at least; columns that nobody reads hold anything)
  static constexpr int kColBytes = N * 128;                // Q or one P tile: [N columns][128 bytes], 128B-swizzled
  static constexpr int kRing = PA_STAGES * PA_STAGE_BYTES;
  static constexpr int kMerge = NQ * PA_ROW * 4;            // this split's result, over the ring once that is used up
  static constexpr int kSmem = 1024 + kRing + 3 * kColBytes;
  static constexpr int kTmemCols = 4 * N;                  // two S tiles, the two pages' O
  static_assert(kMerge <= kRing && kTmemCols <= 512, "fits");
  // D = fp32, A = B = e4m3, N >> 3 at bit 17, M >> 4 at bit 24; values: A is MN-major (bit 15)
  static constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  static constexpr uint32_t kIdescO = kIdescS | (1u << 15);
};

__device__ __forceinline__ void umma_e4m3(uint32_t tmem_d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 da, db;\n"
      "mov.b64 da, {%1, %5};\n"
      "mov.b64 db, {%2, %5};\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(UMMA_DESC_HI)
      : "memory");
}
// COLS consecutive columns of this warp's 32 lanes
template <int COLS>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&v)[COLS]) {
  static_assert(COLS == 4 || COLS == 8 || COLS == 16 || COLS == 32, "");
  if constexpr (COLS == 4)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(taddr));
  else if constexpr (COLS == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr));
  else if constexpr (COLS == 16)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
          "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
  else
    tmem_ld_32x32b_x32_nowait(taddr, v);
}
// barrier of the 128 threads of a group; true if any of them says so
template <int ID>
__device__ __forceinline__ bool group_sync_or_id(bool v) {
  uint32_t r;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.u32 p, %1, 0;\n"
      "barrier.cta.red.or.pred q, %2, 128, p;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(r)
      : "r"((uint32_t)v), "n"(ID)
      : "memory");
  return r != 0;
}
template <int G>
__device__ __forceinline__ bool group_sync_or(int group, bool v) {
  if (group == 0) return group_sync_or_id<1>(v);
  if (G == 2 || group == 1) return group_sync_or_id<2>(v);
  if (group == 2) return group_sync_or_id<3>(v);
  return group_sync_or_id<4>(v);
}
// two weights times 256 as codes.  (Through fp16, whose 11 bits hold more than the two parts do.)
__device__ __forceinline__ void weight_parts(float w0, float w1, uint16_t& hi, uint16_t& lo) {
  uint32_t w, h, r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(w1), "f"(w0));
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(hi) : "r"(w));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(hi));
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(h));
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(r), "r"(0x4c004c00u));  // times 16
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(lo) : "r"(r));
}
template <int AT>
__device__ __forceinline__ void st_shared_u8(uint32_t addr, uint16_t v) {
  asm volatile("st.shared.u8 [%0 + %2], %1;" ::"r"(addr), "h"(v), "n"(AT) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

__device__ __forceinline__ uint64_t pair_of(uint32_t x, uint32_t y) { return pair(__uint_as_float(x), __uint_as_float(y)); }
template <int N, typename F>
__device__ __forceinline__ void unrolled(F f) {  // f(0) .. f(N - 1), constants
  if constexpr (N > 0) {
    unrolled<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// The warp's v[i] combined over its lanes, column i in lanes i * (32 / Q) and on.  Each step halves what is sent: Q + 4 - log2 Q shuffles.
template <int Q, typename F>
__device__ __forceinline__ float by_column(float (&v)[Q], int lane, F op) {
  int o = 16;
#pragma unroll
  for (int w = Q / 2; w >= 1; w /= 2, o /= 2) {
    const bool upper = lane & o;
#pragma unroll
    for (int i = 0; i < w; ++i) {
      const float other = __shfl_xor_sync(0xffffffffu, upper ? v[i] : v[i + w], o);
      v[i] = op(upper ? v[i + w] : v[i], other);
    }
  }
#pragma unroll
  for (; o >= 1; o /= 2) v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
  return v[0];
}

// Byte k of column c: its 128 bytes are one row of a 128B-swizzled K-major tile
__device__ __forceinline__ uint32_t pa_col(int c, int k) { return (uint32_t)(((c >> 3) << 10) + ((c & 7) << 7) + (((k >> 4) ^ (c & 7)) << 4) + (k & 15)); }

template <int NQ>
__global__ void __launch_bounds__(PaCfg<NQ>::kThreads, PaCfg<NQ>::kResident) paged_attn_kernel(const __grid_constant__ CUtensorMap map_kv, const PagedAttnParams p) {
  using Cfg = PaCfg<NQ>;
  constexpr int Q = Cfg::Q, N = Cfg::N, SOFT = Cfg::kSoftWarps;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem + Cfg::kRing;
  uint8_t* sP = sQ + Cfg::kColBytes;  // [2]
  __shared__ uint64_t kv_full[PA_STAGES], kv_empty[PA_STAGES], q_full, s_full[2], p_full, o_full;
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up;
  __shared__ float page_scale[PA_STAGES][4];              // keys of page 0, 1, values of page 0, 1 of the stage's tile
  __shared__ float q_scale[NQ];                           // a query row's scale, times the softmax scale, in log2 units
  __shared__ float warp_most[2][NQ][4];                   // by tile parity
  __shared__ float sums[4][NQ];
  // Values that are no numbers, of keys that not all tokens of the tile see, are taken out (0 * NaN is not 0) and noted by dimension: a bit for each token of the tile behind
  // its first, and for each place from the beginning of the first one's window on
  __shared__ uint32_t nan_new[kHeadDim], nan_old[kHeadDim];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int split = blockIdx.x, splits = gridDim.x, g = blockIdx.y % p.KV, qt = blockIdx.y / p.KV, b = blockIdx.z;
  const int R = p.H / p.KV;
  if (tid < kHeadDim) nan_new[tid] = nan_old[tid] = 0;
  if (tid == 0) {
    for (int i = 0; i < PA_STAGES; ++i) {
      mbar_init(&kv_full[i], 2);  // the copies' arrival and the scales'
      mbar_init(&kv_empty[i], 1);
    }
    mbar_init(&q_full, SOFT);
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(&p_full, SOFT);
    mbar_init(&o_full, 1);
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_kv) : "memory");
  }
  if (warp == SOFT + 1) tmem_alloc(&tmem_slot, Cfg::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_trigger();  // behind the columns' allocation: a dependent that takes its own may come onto this SM (us ahead of it and here: one token over 4096 8.74, 8.73; 32 over 1106 16.9, 16.9)
  pdl_wait();

  const int t_first = p.q_start[b], n_all = p.q_start[b + 1] - t_first, past = p.seqpos[b], row = p.rows[b];
  const int i0 = qt * p.tokens;
  const int n = t_first < 0 || n_all < 0 || n_all > p.T - t_first || past < 0 ? 0 : min(p.tokens, n_all - i0);  // tokens of this tile
  if (n <= 0) {  // the whole cluster alike
    __syncthreads();
    if (warp == SOFT + 1) tmem_dealloc(tmem, Cfg::kTmemCols);
    return;
  }
  if (i0 + p.tokens < n_all && blockIdx.y / p.KV == gridDim.y / p.KV - 1 && split == 0) {  // more tokens than there are tiles for
    if (tid == 0 && p.status) atomicOr(p.status, PG_TOO_LONG);
    no_numbers(p.out + (int64_t)t_first * p.H * kHeadDim + g * R * kHeadDim, i0 + p.tokens, n_all, p.H, R);
  }
  const int nq = n * R, tok0 = t_first + i0;
  const int pos0 = past + i0, hi = pos0 + n;                                   // the tile's first position, one past its last
  const int lo = p.window > 0 ? max(0, pos0 + 1 - p.window) : 0;               // the first position that any query sees
  const int page_lo = lo / PG_TOKENS, n_pages = (hi + PG_TOKENS - 1) / PG_TOKENS - page_lo;
  const int first = page_lo + n_pages * split / splits, last = page_lo + n_pages * (split + 1) / splits;  // this split's pages (n_pages < 2^25)
  const int tiles = (last - first + 1) / 2;

  uint64_t o[Q / 2], l[Q / 2], less[Q / 2];  // of two queries each; less: minus the score that has weight 1
  const int group = warp >> 2, key_at = tid & 127;  // of the softmax threads
  if (warp == SOFT) {
    // ================= producer =================
    const bool row_ok = row >= 0 && row < p.R;
    int page = 0;
    float ks = 0.f, vs = 0.f;
    for (int t = 0; t < tiles; ++t) {
      if ((t & 15) == 0) {  // the next 32 pages, one a lane; their scales arrive while the first tile's bytes do
        const int at = first + 2 * t + lane;
        page = -1;
        if (at < last && row_ok && at < p.P) page = p.table[(int64_t)row * p.P + at];
        const bool ok = page >= 0 && page < p.n_pages;
        if (!ok) page = 0;  // a page that is none: nothing is read out of bounds, and what it weighs is no number
        const float* s = p.scale + ((int64_t)page * p.KV + g) * 2;
        ks = ok ? s[0] : __int_as_float(0x7fffffff);
        vs = ok ? s[1] : __int_as_float(0x7fffffff);
      }
      const int st = t % PA_STAGES, two = first + 2 * t + 1 < last, src = (2 * t) & 31;
      const int page0 = __shfl_sync(0xffffffffu, page, src), page1 = __shfl_sync(0xffffffffu, page, src + 1);
      if (!__all_sync(0xffffffffu, bounded_wait(&kv_empty[st], ((t / PA_STAGES) & 1) ^ 1, &gave_up))) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&kv_full[st], (two ? 4 : 2) * PG_BYTES);
        uint8_t* dst = smem + st * PA_STAGE_BYTES;
        const int r0 = (page0 * p.KV + g) * 2 * PG_TOKENS, r1 = (page1 * p.KV + g) * 2 * PG_TOKENS;
        tma_load_2d(dst, &map_kv, &kv_full[st], 0, r0);
        if (two) tma_load_2d(dst + PG_BYTES, &map_kv, &kv_full[st], 0, r1);
        tma_load_2d(dst + 2 * PG_BYTES, &map_kv, &kv_full[st], 0, r0 + PG_TOKENS);
        if (two) tma_load_2d(dst + 3 * PG_BYTES, &map_kv, &kv_full[st], 0, r1 + PG_TOKENS);
      }
      const float ks0 = __shfl_sync(0xffffffffu, ks, src), ks1 = __shfl_sync(0xffffffffu, ks, src + 1);
      const float vs0 = __shfl_sync(0xffffffffu, vs, src), vs1 = __shfl_sync(0xffffffffu, vs, src + 1);
      if (lane == 0) {
        page_scale[st][0] = ks0;
        page_scale[st][1] = ks1;
        page_scale[st][2] = vs0;
        page_scale[st][3] = vs1;
        mbar_arrive(&kv_full[st]);
      }
      __syncwarp();
    }
  } else if (warp == SOFT + 1) {
    // ================= MMA issuer =================
    bool ok = tiles == 0 || bounded_wait(&q_full, 0, &gave_up);
    const uint32_t q_desc = umma_desc_lo(smem_u32(sQ));
    auto issue_s = [&](int t) {
      const int st = t % PA_STAGES;
      ok = ok && bounded_wait(&kv_full[st], (t / PA_STAGES) & 1, &gave_up);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      tc_fence_after();
      const uint32_t k_desc = umma_desc_lo(smem_u32(smem + st * PA_STAGE_BYTES));
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_e4m3(tmem + (t & 1) * N, k_desc + k * 2, q_desc + k * 2, Cfg::kIdescS, k ? 1u : 0u);
        umma_commit(&s_full[t & 1]);
      }
      __syncwarp();
    };
    // What values that a query does not see hold must not reach its sums: 0 * NaN is not 0.  Done while the softmax warps have the tile's scores.
    auto hide_values = [&](int t) {
      const int key0 = (first + 2 * t) * PG_TOKENS, end = min(hi, last * PG_TOKENS);
      if (key0 >= lo && key0 + PA_KEYS <= pos0 + 1 && (p.window <= 0 || key0 >= pos0 + n - p.window)) return;  // every query sees every key
      uint8_t* v = smem + t % PA_STAGES * PA_STAGE_BYTES + 2 * PG_BYTES;
      for (int r = lane >> 3; r < PA_KEYS; r += 4)  // rows that no query sees, eight lanes each
        if (key0 + r < lo || key0 + r >= end) *reinterpret_cast<uint4*>(v + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
      // rows that some queries see: later tokens of the tile, and what the later tokens' windows have left behind, a lane each
      auto scan = [&](int key, uint32_t* whose) {
        uint4* row = reinterpret_cast<uint4*>(v + (key - key0) * 128);
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          const int chunk = (i + lane) & 7;
          uint4 x = row[chunk];
          const uint32_t bad[4] = {__vcmpeq4(x.x & 0x7f7f7f7fu, 0x7f7f7f7fu), __vcmpeq4(x.y & 0x7f7f7f7fu, 0x7f7f7f7fu), __vcmpeq4(x.z & 0x7f7f7f7fu, 0x7f7f7f7fu),
                                   __vcmpeq4(x.w & 0x7f7f7f7fu, 0x7f7f7f7fu)};
          if ((bad[0] | bad[1] | bad[2] | bad[3]) == 0) continue;
          row[chunk] = make_uint4(x.x & ~bad[0], x.y & ~bad[1], x.z & ~bad[2], x.w & ~bad[3]);
          for (int c = 0; c < 16; ++c)
            if (bad[c >> 2] >> 8 * (c & 3) & 1) atomicOr(whose + (chunk ^ (key - key0 & 7)) * 16 + c, 1u << lane);
        }
      };
      __syncwarp();
      if (n > 1) {
        const int later = pos0 + 1 + lane, left = pos0 + 1 - p.window + lane;
        if (later < hi && later >= key0 && later < min(end, key0 + PA_KEYS)) scan(later, nan_new);
        if (p.window > 0 && lane < n - 1 && left <= pos0 && left >= max(lo, key0) && left < min(end, key0 + PA_KEYS)) scan(left, nan_old);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    };
    if (tiles > 0) issue_s(0);
    if (tiles > 1) issue_s(1);
    for (int t = 0; t < tiles && ok; ++t) {
      hide_values(t);
      ok = bounded_wait(&p_full, t & 1, &gave_up);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const int st = t % PA_STAGES;
      const bool two = first + 2 * t + 1 < last;
      const uint32_t v_desc = umma_desc_lo(smem_u32(smem + st * PA_STAGE_BYTES + 2 * PG_BYTES)), p_desc = umma_desc_lo(smem_u32(sP + (t & 1) * Cfg::kColBytes));
      if (elect_one()) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (h == 0 || two) {
#pragma unroll
            for (int k = 0; k < 2; ++k)  // 32 keys each: 4 KB of values, 32 bytes of a weights' column
              umma_e4m3(tmem + (2 + h) * N, v_desc + ((h * PG_BYTES + k * 4096) >> 4), p_desc + h * 4 + k * 2, Cfg::kIdescO, k ? 1u : 0u);
          }
        umma_commit(&o_full);
        umma_commit(&kv_empty[st]);
      }
      __syncwarp();
      if (t + 2 < tiles) issue_s(t + 2);
    }
  } else {
    // ================= softmax =================
    // queries -> hi and lo parts, a warp per row
    constexpr int ROWS = (NQ + SOFT - 1) / SOFT;
    uint2 raw[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int q = warp + i * SOFT;
      raw[i] = make_uint2(0u, 0u);
      if (q < nq) raw[i] = *reinterpret_cast<const uint2*>(p.q + (int64_t)(tok0 + q / R) * p.ldq + (int64_t)(g * R + q % R) * kHeadDim + lane * 4);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int q = warp + i * SOFT;
      if (q >= NQ) break;
      const uint2 u = raw[i];
      const float x[4] = {bf16lo(u.x), bf16hi(u.x), bf16lo(u.y), bf16hi(u.y)};
      const int e = e4m3_exponent(warp_max_f32(fmaxf(fmaxf(finite_abs(x[0]), finite_abs(x[1])), fmaxf(finite_abs(x[2]), finite_abs(x[3])))));
      const float inv = pow2i(-e);
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = scaled(x[j], inv);
      const uint32_t h0 = to_e4m3x2(y[0], y[1]), h1 = to_e4m3x2(y[2], y[3]);
      const float2 f0 = from_e4m3x2(h0), f1 = from_e4m3x2(h1);
      const uint32_t l0 = to_e4m3x2((y[0] - f0.x) * 16.f, (y[1] - f0.y) * 16.f), l1 = to_e4m3x2((y[2] - f1.x) * 16.f, (y[3] - f1.y) * 16.f);
      const int c = q / Q * 2 * Q + q % Q;
      *reinterpret_cast<uint32_t*>(sQ + pa_col(c, lane * 4)) = h0 | h1 << 16;
      *reinterpret_cast<uint32_t*>(sQ + pa_col(c + Q, lane * 4)) = l0 | l1 << 16;
      if (lane == 0) q_scale[q] = pow2i(e) * p.scale_log2;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(&q_full);
    bool ok = bounded_wait(&q_full, 0, &gave_up);  // q_scale of all rows
    uint64_t qs[Q / 2];
#pragma unroll
    for (int i = 0; i < Q; i += 2) {
      o[i / 2] = l[i / 2] = pair(0.f, 0.f);
      less[i / 2] = pair(-PA_NOTHING, -PA_NOTHING);
      qs[i / 2] = pair(q_scale[group * Q + i], q_scale[group * Q + i + 1]);
    }
    const int most_at = lane % (4 * Q);  // the maximum that this lane looks at: column most_at / 4, warp most_at % 4
    float most = PA_NOTHING, peak = PA_NOTHING;  // of column most_at / 4: the score that has weight 1 (times 256), the maximum
    const uint64_t sixteenth = pair(0.0625f, 0.0625f), eight = pair(8.f, 8.f);
    // Byte key_at of column j of the group: its 128 bytes are row j of a 128B-swizzled K-major tile, which pa_col(group * 2 Q + j, key_at) says in full
    const uint32_t p_at = smem_u32(sP) + group * 2 * Q * 128 + (key_at ^ (Q == 2 ? group << 6 : 0));
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + group * 2 * Q;
    float vs0 = 0.f, vs1 = 0.f;  // value scales of the tile before
    bool two_before = false;
    auto add_values = [&](int t) {  // the sums of tile t, relative to m as it stood then
      ok = ok && bounded_wait(&o_full, t & 1, &gave_up);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      tc_fence_after();
      uint32_t a[2 * Q], z[2 * Q];
      tmem_ld_cols<2 * Q>(lanes + 2 * N, a);
      if (two_before) tmem_ld_cols<2 * Q>(lanes + 3 * N, z);
      tmem_wait_ld();
      const uint64_t by0 = pair(vs0, vs0), by1 = pair(vs1, vs1);
#pragma unroll
      for (int i = 0; i < Q; i += 2) o[i / 2] = fma_pair(fma_pair(pair_of(a[Q + i], a[Q + i + 1]), sixteenth, pair_of(a[i], a[i + 1])), by0, o[i / 2]);
      if (two_before) {
#pragma unroll
        for (int i = 0; i < Q; i += 2) o[i / 2] = fma_pair(fma_pair(pair_of(z[Q + i], z[Q + i + 1]), sixteenth, pair_of(z[i], z[i + 1])), by1, o[i / 2]);
      }
    };
    for (int t = 0; t < tiles; ++t) {
      const int st = t % PA_STAGES;
      const int key0 = (first + 2 * t) * PG_TOKENS, key = key0 + key_at;
      const bool here = first + 2 * t + (key_at >> 6) < last;   // the tile's second page may be none
      const bool seen = here && key >= lo && key < hi;          // by any query
      const bool two = first + 2 * t + 1 < last;
      const bool edge = !two || key0 + PA_KEYS > pos0 + 1 || (p.window > 0 && key0 < pos0 + n - p.window);  // (uniform) some query does not see some key
      float s[Q];
      ok = ok && bounded_wait(&kv_full[st], (t / PA_STAGES) & 1, &gave_up) && bounded_wait(&s_full[t & 1], (t >> 1) & 1, &gave_up);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        const float ks = page_scale[st][key_at >> 6];
        uint32_t a[2 * Q];
        tmem_ld_cols<2 * Q>(lanes + (t & 1) * N, a);
        tmem_wait_ld();
        const uint64_t by = pair(ks, ks);
#pragma unroll
        for (int i = 0; i < Q; i += 2) {
          const float2 f = unpair(mul_pair(fma_pair(pair_of(a[Q + i], a[Q + i + 1]), sixteenth, pair_of(a[i], a[i + 1])), mul_pair(by, qs[i / 2])));
          s[i] = f.x;
          s[i + 1] = f.y;
        }
        if (edge) {
#pragma unroll
          for (int i = 0; i < Q; ++i) {
            bool sees = seen;
            if (n > 1) {  // (of one token every key in [lo, hi) is seen)
              const int pos = pos0 + (group * Q + i) / R;
              sees = seen && key <= pos && (p.window <= 0 || key > pos - p.window);
            }
            s[i] = sees ? s[i] : -INFINITY;
          }
        }
        if constexpr (NQ == 16) {  // (2 tokens of 6 heads a group, 8 requests behind 8400: 35.7 us, 39.1 by the instruction below; 32 columns: 58.6 and 55.6)
          float w[Q];
#pragma unroll
          for (int i = 0; i < Q; ++i) w[i] = s[i];
          const float most_here = by_column<Q>(w, lane, [](float x, float y) { return fmaxf(x, y); });
          if (lane % (32 / Q) == 0) warp_most[t & 1][group * Q + lane / (32 / Q)][warp & 3] = most_here;
        } else {
#pragma unroll
          for (int i = 0; i < Q; ++i) {
            const float w = warp_max_f32(s[i]);
            if (lane == 0) warp_most[t & 1][group * Q + i][warp & 3] = w;
          }
        }
      }
      if (group_sync_or<Cfg::G>(group, !ok)) {
        ok = false;
        break;
      }
      // The group's maxima, a column and warp a lane; broadcast only where one has moved.  (All of them by every thread: 40 instructions of some 350 a tile and thread.)
      float top = warp_most[t & 1][group * Q + most_at / 4][most_at % 4];
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      float to = top;
      bool moves = top > most;
      if (t >= PA_NEAR_TILES) {
        to = fmaxf(top, peak - PA_DOWN);
        moves |= top > PA_NOTHING && to < most - PA_FAR;
      }
      const bool moved = __any_sync(0xffffffffu, moves);  // (the same in all threads of the group)
      uint64_t alpha[Q / 2];
      if (moved) {
        if (moves) most = to;
        peak = fmaxf(peak, most);
#pragma unroll
        for (int i = 0; i < Q; i += 2) {
          const float m0 = __shfl_sync(0xffffffffu, most, i * 4), m1 = __shfl_sync(0xffffffffu, most, i * 4 + 4);
          const float2 was = unpair(less[i / 2]);
          alpha[i / 2] = pair(exp2_ftz(-was.x - m0), exp2_ftz(-was.y - m1));
          l[i / 2] = mul_pair(l[i / 2], alpha[i / 2]);
          less[i / 2] = pair(-m0, -m1);
        }
      }
      const uint32_t P = p_at + (t & 1) * Cfg::kColBytes;
      unrolled<Q / 2>([&](auto at) {
        constexpr int i = 2 * decltype(at)::value;
        const float2 x = unpair(add_pair(add_pair(pair(s[i], s[i + 1]), less[i / 2]), eight));
        const float e0 = exp2_ftz(x.x), e1 = exp2_ftz(x.y);  // weights times 256: the whole of e4m3's range
        l[i / 2] = add_pair(l[i / 2], pair(e0, e1));
        uint16_t hi, lo;
        weight_parts(e0, e1, hi, lo);
        st_shared_u8<i * 128>(P ^ ((i & 7) << 4), hi);
        st_shared_u8<i * 128 + 128>(P ^ ((i + 1 & 7) << 4), hi >> 8);
        st_shared_u8<(i + Q) * 128>(P ^ ((i + Q & 7) << 4), lo);
        st_shared_u8<(i + Q) * 128 + 128>(P ^ ((i + Q + 1 & 7) << 4), lo >> 8);
      });
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (t > 0) add_values(t - 1);
      if (moved) {
#pragma unroll
        for (int i = 0; i < Q / 2; ++i) o[i] = mul_pair(o[i], alpha[i]);
      }
      vs0 = page_scale[st][2];
      vs1 = page_scale[st][3];
      two_before = two;
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && ok) mbar_arrive(&p_full);
    }
    if (tiles > 0 && ok) add_values(tiles - 1);
    if (!__all_sync(0xffffffffu, ok)) {
#pragma unroll
      for (int i = 0; i < Q / 2; ++i) o[i] = pair(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff));
      if (lane == 0 && p.status) atomicOr(p.status, PA_GAVE_UP);
    }
    float all[Q];
#pragma unroll
    for (int i = 0; i < Q; i += 2) {
      const float2 x = unpair(l[i / 2]);
      all[i] = x.x;
      all[i + 1] = x.y;
    }
    const float sum = by_column<Q>(all, lane, [](float x, float y) { return x + y; });
    if (lane % (32 / Q) == 0) sums[warp & 3][group * Q + lane / (32 / Q)] = sum;
  }
  tc_fence_before();
  __syncthreads();
  if (gave_up && tid == 0) {  // copies of this CTA may still be in flight: they end before its shared memory does
    for (int i = 0; i < PA_STAGES; ++i)
      for (uint32_t k = 0; k < 2; ++k)
        for (uint32_t spin = 0; spin < 4096 && !mbar_try_wait(&kv_full[i], k); ++spin) {}
  }
  if (warp == SOFT + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::kTmemCols);
  }
  // ================= merge the splits =================
  // this split's results over the ring, which is used up
  float* mine = reinterpret_cast<float*>(smem);
  if (warp < SOFT) {
    const uint32_t in_new = nan_new[key_at], in_old = nan_old[key_at];
    if (__any_sync(0xffffffffu, (in_new | in_old) != 0)) {
      unrolled<Q / 2>([&](auto at) {
        float2 x = unpair(o[decltype(at)::value]);
        for (int half = 0; half < 2; ++half) {
          const int i = (group * Q + 2 * decltype(at)::value + half) / R;  // token of the tile
          uint32_t sees = (1u << i) - 1;  // the tokens before it but for the first, whose values every query sees or has left behind
          if (p.window > 0 && i >= p.window) sees &= ~((1u << (i - p.window)) - 1);
          if ((in_new & sees) != 0 || in_old >> i != 0) (half ? x.y : x.x) = __int_as_float(0x7fffffff);
        }
        o[decltype(at)::value] = pair(x.x, x.y);
      });
    }
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const int q = group * Q + i;
      if (q < nq) {
        const float sum = sums[0][q] + sums[1][q] + sums[2][q] + sums[3][q], mine_o = i & 1 ? unpair(o[i / 2]).y : unpair(o[i / 2]).x;
        if (splits == 1) {
          p.out[((int64_t)(tok0 + q / R) * p.H + g * R + q % R) * kHeadDim + key_at] = __float2bfloat16_rn(sum == 0.f ? 0.f : mine_o / sum);
        } else {
          mine[q * PA_ROW + 4 + key_at] = mine_o;
          if (key_at == 0) {
            mine[q * PA_ROW] = -(i & 1 ? unpair(less[i / 2]).y : unpair(less[i / 2]).x);
            mine[q * PA_ROW + 1] = sum;
          }
        }
      }
    }
  }
  if (splits == 1) return;
  cluster_sync_all();
  // The results are dealt to all warps of the cluster: a quarter of a query's to each where there are as many warps (one query of 4 heads, 16 splits: 7.9 us, 8.5
  // by whole queries), else a query (drafts of 8 requests in 2 splits: 21.5 us, 23.0 by quarters, four to a warp).  Maxima and sums of all splits come by one
  // load, a split a lane, and the loads of their sums of values do not wait for one another.  (A loop over the splits in every thread: 4500 clocks for 16 of them.)
  auto merge = [&](auto wide) {
    constexpr int D = decltype(wide)::value, PARTS = kHeadDim / (32 * D);  // D dimensions a lane
    const uint32_t base = smem_u32(mine);
    for (int part = split * SOFT + warp; part < nq * PARTS; part += splits * SOFT) {
      const int q = part / PARTS, d = (part % PARTS * 32 + lane) * D;
      const uint32_t at = base + q * PA_ROW * 4;
      const uint32_t from = map_to_rank(at, lane < splits ? lane : 0);
      const float mine_m = lane < splits ? ld_cluster_f32(from) : PA_NOTHING, mine_l = lane < splits ? ld_cluster_f32(from + 4) : 0.f;
      float v[PA_MAX_SPLITS][D], acc[D];
#pragma unroll
      for (int r = 0; r < PA_MAX_SPLITS; ++r) {
        const uint32_t src = map_to_rank(at + 16 + d * 4, r < splits ? r : 0);
        if constexpr (D == 1) {
          v[r][0] = r < splits ? ld_cluster_f32(src) : 0.f;
        } else {
          const float4 x = r < splits ? ld_cluster_f32x4(src) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[r][0] = x.x, v[r][1] = x.y, v[r][2] = x.z, v[r][3] = x.w;
        }
      }
      const float f = exp2_ftz(mine_m - warp_max_f32(mine_m));  // (a split without a key: its sums are 0)
      const float sum = warp_sum(f * mine_l), inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int i = 0; i < D; ++i) acc[i] = 0.f;
#pragma unroll
      for (int r = 0; r < PA_MAX_SPLITS; ++r) {
        const float w = __shfl_sync(0xffffffffu, f, r);
#pragma unroll
        for (int i = 0; i < D; ++i) acc[i] = fmaf(w, v[r][i], acc[i]);
      }
#pragma unroll
      for (int i = 0; i < D; ++i) acc[i] = sum == 0.f ? 0.f : acc[i] * inv;
      bf16* to = p.out + ((int64_t)(tok0 + q / R) * p.H + g * R + q % R) * kHeadDim + d;
      if constexpr (D == 1) *to = __float2bfloat16_rn(acc[0]);
      else *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
    }
  };
  if (warp < SOFT) {
    if (nq * 4 <= splits * SOFT) merge(std::integral_constant<int, 1>{});
    else merge(std::integral_constant<int, 4>{});
  }
  cluster_sync_all();  // nobody leaves while its results are read
}

// the pool as rows of 128 bytes; box = one head's keys or values of a page, 128-byte swizzle
inline int make_pool_map(CUtensorMap* map, const void* kv, int64_t n_pages, int64_t KV) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (enc == nullptr) return fail(MB200_E_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const cuuint64_t dims[2] = {(cuuint64_t)kHeadDim, (cuuint64_t)(n_pages * KV * 2 * PG_TOKENS)};
  const cuuint64_t strides[1] = {(cuuint64_t)kHeadDim};
  const cuuint32_t box[2] = {(cuuint32_t)kHeadDim, (cuuint32_t)PG_TOKENS};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(kv), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MB200_E_CUDA, "cuTensorMapEncodeTiled (pages) failed (%d)", (int)r);
  return MB200_OK;
}

// Clusters of `splits` CTAs that run at once on the current device where each CTA has an SM to itself; 0: unknown
template <int NQ>
inline int paged_attn_clusters_apart(int splits) {
  static std::atomic<int> known[device_info::MAX_DEVICES][PA_MAX_SPLITS + 1];
  const int dev = device_info::current();
  if (dev < 0 || dev >= device_info::MAX_DEVICES || device_info::sm_count() == 0) return 0;
  std::atomic<int>& here = known[dev][splits];
  if (here.load(std::memory_order_relaxed) > 0) return here.load(std::memory_order_relaxed);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)splits);
  cfg.blockDim = dim3(PaCfg<NQ>::kThreads);
  cfg.dynamicSmemBytes = PaCfg<NQ>::kSmem;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int n = 0;
  if (device_info::allow_shared<paged_attn_kernel<NQ>>(PaCfg<NQ>::kSmem) != cudaSuccess || allow_wide_clusters<paged_attn_kernel<NQ>>() != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, paged_attn_kernel<NQ>, &cfg) != cudaSuccess) {
    cudaGetLastError();  // (not this call's: the caller has an estimate of its own)
    return 0;
  }
  here.store(n, std::memory_order_relaxed);
  return n;
}
// Clusters that run at once: where two CTAs share an SM, two layers of them, or clusters of half as many SMs (all but a few of those: 72 of 74 clusters of 4 did not, 32 of 33 of 8 did)
template <int NQ>
inline int paged_attn_clusters(int splits) {
  const int apart = paged_attn_clusters_apart<NQ>(splits);
  if (PaCfg<NQ>::kResident == 1) return apart;
  const int half = splits % 2 == 0 && splits > 2 ? paged_attn_clusters_apart<NQ>(splits / 2) * 97 / 100 : 0;
  return 2 * apart > half ? 2 * apart : half;
}

template <int NQ>
inline int launch_paged_attn(const PagedAttnParams& p, const CUtensorMap& map, int64_t q_tiles, int splits, cudaStream_t st) {
  MB_CHECK_CUDA(device_info::allow_shared<paged_attn_kernel<NQ>>(PaCfg<NQ>::kSmem));
  if (splits > 8) MB_CHECK_CUDA(allow_wide_clusters<paged_attn_kernel<NQ>>());
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)splits, (unsigned)(p.KV * q_tiles), (unsigned)p.B);
  cfg.blockDim = dim3(PaCfg<NQ>::kThreads);
  cfg.dynamicSmemBytes = PaCfg<NQ>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  MB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_attn_kernel<NQ>, map, p));
  return MB200_OK;
}

}  // namespace mb200
