// Block tables and slot maps from request lengths, on the GPU.
//
// State: table [R, P] page ids (-1 behind a row's last page), lens [R] tokens of each row, free [N] a stack of page ids, n_free [1].
//   extend    request b (row r_b) takes add_b more tokens.  Pages are taken in request order: the a-th new page of the call is free[n_free - 1 - a], so the
//             result is the same in every run.  Per token: its position, and its slot = page * 64 + place in the page (-1 where the stack held no page's id).
//   truncate  request b keeps keep_b tokens; pages go back so that the next extend by the same requests finds them again: the exact inverse of extend.
// A call that cannot be done (a row twice or out of range, a negative or too large length, too few free pages or an n_free that no stack of N has, more tokens than there is room for) changes
// nothing and says why in `status`.
//
// Nothing but latency bounds it: the lengths are a few hundred bytes, and each of the dependent steps (lengths -> prefix sums -> page -> slot) is one trip to L2.  So it is
// ONE launch (8 requests' step and its truncate 8.0 us together, 64 prompts of 1000 tokens 12.5): every CTA forms the prefix sums of all requests for itself in
// shared memory, reads only the state as it was, and the last CTA to be done commits.
#pragma once
#include "paged_common.cuh"
#include "plan_layout.cuh"

namespace mb200 {

constexpr int PLAN_THREADS = 256, PLAN_TOKENS_PER_CTA = 1024, PLAN_MAX_CTAS = 148;

struct PlanParams {
  int32_t *table, *lens, *free, *n_free;
  int32_t* scratch;     // [1]: CTAs of an extend that are done (zero between calls)
  const int32_t* rows;  // [B] or null: request b is row b
  const int32_t* count; // [B] tokens to add, or to keep
  int32_t *positions, *slots, *q_start, *seqpos, *status;
  int B, T, R, P, N;
};

enum { PLAN_OK = 0, PLAN_BAD_ROW = 1, PLAN_BAD_LENGTH = 2, PLAN_NO_ROOM = 3, PLAN_NO_PAGES = 4 };

// exclusive prefix sums of `v` over the block, and their total
__device__ __forceinline__ long long block_scan(long long v, long long* sums, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  long long before = 0;
  total = 0;
  for (int w = 0; w < nw; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  return before + x - v;
}

__device__ __forceinline__ int pages_of(int tokens) { return (tokens + PG_TOKENS - 1) / PG_TOKENS; }

// What both kernels begin with: lengths and prefix sums of all requests in shared memory.  Returns the status of the call, the same in every CTA.
// (plan_layout.cuh says what lies where)
template <bool EXTEND>
__device__ __forceinline__ int plan_requests(const PlanParams& p, int* sm, int& n_free, int& n_moved) {
  int *len = sm, *first = sm + plan_first_at(p.B), *moved = sm + plan_moved_at(p.B);
  __shared__ long long sums[32];
  const int per = (p.B + (int)blockDim.x - 1) / (int)blockDim.x, b0 = min((int)threadIdx.x * per, p.B), b1 = min(b0 + per, p.B);
  n_free = *p.n_free;
  int bad = 0;
  long long tokens = 0, pages = 0;
  uint32_t* named = reinterpret_cast<uint32_t*>(sm + plan_named_at(p.B));
  for (int i = threadIdx.x; i < plan_named_words(p.R); i += blockDim.x) named[i] = 0;
  __syncthreads();
  for (int b = b0; b < b1; ++b) {
    const int r = p.rows ? p.rows[b] : b, c = p.count[b];
    if (r < 0 || r >= p.R) {
      bad |= 1 << PLAN_BAD_ROW;
      len[b] = 0;
      continue;
    }
    if (atomicOr(named + r / 32, 1u << (r & 31)) >> (r & 31) & 1) bad |= 1 << PLAN_BAD_ROW;  // (shared memory: the same answer in every CTA)
    const int l = p.lens[r];
    len[b] = l;
    const bool fits = EXTEND ? (c >= 0 && c <= p.P * PG_TOKENS - l) : (c >= 0 && c <= l);
    if (l < 0 || l > p.P * PG_TOKENS || !fits) {
      bad |= 1 << PLAN_BAD_LENGTH;
      continue;
    }
    tokens += c;
    pages += EXTEND ? pages_of(l + c) - pages_of(l) : pages_of(l) - pages_of(c);
  }
  bad = (__syncthreads_or(bad & (1 << PLAN_BAD_ROW)) ? PLAN_BAD_ROW : 0) | (__syncthreads_or(bad & (1 << PLAN_BAD_LENGTH)) ? 16 : 0);
  if (bad) return bad & PLAN_BAD_ROW ? PLAN_BAD_ROW : PLAN_BAD_LENGTH;
  long long n_tokens, n_pages;
  long long t = block_scan(tokens, sums, n_tokens), a = block_scan(pages, sums, n_pages);
  if (EXTEND && n_tokens > p.T) return PLAN_NO_ROOM;
  if (n_free < 0 || n_free > p.N || (EXTEND ? n_pages > n_free : n_free + n_pages > p.N)) return PLAN_NO_PAGES;
  for (int b = b0; b < b1; ++b) {
    const int c = p.count[b], l = len[b];
    first[b] = (int)t;
    moved[b] = (int)a;
    t += c;
    a += EXTEND ? pages_of(l + c) - pages_of(l) : pages_of(l) - pages_of(c);
  }
  if (threadIdx.x == 0) {
    first[p.B] = (int)n_tokens;
    moved[p.B] = (int)n_pages;
  }
  n_moved = (int)n_pages;
  __syncthreads();
  return PLAN_OK;
}

__global__ void __launch_bounds__(PLAN_THREADS) page_extend_kernel(PlanParams p) {
  extern __shared__ int plan_sm[];
  const int *len = plan_sm, *first = plan_sm + plan_first_at(p.B), *moved = plan_sm + plan_moved_at(p.B);
  pdl_trigger();
  pdl_wait();
  int n_free, n_new;
  const int status = plan_requests<true>(p, plan_sm, n_free, n_new);
  const int at = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
  if (status != PLAN_OK) {
    for (int i = at; i < p.T; i += step) {
      p.positions[i] = 0;
      p.slots[i] = -1;
    }
    for (int b = at; b <= p.B; b += step) {
      p.q_start[b] = 0;
      if (b < p.B) p.seqpos[b] = len[b];
    }
    if (at == 0) *p.status = status;
    return;
  }
  auto row_of = [&](int b) { return (int64_t)(p.rows ? p.rows[b] : b) * p.P; };
  for (int i = at; i < p.T; i += step) {
    int pos = 0, slot = -1;  // places behind the last token (fewer tokens than there is room for)
    if (i < first[p.B]) {
      const int b = last_not_above(p.B, i, [&](int j) { return first[j]; });  // (of requests without tokens the last, which has some)
      pos = len[b] + i - first[b];
      const int j = pos / PG_TOKENS, had = pages_of(len[b]);
      const int page = j < had ? p.table[row_of(b) + j] : p.free[n_free - 1 - (moved[b] + j - had)];
      slot = page < 0 || page > 0x7fffffff / PG_TOKENS ? -1 : page * PG_TOKENS + pos % PG_TOKENS;  // (an id past that would wrap into another page's slots)
    }
    p.positions[i] = pos;
    p.slots[i] = slot;
  }
  for (int a = at; a < n_new; a += step) {
    const int b = last_not_above(p.B, a, [&](int j) { return moved[j]; });
    p.table[row_of(b) + pages_of(len[b]) + a - moved[b]] = p.free[n_free - 1 - a];
  }
  for (int b = at; b <= p.B; b += step) {
    p.q_start[b] = first[b];
    if (b < p.B) p.seqpos[b] = len[b];
  }
  if (at == 0) *p.status = PLAN_OK;
  // the last CTA commits: nobody reads the lengths any more
  __shared__ int last;
  __syncthreads();
  if (threadIdx.x == 0) {
    last = 1;
    if (gridDim.x > 1) {
      __threadfence();
      last = atomicAdd(p.scratch, 1) == (int)gridDim.x - 1;
      if (last) *p.scratch = 0;
    }
  }
  __syncthreads();
  if (!last) return;
  for (int b = threadIdx.x; b < p.B; b += blockDim.x) p.lens[p.rows ? p.rows[b] : b] = len[b] + first[b + 1] - first[b];
  if (threadIdx.x == 0) *p.n_free = n_free - n_new;
}

// One CTA: what goes back is a few pages (drafted tokens) or a few hundred (a request that has ended).
__global__ void __launch_bounds__(1024) page_truncate_kernel(PlanParams p) {
  extern __shared__ int plan_sm[];
  const int *len = plan_sm, *first = plan_sm + plan_first_at(p.B), *moved = plan_sm + plan_moved_at(p.B);
  pdl_trigger();
  pdl_wait();
  int n_free, n_back;
  const int status = plan_requests<false>(p, plan_sm, n_free, n_back);
  if (threadIdx.x == 0) *p.status = status;
  if (status != PLAN_OK) return;
  for (int a = threadIdx.x; a < n_back; a += blockDim.x) {
    const int b = last_not_above(p.B, a, [&](int j) { return moved[j]; });
    int32_t* entry = p.table + (int64_t)(p.rows ? p.rows[b] : b) * p.P + pages_of(first[b + 1] - first[b]) + a - moved[b];
    p.free[n_free + n_back - 1 - a] = *entry;
    *entry = -1;
  }
  for (int b = threadIdx.x; b < p.B; b += blockDim.x) p.lens[p.rows ? p.rows[b] : b] = first[b + 1] - first[b];
  if (threadIdx.x == 0) *p.n_free = n_free + n_back;
}

}  // namespace mb200
