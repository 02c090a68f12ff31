// libmb200_paged.so -- the C ABI declared in include/mistral_b200_paged.h.  Argument checking + kernel dispatch only.
#include "paged_attn.cuh"
#include "paged_plan.cuh"
#include "paged_prompt.cuh"
#include "paged_write.cuh"
#include "token_scores.cuh"

namespace mb200 {
thread_local char g_err[512] = "";

static int run_plan(bool extend, PlanParams p, cudaStream_t st) {
  const char* what = extend ? "pages_extend" : "pages_truncate";
  MB_CHECK_ARG(p.table && p.lens && p.free && p.n_free && p.scratch && p.count && p.status, "%s: null pointer", what);
  MB_CHECK_ARG(p.B >= 1 && p.B <= MBP_MAX_REQUESTS, "%s: %d requests (1 to %d)", what, p.B, MBP_MAX_REQUESTS);
  const size_t smem = sizeof(int) * (size_t)plan_words(p.B, p.R);
  if (extend) {
    // one CTA fills a thousand places as fast as a launch of many starts
    const int ctas = p.T <= PLAN_TOKENS_PER_CTA ? 1 : (ceil_div(p.T, PLAN_TOKENS_PER_CTA) < PLAN_MAX_CTAS ? ceil_div(p.T, PLAN_TOKENS_PER_CTA) : PLAN_MAX_CTAS);
    MB_CHECK_CUDA(launch_pdl(page_extend_kernel, dim3((unsigned)ctas), dim3(PLAN_THREADS), smem, st, p));
  } else {
    MB_CHECK_CUDA(launch_pdl(page_truncate_kernel, dim3(1), dim3(1024), smem, st, p));
  }
  return MB200_OK;
}

static int plan_state(PlanParams& p, const char* what, int32_t* table, int32_t* lens, int32_t* free_pages, int32_t* n_free, int32_t* scratch, const int32_t* rows,
                      const int32_t* count, int64_t B, int64_t R, int64_t P, int64_t n_pages, int32_t* status) {
  MB_CHECK_ARG(R >= 1 && P >= 1 && n_pages >= 1 && R <= MBP_MAX_ROWS && P < (1 << 24) && n_pages <= 0x7fffffff / PG_TOKENS, "%s: %lld rows of %lld pages, %lld pages", what,
               (long long)R, (long long)P, (long long)n_pages);
  MB_CHECK_ARG(B >= 1 && B <= MBP_MAX_REQUESTS && (rows || B <= R), "%s: %lld requests (1 to %d, without a list of rows at most %lld)", what, (long long)B, MBP_MAX_REQUESTS,
               (long long)R);
  p = PlanParams{};
  p.table = table;
  p.lens = lens;
  p.free = free_pages;
  p.n_free = n_free;
  p.scratch = scratch;
  p.rows = rows;
  p.count = count;
  p.status = status;
  p.B = (int)B;
  p.R = (int)R;
  p.P = (int)P;
  p.N = (int)n_pages;
  return MB200_OK;
}
// Entries of a segment: a multiple of 16 bytes a thread, of the fewest segments a row that shared memory holds, all alike.  (As many as fill the last round over the
// CTAs that run at once: 500 rows of 32768 bf16 22.3 us for 17.9, 40 of 131072 15.7 for 14.7; fp32 2000 of 32000 66.1 for 69.2, 32 of 131072 13.0 for 14.4.)
static int64_t score_segment_length(int64_t vocab, int64_t size) {
  const int64_t step = TS_THREADS * (16 / size), most = TS_BYTES / size, n = (vocab + most - 1) / most;
  return ((vocab + n - 1) / n + step - 1) / step * step;
}

// Few rows: segments of a row that can be a cluster (a power of two up to 16), all of them at once, one to an SM; 0: there are too many.  (32000 x 1: a launch less, 20.5 us of the
// host's time 18.4; but 25 rows of 131072 as 400 CTAs in clusters of 16 20.5 us of the GPU's, as segments and a second kernel 13.2.)
static int score_cluster(int64_t T, int64_t vocab, int64_t size) {
  const int64_t step = TS_THREADS * (16 / size), room = device_info::sm_count();
  int best = 0;
  for (int64_t n = 1; n <= 16 && T * n <= room; n *= 2) {
    const int64_t length = ((vocab + n - 1) / n + step - 1) / step * step;
    if (length <= TS_BYTES / size && (n - 1) * length < vocab) best = (int)n;  // (no segment is empty)
  }
  return best;
}

template <auto Kernel, bool JOINS>
static int launch_score_segments(const TokenScoresParams& p, int size, cudaStream_t st) {
  const int64_t items = (int64_t)p.T * p.segments, room = (int64_t)device_info::sm_count() * TS_CTAS;
  const size_t lists = JOINS ? sizeof(unsigned long long) * (size_t)p.segments * p.top : 0, data = (size_t)p.length * size;
  MB_CHECK_CUDA(device_info::allow_shared<Kernel>(TS_BYTES));
  if (JOINS && p.segments > 8) MB_CHECK_CUDA(allow_wide_clusters<Kernel>());
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(JOINS || items < room ? items : room));
  cfg.blockDim = dim3(TS_THREADS);
  cfg.dynamicSmemBytes = data > lists ? data : lists;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (JOINS) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = (unsigned)p.segments;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  MB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, Kernel, p));
  return MB200_OK;
}
template <typename ST, bool JOINS>
static int launch_score_segments(const TokenScoresParams& p, cudaStream_t st) {
  const uint64_t apart = (uintptr_t)p.logits | (p.T > 1 ? (uint64_t)p.ld * sizeof(ST) : 0);
  return apart % 16 == 0  ? launch_score_segments<token_scores_segment_kernel<ST, 16, JOINS>, JOINS>(p, sizeof(ST), st)
         : apart % 4 == 0 ? launch_score_segments<token_scores_segment_kernel<ST, 4, JOINS>, JOINS>(p, sizeof(ST), st)
                          : launch_score_segments<token_scores_segment_kernel<ST, 0, JOINS>, JOINS>(p, sizeof(ST), st);
}

template <typename ST>
static int launch_token_scores(TokenScoresParams p, cudaStream_t st) {
  if (p.V <= TS_SHORT) {
    const dim3 grid((unsigned)((p.T + TS_SHORT_WARPS - 1) / TS_SHORT_WARPS)), block(TS_SHORT_WARPS * 32);
    if (p.V <= TS_SHORT / 2) {
      MB_CHECK_CUDA(launch_pdl(token_scores_short_kernel<ST, TS_SHORT / 64>, grid, block, 0, st, p));
    } else {
      MB_CHECK_CUDA(launch_pdl(token_scores_short_kernel<ST, TS_SHORT / 32>, grid, block, 0, st, p));
    }
    return MB200_OK;
  }
  const int cluster = score_cluster(p.T, p.V, sizeof(ST));
  if (cluster > 0) {
    const int step = TS_THREADS * (16 / (int)sizeof(ST));
    p.length = ((p.V + cluster - 1) / cluster + step - 1) / step * step;
    p.segments = cluster;
    return launch_score_segments<ST, true>(p, st);
  }
  p.length = (int)score_segment_length(p.V, sizeof(ST));
  p.segments = (int)((p.V + p.length - 1) / p.length);
  const int rc = launch_score_segments<ST, false>(p, st);
  if (rc) return rc;
  const size_t lists = p.segments <= TS_JOIN_SEGMENTS ? sizeof(unsigned long long) * (size_t)p.segments * p.top : 0;
  MB_CHECK_CUDA(launch_pdl(token_scores_join_kernel<ST>, dim3((unsigned)p.T), dim3(32), lists, st, p));
  return MB200_OK;
}

// How a call's attention is cut: columns of a query tile (the fewest that hold a request's tokens, 32 at most), its tokens, tiles of queries, splits of the keys (as many as run
// at once, two tiles of keys each at least; a cluster lies within one GPC, so fewer run than the SMs hold CTAs: powers of two by the SMs alone took 60 us for drafts of 5 x 48 heads
// for 5 requests behind 9000, now 44, 41.7 for 9 single tokens behind 9000, now 30.8, and 18.4 for 2, now 12.1), and whether its pages go through 16-bit rings.
struct AttnCut {
  int nq, tokens, splits;
  int64_t q_tiles, keys;
  bool rings;
};
static AttnCut attn_cut(int64_t B, int64_t T, int64_t longest, int64_t most, int64_t P, int64_t n_heads, int64_t n_kv_heads, int64_t window) {
  AttnCut c;
  const int64_t rep = n_heads / n_kv_heads, want = longest * rep, sms = device_info::sm_count() > 0 ? device_info::sm_count() : 148;
  c.nq = want <= 4 ? 4 : want <= 8 ? 8 : want <= 16 ? 16 : 32;
  c.tokens = c.nq / (int)rep;
  c.q_tiles = (longest + c.tokens - 1) / c.tokens;
  c.keys = most > 0 && most < P * PG_TOKENS ? most : P * PG_TOKENS;
  if (window > 0 && c.keys > window + longest) c.keys = window + longest;
  // tiles of `rows` tokens that have any: the requests' lengths are not known here, but their sum is
  auto used = [&](int64_t rows, int64_t most_tiles) { return T / rows + B < B * most_tiles ? T / rows + B : B * most_tiles; };
  const int64_t pairs = n_kv_heads * used(c.tokens, c.q_tiles), room = sms * (c.nq < 32 ? 2 : 1);
  c.splits = 1;
  for (int s = PA_MAX_SPLITS; s > 1; --s) {
    if (pairs * s > room || c.keys < (int64_t)s * 2 * PA_KEYS) continue;
    const int fit = c.nq == 4 ? paged_attn_clusters<4>(s) : c.nq == 8 ? paged_attn_clusters<8>(s) : c.nq == 16 ? paged_attn_clusters<16>(s) : paged_attn_clusters<32>(s);
    if (fit == 0 ? (s & (s - 1)) == 0 : pairs <= fit) {
      c.splits = s;
      break;
    }
  }
  // Time of both ways in us, tiles of 128 keys: 1.4 each on 32 query columns, 2.55 each in the prompt kernel (two heads x 128 tokens), and the conversion.  (nemo shape,
  // measured direct and by rings: 1 x 17 tokens behind 8000 33, 186; 1 x 257 behind 2000 66, 58; 1 x 257 behind 300 28, 24; 3 x 65 behind 2000 57, 65; 3 x 129 behind
  // 8000 268, 203; 16 heads over 4, 3 x 100 behind 20000 234, 464.)
  c.rings = false;
  if (c.q_tiles > 1) {
    const double tiles = (double)(c.keys + PA_KEYS - 1) / PA_KEYS;
    const int64_t prompt = n_heads / (rep % 2 == 0 ? 2 : 1) * used(128, (longest + 127) / 128);
    const double direct = (double)((pairs * c.splits + sms - 1) / sms) * (tiles / c.splits * 1.4 + 5) + 3;
    const double rings = (double)((prompt + sms - 1) / sms) * tiles * 2.55 + 12 + (double)B * (double)c.keys * (double)n_kv_heads * (kHeadDim * 2 * 3) / 4e6;
    c.rings = rings < direct || n_kv_heads * c.q_tiles > 65535;
  }
  return c;
}
// Bytes of the rings.  group: requests that share them at a time (1 GB at most, but for one request alone)
static int64_t ring_scratch(int64_t B, int64_t longest, int64_t most, int64_t P, int64_t KV, int64_t window, int64_t* group) {
  const int64_t rows = paged_ring_rows(longest, most > 0 && most < P * PG_TOKENS ? most : P * PG_TOKENS, window), each = rows * KV * kHeadDim * 4;
  int64_t n = ((int64_t)1 << 30) / each;
  n = n < 1 ? 1 : n > B ? B : n;
  *group = n;
  return n * each;
}
}  // namespace mb200

using namespace mb200;

extern "C" {

int mbp_abi_version(void) { return MBP_ABI_VERSION; }
const char* mbp_last_error(void) { return g_err; }

int mbp_pages_extend(int32_t* table, int32_t* lens, int32_t* free_pages, int32_t* n_free, int32_t* scratch, const int32_t* rows, const int32_t* add, int32_t* positions,
                     int32_t* slots, int32_t* q_start, int32_t* seqpos, int32_t* status, int64_t B, int64_t T, int64_t R, int64_t P, int64_t n_pages, void* stream) {
  PlanParams p;
  int rc = plan_state(p, "pages_extend", table, lens, free_pages, n_free, scratch, rows, add, B, R, P, n_pages, status);
  if (rc) return rc;
  MB_CHECK_ARG(T >= 0 && T <= (1 << 30) && (T == 0 || (positions && slots)) && q_start && seqpos, "pages_extend: room for %lld tokens", (long long)T);
  p.positions = positions;
  p.slots = slots;
  p.q_start = q_start;
  p.seqpos = seqpos;
  p.T = (int)T;
  return run_plan(true, p, (cudaStream_t)stream);
}

int mbp_pages_truncate(int32_t* table, int32_t* lens, int32_t* free_pages, int32_t* n_free, int32_t* scratch, const int32_t* rows, const int32_t* keep, int32_t* status,
                       int64_t B, int64_t R, int64_t P, int64_t n_pages, void* stream) {
  PlanParams p;
  int rc = plan_state(p, "pages_truncate", table, lens, free_pages, n_free, scratch, rows, keep, B, R, P, n_pages, status);
  if (rc) return rc;
  return run_plan(false, p, (cudaStream_t)stream);
}

static int check_pool(const char* what, const void* kv, const void* scale, int64_t n_pages, int64_t KV) {
  MB_CHECK_ARG(kv && scale, "%s: null pointer", what);
  MB_CHECK_ARG((uintptr_t)kv % 16 == 0, "%s: the pool must be 16-byte aligned", what);
  // rows of the pool and slots are counted in 32 bits; bytes are not
  MB_CHECK_ARG(n_pages >= 1 && KV >= 1 && KV <= 32767 && n_pages <= 0x7fffffff / (2 * PG_TOKENS * KV), "%s: %lld pages of %lld heads", what, (long long)n_pages, (long long)KV);
  return MB200_OK;
}

int mbp_pages_write(const void* k, int64_t ldk, const void* v, int64_t ldv, void* kv, float* scale, const int32_t* slots, const int32_t* q_start, const int32_t* seqpos,
                    int64_t B, int64_t T, int64_t n_kv_heads, int64_t head_dim, int64_t n_pages, void* stream) {
  int rc = check_pool("pages_write", kv, scale, n_pages, n_kv_heads);
  if (rc) return rc;
  MB_CHECK_ARG(head_dim == kHeadDim, "pages_write: head_dim=%lld unsupported (128 only)", (long long)head_dim);
  MB_CHECK_ARG(k && v && slots && q_start && seqpos, "pages_write: null pointer");
  MB_CHECK_ARG(B >= 1 && B <= MBP_MAX_REQUESTS && T >= 0 && T <= 0x7fffffff - PG_TOKENS, "pages_write: %lld requests, %lld tokens", (long long)B, (long long)T);
  MB_CHECK_ARG(((uintptr_t)k | (uintptr_t)v) % 16 == 0 && ldk % 8 == 0 && ldv % 8 == 0 && ldk >= n_kv_heads * head_dim && ldv >= n_kv_heads * head_dim,
               "pages_write: rows of keys and values must be 16-byte aligned and not overlap (%lld, %lld elements apart)", (long long)ldk, (long long)ldv);
  if (T == 0) return MB200_OK;
  PagedWriteParams p;
  p.k = (const bf16*)k;
  p.v = (const bf16*)v;
  p.ldk = ldk;
  p.ldv = ldv;
  p.kv = (uint8_t*)kv;
  p.scale = scale;
  p.slots = slots;
  p.q_start = q_start;
  p.seqpos = seqpos;
  p.B = (int)B;
  p.T = (int)T;
  p.KV = (int)n_kv_heads;
  p.n_pages = (int)n_pages;
  const int64_t items = T / PG_TOKENS + 2 * B, ctas = T <= PW_FEW * B ? items * ((2 * n_kv_heads + PW_WARPS - 1) / PW_WARPS) : items * 2 * n_kv_heads;
  MB_CHECK_ARG(ctas <= 0x7fffffff, "pages_write: %lld tokens of %lld heads", (long long)T, (long long)n_kv_heads);
  const cudaStream_t st = (cudaStream_t)stream;
  if (T <= PW_FEW * B) {
    MB_CHECK_CUDA(launch_pdl(page_write_kernel<32>, dim3((unsigned)ctas), dim3(PW_THREADS), 0, st, p));
  } else {
    MB_CHECK_CUDA(launch_pdl(page_write_kernel<PW_THREADS>, dim3((unsigned)ctas), dim3(PW_THREADS), 0, st, p));
  }
  return MB200_OK;
}

int64_t mbp_attn_pages_scratch(int64_t B, int64_t T, int64_t longest, int64_t most, int64_t P, int64_t n_heads, int64_t n_kv_heads, int64_t window) {
  int64_t group;
  if (B < 1 || T < 1 || longest < 1 || P < 1 || n_kv_heads < 1 || n_heads < n_kv_heads || n_heads > 32 * n_kv_heads || n_heads % n_kv_heads || window < 0) return 0;
  return attn_cut(B, T, longest, most, P, n_heads, n_kv_heads, window).rings ? ring_scratch(B, longest, most, P, n_kv_heads, window, &group) : 0;
}

int mbp_attn_pages(const void* q, int64_t ldq, const void* kv, const float* scale, const int32_t* table, const int32_t* rows, const int32_t* q_start, const int32_t* seqpos,
                   void* out, int32_t* status, int64_t B, int64_t T, int64_t longest, int64_t most, int64_t R, int64_t P, int64_t n_pages, int64_t n_heads, int64_t n_kv_heads,
                   int64_t head_dim, int64_t window, float softmax_scale, void* scratch, int64_t scratch_bytes, void* stream) {
  int rc = check_pool("attn_pages", kv, scale, n_pages, n_kv_heads);
  if (rc) return rc;
  MB_CHECK_ARG(head_dim == kHeadDim, "attn_pages: head_dim=%lld unsupported (128 only)", (long long)head_dim);
  MB_CHECK_ARG(q && table && rows && q_start && seqpos && out, "attn_pages: null pointer");
  MB_CHECK_ARG(n_heads >= 1 && n_heads % n_kv_heads == 0 && n_heads / n_kv_heads <= 32, "attn_pages: H=%lld KV=%lld (H a multiple of KV, at most 32 times it)",
               (long long)n_heads, (long long)n_kv_heads);
  MB_CHECK_ARG(B >= 1 && B <= MBP_MAX_REQUESTS && T >= 0 && T <= 0x7fffffff && longest >= 1 && R >= 1 && P >= 1 && P < (1 << 24) && window >= 0 && window <= 0x7fffffff,
               "attn_pages: B=%lld T=%lld longest=%lld R=%lld P=%lld window=%lld", (long long)B, (long long)T, (long long)longest, (long long)R, (long long)P, (long long)window);
  MB_CHECK_ARG(((uintptr_t)q) % 8 == 0 && ldq % 4 == 0 && ldq >= n_heads * head_dim, "attn_pages: rows of queries must be 8-byte aligned and not overlap (%lld elements apart)",
               (long long)ldq);
  MB_CHECK_ARG(((uintptr_t)out) % 8 == 0, "attn_pages: the output must be 8-byte aligned");
  MB_CHECK_ARG(softmax_scale > 0.f && softmax_scale < 3.4e38f, "attn_pages: scale %g", (double)softmax_scale);
  if (T == 0) return MB200_OK;
  const AttnCut cut = attn_cut(B, T, longest, most, P, n_heads, n_kv_heads, window);
  // (rows of queries that the copy engine cannot take stay with the kernel below)
  if (cut.rings && (uintptr_t)q % 16 == 0 && ldq % 8 == 0 && (uintptr_t)out % 16 == 0) {
    int64_t group = 0;
    const int64_t need = ring_scratch(B, longest, most, P, n_kv_heads, window, &group);
    if (scratch == nullptr || scratch_bytes < need || (uintptr_t)scratch % 256 != 0)
      return fail(MB200_E_WORKSPACE, "attn_pages: scratch %lld < %lld, or not 256-byte aligned", (long long)scratch_bytes, (long long)need);
    PagedRingParams p;
    p.kv = (const uint8_t*)kv;
    p.scale = scale;
    p.table = table;
    p.rows = rows;
    p.q_start = q_start;
    p.seqpos = seqpos;
    p.status = status;
    p.T = (int)T;
    p.R = (int)R;
    p.P = (int)P;
    p.n_pages = (int)n_pages;
    p.KV = (int)n_kv_heads;
    p.window = (int)window;
    p.W = (int)paged_ring_rows(longest, most > 0 && most < P * PG_TOKENS ? most : P * PG_TOKENS, window);
    for (int64_t b0 = 0; b0 < B; b0 += group) {
      rc = launch_paged_prompt(p, q, ldq, (bf16*)out, b0, B - b0 < group ? B - b0 : group, longest, (int)n_heads, softmax_scale * 1.4426950408889634f, scratch, (cudaStream_t)stream);
      if (rc) return rc;
    }
    return MB200_OK;
  }
  MB_CHECK_ARG(n_kv_heads * cut.q_tiles <= 65535, "attn_pages: %lld tiles of queries", (long long)(n_kv_heads * cut.q_tiles));
  PagedAttnParams p;
  p.q = (const bf16*)q;
  p.ldq = ldq;
  p.scale = scale;
  p.table = table;
  p.rows = rows;
  p.q_start = q_start;
  p.seqpos = seqpos;
  p.out = (bf16*)out;
  p.status = status;
  p.T = (int)T;
  p.B = (int)B;
  p.R = (int)R;
  p.P = (int)P;
  p.n_pages = (int)n_pages;
  p.H = (int)n_heads;
  p.KV = (int)n_kv_heads;
  p.window = (int)window;
  p.tokens = cut.tokens;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  CUtensorMap map;
  rc = make_pool_map(&map, kv, n_pages, n_kv_heads);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  switch (cut.nq) {
    case 4: return launch_paged_attn<4>(p, map, cut.q_tiles, cut.splits, st);
    case 8: return launch_paged_attn<8>(p, map, cut.q_tiles, cut.splits, st);
    case 16: return launch_paged_attn<16>(p, map, cut.q_tiles, cut.splits, st);
    default: return launch_paged_attn<32>(p, map, cut.q_tiles, cut.splits, st);
  }
}

int mbp_token_scores_sizes(int64_t T, int64_t vocab, int64_t top, int64_t* bytes) {
  MB_CHECK_ARG(T >= 0 && vocab >= 1 && vocab <= MBP_MAX_VOCAB && top >= 0 && top <= TS_MAX_TOP && top <= vocab && bytes, "token_scores: T=%lld vocab=%lld top=%lld (at most %d)", (long long)T,
               (long long)vocab, (long long)top, TS_MAX_TOP);
  const int64_t segments = vocab / (TS_BYTES / 4) + 1 > 16 ? vocab / (TS_BYTES / 4) + 1 : 16;  // at most: of the wider type, or a cluster's
  *bytes = T * segments * (8 * top + 12);
  return MB200_OK;
}

int mbp_token_scores(const void* logits, int64_t ld, int dtype, const int64_t* target, float* logprob, float* entropy, int64_t* top_ids, float* top_logprobs, int64_t T,
                     int64_t vocab, int64_t top, void* scratch, void* stream) {
  int64_t bytes = 0;
  int rc = mbp_token_scores_sizes(T, vocab, top, &bytes);
  if (rc) return rc;
  MB_CHECK_ARG(logits && scratch && (uintptr_t)scratch % 8 == 0 && (logprob == nullptr || target) && (top == 0 || (top_ids && top_logprobs)), "token_scores: null pointer");
  MB_CHECK_ARG((uintptr_t)logits % (dtype == 0 ? 2 : 4) == 0, "token_scores: logits that are not aligned to their type");
  MB_CHECK_ARG(ld >= vocab && (dtype == 0 || dtype == 1), "token_scores: rows %lld elements apart of %lld, dtype %d", (long long)ld, (long long)vocab, dtype);
  MB_CHECK_ARG(T <= 65535, "token_scores: %lld rows (at most 65535)", (long long)T);
  if (T == 0) return MB200_OK;
  TokenScoresParams p = {};
  p.logits = logits;
  p.ld = ld;
  p.target = target;
  p.T = (int)T;
  p.V = (int)vocab;
  p.top = (int)top;
  const int64_t most = bytes / (T * (8 * top + 12));  // segments that there is room for
  p.best = (unsigned long long*)scratch;
  p.sums = (float*)(p.best + T * most * top);
  p.logprob = logprob;
  p.entropy = entropy;
  p.top_ids = top_ids;
  p.top_logprobs = top_logprobs;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == 0 ? launch_token_scores<bf16>(p, st) : launch_token_scores<float>(p, st);
}

}  // extern "C"
