// libmb200_rows8.so -- the C ABI declared in include/mistral_b200_rows8.h.  Argument checking + kernel dispatch only.
#include "rows8_quantise.cuh"
#include "rows8_pair.cuh"
#include "rows8_rotate.cuh"
#include "rows8_stream.cuh"
#include "rows8_product.cuh"

namespace mb200 {
thread_local char g_err[512] = "";

static int check_sizes(const char* what, int64_t T, int64_t N, int64_t K) {
  MB_CHECK_ARG(T >= 0 && T <= MB8_MAX_ROWS && N >= 1 && N <= MB8_MAX_ROWS && K >= 1 && K <= MB8_MAX_ROWS, "%s: %lld rows, %lld features, %lld entries (at most %d)", what, (long long)T,
               (long long)N, (long long)K, MB8_MAX_ROWS);
  return MB200_OK;
}
static int check_rows(const char* what, const void* codes, const void* scales) {
  MB_CHECK_ARG(codes && scales, "%s: null pointer", what);
  MB_CHECK_ARG(((uintptr_t)codes | (uintptr_t)scales) % 16 == 0, "%s: codes and scales start on 16 bytes", what);
  return MB200_OK;
}
static int check_numbers(const char* what, const void* x, int dtype, int64_t ld, int64_t T, int64_t K) {
  MB_CHECK_ARG(dtype == 0 || dtype == 1, "%s: dtype %d", what, dtype);
  MB_CHECK_ARG(x, "%s: null pointer", what);
  MB_CHECK_ARG((uintptr_t)x % (dtype == 0 ? 2 : 4) == 0, "%s: numbers that are not aligned to their type", what);
  MB_CHECK_ARG(T <= 1 || ld >= K, "%s: rows %lld elements apart of %lld", what, (long long)ld, (long long)K);
  return MB200_OK;
}

template <int OUT>
static int product(const ProductParams& p, const void* xc, const void* xs, const void* wc, const void* ws, bool fixed, void* scratch, int64_t scratch_bytes, cudaStream_t st) {
  const int sms = device_info::sm_count();
  MB_CHECK_ARG(sms > 1, "product: the device does not say how many SMs it has");
  return p.T <= RS_MAX_T ? launch_rows8_stream<OUT>(p, xc, xs, wc, ws, fixed, sms, st) : launch_rows8_pair<OUT>(p, xc, xs, wc, ws, scratch, scratch_bytes, sms, st);
}
static int product(const char* what, int form, const ProductParams& p, const void* xc, const void* xs, const void* wc, const void* ws, int fixed, void* scratch, int64_t scratch_bytes,
                   cudaStream_t st) {
  int rc = check_rows(what, xc, xs);
  if (!rc) rc = check_rows(what, wc, ws);
  if (rc) return rc;
  switch (form) {
    case R8_OUT_BF16: return product<R8_OUT_BF16>(p, xc, xs, wc, ws, fixed != 0, scratch, scratch_bytes, st);
    case R8_OUT_F32: return product<R8_OUT_F32>(p, xc, xs, wc, ws, fixed != 0, scratch, scratch_bytes, st);
    default: return product<R8_OUT_GATE>(p, xc, xs, wc, ws, fixed != 0, scratch, scratch_bytes, st);
  }
}
}  // namespace mb200

using namespace mb200;

extern "C" {

int mb8_abi_version(void) { return MB8_ABI_VERSION; }
const char* mb8_last_error(void) { return g_err; }

int mb8_quantise(const void* x, int64_t ld, int dtype, void* codes, void* scales, int64_t T, int64_t K, void* stream) {
  int rc = check_sizes("quantise", T, 1, K);
  if (rc || T == 0) return rc;
  rc = check_numbers("quantise", x, dtype, ld, T, K);
  if (!rc) rc = check_rows("quantise", codes, scales);
  if (rc) return rc;
  QuantiseParams p = {};
  p.x = x;
  p.codes = (uint8_t*)codes;
  p.scales = (uint8_t*)scales;
  p.T = (int)T;
  p.K = (int)K;
  p.ld = ld;
  p.width = (int)r8_width(K);
  p.quads = (int)r8_quads(K);
  return dtype == 0 ? launch_rows8_quantise<bf16>(p, (cudaStream_t)stream) : launch_rows8_quantise<float>(p, (cudaStream_t)stream);
}

int mb8_norm(const void* x, int64_t ld, const void* add, int64_t ld_add, const void* w, int dtype, void* h_out, void* codes, void* scales, int64_t T, int64_t K, float eps,
             void* stream) {
  static_assert(MB8_MAX_NORM == RN8_MAX_K, "what a CTA keeps in registers");
  int rc = check_sizes("norm", T, 1, K);
  MB_CHECK_ARG(K <= MB8_MAX_NORM, "norm: rows of %lld entries (at most %d)", (long long)K, MB8_MAX_NORM);
  if (rc || T == 0) return rc;
  rc = check_numbers("norm", x, dtype, ld, T, K);
  if (!rc) rc = check_numbers("norm", w, dtype, K, 1, K);
  if (!rc) rc = check_rows("norm", codes, scales);
  if (!rc && add) rc = check_numbers("norm", add, dtype, ld_add, T, K);
  if (!rc && add) rc = check_numbers("norm", h_out, dtype, K, T, K);
  if (rc) return rc;
  NormParams p = {};
  p.x = x;
  p.add = add;
  p.w = w;
  p.stream = h_out;
  p.codes = (uint8_t*)codes;
  p.scales = (uint8_t*)scales;
  p.T = (int)T;
  p.K = (int)K;
  p.ld = ld;
  p.ld_add = ld_add;
  p.width = (int)r8_width(K);
  p.quads = (int)r8_quads(K);
  p.eps = eps;
  return dtype == 0 ? launch_rows8_norm<bf16>(p, (cudaStream_t)stream) : launch_rows8_norm<float>(p, (cudaStream_t)stream);
}

int64_t mb8_product_scratch(int64_t T, int64_t N, int64_t K) {
  const int sms = device_info::sm_count();
  return T <= RS_MAX_T || T > MB8_MAX_ROWS || N < 1 || N > MB8_MAX_ROWS || K < 1 || K > MB8_MAX_ROWS || sms < 2 ? 0 : rows8_pair_scratch(T, N, K, sms);
}

int mb8_multiply(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales, void* out, int64_t ld, int dtype, int64_t T, int64_t N, int64_t K, int w_fixed,
                 void* scratch, int64_t scratch_bytes, void* stream) {
  int rc = check_sizes("multiply", T, N, K);
  if (rc || T == 0) return rc;
  rc = check_numbers("multiply", out, dtype, ld, T, N);
  if (rc) return rc;
  ProductParams p = {};
  p.T = (int)T;
  p.N = (int)N;
  p.K = (int)K;
  p.ld = ld;
  p.out = out;
  return product("multiply", dtype, p, x_codes, x_scales, w_codes, w_scales, w_fixed, scratch, scratch_bytes, (cudaStream_t)stream);
}

int mb8_gate(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales, void* codes, void* scales, int64_t T, int64_t H, int64_t K, int w_fixed,
             void* scratch, int64_t scratch_bytes, void* stream) {
  int rc = check_sizes("gate", T, H < 1 || H > MB8_MAX_ROWS ? 0 : 2 * H, K);
  if (rc || T == 0) return rc;
  rc = check_rows("gate", codes, scales);
  if (rc) return rc;
  ProductParams p = {};
  p.T = (int)T;
  p.N = (int)(2 * H);
  p.K = (int)K;
  p.codes = (uint8_t*)codes;
  p.scales = (uint8_t*)scales;
  p.width = (int)r8_width(H);
  p.quads = (int)r8_quads(H);
  return product("gate", R8_OUT_GATE, p, x_codes, x_scales, w_codes, w_scales, w_fixed, scratch, scratch_bytes, (cudaStream_t)stream);
}

int mb8_rotate(const void* qkv, const float* rope, const int32_t* positions, const int32_t* rows, void* q, void* k, void* v, int64_t T, int64_t n_heads, int64_t n_kv_heads,
               void* stream) {
  MB_CHECK_ARG(T >= 0 && T <= MB8_MAX_ROWS && n_heads >= 1 && n_kv_heads >= 1 && n_heads <= 65536 && n_kv_heads <= 65536 && n_heads + 2 * n_kv_heads <= 65536, "rotate: %lld tokens, %lld + 2 * %lld heads", (long long)T,
               (long long)n_heads, (long long)n_kv_heads);
  if (T == 0) return MB200_OK;
  MB_CHECK_ARG(qkv && rope && positions && q && k && v, "rotate: null pointer");
  MB_CHECK_ARG(((uintptr_t)qkv | (uintptr_t)rope | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 == 0, "rotate: matrices start on 16 bytes");
  RotateParams p;
  p.qkv = (const uint4*)qkv;
  p.rope = (const float4*)rope;
  p.positions = positions;
  p.rows = rows;
  p.q = (uint4*)q;
  p.k = (uint4*)k;
  p.v = (uint4*)v;
  p.T = (int)T;
  p.H = (int)n_heads;
  p.KV = (int)n_kv_heads;
  const int threads = (p.H + 2 * p.KV) * 16;
  MB_CHECK_CUDA(launch_pdl(rows8_rotate_kernel, dim3((unsigned)T, (unsigned)((threads + RR_THREADS - 1) / RR_THREADS)), dim3(RR_THREADS), 0, (cudaStream_t)stream, p));
  return MB200_OK;
}

}  // extern "C"
