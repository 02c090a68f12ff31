/* libmb200_rows8.so: Linears of 8-bit numbers.
 *
 * Conventions as in mistral_b200.h: plain C types, device pointers, work enqueued on `stream`, 0 or a negative MB200_E_* code, mb8_last_error() for this thread's
 * message, nothing allocated, nothing thrown.  All tensors of a call lie on the current device.
 *
 * Rows.  R rows of K numbers are codes [R, W] e4m3, W = K rounded up to 128, zeros behind the K-th, and a power of two for every 128 of them: number = code * power.  Powers are bytes b,
 * 2^(b - 127), in tiles of 128 rows by 4 blocks of 128 entries, [ceil(R / 128)][ceil(K / 512)][512 bytes]: row 32 j + i and block c of a tile at byte 16 i + 4 j + c.  Places of no row or no
 * block hold 127.  Calls that write rows write all of it.  Both arrays start on 16 bytes.
 */
#ifndef MISTRAL_B200_ROWS8_H_
#define MISTRAL_B200_ROWS8_H_
#include <stddef.h>
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

#define MB8_ABI_VERSION 1
#define MB8_MAX_ROWS (1 << 24)  /* rows, and entries of a row, of any matrix */
#define MB8_MAX_NORM 65536      /* entries of a row that is normed */

int mb8_abi_version(void);
const char* mb8_last_error(void);

/* Rows of x [T, K] (dtype 0 bf16, 1 fp32; rows ld elements apart).  A block's power is 2^e, e >= -100 the smallest with max |x| <= 448 * 2^e; codes are rounded to nearest, ties to
 * even.  A block that holds a NaN or an infinity becomes NaN. */
int mb8_quantise(const void* x, int64_t ld, int dtype, void* codes, void* scales, int64_t T, int64_t K, void* stream);

/* h = x + add (rounded to dtype; add NULL: h = x, and nothing is written to h_out), rows of h * rsqrt(mean(h^2) + eps) * w.  x, add, h_out [T, K] and w [K] of one dtype; h_out
 * contiguous, and no part of x or add but all of one of them with the same rows. */
int mb8_norm(const void* x, int64_t ld, const void* add, int64_t ld_add, const void* w, int dtype, void* h_out, void* codes, void* scales, int64_t T, int64_t K, float eps,
             void* stream);

/* Products.  w_fixed: 0, or 1 where everything that ever wrote w has ended (as a loaded model's weights): then w may be read before the call's turn on its stream.
 * scratch: mb8_product_scratch(T, rows of w, K) bytes on 16, for the call alone (0: NULL).
 */
int64_t mb8_product_scratch(int64_t T, int64_t N, int64_t K); /* on the current device */

/* out [T, N] (dtype 0 bf16, 1 fp32; rows ld elements apart) = x [T, K] times w [N, K] transposed, summed in fp32. */
int mb8_multiply(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales, void* out, int64_t ld, int dtype, int64_t T, int64_t N, int64_t K, int w_fixed,
                 void* scratch, int64_t scratch_bytes, void* stream);

/* Rows [T, H] of silu(y[2 i]) * y[2 i + 1], y = x [T, K] times w [2 H, K] transposed. */
int mb8_gate(const void* x_codes, const void* x_scales, const void* w_codes, const void* w_scales, void* codes, void* scales, int64_t T, int64_t H, int64_t K, int w_fixed,
             void* scratch, int64_t scratch_bytes, void* stream);

/* Queries and keys of qkv [T, (n_heads + 2 n_kv_heads) * 128] bf16, rotated by rope [positions, 64, 2] fp32 (cosine, sine of a pair) at positions [T], and its values: q [T, n_heads * 128],
 * k, v [.., n_kv_heads * 128], token t in row rows[t] of them (-1: nowhere), or in row t (rows NULL). */
int mb8_rotate(const void* qkv, const float* rope, const int32_t* positions, const int32_t* rows, void* q, void* k, void* v, int64_t T, int64_t n_heads, int64_t n_kv_heads,
               void* stream);

#ifdef __cplusplus
}
#endif
#endif
