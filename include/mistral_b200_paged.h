/* libmb200_paged.so: requests of different lengths served from a pool of 8-bit pages, and scores of tokens.
 *
 * Conventions as in mistral_b200.h: plain C types, device pointers, work enqueued on `stream`, 0 or a negative MB200_E_* code, mbp_last_error() for this thread's
 * message, nothing allocated, nothing thrown.  All tensors of a call lie on the current device.
 *
 * Pages.  A page holds 64 tokens.  One layer's pool: kv [n_pages, KV, 2 (keys, values), 64, 128] e4m3 and scale [n_pages, KV, 2] fp32, powers of two; a number is its code
 * times the scale of its page, head and kind.  table [R, P] int32: row r names the pages of the request in it, in order, -1 behind the last.  lens [R] int32: its
 * tokens.  free_pages [n_pages] int32: a stack of n_free[0] page ids, the last one is taken first.  scratch [1] int32: zero once, this state's own.
 * Calls on one state, and on pools that its pages name, are ordered on one stream (or by events).
 */
#ifndef MISTRAL_B200_PAGED_H_
#define MISTRAL_B200_PAGED_H_
#include <stddef.h>
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

#define MBP_ABI_VERSION 1
#define MBP_MAX_REQUESTS 4000 /* requests of a call */
#define MBP_MAX_ROWS 131072   /* rows of a state */
#define MBP_MAX_VOCAB (1 << 24)

int mbp_abi_version(void);
const char* mbp_last_error(void);

/* Request b = 0 .. B - 1, in row rows[b] (rows NULL: row b), takes add[b] >= 0 more tokens.  Pages are taken in the order of the requests.
 *   positions, slots [T]  of the new tokens, request after request: position in the request, and page * 64 + place in the page; places behind the last new token 0, -1
 *   q_start [B + 1]       prefix sums of add;  seqpos [B]: lengths before
 *   status [1]            0, or why nothing was changed: 1 a row out of range or named twice, 2 a length that is negative or longer than P pages,
 *                         3 more tokens than T, 4 too few free pages, or n_free is not within 0 .. n_pages; then q_start is 0 and every slot -1: writes and attention by this plan do nothing. */
int mbp_pages_extend(int32_t* table, int32_t* lens, int32_t* free_pages, int32_t* n_free, int32_t* scratch, const int32_t* rows, const int32_t* add, int32_t* positions,
                     int32_t* slots, int32_t* q_start, int32_t* seqpos, int32_t* status, int64_t B, int64_t T, int64_t R, int64_t P, int64_t n_pages, void* stream);
/* Request b keeps its first keep[b] tokens (at most what it has); pages that hold none of them go back on the stack, so that an extend by the same requests would take
 * them again in the same order.  status as above. */
int mbp_pages_truncate(int32_t* table, int32_t* lens, int32_t* free_pages, int32_t* n_free, int32_t* scratch, const int32_t* rows, const int32_t* keep, int32_t* status,
                       int64_t B, int64_t R, int64_t P, int64_t n_pages, void* stream);

/* Keys and values of a plan's tokens into one layer's pool.  k, v [T, KV * 128] bf16, rows ldk, ldv elements apart (16-byte aligned).  scale = 2^e, e >= -100 the smallest with
 * max |x| <= 448 * 2^e over the page's new numbers, and no smaller than the page's scale where it holds earlier tokens, whose codes are rounded to a grown scale; codes are
 * rounded to nearest even.  Infinities and NaNs become NaN.  Tokens with slot -1 are left out.  Plans are written in the order in
 * which they were made; the last one may be written again (the same result). */
int mbp_pages_write(const void* k, int64_t ldk, const void* v, int64_t ldv, void* kv, float* scale, const int32_t* slots, const int32_t* q_start, const int32_t* seqpos,
                    int64_t B, int64_t T, int64_t n_kv_heads, int64_t head_dim, int64_t n_pages, void* stream);

/* Bytes of scratch that mbp_attn_pages needs for these sizes (0: none): portions of prompts go through 16-bit rings. */
int64_t mbp_attn_pages_scratch(int64_t B, int64_t T, int64_t longest, int64_t most, int64_t P, int64_t n_heads, int64_t n_kv_heads, int64_t window);
/* Causal attention of a plan's tokens over one layer's pool, their own keys and values written before.  q [T, H * 128] bf16, rows ldq elements apart (8-byte aligned); out
 * [T, H * 128] bf16, 8-byte aligned.  The query at position p sees positions (p - window, p]; window 0: all.  longest: no request has more tokens in this plan; most: none has more in all
 * (0: unknown).  status [1] or NULL: 16 is set when a wait inside ran out, 32 when a request has more tokens than longest or most say: those it
 * has no room for, or all of its results, are NaN.  scratch:
 * mbp_attn_pages_scratch bytes, 256-byte aligned, of any content and this call's own until it has run.  A page id out of range makes the results that need it NaN (and
 * perhaps those of a few tokens of its request ahead of it).  So does a NaN among the
 * values, in its column, of the queries that see it (by rings also of others up to 127 positions from those); rows of out behind
 * q_start[B] are left as they are. */
int mbp_attn_pages(const void* q, int64_t ldq, const void* kv, const float* scale, const int32_t* table, const int32_t* rows, const int32_t* q_start, const int32_t* seqpos,
                   void* out, int32_t* status, int64_t B, int64_t T, int64_t longest, int64_t most, int64_t R, int64_t P, int64_t n_pages, int64_t n_heads, int64_t n_kv_heads,
                   int64_t head_dim, int64_t window, float softmax_scale, void* scratch, int64_t scratch_bytes, void* stream);

/* Scores of the rows of logits [T, vocab] (dtype 0: bf16, 1: fp32; rows ld elements apart), each output NULL or
 *   logprob [T]: log_softmax(logits[t])[target[t]], 0 where target[t] < 0, NaN for a target past the vocabulary
 *   entropy [T]: of softmax(logits[t]), in nats
 *   top_ids [T, top] int64, top_logprobs [T, top]: the largest logits, the lowest index first where they are equal, NaN before all, and their log-probabilities
 * all sums in fp32.  An entry of -infinity weighs nothing; a row of nothing else, or with NaN or +infinity, scores NaN.  top <= 64, T <= 65535.
 * scratch: mbp_token_scores_sizes bytes, 8-byte aligned, this call's own until it has run. */
int mbp_token_scores_sizes(int64_t T, int64_t vocab, int64_t top, int64_t* bytes);
int mbp_token_scores(const void* logits, int64_t ld, int dtype, const int64_t* target, float* logprob, float* entropy, int64_t* top_ids, float* top_logprobs, int64_t T,
                     int64_t vocab, int64_t top, void* scratch, void* stream);

#ifdef __cplusplus
}
#endif
#endif
