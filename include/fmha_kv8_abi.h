/*
 * C ABI of the operators around a key/value cache held in 8 bits (head dim 128), beside the 4-bit one of fmha_kv4_abi.h in the same library: append, read back and
 * attention over the cache. Sequences, tables, lengths, rows and counts mean what they mean there, and so do streams, the scratch memory and the return codes.
 *
 * The cache. A page of `page` tokens (16, 32, 64 or 128) is page / 16 blocks for each KV head, head after head; a block of 16 tokens and a head is 4112 bytes:
 *
 *   [ 2048  K codes | 2048  V codes | f32 K scale | f32 V scale | u16 K mask | u16 V mask | 4 bytes of nothing ]
 *
 * Codes are OCP e4m3, value = code * scale, one scale for all of the block's K and one for its V, powers of two from 2^-90 to 2^119. Bit t of a mask: token t of the block
 * holds no numbers in K (V): all of its 128 elements are NaN, its codes 0. K's byte of token t and element d lies at 128 t + 16 ((d / 16) ^ (t % 8)) + d % 16; V's tokens
 * lie in pairs, j = t / 2: 256 j + 16 ((d / 8) ^ s) + 2 (d % 8) + t % 2 with s = j % 2 + 4 (j / 2 % 2). So the matrix instructions' operands are found without regrouping, K's rows
 * and V's columns, and shared memory is read without conflicts. What lies behind a sequence's length is never looked at: a pool needs no initial contents.
 */
#ifndef FMHA_KV8_ABI_H
#define FMHA_KV8_ABI_H

#include "fmha_kv4_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FMHA_KV8_BLOCK_TOKENS 16u
#define FMHA_KV8_BLOCK_BYTES 4112u   /* of 16 tokens and a KV head: 257 a token */

/* the fields of the 4-bit cache; pool is uint8 [pages][HK][257 * page] */
typedef fmha_kv4_cache fmha_kv8_cache;

/*
 * append: rounds K and V rows [B][S][HK] into the cache's tokens (lengths have been raised by the caller). Of each block that gets tokens, K and V for themselves:
 *   scale = the smallest power of two with largest <= 448 * scale over the new tokens' elements (2^-90 to 2^119: beyond that elements are cut to 448 * scale), or the block's
 *   scale if that is larger and the block has tokens in front of the new ones. code = e4m3, nearest, ties to even. Where the scale grows, the older tokens' codes become
 *   e4m3(code * old scale / new scale): a shift of their exponents, which loses bits only below 2^-6 of the new scale. Of a token with Inf or NaN all elements become NaN, and it
 *   does not count for the scale.
 * read: the values that the cache holds, exact in bf16, as fmha_kv4_read gives them.
 */
int fmha_kv8_append(const fmha_kv8_cache* cache, const fmha_kv4_rows* k, const fmha_kv4_rows* v, uint32_t S, const int32_t* counts, void* stream, char* err, size_t cap);
int fmha_kv8_read(const fmha_kv8_cache* cache, const fmha_kv4_rows* k, const fmha_kv4_rows* v, uint32_t S, int last, const int32_t* counts, void* stream, char* err, size_t cap);

/*
 * attend: out[b][i][h] = softmax_t(scale * q . k_t) v over the tokens t < length, with `causal` over t <= length - n + i only; KV head = h / (H / HK), H / HK from 1 to 16. Rows from n
 *   on, and rows that see no token, get zeros (log-sum-exp -inf).
 *   lse: NULL or f32 [B][H][S], natural.
 *   NaN: a token without numbers in V makes the rows that see it NaN, whatever its weight, in K their log-sum-exps too; so does a page that the pool does not have. Tokens that a row
 *   does not see leave nothing in it.
 *   Ranges: the products run in f16, codes as they are, the query rows against a power of two that is taken out (exact down to 2^-30 of a row's largest element). Softmax weights are
 *   rounded to f16 in front of V, times V's scale against the row's largest such product; one that is less than 2^-35 of it (2^-30 with more than 32 query rows of a KV head) leaves
 *   nothing in out. In their sum (log-sum-exp) they are not rounded. Scores have to stay below 2^90 in size.
 *   workspace: fmha_kv8_attend_workspace() bytes of device memory, 16-byte aligned; scratch, no initial contents.
 */
typedef struct fmha_kv8_attend_args {
    fmha_kv4_rows q;        /* [B][S][H][128] */
    void* out;              /* bf16 [B][S][H][128], packed, 16-byte aligned; shares no memory with q, or is q, packed */
    const int32_t* counts;
    float* lse;
    void* workspace;
    uint64_t workspace_bytes;
    uint32_t S, H, causal;
    float scale;
} fmha_kv8_attend_args;
uint64_t fmha_kv8_attend_workspace(const fmha_kv8_cache* cache, const fmha_kv8_attend_args* args);
int fmha_kv8_attend(const fmha_kv8_cache* cache, const fmha_kv8_attend_args* args, void* stream, char* err, size_t cap);

#ifdef __cplusplus
}
#endif
#endif /* FMHA_KV8_ABI_H */
