/*
 * C ABI of the operators around a key/value cache held in 4 bits (head dim 128), next to the MXFP8 attention path of fmha_mxfp8_abi.h in the same
 * library: append, read back, attention over the cache, eviction by accumulated attention weight.
 *
 * The cache. Tokens live in pages of `page` tokens (16, 32, 64 or 128). `table` gives for each sequence the pages that hold its tokens in order, and
 * `lengths` how many tokens it has. A page is HK records of 136 * page bytes, one per KV head, one behind the other:
 *
 *   [ 64 * page  K codes | 64 * page  V codes | 4 * page  K scales | 4 * page  V scales ]
 *
 * A token's 128 elements of K (or V) are OCP MXFP4: 64 bytes of e2m1 codes and four E8M0 scales, one per 32 elements; value = code * 2^(scale - 127).
 * Scale 255 with codes of 0, as append writes it, makes the block's elements NaN, scale 0 makes them zero. Byte 8 g + 2 b + r of the 64 holds the elements 32 b + 4 g + 2 r (low nibble)
 * and 32 b + 4 g + 2 r + 1: with it a lane of the matrix instructions' operand layouts finds its elements of all four blocks side by side, for K
 * (16 bytes) and for V (8 bytes) alike, and a token's bytes are its own, so that appending one token never rewrites a neighbour's byte.
 *
 * Every call is enqueued on `stream`, allocates nothing and waits for nothing. attend and evict enqueue several kernels, which hand on to one another what they leave in the
 * scratch memory they are given (`workspace`, `kept`): two calls may share it only if all kernels of one are enqueued, on the same stream, before those of the other, not from two
 * threads at a time. Lengths, counts and page numbers are read on the device: a length
 * above table_width * page or below 0 is cut to that range, a page number outside the pool is never followed (append drops the token, the others see
 * NaN in its place).
 *
 * Return codes: 0 ok, > 0 FMHA_MXFP8_E_ARG with a message in `err`, < 0 minus a cudaError_t.
 */
#ifndef FMHA_KV4_ABI_H
#define FMHA_KV4_ABI_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FMHA_KV4_TOKEN_BYTES 136u   /* bytes of a token and KV head */

typedef struct fmha_kv4_cache {
    void* pool;             /* uint8 [pages][HK][136 * page], 16-byte aligned */
    const int32_t* table;   /* [B][table_width] */
    int32_t* lengths;       /* [B]; only fmha_kv4_evict writes them (those of `into`) */
    uint64_t pages;
    uint32_t B, HK, page, table_width;
} fmha_kv4_cache;

/* bf16 [B][S][heads][128]: strides in elements, the last dimension dense; pointer and strides multiples of 16 bytes */
typedef struct fmha_kv4_rows {
    void* data;
    int64_t stride_b, stride_s, stride_h;
} fmha_kv4_rows;

/*
 * The S rows of a sequence are its newest tokens: with n = counts[b] (cut to min(S, length); counts NULL: n = min(S, length)) row i < n stands for token
 * length - n + i, and rows from n on for nothing. S may be 0 (and the rows' pointers then NULL): there is nothing to do but to carry weights_in over to weights.
 *
 * append: rounds K and V rows [B][S][HK] into the cache's tokens (lengths have been raised by the caller). scale = clamp(floor(log2 amax) - 2 + 127,
 *   1, 252), code = e2m1, nearest, ties to even, saturating at 6; a block that holds Inf or NaN becomes NaN.
 * read: the values that the cache holds, exact in bf16. last != 0: row i as above. last == 0: row i is token i (counts must be NULL). Rows that stand for
 *   nothing are written as zeros.
 */
int fmha_kv4_append(const fmha_kv4_cache* cache, const fmha_kv4_rows* k, const fmha_kv4_rows* v, uint32_t S, const int32_t* counts, void* stream, char* err, size_t cap);
int fmha_kv4_read(const fmha_kv4_cache* cache, const fmha_kv4_rows* k, const fmha_kv4_rows* v, uint32_t S, int last, const int32_t* counts, void* stream, char* err, size_t cap);

/*
 * attend: out[b][i][h] = softmax_t(scale * q . k_t) v over the tokens t < length, with `causal` over t <= length - n + i only; KV head = h / (H / HK),
 *   H / HK from 1 to 16. Rows from n on, and rows that see no token, get zeros (log-sum-exp -inf).
 *   lse: NULL or f32 [B][H][S], natural.
 *   weights: NULL or f32 [B][HK][weights_width]: weights[b][kv][t] = old + (sum of the softmax weights of token t over the rows and the query heads of the
 *     KV head), for t < length; nothing is written behind the length. old = weights_in[b][kv][t] (same width; the same array, or one that shares no memory with it), 0 where weights_in is
 *     NULL and, with `causal`, for the n newest tokens. Sums in a fixed order: the same bits every time.
 *   NaN: a block of V that is NaN makes its 32 elements NaN in the rows that see the token, whatever the weight, and nothing else; NaN in K makes all of these rows NaN.
 *   Ranges: the products run in f16 against powers of two that are taken out. What is exact is a query row's elements down to 2^-30 of its largest, V's down to 2^-33 of the largest
 *     scale among 32 neighbouring tokens (128 with more than 32 query rows of a KV head, then K's as well); smaller ones count as less. Keys have to stay below 2^100, scores below 2^90
 *     in size, and with `weights` of more than 8 rows of a KV head the products q . k, without the scale, within f32.
 *     In front of V the softmax weights are rounded to f16, in their sum (log-sum-exp, `weights`) they are not. A token whose weight times V's scale is less than 2^-25 of the row's largest such
 *     product leaves nothing in out, at most 1.5 * 2^-25 of that product each: 0.3 % of it if 65536 tokens are all that small.
 *   workspace: fmha_kv4_attend_workspace() bytes of device memory, 16-byte aligned; scratch, no initial contents.
 */
typedef struct fmha_kv4_attend_args {
    fmha_kv4_rows q;        /* [B][S][H][128] */
    void* out;              /* bf16 [B][S][H][128], packed, 16-byte aligned; shares no memory with q, or is q, packed, without weights or with up to 8 rows of a KV head */
    const int32_t* counts;
    float* lse;
    float* weights;
    const float* weights_in;
    void* workspace;
    uint64_t workspace_bytes, weights_width;
    uint32_t S, H, causal;
    float scale;
} fmha_kv4_attend_args;
uint64_t fmha_kv4_attend_workspace(const fmha_kv4_cache* cache, const fmha_kv4_attend_args* args);
int fmha_kv4_attend(const fmha_kv4_cache* cache, const fmha_kv4_attend_args* args, void* stream, char* err, size_t cap);

/*
 * evict: of each sequence and KV head the first `first` and the last `recent` tokens stay, and of the others the ones with the most weight, `keep` tokens in
 *   all (all of a sequence that has no more); equal weights: the earlier token; NaN counts as more than any number. They are copied, in their order, to the
 *   tokens 0, 1, ... of `into`, whose lengths become min(length, keep). `into` has the same B, HK and page, room for `keep` tokens, and its pages must not be
 *   pages that `cache` reads (the pool may be the same).
 *   weights f32 [B][HK][weights_width]. kept: int32 [B][HK][keep], the positions that stayed, -1 behind them (scratch that must be there).
 *   weights_out: NULL or f32 [B][HK][weights_out_width], the weights of the tokens that stayed; nothing is written behind the new length. It must not share memory
 *   with `weights` (the copies run in no order).
 */
typedef struct fmha_kv4_evict_args {
    const float* weights;
    int32_t* kept;
    float* weights_out;
    uint64_t weights_width, weights_out_width;
    uint32_t keep, recent, first;
} fmha_kv4_evict_args;
int fmha_kv4_evict(const fmha_kv4_cache* cache, const fmha_kv4_cache* into, const fmha_kv4_evict_args* args, void* stream, char* err, size_t cap);

#ifdef __cplusplus
}
#endif
#endif /* FMHA_KV4_ABI_H */
