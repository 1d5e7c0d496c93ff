/*
 * C ABI of rotary positions, in the library of fmha_mxfp8_abi.h: queries and keys are turned by their tokens' positions before they go to the attention or the cache.
 *
 * Of each row (a token's head of head_dim elements) the first `rotary` elements are n = rotary / 2 pairs (a, b): elements i and n + i, or 2 i and 2 i + 1 (`interleaved`). With
 * t = position * (frequency of pair i, in turns):
 *
 *   a' = factor * (a cos 2 pi t - b sin 2 pi t),   b' = factor * (a sin 2 pi t + b cos 2 pi t)
 *
 * and with `backward` the transposed matrix: what turns the gradient of (a', b') into that of (a, b). Elements from `rotary` on stay as they are.
 *
 * `turns` holds the frequencies as fractions of a turn per position, times 2^64. The product with the position, in 64 bits without the whole turns, is the angle to 2^-33 of a turn
 * for any position of 32 bits: far positions cost no accuracy. Sums in f32, rounded once.
 */
#ifndef FMHA_ROPE_ABI_H
#define FMHA_ROPE_ABI_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FMHA_ROPE_BF16 0u
#define FMHA_ROPE_F16 1u
#define FMHA_ROPE_F32 2u
#define FMHA_ROPE_MAX_HEAD_DIM 512u

/* [B][S][heads][head_dim]: strides in elements, not negative, the last dimension dense; aligned as an element is */
typedef struct fmha_rope_rows {
    void* data;
    int64_t stride_b, stride_s, stride_h;
} fmha_rope_rows;

/*
 * x goes to x_out and y, where heads_y is not 0, to y_out. An output is its input (same address, same strides) or shares no memory with it, no element of the outputs stands twice
 * in them, and an output and the other input or output share no element.
 * Enqueued on `stream`; allocates nothing and waits for nothing. Returns 0, > 0 FMHA_MXFP8_E_ARG with a message in `err`, < 0 minus a cudaError_t. B or S of 0: nothing to do.
 */
typedef struct fmha_rope_args {
    fmha_rope_rows x, x_out, y, y_out;
    const uint64_t* turns;       /* [rotary / 2], device memory */
    const void* positions;       /* int32 or int64 [B][S], strides in elements (0: the same for all) */
    int64_t positions_stride_b, positions_stride_s;
    uint32_t positions_64, B, S, heads_x, heads_y, head_dim, rotary, type, interleaved, backward;
    float factor;
} fmha_rope_args;
int fmha_rope_rotate(const fmha_rope_args* args, void* stream, char* err, size_t cap);

#ifdef __cplusplus
}
#endif
#endif /* FMHA_ROPE_ABI_H */
