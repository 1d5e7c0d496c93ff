// Attention of few query rows over the 4-bit cache: decode, and drafts of a few tokens, up to 32 rows of a KV head (kv4_prefill.cu has more).
//
// Work. An item is one sequence and KV head; its tokens are cut in tiles of 128. All tiles of all items, in order, are dealt out in equal runs to the CTAs, from the
// lengths on the device: a batch of ragged sequences keeps every CTA busy for the same time, one long sequence as well. An item that more than one CTA worked on is put
// together from f32 partials by the combine kernel.
//
// Copies of whole page records (cp.async.bulk) bring a tile, 17408 bytes, to a ring of three in shared memory; the warps take turns in issuing them. A warp takes 32 of
// the tile's tokens and computes both products transposed, so that the tokens are the rows of the matrix instruction and the few query rows its 8 columns:
//   S^T [16 tokens x 8 rows] = K [16 x 128] Q^T      K's codes become f16 by the conversion instruction, two per byte; the E8M0 factor of a token's 32 elements
//                                                     multiplies the two products' sum in f32
//   O^T [128 x 8 rows] += V^T [128 x 16 tokens] P^T  P goes from S^T's layout to the operand's by an 8 x 8 transpose between lanes; V's factors multiply P
// Q goes in as f16 with a power of two per row taken out, which is exact for bf16 elements down to 2^-30 of the row's largest.
//
// Softmax in base 2 with a running reference per row. P V wants P times V's factor in f16: the reference M follows s + e, e the exponent of the largest V factor of
// the 32 tokens, so that P 2^e is at most 2^4 however large V is; the factors relative to 2^e are exact in f16 down to 2^-34. M moves when a value exceeds it by more
// than 2^4, by a vote of the warp; the sums and O are rescaled then.
//
// With one group of 8 columns the bound is latency, not the bytes and no pipe: 64 sequences x 8 heads of 16384 tokens take 237 to 257 us by box, 4.4 to 4.8 TB/s of the 6.5 that a copy reaches; 594
// instructions per 32 tokens of a warp (301 of them conversions, packing and logic, a pipe at half rate that is busy 56 % of the time), issued in 56 % of the cycles by 16 warps an SM. Four CTAs an SM
// are what the registers allow; three of them took 226 us where four took 236, but 71 in place of 68 on ragged sequences in pages of 16, five and six with two stages 470 to 610 (spills). The kernels
// taken spill too: 68 and 80 bytes stored and loaded with one group, 84 and 124, 60 and 92, 292 and 424 with two, three and four.
// Groups of 8 rows more cost their products and softmax: 32 rows over 16 x 4096 tokens 65 us, against 100 with the tiles of 128 rows.
#include "kv4.cuh"
#include "kv4_schedule.cuh"
#include "ptx_sm100.cuh"

#include <atomic>

namespace b200mx {

namespace {

using namespace kv4;

constexpr unsigned kWarps = 4, kThreads = kWarps * 32;
constexpr unsigned kUnit = 32;                    // tokens of a warp at a time
constexpr unsigned kTile = kWarps * kUnit;
static_assert(kTile == kStepTokens, "a step is a tile");
constexpr unsigned kStages = 3;                    // (a segment's first kStages - 1 tiles are brought by a warp each)
static_assert(kStages - 1 <= kWarps, "a warp for each of the first tiles");
constexpr unsigned kTileBytes = kTile * FMHA_KV4_TOKEN_BYTES;
constexpr float kSlack = 4.0f;
constexpr float kLeast = 1e-37f;                  // of a row's factor: times a masked score it is still -inf
constexpr float kVanishes = 2.98023223876953125e-8f;   // 2^-25: becomes 0 in f16
constexpr float kLn2 = 0.69314718055994531f;

// What a unit's 32 lanes work out for its tokens, one lane a token
struct TokenFactors {
    float4 k[kUnit];           // 2^(E - 127) of the four K blocks
    uint32_t r[kUnit / 2][4];  // [token pair][block]: V's factors over 2^(e - kUp), f16, of the pair's tokens in the operand's order
};

// Row r of the matrix instructions' token operands is token row_token(r) of its eight: neighbours in a pair (rows 2 j, 2 j + 1) stay neighbours, and the first tokens of the four
// pairs, which one load of V codes reads, are two even and two odd ones: their 64-byte rows then meet in the banks in twos, not in fours.
__device__ __forceinline__ uint32_t row_token(uint32_t r) { return r ^ ((r >> 1) & 1u); }

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Query rows of an item as the matrix instruction's operand: rows gid of each of NT groups of eight, elements 32 blk + 8 tig .. + 7 of each block. Two and more groups keep
// the elements in shared memory (a lane reads back what it would hold): the registers are O's.
template <int NT>
struct QueryRows {
    static constexpr bool kShared = NT >= 2;
    uint4 q[kShared ? 1 : NT][4];   // [group][block]
    float factor[NT][2];            // of the columns 2 tig, 2 tig + 1: scale * log2(e) * the power of two taken out
    uint32_t limit[NT][2];          // tokens that the columns see
};
template <int NT>
__device__ __forceinline__ void load_rows(QueryRows<NT>& x, uint4* q_shared, const Kv4AttendParams& p, uint32_t b, uint32_t head, uint32_t row0, uint32_t length, uint32_t n) {
    const unsigned lane = threadIdx.x & 31u, gid = lane >> 2, tig = lane & 3u;
    const uint32_t rows = p.S * p.group;
#pragma unroll
    for (int g = 0; g < NT; ++g) {
        const uint32_t row = row0 + 8u * g + gid, i = row / p.group;
        const bool live = row < rows && i < n;
        uint4 raw[4];
        uint32_t amax = 0;
#pragma unroll
        for (int blk = 0; blk < 4; ++blk) {
            raw[blk] = make_uint4(0u, 0u, 0u, 0u);
            if (live) raw[blk] = ld_v4(p.q.data + b * p.q.stride_b + i * p.q.stride_s + (head * p.group + row % p.group) * p.q.stride_h + 64u * blk + 16u * tig);
            const uint32_t w[4] = {raw[blk].x, raw[blk].y, raw[blk].z, raw[blk].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) amax = max(amax, max((w[k] << 16) & 0x7FFFFFFFu, w[k] & 0x7FFF0000u));
        }
        amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
        const float2 f = row_factors(amax);
#pragma unroll
        for (int blk = 0; blk < 4; ++blk) {
            uint32_t w[4] = {raw[blk].x, raw[blk].y, raw[blk].z, raw[blk].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = pack_f16x2(__uint_as_float(w[k] << 16) * f.x, __uint_as_float(w[k] & 0xFFFF0000u) * f.x);
            const uint4 packed = make_uint4(w[0], w[1], w[2], w[3]);
            if (QueryRows<NT>::kShared) q_shared[(g * 4 + blk) * 32 + lane] = packed;   // (all warps write the same)
            else x.q[QueryRows<NT>::kShared ? 0 : g][blk] = packed;
        }
        const uint32_t lim = !live ? 0u : p.causal ? length - n + i + 1u : length;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int src = static_cast<int>(2u * tig + j) * 4;   // a lane that holds that row
            x.factor[g][j] = fmaxf(__shfl_sync(0xFFFFFFFFu, f.y, src) * p.scale_log2, kLeast);
            x.limit[g][j] = __shfl_sync(0xFFFFFFFFu, lim, src);
        }
    }
    if (QueryRows<NT>::kShared) __syncwarp();
}

// S^T of 32 tokens: the K codes at `codes` (row-major, 64 bytes a token), the second 16 tokens `granule` bytes on, factors f[0 .. 31]
template <int NT>
__device__ __forceinline__ void scores(float (&s)[2][NT][4], const uint8_t* codes, uint32_t granule, const float4* f, const QueryRows<NT>& x, const uint4* q_shared) {
    const unsigned lane = threadIdx.x & 31u, gid = lane >> 2, tig = lane & 3u;
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t row = row_token(gid);
    uint4 top[2], bot[2];
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
        top[gr] = *reinterpret_cast<const uint4*>(codes + gr * granule + 64u * row + 16u * tig);
        bot[gr] = *reinterpret_cast<const uint4*>(codes + gr * granule + 64u * (row + 8u) + 16u * tig);
    }
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
        uint4 q[NT];
#pragma unroll
        for (int g = 0; g < NT; ++g) q[g] = QueryRows<NT>::kShared ? q_shared[(g * 4 + blk) * 32 + lane] : x.q[QueryRows<NT>::kShared ? 0 : g][blk];
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
            const uint32_t t0 = blk < 2 ? top[gr].x : top[gr].y, t1 = blk < 2 ? top[gr].z : top[gr].w, b0 = blk < 2 ? bot[gr].x : bot[gr].y, b1 = blk < 2 ? bot[gr].z : bot[gr].w;
            uint32_t a[8];
            if (blk & 1) {
                a[0] = e2m1x2_to_f16x2<2>(t0), a[1] = e2m1x2_to_f16x2<2>(b0), a[2] = e2m1x2_to_f16x2<3>(t0), a[3] = e2m1x2_to_f16x2<3>(b0);
                a[4] = e2m1x2_to_f16x2<2>(t1), a[5] = e2m1x2_to_f16x2<2>(b1), a[6] = e2m1x2_to_f16x2<3>(t1), a[7] = e2m1x2_to_f16x2<3>(b1);
            } else {
                a[0] = e2m1x2_to_f16x2<0>(t0), a[1] = e2m1x2_to_f16x2<0>(b0), a[2] = e2m1x2_to_f16x2<1>(t0), a[3] = e2m1x2_to_f16x2<1>(b0);
                a[4] = e2m1x2_to_f16x2<0>(t1), a[5] = e2m1x2_to_f16x2<0>(b1), a[6] = e2m1x2_to_f16x2<1>(t1), a[7] = e2m1x2_to_f16x2<1>(b1);
            }
            const float *ft = reinterpret_cast<const float*>(f + 16 * gr + row), *fb = reinterpret_cast<const float*>(f + 16 * gr + row + 8u);
            const float st = ft[blk], sb = fb[blk];
#pragma unroll
            for (int g = 0; g < NT; ++g) {
                float d[4];
                mma_f16(d, a[0], a[1], a[2], a[3], q[g].x, q[g].y, zero);
                mma_f16(d, a[4], a[5], a[6], a[7], q[g].z, q[g].w, d);
                if (blk == 0) {
                    s[gr][g][0] = d[0] * st, s[gr][g][1] = d[1] * st, s[gr][g][2] = d[2] * sb, s[gr][g][3] = d[3] * sb;
                } else {
                    s[gr][g][0] = fmaf(d[0], st, s[gr][g][0]), s[gr][g][1] = fmaf(d[1], st, s[gr][g][1]);
                    s[gr][g][2] = fmaf(d[2], sb, s[gr][g][2]), s[gr][g][3] = fmaf(d[3], sb, s[gr][g][3]);
                }
            }
        }
    }
}

// One lane a token: its factors, from the unit's scale bytes; e of the unit. A token behind the length is masked later; its V factors have to be finite.
__device__ __forceinline__ int token_factors(TokenFactors& f, uint32_t kw, uint32_t vw, bool live) {
    const unsigned t = threadIdx.x & 31u;
    f.k[t] = make_float4(scale_f32(kw, 0), scale_f32(kw, 1), scale_f32(kw, 2), scale_f32(kw, 3));
    if (!live) vw = 0u;
    const uint32_t largest = largest_byte(vw);
    uint32_t met = largest;
    if (largest == 255u) met = largest_byte(vw & ~nan_bytes(vw));   // (a token's other blocks count)
    const int e = group_exponent(__reduce_max_sync(0xFFFFFFFFu, met));
    const ValueFactors vf = value_factors(vw, largest, e);
    // an even lane takes blocks 0 and 1 of its pair, the odd one 2 and 3; pairs whose operand rows are the other way round are stored so
    const bool odd = t & 1u, flip = (t >> 1) & 1u;
    const uint32_t mine = odd ? vf.r23 : vf.r01, got = __shfl_xor_sync(0xFFFFFFFFu, odd ? vf.r01 : vf.r23, 1);
    const uint32_t first = odd != flip ? got : mine, second = odd != flip ? mine : got;
    *reinterpret_cast<uint2*>(&f.r[t >> 1][odd ? 2 : 0]) = make_uint2(__byte_perm(first, second, 0x5410), __byte_perm(first, second, 0x7632));
    return e;
}

template <int NT>
struct alignas(128) CtaShared {
    uint8_t ring[kStages][kTileBytes];
    TokenFactors f[kWarps];
    uint4 q[QueryRows<NT>::kShared ? NT * 4 * 32 : 1];
    float m[kWarps][8 * NT], l[kWarps][8 * NT];
    Sums part[kWarps];
    unsigned long long full[kStages], empty[kStages];
    uint32_t failed;
};

// What stands in for a page that the pool does not have: codes of 0, scales of 255, so that everything in it is NaN
template <int kPage>
struct LostPage {
    uint8_t bytes[FMHA_KV4_TOKEN_BYTES * kPage];
    constexpr LostPage() : bytes{} {
        for (int i = 128 * kPage; i < 136 * kPage; ++i) bytes[i] = 0xFF;
    }
};
struct LostPages {
    alignas(16) LostPage<16> p16;
    alignas(16) LostPage<32> p32;
    alignas(16) LostPage<64> p64;
    alignas(16) LostPage<128> p128;
};
__device__ const LostPages kNowhere;

// 32 tokens: scores, softmax, and their part of O
template <int NT, bool kEdge>
__device__ __forceinline__ void attend_unit(float (&o)[NT][8][4], float (&m)[NT][2], float (&l)[NT][2], const QueryRows<NT>& x, const uint8_t* k_codes, const uint8_t* v_codes, uint32_t granule,
                                            const TokenFactors& f, int e, uint32_t tok0, const uint4* q_shared, float* kept_scores, uint32_t kept_rows, uint32_t length, Exponents& seen) {
    seen.add(e);
    const unsigned lane = threadIdx.x & 31u, gid = lane >> 2, tig = lane & 3u;
    const uint32_t row = row_token(gid);
    float s[2][NT][4];
    scores<NT>(s, k_codes, granule, f.k, x, q_shared);
    const float ef = static_cast<float>(e), inv = seen.wide ? 0.0f : __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
#pragma unroll
        for (int g = 0; g < NT; ++g) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (kEdge && tok0 + 16u * gr + 8u * (i >> 1) + row >= x.limit[g][i & 1]) s[gr][g][i] = -INFINITY;
            }
        }
    }
    if (NT == 1 && kept_scores != nullptr && 2u * tig < kept_rows) {   // for the attention weights: scores in base 2, [token][rows]
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t t = 16u * gr + 8u * i + row;
                if (kEdge && tok0 + t >= length) continue;
                *reinterpret_cast<float2*>(kept_scores + t * kept_rows + 2u * tig) = make_float2(s[gr][0][2 * i] * x.factor[0][0], s[gr][0][2 * i + 1] * x.factor[0][1]);
            }
        }
    }
    bool over = seen.wide;
    float top[NT][2];
#pragma unroll
    for (int g = 0; g < NT; ++g) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            top[g][j] = fmaf(fmaxf(fmaxf(s[0][g][j], s[0][g][2 + j]), fmaxf(s[1][g][j], s[1][g][2 + j])), x.factor[g][j], ef);
            over |= top[g][j] > m[g][j] + kSlack;
        }
    }
    if (__any_sync(0xFFFFFFFFu, over)) {
#pragma unroll
        for (int g = 0; g < NT; ++g) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float t = top[g][j];
                t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 4));
                t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 8));
                t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 16));
                t = fmaxf(t, m[g][j]);
                const float c = ex2(m[g][j] - t), cl = sum_factor(l[g][j], m[g][j] - t);
                m[g][j] = t;
                l[g][j] *= cl;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[g][i][j] *= c, o[g][i][2 + j] *= c;
            }
        }
        if (seen.wide) {
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
#pragma unroll
                for (int g = 0; g < NT; ++g) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float up = static_cast<float>(kWide) - m[g][j];
                        l[g][j] = fmaf(ex2_wide(fmaf(s[gr][g][j], x.factor[g][j], up)) + ex2_wide(fmaf(s[gr][g][2 + j], x.factor[g][j], up)), kWideDown, l[g][j]);
                    }
                }
            }
        }
    }
    const uint32_t t0 = row_token(2u * tig), t1 = t0 ^ 1u;
    float sum[NT][2];
#pragma unroll
    for (int g = 0; g < NT; ++g) sum[g][0] = sum[g][1] = 0.0f;
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
        uint32_t pt[NT][2];
#pragma unroll
        for (int g = 0; g < NT; ++g) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = ex2(fmaf(s[gr][g][i], x.factor[g][i & 1], ef - m[g][i & 1]));
                sum[g][i & 1] += w[i];
                if (kEdge && w[i] <= kVanishes && s[gr][g][i] != -INFINITY) w[i] = -0.0f;   // seen all the same: 0 is for masked tokens
            }
            pt[g][0] = transpose_8x8(pack_f16x2(w[0], w[1]));
            pt[g][1] = transpose_8x8(pack_f16x2(w[2], w[3]));
        }
        const uint8_t* codes = v_codes + gr * granule + 8u * gid;
        const uint2 w0 = *reinterpret_cast<const uint2*>(codes + 64u * t0), w1 = *reinterpret_cast<const uint2*>(codes + 64u * t1);
        const uint2 w2 = *reinterpret_cast<const uint2*>(codes + 64u * (t0 + 8u)), w3 = *reinterpret_cast<const uint2*>(codes + 64u * (t1 + 8u));
        const uint4 ra = *reinterpret_cast<const uint4*>(f.r[8 * gr + tig]), rb = *reinterpret_cast<const uint4*>(f.r[8 * gr + 4 + tig]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t x0 = half ? w0.y : w0.x, x1 = half ? w1.y : w1.x, x2 = half ? w2.y : w2.x, x3 = half ? w3.y : w3.x;
            // bytes of (first token, second token) of a pair: even elements, odd elements
            const uint32_t ev0 = (x0 & 0x0F0F0F0Fu) | ((x1 << 4) & 0xF0F0F0F0u), od0 = ((x0 >> 4) & 0x0F0F0F0Fu) | (x1 & 0xF0F0F0F0u);
            const uint32_t ev1 = (x2 & 0x0F0F0F0Fu) | ((x3 << 4) & 0xF0F0F0F0u), od1 = ((x2 >> 4) & 0x0F0F0F0Fu) | (x3 & 0xF0F0F0F0u);
#pragma unroll
            for (int bb = 0; bb < 2; ++bb) {
                const int blk = 2 * half + bb;
                const uint32_t r0 = blk == 0 ? ra.x : blk == 1 ? ra.y : blk == 2 ? ra.z : ra.w, r1 = blk == 0 ? rb.x : blk == 1 ? rb.y : blk == 2 ? rb.z : rb.w;
                uint32_t a[8];
                if (bb) {
                    a[0] = e2m1x2_to_f16x2<2>(ev0), a[1] = e2m1x2_to_f16x2<2>(od0), a[2] = e2m1x2_to_f16x2<2>(ev1), a[3] = e2m1x2_to_f16x2<2>(od1);
                    a[4] = e2m1x2_to_f16x2<3>(ev0), a[5] = e2m1x2_to_f16x2<3>(od0), a[6] = e2m1x2_to_f16x2<3>(ev1), a[7] = e2m1x2_to_f16x2<3>(od1);
                } else {
                    a[0] = e2m1x2_to_f16x2<0>(ev0), a[1] = e2m1x2_to_f16x2<0>(od0), a[2] = e2m1x2_to_f16x2<0>(ev1), a[3] = e2m1x2_to_f16x2<0>(od1);
                    a[4] = e2m1x2_to_f16x2<1>(ev0), a[5] = e2m1x2_to_f16x2<1>(od0), a[6] = e2m1x2_to_f16x2<1>(ev1), a[7] = e2m1x2_to_f16x2<1>(od1);
                }
#pragma unroll
                for (int g = 0; g < NT; ++g) {
                    uint32_t p0 = mul_f16x2(pt[g][0], r0), p1 = mul_f16x2(pt[g][1], r1);
                    if (kEdge) {   // a weight of 0 (not -0) hides what it multiplies, NaN too
                        p0 = (pt[g][0] & 0xFFFFu ? p0 & 0xFFFFu : 0u) | (pt[g][0] & 0xFFFF0000u ? p0 & 0xFFFF0000u : 0u);
                        p1 = (pt[g][1] & 0xFFFFu ? p1 & 0xFFFFu : 0u) | (pt[g][1] & 0xFFFF0000u ? p1 & 0xFFFF0000u : 0u);
                    }
                    mma_f16(o[g][2 * blk], a[0], a[1], a[2], a[3], p0, p1, o[g][2 * blk]);
                    mma_f16(o[g][2 * blk + 1], a[4], a[5], a[6], a[7], p0, p1, o[g][2 * blk + 1]);
                }
            }
        }
    }
#pragma unroll
    for (int g = 0; g < NT; ++g) l[g][0] = fmaf(sum[g][0], inv, l[g][0]), l[g][1] = fmaf(sum[g][1], inv, l[g][1]);
}

template <int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : NT == 2 ? 3 : 2) kv4_attend_kernel(const __grid_constant__ Kv4AttendParams p) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    CtaShared<NT>& sh = *reinterpret_cast<CtaShared<NT>*>(smem_raw);
    const unsigned lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, gid = lane >> 2, tig = lane & 3u;
    const uint32_t full0 = sm100::smem_u32(sh.full), empty0 = sm100::smem_u32(sh.empty), ring0 = sm100::smem_u32(sh.ring[0]);
    if (threadIdx.x == 0u) {
        for (unsigned i = 0; i < kStages; ++i) sm100::mbar_init(full0 + 8u * i, 1u), sm100::mbar_init(empty0 + 8u * i, kWarps);
        sm100::fence_mbar_init();
        sh.failed = 0u;
    }
    pdl_launch();
    pdl_wait();
    __syncthreads();
    const Deal deal{8u * NT, 1u};
    const uint32_t all = sum_steps(p, deal, 0u, sh.part).all;
    const uint32_t n_work = workers(all, gridDim.x);
    clear_empty_entries(p, deal);
    if (threadIdx.x == 0u) begin_nothing(p, deal);
    if (blockIdx.x >= n_work) return;
    const uint32_t begin = run_begin(all, n_work, blockIdx.x), end = run_begin(all, n_work, blockIdx.x + 1u);
    uint32_t left = end - begin;
    Place at = find_step(p, deal, begin);
    // where this warp's 32 tokens of a tile lie in a stage: their K codes (the second 16 `granule` bytes on), from there to the V codes, and a lane's scales
    const uint32_t page = 1u << p.c.page_log2, record_bytes = FMHA_KV4_TOKEN_BYTES << p.c.page_log2, pages = static_cast<uint32_t>(p.c.pages), page_bytes = static_cast<uint32_t>(p.c.page_bytes);
    const uint32_t in_tile = warp * kUnit, unit_at = (in_tile >> p.c.page_log2) * record_bytes + (in_tile & (page - 1u)) * 64u;
    const uint32_t granule = page == 16u ? record_bytes : 1024u, v_codes = 64u * page;
    const uint32_t my_token = in_tile + lane, scales_at = (my_token >> p.c.page_log2) * record_bytes + 128u * page + (my_token & (page - 1u)) * 4u, v_scales = 4u * page;
    const uint8_t* nowhere = page == 16u ? kNowhere.p16.bytes : page == 32u ? kNowhere.p32.bytes : page == 64u ? kNowhere.p64.bytes : kNowhere.p128.bytes;
    const uint32_t kept_rows = (p.S * p.group + 1u) & ~1u;
    uint32_t stage = 0, phase = 0, filled = 0;   // of the next tile: its stage and the parity of the stage's barriers; tiles so far

    while (left > 0u) {
        const uint32_t pos = end - left;
        const Segment seg = next_segment(p, deal, at, left);
        if (threadIdx.x == 0u) begin_item(p, deal, seg, pos, all, n_work);
        const uint32_t b = seg.b, head = seg.head, row0 = seg.row0, first = seg.first, n_tiles = seg.steps;
        const uint32_t length = length_of(p.c, b), n_rows = count_of(p.counts, b, p.S, length);
        const int32_t* row_of_table = p.c.table + static_cast<size_t>(b) * p.c.table_width;
        const uint8_t* heads = p.c.pool + static_cast<size_t>(head) * record_bytes;
        // The copies of tile i of the segment: lane r brings the tile's r-th record; its page was looked up when the warp last had its turn
        int id = 0;
        auto look_up = [&](uint32_t i) {
            const uint32_t t = (first + i) * kTile + lane * page;
            if (i < n_tiles && lane * page < kTile && t < length) id = ld_i32(row_of_table + (t >> p.c.page_log2));
        };
        auto issue = [&](uint32_t i, uint32_t into) {
            const uint32_t t = (first + i) * kTile, records = min(max(kTile >> p.c.page_log2, 1u), (length - t + page - 1u) >> p.c.page_log2);
            if (lane == 0u) sm100::mbar_arrive_expect_tx(full0 + 8u * into, records * record_bytes);
            __syncwarp();
            if (lane < records) {
                const uint8_t* rec = static_cast<uint32_t>(id) < pages ? heads + static_cast<uint64_t>(static_cast<uint32_t>(id)) * page_bytes : nowhere;
                bulk_load(ring0 + into * kTileBytes + lane * record_bytes, rec, record_bytes, full0 + 8u * into);
            }
        };
        // warp w issues the tiles w, w + 4, ...; at the start of a segment the ring is empty
        look_up(warp);
        if (warp < kStages - 1u && warp < n_tiles) {
            issue(warp, (stage + warp) % kStages);
            look_up(warp + kWarps);
        }
        QueryRows<NT> x;
        load_rows<NT>(x, sh.q, p, b, head, row0, length, n_rows);
        uint32_t low = 0xFFFFFFFFu;   // tokens that every live column sees
#pragma unroll
        for (int g = 0; g < NT; ++g) {
#pragma unroll
            for (int j = 0; j < 2; ++j) low = min(low, x.limit[g][j] == 0u ? 0xFFFFFFFFu : x.limit[g][j]);
        }
        low = min(__reduce_min_sync(0xFFFFFFFFu, low), length);

        float o[NT][8][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int g = 0; g < NT; ++g) {
            m[g][0] = m[g][1] = kLowest;
            l[g][0] = l[g][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[g][i][0] = o[g][i][1] = o[g][i][2] = o[g][i][3] = 0.0f;
        }
        float* kept = p.scores == nullptr ? nullptr : p.scores + ((static_cast<size_t>(b) * p.c.HK + head) * (static_cast<size_t>(p.c.table_width) << p.c.page_log2) + first * kTile + in_tile) * kept_rows;
        bool ok = true;
        Exponents seen;
        uint32_t tok0 = first * kTile + in_tile, my_turn = (warp + 2u * kWarps - (kStages - 1u)) % kWarps;   // tiles until this warp brings one
        for (uint32_t i = 0; i < n_tiles; ++i, tok0 += kTile) {
            if (!sm100::mbar_wait(full0 + 8u * stage, phase, &sh.failed)) {
                ok = false;
                break;
            }
            if (tok0 < length) {
                const uint8_t* raw = sh.ring[stage];
                const int e = token_factors(sh.f[warp], *reinterpret_cast<const uint32_t*>(raw + scales_at), *reinterpret_cast<const uint32_t*>(raw + scales_at + v_scales), tok0 + lane < length);
                __syncwarp();
                const uint8_t* codes = raw + unit_at;
                if (tok0 + kUnit <= low) {
                    attend_unit<NT, false>(o, m, l, x, codes, codes + v_codes, granule, sh.f[warp], e, tok0, sh.q, kept == nullptr ? nullptr : kept + i * kTile * kept_rows, kept_rows, length, seen);
                } else {
                    attend_unit<NT, true>(o, m, l, x, codes, codes + v_codes, granule, sh.f[warp], e, tok0, sh.q, kept == nullptr ? nullptr : kept + i * kTile * kept_rows, kept_rows, length, seen);
                }
            }
            __syncwarp();   // this warp is done with the stage and its factors
            if (lane == 0u) sm100::mbar_arrive(empty0 + 8u * stage);
            // its turn to bring the tile kStages - 1 tiles on, into the stage of the tile before this one
            const uint32_t ahead = i + kStages - 1u, into = stage == 0u ? kStages - 1u : stage - 1u;
            if (my_turn-- == 0u) {
                my_turn = kWarps - 1u;
                if (ahead < n_tiles) {
                    // (the tile before this one has the phase before this stage's, or this stage's where it lies behind it; a stage's first tile finds it empty)
                    if (filled + i > 0u && !sm100::mbar_wait(empty0 + 8u * into, stage == 0u ? phase ^ 1u : phase, &sh.failed)) {
                        ok = false;
                        break;
                    }
                    issue(ahead, into);
                    look_up(ahead + kWarps);
                }
            }
            if (++stage == kStages) stage = 0u, phase ^= 1u;
        }
        filled += n_tiles;
        if (!ok) {
            if (lane == 0u) atomicOr(p.status, 1u);
        }

        // the warps' sums of the item come together
#pragma unroll
        for (int g = 0; g < NT; ++g) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                l[g][j] += __shfl_xor_sync(0xFFFFFFFFu, l[g][j], 4);
                l[g][j] += __shfl_xor_sync(0xFFFFFFFFu, l[g][j], 8);
                l[g][j] += __shfl_xor_sync(0xFFFFFFFFu, l[g][j], 16);
                if (gid == 0u) sh.m[warp][8 * g + 2 * tig + j] = m[g][j], sh.l[warp][8 * g + 2 * tig + j] = l[g][j];
            }
        }
        __syncthreads();
        if (sh.failed != 0u) return;   // (the same for all: it was raised in front of the barrier)
        const bool whole = n_tiles == seg.of;
        const uint32_t slot = first == 0u ? 1u : 0u;
        float* part = slot_of(p.ws, gridDim.x, blockIdx.x, slot, 8u * NT);
#pragma unroll
        for (int g = 0; g < NT; ++g) {
            float* mine_o = reinterpret_cast<float*>(sh.ring[0]) + warp * 1024u;   // [8 rows][128], the ring is empty
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = 8 * g + 2 * static_cast<int>(tig) + j;
                float top = fmaxf(fmaxf(sh.m[0][row], sh.m[1][row]), fmaxf(sh.m[2][row], sh.m[3][row]));
                const float f = ex2(m[g][j] - top);
#pragma unroll
                for (int blk = 0; blk < 4; ++blk) {
                    *reinterpret_cast<float4*>(mine_o + (2u * tig + j) * 128u + 32u * blk + 4u * gid) =
                        make_float4(o[g][2 * blk][j] * f, o[g][2 * blk][2 + j] * f, o[g][2 * blk + 1][j] * f, o[g][2 * blk + 1][2 + j] * f);
                }
            }
            __syncthreads();
            {
                const uint32_t r = threadIdx.x >> 4, d = (threadIdx.x & 15u) * 8u, row = row0 + 8u * g + r;
                const float top = fmaxf(fmaxf(sh.m[0][8 * g + r], sh.m[1][8 * g + r]), fmaxf(sh.m[2][8 * g + r], sh.m[3][8 * g + r]));
                float total = 0.0f, acc[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[k] = 0.0f;
#pragma unroll
                for (unsigned w = 0; w < kWarps; ++w) {
                    float l_w = sh.l[w][8 * g + r];
                    const float f = sum_factor(l_w, sh.m[w][8 * g + r] - top);
                    total = fmaf(l_w, f, total);
                    const float4* src = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sh.ring[0]) + w * 1024u + r * 128u + d);
                    const float4 a = src[0], c = src[1];
                    acc[0] += a.x, acc[1] += a.y, acc[2] += a.z, acc[3] += a.w, acc[4] += c.x, acc[5] += c.y, acc[6] += c.z, acc[7] += c.w;
                }
                if (row < p.S * p.group) {
                    if (whole) {
                        const bool none = total == 0.0f || row / p.group >= n_rows;   // sees nothing, or stands for nothing
                        const uint32_t i = row / p.group, h = head * p.group + row % p.group;
                        const float inv = kDown / total;
                        *reinterpret_cast<uint4*>(p.out + ((static_cast<size_t>(b) * p.S + i) * p.H + h) * 128u + d) =
                            none ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv), pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
                        if (p.lse != nullptr && d == 0u) p.lse[(static_cast<size_t>(b) * p.H + h) * p.S + i] = none ? -INFINITY : (top + lg2(total)) * kLn2;
                    } else {
                        float* at = part + (8u * g + r) * 128u + d;
                        *reinterpret_cast<float4*>(at) = make_float4(acc[0] * kDown, acc[1] * kDown, acc[2] * kDown, acc[3] * kDown);
                        *reinterpret_cast<float4*>(at + 4) = make_float4(acc[4] * kDown, acc[5] * kDown, acc[6] * kDown, acc[7] * kDown);
                        if (d == 0u) *reinterpret_cast<float2*>(part + 8u * NT * 128u + (8u * g + r) * 2u) = make_float2(top, total);
                    }
                }
            }
            __syncthreads();
        }
        // what the generic proxy read and wrote in the ring is behind the next copies into it
        sm100::fence_proxy_async_smem();
    }
}

// Puts the items together that more than one CTA of a launch worked on: blockIdx.x is an entry of the workspace, parts come from a launch of `grid` CTAs. kTogether: a CTA of so many
// warps has one row, its warps the parts in turn; 0: a warp has a row and all of its parts. Four parts are in flight at a time. (The CTAs take little shared memory on
// purpose: with 8 KB in place of 2 the attention kernel behind this one took 272 us in place of
// 236, 64 sequences of 16384 tokens.)
template <uint32_t kTogether>
__global__ void __launch_bounds__(kTogether ? 32 * kTogether : 256) kv4_combine_kernel(const __grid_constant__ Kv4AttendParams p, uint32_t rows, uint32_t row_tiles, uint32_t grid) {
    __shared__ float sm_m[kTogether ? kTogether : 1u], sm_l[kTogether ? kTogether : 1u];
    __shared__ float4 sm_o[kTogether ? 4 : 1][32];
    pdl_launch();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t r = kTogether ? blockIdx.y : blockIdx.y * (blockDim.x >> 5) + warp;
    const uint4 begun = ld_v4(begun_at(p.ws, blockIdx.x));
    const uint32_t entry = begun.x / p.c.HK, head = begun.x - entry * p.c.HK, b = entry / row_tiles, row = (entry - b * row_tiles) * rows + r, from = begun.y, last = begun.z;
    if (last == from || row >= p.S * p.group) return;   // (the same in all warps where they meet below)
    const uint32_t i = row / p.group, h = head * p.group + row % p.group;
    const bool sees = i < count_of(p.counts, b, p.S, length_of(p.c, b));
    constexpr uint32_t kStride = kTogether ? kTogether : 1u;
    float m = kLowest, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t w0 = from + (kTogether ? warp : 0u); sees && w0 <= last; w0 += 4u * kStride) {
        float pm[4], pl[4];
        uint4 raw[4];
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
            const uint32_t w = w0 + k * kStride;
            pm[k] = kLowest, pl[k] = 0.0f, raw[k] = make_uint4(0u, 0u, 0u, 0u);
            if (w <= last) {
                const float* src = slot_of(p.ws, grid, w, w == from ? 1u : 0u, rows);
                pm[k] = ld_f32(src + rows * 128u + 2u * r), pl[k] = ld_f32(src + rows * 128u + 2u * r + 1u);
                raw[k] = ld_v4(src + r * 128u + 4u * lane);
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
            const float top = fmaxf(m, pm[k]), a = ex2(m - top), c = ex2(pm[k] - top), al = sum_factor(l, m - top), cl = sum_factor(pl[k], pm[k] - top);
            m = top;
            l = fmaf(l, al, pl[k] * cl);
            o.x = fmaf(o.x, a, __uint_as_float(raw[k].x) * c), o.y = fmaf(o.y, a, __uint_as_float(raw[k].y) * c);
            o.z = fmaf(o.z, a, __uint_as_float(raw[k].z) * c), o.w = fmaf(o.w, a, __uint_as_float(raw[k].w) * c);
        }
    }
    if constexpr (kTogether != 0u) {   // four warps at a time hand over what they have
        if (lane == 0u) sm_m[warp] = m, sm_l[warp] = l;
        if (warp < 4u) sm_o[warp][lane] = o;
        __syncthreads();
        m = sm_m[0];
#pragma unroll
        for (uint32_t w = 1; w < kTogether; ++w) m = fmaxf(m, sm_m[w]);
        const float4 mine = o;
        l = 0.0f;
        o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (uint32_t w0 = 0; w0 < kTogether; w0 += 4u) {
            if (w0 > 0u) {
                __syncthreads();
                if (warp - w0 < 4u) sm_o[warp - w0][lane] = mine;
                __syncthreads();
            }
            if (warp == 0u) {
#pragma unroll
                for (uint32_t w = 0; w < 4u; ++w) {
                    float l_w = sm_l[w0 + w];
                    const float f = ex2(sm_m[w0 + w] - m), fl = sum_factor(l_w, sm_m[w0 + w] - m);
                    const float4 c = sm_o[w][lane];
                    l = fmaf(l_w, fl, l);
                    o.x = fmaf(c.x, f, o.x), o.y = fmaf(c.y, f, o.y), o.z = fmaf(c.z, f, o.z), o.w = fmaf(c.w, f, o.w);
                }
            }
        }
        if (warp != 0u) return;
    }
    const bool none = l == 0.0f;
    const float inv = none ? 0.0f : 1.0f / l;
    *reinterpret_cast<uint2*>(p.out + ((static_cast<size_t>(b) * p.S + i) * p.H + h) * 128u + 4u * lane) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
    if (p.lse != nullptr && lane == 0u) p.lse[(static_cast<size_t>(b) * p.H + h) * p.S + i] = none ? -INFINITY : (m + lg2(l)) * kLn2;
}

// The same for items of many rows of which most have one or two parts: a warp has kRows rows, whose parts come in together, one CTA's behind the other's, in the same order and to the same bits. With a warp a
// row there are kRows times as many CTAs, most of which find nothing to do (4-bit cache, 4096 rows over 8192 tokens, 128 items: 437.2 us and 434.8 so; 4 x 333 ragged rows, 128 items too: alike). Items of more
// parts have a warp a row, whose trips to memory are then under way beside one another (512 rows over 16384 tokens, 32 items: 97.7 us so and 92.7 with a warp a row, 4 x 100 ragged rows, 64 items: 89.3 and 85.6).
template <uint32_t kRows>
__global__ void __launch_bounds__(256) kv4_combine_rows_kernel(const __grid_constant__ Kv4AttendParams p, uint32_t rows, uint32_t row_tiles, uint32_t grid) {
    pdl_launch();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, r0 = (blockIdx.y * 8u + (threadIdx.x >> 5)) * kRows;
    const uint4 begun = ld_v4(begun_at(p.ws, blockIdx.x));
    const uint32_t entry = begun.x / p.c.HK, head = begun.x - entry * p.c.HK, b = entry / row_tiles, row0 = (entry - b * row_tiles) * rows + r0, from = begun.y, last = begun.z;
    if (last == from || row0 >= p.S * p.group) return;
    const uint32_t live = count_of(p.counts, b, p.S, length_of(p.c, b)) * p.group;   // rows that see something
    float m[kRows], l[kRows];
    float4 o[kRows];
#pragma unroll
    for (uint32_t y = 0; y < kRows; ++y) m[y] = kLowest, l[y] = 0.0f, o[y] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (uint32_t w = from; w <= last; ++w) {
        const float* src = slot_of(p.ws, grid, w, w == from ? 1u : 0u, rows);
        float pm[kRows], pl[kRows];
        uint4 raw[kRows];
#pragma unroll
        for (uint32_t y = 0; y < kRows; ++y) {
            pm[y] = kLowest, pl[y] = 0.0f, raw[y] = make_uint4(0u, 0u, 0u, 0u);
            if (row0 + y < live) {
                pm[y] = ld_f32(src + rows * 128u + 2u * (r0 + y)), pl[y] = ld_f32(src + rows * 128u + 2u * (r0 + y) + 1u);
                raw[y] = ld_v4(src + (r0 + y) * 128u + 4u * lane);
            }
        }
#pragma unroll
        for (uint32_t y = 0; y < kRows; ++y) {
            const float top = fmaxf(m[y], pm[y]), a = ex2(m[y] - top), c = ex2(pm[y] - top), al = sum_factor(l[y], m[y] - top), cl = sum_factor(pl[y], pm[y] - top);
            m[y] = top;
            l[y] = fmaf(l[y], al, pl[y] * cl);
            o[y].x = fmaf(o[y].x, a, __uint_as_float(raw[y].x) * c), o[y].y = fmaf(o[y].y, a, __uint_as_float(raw[y].y) * c);
            o[y].z = fmaf(o[y].z, a, __uint_as_float(raw[y].z) * c), o[y].w = fmaf(o[y].w, a, __uint_as_float(raw[y].w) * c);
        }
    }
#pragma unroll
    for (uint32_t y = 0; y < kRows; ++y) {
        const uint32_t row = row0 + y, i = row / p.group, h = head * p.group + row - i * p.group;
        if (row >= p.S * p.group || r0 + y >= rows) break;
        const bool none = l[y] == 0.0f;
        const float inv = none ? 0.0f : 1.0f / l[y];
        *reinterpret_cast<uint2*>(p.out + ((static_cast<size_t>(b) * p.S + i) * p.H + h) * 128u + 4u * lane) = make_uint2(pack_bf16x2(o[y].x * inv, o[y].y * inv), pack_bf16x2(o[y].z * inv, o[y].w * inv));
        if (p.lse != nullptr && lane == 0u) p.lse[(static_cast<size_t>(b) * p.H + h) * p.S + i] = none ? -INFINITY : (m[y] + lg2(l[y])) * kLn2;
    }
}

}  // namespace

// what a launch of `grid` CTAs with items of `slots` rows (8 to 32, one row tile a sequence) or of `per` rows left in p.ws
cudaError_t launch_combine_few(const Kv4AttendParams& p, uint32_t slots, uint32_t grid, cudaStream_t stream) {
    // 4 warps have 16 parts in flight; where an item has more on average, 16 warps (5 rows over 65536 tokens, 74 parts: 28 us in place of 36)
    const uint32_t rows = p.S * p.group, entries = begun_entries(p.c, 1u, grid), some = rows < slots ? rows : slots;
    if (grid / entries > 16u) return kv4_launch(kv4_combine_kernel<16>, dim3(entries, some), 512u, 0, stream, p, slots, 1u, grid);
    return kv4_launch(kv4_combine_kernel<4>, dim3(entries, some), 128u, 0, stream, p, slots, 1u, grid);
}
cudaError_t launch_combine_many(const Kv4AttendParams& p, uint32_t per, uint32_t row_tiles, uint32_t grid, cudaStream_t stream, bool together) {
    constexpr uint32_t kRows = 4;
    const uint32_t rows = p.S * p.group, most = rows < per ? rows : per, entries = begun_entries(p.c, row_tiles, grid), parts = grid / entries;
    const uint64_t items = static_cast<uint64_t>(p.c.B) * p.c.HK * row_tiles;
    if (!together && 2u * items > grid) return kv4_launch(kv4_combine_rows_kernel<kRows>, dim3(entries, (most + 8u * kRows - 1u) / (8u * kRows)), 256u, 0, stream, p, per, row_tiles, grid);
    if (!together) return kv4_launch(kv4_combine_kernel<0>, dim3(entries, (most + 7u) / 8u), 256u, 0, stream, p, per, row_tiles, grid);
    if (parts > 16u) return kv4_launch(kv4_combine_kernel<16>, dim3(entries, most), 512u, 0, stream, p, per, row_tiles, grid);
    return kv4_launch(kv4_combine_kernel<4>, dim3(entries, most), 128u, 0, stream, p, per, row_tiles, grid);
}

namespace {

// Rows of a KV head up to which this kernel is taken; more go to the tensor cores' tiles of 128 rows. 16 sequences of 4096 tokens: 20 rows 49 us here and 100 there, 32 rows 65 and 100;
// one of 65536: 28 and 66, 34 and 67. (The registers end at 32: two passes over the cache would cost as much as the tiles do from about 48 rows on.)
constexpr uint32_t kMostFew = 32;

uint32_t groups_of(uint32_t rows) { return (rows + 7u) / 8u; }

uint32_t attend_grid(const Kv4View& c, uint32_t groups) {
    const unsigned long long tiles = ((static_cast<unsigned long long>(c.table_width) << c.page_log2) + kTile - 1u) / kTile, per_sm = groups == 1u ? 4u : groups == 2u ? 3u : 2u;
    const unsigned long long most = tiles * c.B * c.HK, full = per_sm * static_cast<unsigned long long>(current_sm_count());
    return static_cast<uint32_t>(most < full ? (most ? most : 1ull) : full);
}

template <int NT>
cudaError_t launch_rows(const Kv4AttendParams& p, cudaStream_t stream) {
    const uint32_t grid = attend_grid(p.c, NT);
    const size_t smem = sizeof(CtaShared<NT>);
    static std::atomic<bool> set[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_relaxed)) {
        e = cudaFuncSetAttribute(kv4_attend_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_relaxed);
    }
    e = kv4_launch(kv4_attend_kernel<NT>, dim3(grid), kThreads, smem, stream, p);
    return e != cudaSuccess ? e : launch_combine_few(p, 8u * NT, grid, stream);
}

cudaError_t launch_many(const Kv4AttendParams& p, cudaStream_t stream) {
    const uint32_t rows = p.S * p.group, per = kv4_prefill_rows(), row_tiles = (rows + per - 1u) / per;
    const cudaError_t e = launch_kv4_prefill(p, row_tiles, stream);
    return e != cudaSuccess ? e : launch_combine_many(p, per, row_tiles, kv4_prefill_grid(), stream);
}

uint64_t partial_bytes(const Kv4View& c, uint32_t rows) {
    if (rows > kMostFew) return kv4_partial_bytes(kv4_prefill_grid(), kv4_prefill_rows());
    return kv4_partial_bytes(attend_grid(c, groups_of(rows)), 8u * groups_of(rows));
}
uint64_t lse_bytes(const Kv4View& c, uint32_t S, uint32_t H) { return (static_cast<uint64_t>(c.B) * S * H * 4u + 15u) & ~15ull; }
// Up to 8 rows leave their scores for the weights, at 4 bytes a row and token (16 sequences of 4096 tokens: 4 rows 38 us, 69 where they are computed again; 8 rows 42 and 71). More rows
// would fill the memory with scores, 4 bytes against the 17 of a token's K and V per row in the group; they are computed again.
uint64_t score_bytes(const Kv4View& c, uint32_t rows) {
    return rows > 8u ? 0u : (static_cast<uint64_t>(c.B) * c.HK * c.table_width << c.page_log2) * ((rows + 1u) & ~1u) * 4u;
}

}  // namespace

uint64_t kv4_attend_workspace(const Kv4View& c, uint32_t S, uint32_t H, bool weights, bool lse) {
    const uint32_t rows = S * (H / c.HK);
    return partial_bytes(c, rows) + (weights ? score_bytes(c, rows) + (lse ? 0u : lse_bytes(c, S, H)) : 0u);
}

cudaError_t launch_kv4_attend(const Kv4AttendParams& params, cudaStream_t stream) {
    Kv4AttendParams p = params;
    const uint32_t rows = p.S * p.group;
    p.scores = nullptr;
    if (p.weights != nullptr) {   // the weights go by the rows' log-sum-exps
        uint8_t* more = reinterpret_cast<uint8_t*>(p.ws) + partial_bytes(p.c, rows);
        if (rows <= 8u) p.scores = reinterpret_cast<float*>(more);
        if (p.lse == nullptr) p.lse = reinterpret_cast<float*>(more + score_bytes(p.c, rows));
    }
    const uint32_t groups = groups_of(rows);
    const cudaError_t e = rows > kMostFew ? launch_many(p, stream) : groups == 1u ? launch_rows<1>(p, stream) : groups == 2u ? launch_rows<2>(p, stream) : groups == 3u ? launch_rows<3>(p, stream) : launch_rows<4>(p, stream);
    return e != cudaSuccess || p.weights == nullptr ? e : launch_kv4_weigh(p, stream);
}

}  // namespace b200mx
