// Attention of few query rows over the 8-bit cache: decode, and drafts of a few tokens, up to 32 rows of a KV head (kv8_prefill.cu has more).
//
// Work. An item is one sequence and KV head. Steps of 128 tokens of all items, in order, are dealt out in equal runs to the CTAs, from the lengths on the device; an item that more
// than one CTA worked on is put together from f32 partials by the combine kernel (kv4_schedule.cuh, kv4_attend.cu).
//
// A warp has 32 tokens, two blocks, of each step, and a ring of its own in shared memory that whole blocks come to (cp.async.bulk, 8224 bytes at a time; one copy, or two where pages
// hold 16 tokens). Nothing but the item's end makes the warps wait for one another. Both products are computed transposed, so that the tokens are the rows of the matrix
// instruction and the few query rows its 8 columns:
//   S^T [16 tokens x 8 rows] = K [16 x 128] Q^T       K's codes become f16 two at a time, exactly, and the block's scale multiplies the sum with the row's factor
//   O^T [128 x 8 rows] += V^T [128 x 16 tokens] P^T   P goes from S^T's layout to the operand's by an 8 x 8 transpose between lanes; V's scale is part of the exponent
// The cache keeps K's elements and V's pairs of tokens where a lane's operands are; which element of a head is which k or row of an instruction is of no matter to the products, Q and O
// are permuted alike.
//
// Softmax in base 2 with a running reference per row: w = 2^(c s + e - M), e the exponent of V's scale, goes into the second product, w 2^-e into the sum. M follows the largest c s + e,
// less 2^kUp, since f16 has more room above 1 than a weight needs; it moves when a value exceeds it by another 2^kSlack, by a vote of the warp.
//
// Bound by bytes where sequences are long: 64 of 16384 tokens, 8 KV heads, 4 rows each, 342 to 352 us by box for 2.16 GB, 6.1 to 6.3 TB/s, 0.94 to 0.96 of the copy rate (16 of them: issue 31 %, tensor pipe
// 20 %, 8 warps an SM).
// Ragged and short ones by what a change of item costs: 24 of up to 32768 tokens in pages of 16, 20 rows each, 61 us where the bytes take 32. Two CTAs an SM: three stages of four warps are 99 KB.
#include "kv4_schedule.cuh"
#include "kv8.cuh"
#include "ptx_sm100.cuh"

#include <atomic>

namespace b200mx {

namespace {

using namespace kv8;

constexpr uint32_t kWarps = 4, kThreads = kWarps * 32;
constexpr uint32_t kUnit = 32, kUnitBytes = kUnit / kBlockTokens * kBlockBytes;   // a warp's tokens at a time
static_assert(kWarps * kUnit == kStepTokens, "a step is a unit of each warp");
constexpr uint32_t kStages = 3;
constexpr uint32_t kExtra = 4;   // what a CTA's change to another item costs, in steps (24 ragged drafts of 5 rows in pages of 16: 78 us without, 65, 59, 59 with 2, 4, 6)
constexpr int kTogether = 3;                      // groups of eight rows up to which a unit's two blocks are worked on together
constexpr float kUp = 10.0f, kSlack = 4.0f;
constexpr float kLeast = 1e-37f;                  // of a row's factor: times a masked score it is still -inf
constexpr float kLn2 = 0.69314718055994531f;

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Query rows of an item as the matrix instruction's operand: rows gid of each of NT groups of eight, elements 32 tig .. + 31. Two and more groups keep the elements in shared
// memory (a lane reads back what it would hold): the registers are O's.
template <int NT>
struct QueryRows {
    static constexpr bool kShared = NT >= 2;
    uint4 q[kShared ? 1 : NT][4];   // [group][8 elements: two of the products]
    static constexpr bool kAway = NT >= 4;   // so do these
    float factors[kAway ? 1 : NT][2];        // of the columns 2 tig, 2 tig + 1: scale * log2(e) * the power of two taken out
    uint32_t limits[kAway ? 1 : NT][2];      // tokens that the columns see
    float* away;                             // [group][column of 8] factors, then limits
    __device__ __forceinline__ float factor(int g, int j) const { return kAway ? away[8 * g + 2 * (threadIdx.x & 3u) + j] : factors[kAway ? 0 : g][j]; }
    __device__ __forceinline__ uint32_t limit(int g, int j) const { return kAway ? __float_as_uint(away[8 * NT + 8 * g + 2 * (threadIdx.x & 3u) + j]) : limits[kAway ? 0 : g][j]; }
};
template <int NT>
__device__ __forceinline__ void load_rows(QueryRows<NT>& x, uint4* q_shared, const Kv8AttendParams& p, uint32_t b, uint32_t head, uint32_t row0, uint32_t length, uint32_t n) {
    const unsigned lane = threadIdx.x & 31u, gid = lane >> 2, tig = lane & 3u;
    const uint32_t rows = p.S * p.group;
#pragma unroll
    for (int g = 0; g < NT; ++g) {
        const uint32_t row = row0 + 8u * g + gid, i = row / p.group;
        const bool live = row < rows && i < n;
        uint4 raw[4];
        uint32_t amax = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            raw[k] = make_uint4(0u, 0u, 0u, 0u);
            if (live) raw[k] = ld_v4(p.q.data + b * p.q.stride_b + i * p.q.stride_s + (head * p.group + row % p.group) * p.q.stride_h + 64u * tig + 16u * k);
            const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
            for (int y = 0; y < 4; ++y) amax = max(amax, max((w[y] << 16) & 0x7FFFFFFFu, w[y] & 0x7FFF0000u));
        }
        amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
        const float2 f = row_factors(amax);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
            for (int y = 0; y < 4; ++y) w[y] = pack_f16x2(__uint_as_float(w[y] << 16) * f.x, __uint_as_float(w[y] & 0xFFFF0000u) * f.x);
            const uint4 packed = make_uint4(w[0], w[1], w[2], w[3]);
            if (QueryRows<NT>::kShared) q_shared[(g * 4 + k) * 32 + lane] = packed;   // (all warps write the same)
            else x.q[QueryRows<NT>::kShared ? 0 : g][k] = packed;
        }
        const uint32_t lim = !live ? 0u : p.causal ? length - n + i + 1u : length;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int src = static_cast<int>(2u * tig + j) * 4;   // a lane that holds that row
            const float factor = __shfl_sync(0xFFFFFFFFu, f.y, src) * p.scale_log2;
            const uint32_t seen = __shfl_sync(0xFFFFFFFFu, lim, src);
            if constexpr (QueryRows<NT>::kAway) x.away[8 * g + 2 * tig + j] = factor, x.away[8 * NT + 8 * g + 2 * tig + j] = __uint_as_float(seen);   // (all warps write the same)
            else x.factors[g][j] = factor, x.limits[g][j] = seen;
        }
    }
    if (QueryRows<NT>::kShared) __syncwarp();
}

template <int NT>
struct alignas(128) CtaShared {
    uint8_t ring[kWarps][kStages][kUnitBytes];
    union {
        uint4 q[QueryRows<NT>::kShared ? NT * 4 * 32 : 1];
        float o[2][8 * 128];   // where the warps' parts of an item's O come together, when its rows are no longer needed
    };
    float away[QueryRows<NT>::kAway ? 16 * NT : 1];
    float m[kWarps][8 * NT], l[kWarps][8 * NT];
    Sums part[kWarps];
    unsigned long long full[kWarps][kStages];
    uint32_t failed;
};

// What stands in for the blocks of a page that the pool does not have: tokens without numbers
struct LostBlocks {
    alignas(16) uint8_t bytes[kUnitBytes];
    constexpr LostBlocks() : bytes{} {
        for (uint32_t b = 0; b < kUnitBytes; b += kBlockBytes) {
            bytes[b + kMeta + 2] = bytes[b + kMeta + kVScale + 2] = 0x80, bytes[b + kMeta + 3] = bytes[b + kMeta + kVScale + 3] = 0x3F;   // 1.0
            for (uint32_t i = 0; i < 4; ++i) bytes[b + kMeta + kMasks + i] = 0xFF;
        }
    }
};
__device__ const LostBlocks kNowhere;

// G blocks of 16 tokens: scores, softmax, and their part of O: o[g][i][j], d = 16 gid + 2 i and, from [2 + j], the next, of the column 2 tig + j
template <int NT, int G, bool kEdge>
__device__ __forceinline__ void attend_blocks(float (&o)[NT][8][4], float (&m)[NT][2], float (&l)[NT][2], const QueryRows<NT>& x, const uint8_t* unit, uint32_t tok0, const uint4* q_shared, uint32_t length, Exponents& seen) {
    constexpr int kSums = NT <= 2 ? 2 : 1;
    const unsigned lane = threadIdx.x & 31u, gid = lane >> 2, tig = lane & 3u;
    float s[G][NT][4];
    uint4 meta[G];
    bool dead[G];   // a block behind the length: whatever it holds
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
        meta[gr] = *reinterpret_cast<const uint4*>(unit + gr * kBlockBytes + kMeta);
        dead[gr] = kEdge && tok0 + 16u * gr >= length;
        if (dead[gr]) meta[gr] = make_uint4(0x3F800000u, 0x3F800000u, 0u, 0u);
    }
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
        const uint8_t* row = unit + gr * kBlockBytes + 128u * gid;
        uint4 top[2], bot[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t at = ((2u * tig + h) ^ k_swap(gid)) << 4;
            top[h] = *reinterpret_cast<const uint4*>(row + at);
            bot[h] = *reinterpret_cast<const uint4*>(row + 1024u + at);
        }
        float d[NT][kSums][4];   // two sums, of every other product, where the registers allow it
#pragma unroll
        for (int g = 0; g < NT; ++g) {
#pragma unroll
            for (int y = 0; y < 4; ++y) d[g][0][y] = d[g][kSums - 1][y] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t t[2] = {k & 1 ? top[k >> 1].z : top[k >> 1].x, k & 1 ? top[k >> 1].w : top[k >> 1].y}, u[2] = {k & 1 ? bot[k >> 1].z : bot[k >> 1].x, k & 1 ? bot[k >> 1].w : bot[k >> 1].y};
            uint4 q[NT];
#pragma unroll
            for (int g = 0; g < NT; ++g) q[g] = QueryRows<NT>::kShared ? q_shared[(g * 4 + k) * 32 + lane] : x.q[QueryRows<NT>::kShared ? 0 : g][k];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const uint32_t a0 = e4m3x2_lo(t[y]), a1 = e4m3x2_lo(u[y]), a2 = e4m3x2_hi(t[y]), a3 = e4m3x2_hi(u[y]);
#pragma unroll
                for (int g = 0; g < NT; ++g) mma_f16(d[g][y % kSums], a0, a1, a2, a3, y ? q[g].z : q[g].x, y ? q[g].w : q[g].y, d[g][y % kSums]);
            }
        }
#pragma unroll
        for (int g = 0; g < NT; ++g) {
#pragma unroll
            for (int y = 0; y < 4; ++y) s[gr][g][y] = kSums == 2 ? d[g][0][y] + d[g][kSums - 1][y] : d[g][0][y];
        }
    }
    if (meta[0].z | meta[G - 1].z) {   // tokens without numbers (the same in all lanes)
#pragma unroll 1
        for (uint32_t t = 0; t < G * kBlockTokens; ++t) {
            const uint32_t mask = (t < 16u ? meta[0].z : meta[G - 1].z) >> (t & 15u);
#pragma unroll
            for (int g = 0; g < NT; ++g) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if ((mask & 0x10000u) != 0u && tok0 + t < x.limit(g, j)) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) o[g][i][j] = o[g][i][2 + j] = __uint_as_float(0x7FC00000u);
                    }
#pragma unroll
                    for (int y = 0; y < 2 * G; ++y) {
                        if ((mask & 1u) != 0u && t == 8u * y + gid) s[y >> 1][g][2 * (y & 1) + j] = __uint_as_float(0x7FC00000u);
                    }
                }
            }
        }
    }
    if (kEdge) {
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
#pragma unroll
            for (int g = 0; g < NT; ++g) {
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    if (tok0 + 16u * gr + 8u * (y >> 1) + gid >= x.limit(g, y & 1)) s[gr][g][y] = -INFINITY;
                }
            }
        }
    }
    float c[G][NT][2], e[G], back[G];
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
        if (!dead[gr]) seen.add(exponent_of(meta[gr].y));
    }
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
        const int exponent = exponent_of(meta[gr].y);
        e[gr] = static_cast<float>(exponent), back[gr] = seen.wide ? 0.0f : power_of(-exponent);
#pragma unroll
        for (int g = 0; g < NT; ++g) {
#pragma unroll
            for (int j = 0; j < 2; ++j) c[gr][g][j] = fmaxf(x.factor(g, j) * __uint_as_float(meta[gr].x), kLeast);
        }
    }
    bool over = seen.wide;
    float top[NT][2];
#pragma unroll
    for (int g = 0; g < NT; ++g) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            top[g][j] = fmaf(fmaxf(s[0][g][j], s[0][g][2 + j]), c[0][g][j], e[0]) - kUp;
            if (G == 2) top[g][j] = fmaxf(top[g][j], fmaf(fmaxf(s[G - 1][g][j], s[G - 1][g][2 + j]), c[G - 1][g][j], e[G - 1]) - kUp);
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
                const float f = ex2(m[g][j] - t), fl = sum_factor(l[g][j], m[g][j] - t);
                m[g][j] = t;
                l[g][j] *= fl;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[g][i][j] *= f, o[g][i][2 + j] *= f;
            }
        }
        if (seen.wide) {
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
#pragma unroll
                for (int g = 0; g < NT; ++g) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float up = static_cast<float>(kWide) - m[g][j], more = ex2_wide(fmaf(s[gr][g][j], c[gr][g][j], up)) + ex2_wide(fmaf(s[gr][g][2 + j], c[gr][g][j], up));
                        l[g][j] = fmaf(more, kWideDown, l[g][j]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
        if (dead[gr]) continue;
        uint32_t pt[NT][2];
#pragma unroll
        for (int g = 0; g < NT; ++g) {
            float w[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) w[y] = ex2(fmaf(s[gr][g][y], c[gr][g][y & 1], e[gr] - m[g][y & 1]));
#pragma unroll
            for (int j = 0; j < 2; ++j) l[g][j] = fmaf(w[j] + w[2 + j], back[gr], l[g][j]);
            pt[g][0] = transpose_8x8(pack_f16x2(w[0], w[1]));
            pt[g][1] = transpose_8x8(pack_f16x2(w[2], w[3]));
        }
        const uint8_t* pair = unit + gr * kBlockBytes + kVCodes + 256u * tig;
        uint32_t keep[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};   // codes behind the length may be anything, NaN too
        if (kEdge) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const uint32_t t = tok0 + 16u * gr + 8u * y + 2u * tig;
                keep[y] = (t < length ? 0x00FF00FFu : 0u) | (t + 1u < length ? 0xFF00FF00u : 0u);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t at = ((2u * gid + h) ^ v_swap(tig)) << 4;
            const uint4 va = *reinterpret_cast<const uint4*>(pair + at), vb = *reinterpret_cast<const uint4*>(pair + 1024u + at);
            uint32_t a[4] = {va.x, va.y, va.z, va.w}, b[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (kEdge) a[i] &= keep[0], b[i] &= keep[1];
                const uint32_t a0 = e4m3x2_lo(a[i]), a1 = e4m3x2_hi(a[i]), a2 = e4m3x2_lo(b[i]), a3 = e4m3x2_hi(b[i]);
#pragma unroll
                for (int g = 0; g < NT; ++g) mma_f16(o[g][4 * h + i], a0, a1, a2, a3, pt[g][0], pt[g][1], o[g][4 * h + i]);
            }
        }
    }
}

// a unit's 32 tokens: both blocks together, or with many groups one after the other, which takes fewer registers
template <int NT, bool kEdge>
__device__ __forceinline__ void attend_unit(float (&o)[NT][8][4], float (&m)[NT][2], float (&l)[NT][2], const QueryRows<NT>& x, const uint8_t* unit, uint32_t tok0, const uint4* q_shared, uint32_t length, Exponents& seen) {
    if constexpr (NT <= kTogether) {
        attend_blocks<NT, 2, kEdge>(o, m, l, x, unit, tok0, q_shared, length, seen);
    } else {
#pragma unroll 1
        for (uint32_t b = 0; b < 2u && (!kEdge || tok0 + b * kBlockTokens < length); ++b) attend_blocks<NT, 1, kEdge>(o, m, l, x, unit + b * kBlockBytes, tok0 + b * kBlockTokens, q_shared, length, seen);
    }
}

constexpr uint32_t kCtasPerSm = 2;

template <int NT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) kv8_attend_kernel(const __grid_constant__ Kv8AttendParams p, bool whole_items) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    CtaShared<NT>& sh = *reinterpret_cast<CtaShared<NT>*>(smem_raw);
    const unsigned lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, gid = lane >> 2, tig = lane & 3u;
    const uint32_t full0 = sm100::smem_u32(sh.full[warp]), ring0 = sm100::smem_u32(sh.ring[warp][0]);
    if (lane == 0u) {
        for (uint32_t i = 0; i < kStages; ++i) sm100::mbar_init(full0 + 8u * i, 1u);
        sm100::fence_mbar_init();
    }
    if (threadIdx.x == 0u) sh.failed = 0u;
    pdl_launch();
    pdl_wait();
    __syncthreads();
    const DealOf<kStepTokens, kExtra> deal{8u * NT, 1u};
    // Steps are dealt out evenly, or, where the host has found that no item can have many, items as they are: nothing has to be put together then
    const uint32_t all = whole_items ? 0u : sum_steps(p, deal, 0u, sh.part).all, n_work = workers(all, gridDim.x), items = p.c.B * p.c.HK;
    clear_empty_entries(p, deal, !whole_items);
    if (!whole_items && threadIdx.x == 0u) begin_nothing(p, deal);
    if (!whole_items && blockIdx.x >= n_work) return;
    const uint32_t begin = whole_items ? 0u : run_begin(all, n_work, blockIdx.x), end = whole_items ? 0u : run_begin(all, n_work, blockIdx.x + 1u);
    uint32_t left = end - begin, item = blockIdx.x;
    Place at = {0u, 0u};
    if (!whole_items) at = find_step(p, deal, begin);
    const auto next = [&](Segment& seg) {
        if (whole_items) {
            for (; item < items; item += gridDim.x) {
                const uint32_t b = item / p.c.HK, dealt = steps_of(p, deal, b), steps = max(dealt, kExtra) - kExtra;
                if (steps == 0u) continue;
                seg = {b, item - b * p.c.HK, 0u, 0u, steps, steps, 0u};
                item += gridDim.x;
                return true;
            }
            return false;
        }
        while (left > 0u) {
            const uint32_t pos = end - left;
            seg = next_segment(p, deal, at, left);
            if (seg.steps == 0u) continue;
            if (threadIdx.x == 0u) begin_item(p, deal, seg, pos, all, n_work);
            return true;
        }
        return false;
    };
    const uint32_t page = 1u << p.c.page_log2, pages = static_cast<uint32_t>(p.c.pages);
    const bool small_pages = page < kUnit;
    uint32_t stage = 0, phase = 0;   // of the warp's next unit: its stage and the parity of the stage's barrier

    // A warp's copies of a segment: its units are the tokens start + 128 k, as far as the sequence goes
    struct Feed {
        const int32_t* row_of_table;
        const uint8_t* blocks;
        uint32_t start, units, length;
        int id, id_second, next_id, next_second;   // page numbers of 32 units at a time, one a lane (two where a unit has two pages), and those of the next 32 ahead
    } feed = {};
    const auto look_up = [&](uint32_t k) {
        const uint32_t t = feed.start + k * kStepTokens;
        if (k < feed.units) {
            feed.next_id = ld_i32(feed.row_of_table + (t >> p.c.page_log2));
            if (small_pages && t + kBlockTokens < feed.length) feed.next_second = ld_i32(feed.row_of_table + (t >> p.c.page_log2) + 1);
        }
    };
    const auto issue = [&](uint32_t k, uint32_t into) {
        if ((k & 31u) == 0u) {
            feed.id = feed.next_id, feed.id_second = feed.next_second;
            look_up(k + 32u + lane);
        }
        const uint32_t t = feed.start + k * kStepTokens, mine = __shfl_sync(0xFFFFFFFFu, feed.id, k & 31u), second = __shfl_sync(0xFFFFFFFFu, feed.id_second, k & 31u);
        if (lane == 0u) {
            auto source = [&](uint32_t number) {
                return number < pages ? feed.blocks + number * p.c.page_bytes + (t & (page - 1u)) / kBlockTokens * kBlockBytes : kNowhere.bytes;
            };
            const uint32_t bar = full0 + 8u * into, dst = ring0 + into * kUnitBytes;
            if (!small_pages) {
                sm100::mbar_arrive_expect_tx(bar, kUnitBytes);
                bulk_load(dst, source(mine), kUnitBytes, bar);
            } else {
                const bool two = t + kBlockTokens < feed.length;
                sm100::mbar_arrive_expect_tx(bar, two ? kUnitBytes : kBlockBytes);
                bulk_load(dst, source(mine), kBlockBytes, bar);
                if (two) bulk_load(dst + kBlockBytes, source(second), kBlockBytes, bar);
            }
        }
    };
    // the first copies of a segment, into a ring that the warp has emptied
    const auto open = [&](const Segment& seg) {
        feed.length = length_of(p.c, seg.b);
        feed.row_of_table = p.c.table + static_cast<size_t>(seg.b) * p.c.table_width;
        feed.blocks = p.c.pool + static_cast<uint64_t>(seg.head) * (page / kBlockTokens) * kBlockBytes;
        feed.start = seg.first * kStepTokens + warp * kUnit;
        const uint32_t stop = min(feed.length, (seg.first + seg.steps) * kStepTokens);
        feed.units = feed.start < stop ? (stop - feed.start + kStepTokens - 1u) / kStepTokens : 0u;
        feed.id = feed.id_second = feed.next_id = feed.next_second = -1;
        look_up(lane);
#pragma unroll 1
        for (uint32_t k = 0; k < kStages && k < feed.units; ++k) issue(k, (stage + k) % kStages);
    };

    Segment coming;
    bool have = next(coming);
    if (have) open(coming);
    while (have) {
        const Segment seg = coming;
        const uint32_t b = seg.b, head = seg.head, row0 = seg.row0, first = seg.first, start = feed.start, units = feed.units, length = feed.length;
        const uint32_t n_rows = count_of(p.counts, b, p.S, length);
        QueryRows<NT> x;
        x.away = sh.away;
        load_rows<NT>(x, sh.q, p, b, head, row0, length, n_rows);
        uint32_t low = 0xFFFFFFFFu;   // tokens that every live column sees
#pragma unroll
        for (int g = 0; g < NT; ++g) {
#pragma unroll
            for (int j = 0; j < 2; ++j) low = min(low, x.limit(g, j) == 0u ? 0xFFFFFFFFu : x.limit(g, j));
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
        bool ok = true;
        Exponents seen;
#pragma unroll 1
        for (uint32_t k = 0; k < units; ++k) {
            ok = __all_sync(0xFFFFFFFFu, sm100::mbar_wait(full0 + 8u * stage, phase, &sh.failed));
            if (!ok) break;
            const uint32_t tok0 = start + k * kStepTokens;
            const uint8_t* unit = sh.ring[warp][stage];
            if (tok0 + kUnit <= low) attend_unit<NT, false>(o, m, l, x, unit, tok0, sh.q, length, seen);
            else attend_unit<NT, true>(o, m, l, x, unit, tok0, sh.q, length, seen);
            __syncwarp();   // the warp is done with the stage
            if (k + kStages < units) issue(k + kStages, stage);
            if (++stage == kStages) stage = 0u, phase ^= 1u;
        }
        if (!ok && lane == 0u) atomicOr(p.status, 1u);
        // the next segment's first copies are under way while this one's sums come together
        have = ok && next(coming);
        if (have) open(coming);

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
        if (sh.failed != 0u) break;   // (the same for all: it was raised in front of the barrier)
        const bool whole = seg.steps == seg.of;
        const uint32_t slot = first == 0u ? 1u : 0u;
        float* part = slot_of(p.ws, gridDim.x, blockIdx.x, slot, 8u * NT);
#pragma unroll
        for (int g = 0; g < NT; ++g) {
            // warps 2 and 3 hand their O, relative to the item's reference, to 0 and 1, which leave the sums there
            float* sums = sh.o[warp & 1u];   // [8 rows][128]
#pragma unroll
            for (uint32_t turn = 0; turn < 2u; ++turn) {
                if ((warp >> 1) != turn) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int row = 8 * g + 2 * static_cast<int>(tig) + j;
                        const float top = fmaxf(fmaxf(sh.m[0][row], sh.m[1][row]), fmaxf(sh.m[2][row], sh.m[3][row]));
                        const float f = ex2(m[g][j] - top);
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) {
                            // (pieces of 16 bytes change places within a row, so that the lanes of a column meet different banks)
                            float4* at = reinterpret_cast<float4*>(sums + (2u * tig + j) * 128u) + ((4u * gid + i) ^ ((2u * tig + j) & 7u));
                            float4 v = make_float4(o[g][2 * i][j] * f, o[g][2 * i][2 + j] * f, o[g][2 * i + 1][j] * f, o[g][2 * i + 1][2 + j] * f);
                            if (turn == 1u) {
                                const float4 more = *at;
                                v.x += more.x, v.y += more.y, v.z += more.z, v.w += more.w;
                            }
                            *at = v;
                        }
                    }
                }
                __syncthreads();
            }
            {
                const uint32_t r = threadIdx.x >> 4, d = (threadIdx.x & 15u) * 8u, row = row0 + 8u * g + r;
                const float top = fmaxf(fmaxf(sh.m[0][8 * g + r], sh.m[1][8 * g + r]), fmaxf(sh.m[2][8 * g + r], sh.m[3][8 * g + r]));
                float total = 0.0f, acc[8];
#pragma unroll
                for (unsigned w = 0; w < kWarps; ++w) {
                    float l_w = sh.l[w][8 * g + r];
                    const float f = sum_factor(l_w, sh.m[w][8 * g + r] - top);
                    total = fmaf(l_w, f, total);
                }
#pragma unroll
                for (uint32_t y = 0; y < 2u; ++y) {
                    const uint32_t piece = (2u * (threadIdx.x & 15u) + y) ^ (r & 7u);
                    const float4 a = reinterpret_cast<const float4*>(sh.o[0] + r * 128u)[piece], c = reinterpret_cast<const float4*>(sh.o[1] + r * 128u)[piece];
                    acc[4 * y] = a.x + c.x, acc[4 * y + 1] = a.y + c.y, acc[4 * y + 2] = a.z + c.z, acc[4 * y + 3] = a.w + c.w;
                }
                if (row < p.S * p.group) {
                    if (whole) {
                        const bool none = total == 0.0f || row / p.group >= n_rows;   // sees nothing, or stands for nothing
                        const uint32_t i = row / p.group, h = head * p.group + row % p.group;
                        const float inv = 1.0f / total;
                        *reinterpret_cast<uint4*>(p.out + ((static_cast<size_t>(b) * p.S + i) * p.H + h) * 128u + d) =
                            none ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv), pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
                        if (p.lse != nullptr && d == 0u) p.lse[(static_cast<size_t>(b) * p.H + h) * p.S + i] = none ? -INFINITY : (top + lg2(total)) * kLn2;
                    } else {
                        float* to = part + (8u * g + r) * 128u + d;
                        *reinterpret_cast<float4*>(to) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                        *reinterpret_cast<float4*>(to + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
                        if (d == 0u) *reinterpret_cast<float2*>(part + 8u * NT * 128u + (8u * g + r) * 2u) = make_float2(top, total);
                    }
                }
            }
            __syncthreads();
        }
    }
    // after a failure: no copy may land in shared memory that is another CTA's by then. (A copy that was issued ends by itself; the wait for it has a limit.)
    if (sh.failed != 0u) {
        uint32_t again = 0;
        for (uint32_t i = 0; i < kStages; ++i) (void)sm100::mbar_wait(full0 + 8u * i, i < stage ? phase ^ 1u : phase, &again, 20000000LL);
    }
}

// Rows of a KV head up to which this kernel is taken; more go to the tensor cores' tiles of 256 rows. (24 ragged sequences of up to 32768 tokens: 20, 24, 28 and 32 rows 62, 64, 100 and 102 us here, 36
// rows 120 there; of up to 8192 tokens 34 to 54 and 56; 64 of up to 2048 32 to 53 and 63. Above 24 rows registers spill, which is a part of the 100.)
constexpr uint32_t kMostFew = 32;

uint32_t groups_of(uint32_t rows) { return (rows + 7u) / 8u; }

// Items of up to so many steps, which is up to 512 tokens, are not cut: a launch and the way through memory are saved, 2 heads of 256 tokens 9.7 us in place of 11.8
constexpr uint32_t kWholeSteps = 4;
uint32_t most_steps(const Kv4View& c) { return static_cast<uint32_t>(((static_cast<unsigned long long>(c.table_width) << c.page_log2) + kStepTokens - 1u) / kStepTokens); }
uint32_t attend_grid(const Kv4View& c) {
    const unsigned long long steps = most_steps(c);
    const unsigned long long most = (steps <= kWholeSteps ? 1ull : steps) * c.B * c.HK, full = static_cast<unsigned long long>(kCtasPerSm) * static_cast<unsigned long long>(current_sm_count());
    return static_cast<uint32_t>(most < full ? (most ? most : 1ull) : full);
}

template <int NT>
cudaError_t launch_rows(const Kv8AttendParams& p, cudaStream_t stream) {
    const uint32_t grid = attend_grid(p.c);
    const size_t smem = sizeof(CtaShared<NT>);
    static std::atomic<bool> set[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_relaxed)) {
        e = cudaFuncSetAttribute(kv8_attend_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_relaxed);
    }
    const bool whole = most_steps(p.c) <= kWholeSteps;
    e = kv4_launch(kv8_attend_kernel<NT>, dim3(grid), kThreads, smem, stream, p, whole);
    return e != cudaSuccess || whole ? e : launch_combine_few(p, 8u * NT, grid, stream);
}

// Puts the prefill kernel's items together that a few CTAs each have a part of, whose parts lie by columns: a warp has 32 rows, a lane's own, and 16 columns
__global__ void __launch_bounds__(256) kv8_combine_columns_kernel(const __grid_constant__ Kv8AttendParams p, uint32_t rows, uint32_t row_tiles, uint32_t grid) {
    pdl_launch();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, r = blockIdx.y * 32u + lane;
    const uint4 begun = ld_v4(begun_at(p.ws, blockIdx.x));
    const uint32_t entry = begun.x / p.c.HK, head = begun.x - entry * p.c.HK, b = entry / row_tiles, row = (entry - b * row_tiles) * rows + r, from = begun.y, last = begun.z;
    if (last == from || row >= p.S * p.group) return;
    const uint32_t i = row / p.group, h = head * p.group + row - i * p.group;
    const bool sees = i < count_of(p.counts, b, p.S, length_of(p.c, b));
    float m = kLowest, l = 0.0f, o[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) o[x] = 0.0f;
    for (uint32_t w0 = from; sees && w0 <= last; w0 += 2u) {   // two parts in flight
        uint2 ml[2];
        uint4 raw[2][4];
#pragma unroll
        for (uint32_t k = 0; k < 2u; ++k) {
            const uint32_t w = min(w0 + k, last);
            const float* src = slot_of(p.ws, grid, w, w == from ? 1u : 0u, rows);
            ml[k] = ld_v2(src + rows * 128u + 2u * r);
#pragma unroll
            for (uint32_t y = 0; y < 4u; ++y) raw[k][y] = ld_v4(src + ((4u * warp + y) * rows + r) * 4u);
        }
#pragma unroll
        for (uint32_t k = 0; k < 2u; ++k) {
            if (w0 + k > last) break;
            const float pm = __uint_as_float(ml[k].x), top = fmaxf(m, pm), a = ex2(m - top), c = ex2(pm - top);
            float pl = __uint_as_float(ml[k].y);
            const float al = sum_factor(l, m - top), cl = sum_factor(pl, pm - top);
            m = top;
            l = fmaf(l, al, pl * cl);
#pragma unroll
            for (uint32_t y = 0; y < 4u; ++y) {
                const uint4 v = raw[k][y];
                o[4 * y] = fmaf(o[4 * y], a, __uint_as_float(v.x) * c), o[4 * y + 1] = fmaf(o[4 * y + 1], a, __uint_as_float(v.y) * c);
                o[4 * y + 2] = fmaf(o[4 * y + 2], a, __uint_as_float(v.z) * c), o[4 * y + 3] = fmaf(o[4 * y + 3], a, __uint_as_float(v.w) * c);
            }
        }
    }
    const bool none = l == 0.0f;
    const float inv = none ? 0.0f : 1.0f / l;
    uint32_t y[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) y[x] = pack_bf16x2(o[2 * x] * inv, o[2 * x + 1] * inv);
    uint4* to = reinterpret_cast<uint4*>(p.out + ((static_cast<size_t>(b) * p.S + i) * p.H + h) * 128u + 16u * warp);
    to[0] = make_uint4(y[0], y[1], y[2], y[3]), to[1] = make_uint4(y[4], y[5], y[6], y[7]);
    if (p.lse != nullptr && warp == 0u) p.lse[(static_cast<size_t>(b) * p.H + h) * p.S + i] = none ? -INFINITY : (m + lg2(l)) * kLn2;
}

cudaError_t launch_many(const Kv8AttendParams& p, cudaStream_t stream) {
    const uint32_t rows = p.S * p.group, per = kv8_prefill_rows(), row_tiles = (rows + per - 1u) / per, grid = kv8_prefill_grid(), most = rows < per ? rows : per;
    const cudaError_t e = launch_kv8_prefill(p, row_tiles, stream);
    if (e == cudaSuccess && few_parts(p.c, row_tiles, grid)) return kv4_launch(kv8_combine_columns_kernel, dim3(begun_entries(p.c, row_tiles, grid), (most + 31u) / 32u), 256u, 0, stream, p, per, row_tiles, grid);
    return e != cudaSuccess ? e : launch_combine_many(p, per, row_tiles, kv8_prefill_grid(), stream, /*together=*/true);   // (48 rows over 30000 tokens: 25.5 us, 105.8 with a warp a row)
}

}  // namespace

uint64_t kv8_attend_workspace(const Kv4View& c, uint32_t S, uint32_t H) {
    const uint32_t rows = S * (H / c.HK);
    if (rows > kMostFew) return kv4_partial_bytes(kv8_prefill_grid(), kv8_prefill_rows());
    return kv4_partial_bytes(attend_grid(c), 8u * groups_of(rows));
}

cudaError_t launch_kv8_attend(const Kv8AttendParams& p, cudaStream_t stream) {
    const uint32_t rows = p.S * p.group, groups = groups_of(rows);
    if (rows > kMostFew) return launch_many(p, stream);
    return groups == 1u ? launch_rows<1>(p, stream) : groups == 2u ? launch_rows<2>(p, stream) : groups == 3u ? launch_rows<3>(p, stream) : launch_rows<4>(p, stream);
}

}  // namespace b200mx
