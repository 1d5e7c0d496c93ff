// Attention of many query rows over the 4-bit cache: prompts and chunks of them, on the tcgen05 tensor cores.
//
//   S = Q K'^T,  P = 2^(c S + e - m),  O += P V',  l += sum P 2^-e,  out = O / l,   c = scale * log2(e) * what was taken out of Q and K, m a running reference per row
//
// All operands are f16: Q with a power of two per row taken out, K' and V' relative to the largest factor of the step's 128 tokens, all exact down to 2^-30 of the row's
// or the step's largest.
//
// A CTA has 256 query rows of one KV head (rows of the sequence and of the head's group packed, whatever the group's size) as two tiles of 128 and goes over the tokens
// 128 at a time. Per step four warps turn the step's K and V codes into f16 in shared memory, once for both tiles; one thread issues the products, S from shared
// memory, P V with P from tensor memory; and two groups of four warps do the softmax, one tile each, a thread a row, so that the tensor cores work on one tile while the
// other's softmax runs. P overwrites S in tensor memory and goes over in two halves of 64 tokens, the first while the second is still being computed. m moves only
// when a row's maximum exceeds it by 2^8, so O is hardly ever rescaled.
//
// Bounds: a step of 256 rows and 128 tokens takes about 3750 clocks, of which the tensor cores work 2048 and the exponentials need as many; a tile's scores, softmax and product
// follow one another, since the 512 columns of tensor memory are O and one S of both tiles. A CTA's change from one item to the next costs about 16000 clocks more. 4096 rows
// over 8192 tokens, 32 heads on 8: 445 us = 0.93 PFLOP/s, 0.57 of the measured bf16 rate; 512 rows over 16384, 16 heads on 4: 91 us, 27.4 steps a CTA. Spills: 296 bytes stored, 596 loaded. Slower: scores in halves of 64 tokens (801 us
// when this took 746), two threads a row (594, then 473), part of the exponentials as polynomials (483, then 463), no turns of the tiles (558), P in one piece (457, then 447),
// K in bf16 (458, with the query rows by asynchronous copies).
//
// Steps are dealt out to one CTA per SM as kv4_schedule.cuh says; items that several CTAs worked on go through f32 partials and the combine kernel.
#include "kv4.cuh"
#include "kv4_schedule.cuh"
#include "ptx_sm100.cuh"

#include <atomic>
#include <cstddef>

namespace b200mx {

namespace {

using namespace kv4;
using namespace sm100;

constexpr uint32_t kTileRows = 128, kItemRows = 256, kStages = 2, kHalf = 64;
// Slots of the steps' exponents. The converters write those of step j + 4 behind the scores of step j + 2, which are behind the P of step j + 1 of the tiles that go on
constexpr uint32_t kFactorSlots = 4;
// Slots of the segments' blocks of NaN. The converters begin segment n behind its step's third forerunner, whose scores both issuing warps have issued: these are in segment n - 3 at least,
// and an issuing warp begins a segment when its tile's softmax has stored the one before
constexpr uint32_t kNanSlots = 4;
constexpr uint32_t kAtomBytes = 128u * 128u, kTileBytes = 2u * kAtomBytes;   // 128 rows x 64 elements with 128-byte swizzle; two of them a tile
constexpr uint32_t kThreads = 512;
// Warps 0-3 and 4-7: softmax of tile 0 and 1; 8-11: codes to f16; 12 and 13: products of tile 0 and 1. The pools of setmaxnreg come out of the launch's 128 registers a thread.
constexpr int kSoftmaxRegs = 176, kConvertRegs = 104, kIssueRegs = 56;
static_assert(8 * kSoftmaxRegs + 4 * kConvertRegs + 4 * kIssueRegs <= 16 * 128, "register shares");
constexpr uint32_t kColS = 0, kColO = 256;   // S of tile q (P in its first half) at 128 q, O at 256 + 128 q
constexpr float kSlack = 8.0f;
constexpr float kLeast = 1e-37f;   // times a masked score it is still -inf
constexpr float kLn2 = 0.69314718055994531f;

// barriers; kPFull by 2 q + half
enum Bar : uint32_t { kKFull = 0, kKEmpty = 2, kVFull = 4, kVEmpty = 6, kSFull = 8, kODone = 10, kPFull = 12, kOFree = 16, kQFull = 18, kQEmpty = 20, kTurn = 22, kDrained = 24, kEFull = 26, kBars = 26 + kFactorSlots };

struct Shared {
    uint8_t q[2][kTileBytes], k[kStages][kTileBytes], v[kStages][kTileBytes];
    uint4 most[kFactorSlots][2];   // the largest scale byte of K and of V that each of the converting warps met
    uint4 nan_from[kNanSlots][4];  // of a segment and a converting warp: the first token that has NaN in each block of its V, all ones where none has
    unsigned long long bars[kBars];
    Sums part[kThreads / 32];
    struct Plan {
        Segment seg;
        uint32_t pos, length, n, number;   // (segments are counted from 1)
    } plan[8];                     // of a softmax warp's next segment
    uint32_t converting[4];        // number of a converting warp's segment
    uint32_t tmem, failed, not_drained;
};

// a = a x + c, b = b x + c in one instruction
__device__ __forceinline__ void fma2(uint32_t& a, uint32_t& b, float x, float c) {
    unsigned long long p, q, r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "r"(a), "r"(b));
    asm("mov.b64 %0, {%1, %1};" : "=l"(q) : "f"(x));
    asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(c));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p) : "l"(p), "l"(q), "l"(r));
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(p));
}
__device__ __forceinline__ void add2(float& a, float& b, float x, float y) {
    unsigned long long p, q;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    asm("mov.b64 %0, {%1, %2};" : "=l"(q) : "f"(x), "f"(y));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(p), "l"(q));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}

// steps of tile q of a segment's item: those that its last live row sees
__device__ __forceinline__ uint32_t tile_steps(const Kv4AttendParams& p, const Segment& s, uint32_t q, uint32_t length, uint32_t n) {
    const uint32_t r0 = s.row0 + q * kTileRows;
    if (r0 >= n * p.group) return 0u;
    const uint32_t last = (min(r0 + kTileRows, n * p.group) - 1u) / p.group;
    const uint32_t of = ((p.causal ? length - n + last + 1u : length) + kStepTokens - 1u) / kStepTokens;
    return of <= s.first ? 0u : min(s.steps, of - s.first);
}

// 8 elements of a block, two bytes of codes in `half` (0, 1) of each word, times the block's factor (twice in f), as f16
__device__ __forceinline__ uint4 to_f16(uint32_t lo, uint32_t hi, bool half, uint32_t f) {
    return make_uint4(mul_f16x2(half ? e2m1x2_to_f16x2<2>(lo) : e2m1x2_to_f16x2<0>(lo), f), mul_f16x2(half ? e2m1x2_to_f16x2<3>(lo) : e2m1x2_to_f16x2<1>(lo), f),
                      mul_f16x2(half ? e2m1x2_to_f16x2<2>(hi) : e2m1x2_to_f16x2<0>(hi), f), mul_f16x2(half ? e2m1x2_to_f16x2<3>(hi) : e2m1x2_to_f16x2<1>(hi), f));
}
// A token's 64 code bytes to its row of a tile
__device__ __forceinline__ void store_row(uint8_t* tile, uint32_t row, const uint4 (&codes)[4], const ValueFactors& factors) {
    uint8_t* at = tile + row * 128u;
    const uint32_t f[4] = {__byte_perm(factors.r01, 0u, 0x1010), __byte_perm(factors.r01, 0u, 0x3232), __byte_perm(factors.r23, 0u, 0x1010), __byte_perm(factors.r23, 0u, 0x3232)};
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
#pragma unroll
        for (uint32_t b = 0; b < 4; ++b) {
            const uint4 x = to_f16(b < 2 ? codes[j].x : codes[j].y, b < 2 ? codes[j].z : codes[j].w, b & 1u, f[b]);
            *reinterpret_cast<uint4*>(at + (b >> 1) * kAtomBytes + (((4u * (b & 1u) + j) ^ (row & 7u)) << 4)) = x;
        }
    }
}

// The first of a warp's 32 tokens, from token `from` on, with NaN in a block of its V (0xFF in that byte of `nan`), where none before had it
__device__ __forceinline__ void note_nan(uint4& first, uint32_t nan, uint32_t from) {
    uint32_t* at = reinterpret_cast<uint32_t*>(&first);
#pragma unroll 1
    for (uint32_t x = 0; x < 4u; ++x) {
        const uint32_t has = __ballot_sync(0xFFFFFFFFu, (nan >> (8u * x) & 1u) != 0u);
        if ((threadIdx.x & 31u) == 0u && has != 0u && at[x] == 0xFFFFFFFFu) at[x] = from + static_cast<uint32_t>(__ffs(static_cast<int>(has))) - 1u;
    }
}

__global__ void __launch_bounds__(kThreads, 1) kv4_prefill_kernel(const __grid_constant__ Kv4AttendParams p, uint32_t row_tiles) {
    extern __shared__ uint8_t smem_raw[];
    Shared& sh = *reinterpret_cast<Shared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~static_cast<uintptr_t>(1023u));
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t bars = smem_u32(sh.bars);
    auto bar = [&](uint32_t i) { return bars + 8u * i; };
    if (threadIdx.x == 0u) {
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(bar(kKFull + i), 128u), mbar_init(bar(kVFull + i), 128u);
            mbar_init(bar(kKEmpty + i), 2u), mbar_init(bar(kVEmpty + i), 2u), mbar_init(bar(kOFree + i), 4u);
            mbar_init(bar(kSFull + i), 1u), mbar_init(bar(kODone + i), 1u), mbar_init(bar(kQFull + i), 4u), mbar_init(bar(kQEmpty + i), 1u);
            mbar_init(bar(kTurn + i), 1u), mbar_init(bar(kDrained + i), 1u);
        }
        for (uint32_t i = 0; i < 4; ++i) mbar_init(bar(kPFull + i), 4u);
        for (uint32_t i = 0; i < kFactorSlots; ++i) mbar_init(bar(kEFull + i), 4u);
        
        fence_mbar_init();
        sh.failed = sh.not_drained = 0u;
        for (uint32_t i = 0; i < 8; ++i) sh.plan[i].number = sh.converting[i & 3u] = 0u;
    }
    if (warp == 12u) tmem_alloc(smem_u32(&sh.tmem), 512u);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, sh.tmem, 0);
    pdl_launch();
    pdl_wait();
    const Deal deal{kItemRows, row_tiles};
    const uint32_t all = sum_steps(p, deal, 0u, sh.part).all;
    const uint32_t n_work = workers(all, gridDim.x);
    volatile uint32_t* failed = &sh.failed;
    clear_empty_entries(p, deal);
    if (threadIdx.x == 0u) begin_nothing(p, deal);
    if (blockIdx.x < n_work) {
        const uint32_t begin = run_begin(all, n_work, blockIdx.x);
        const uint32_t end = run_begin(all, n_work, blockIdx.x + 1u);
        uint32_t left = end - begin;
        Place at = find_step(p, deal, begin);
        if (warp < 8u) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
            const uint32_t q = warp >> 2, r = threadIdx.x & 127u, lanes = (warp & 3u) << 21;   // 32 TMEM lanes per warp, in bits 16 and up
            const uint32_t t_s = tmem + lanes + kColS + 128u * q, t_o = tmem + lanes + kColO + 128u * q;
            uint32_t s_phase = 0, o_phase = 0, q_phase = 0, step0 = 0;   // step0: steps in front of the segment
            bool ok = true;
            // The query rows: asked for while the last products of the segment before are under way, kept in registers over its epilogue. A warp has the rows of its threads, two
            // of them with a load: lane l brings 16 bytes (8 elements, number l mod 16) of row 2 x + l / 16
            uint4 raw[16];
            // Where the next segment is, is worked out while the first scores of this one are computed; the rows are asked for at its end
            auto plan_next = [&]() {
                Shared::Plan x;
                x.pos = end - left;
                x.seg = next_segment(p, deal, at, left);
                x.length = length_of(p.c, x.seg.b), x.n = count_of(p.counts, x.seg.b, p.S, x.length);
                if (lane == 0u) {
                    x.number = sh.plan[warp].number + 1u;
                    sh.plan[warp] = x;
                }
                __syncwarp();
            };
            auto ask_rows = [&](const Segment& seg, uint32_t n) {
                const uint32_t row = seg.row0 + q * kTileRows + (r & 96u) + (lane >> 4);
                uint32_t i = row / p.group, h = row - i * p.group;
                const uint8_t* src = p.q.data + seg.b * p.q.stride_b + seg.head * p.group * p.q.stride_h + 16u * (lane & 15u);
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    raw[x] = i < n ? ld_v4(src + i * p.q.stride_s + h * p.q.stride_h) : make_uint4(0u, 0u, 0u, 0u);
                    for (h += 2u; h >= p.group; h -= p.group) ++i;
                }
            };
            plan_next();
            Shared::Plan now = sh.plan[warp];
            ask_rows(now.seg, now.n);
            uint8_t* mine = sh.q[q] + (r >> 5) * (kTileBytes / 4u);   // a quarter of the rows' place, where this warp turns its part of O round, between two segments
            for (bool more = true; more;) {
                const Segment seg = now.seg;
                const uint32_t pos = now.pos, length = now.length, n = now.n;
                // the tile's four warps are done with the place of the rows; also where a wait has run out in one of them: they leave together
                ok = named_bar_all(2u + q, 128u, ok);
                if (!ok) break;
                if (threadIdx.x == 0u) begin_item(p, deal, seg, pos, all, n_work);
                const uint32_t steps = tile_steps(p, seg, q, length, n), row = seg.row0 + q * kTileRows + r, i = row / p.group;
                const bool exists = row < p.S * p.group;
                const uint32_t limit = !exists || i >= n ? 0u : p.causal ? length - n + i + 1u : length;
                float m = kLowest, l = 0.0f, c_row = 0.0f;
                {
                    uint32_t amax[8];   // sizes as bf16 bits, of rows 2 x and 2 x + 1 of pairs of loads in the halves
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        auto largest = [](const uint4& v) {
                            const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
                            return max(m & 0xFFFFu, m >> 16);
                        };
                        amax[x] = largest(raw[2 * x]) | largest(raw[2 * x + 1]) << 16;
                    }
#pragma unroll
                    for (int y = 1; y < 16; y <<= 1) {
#pragma unroll
                        for (int x = 0; x < 8; ++x) amax[x] = __vmaxu2(amax[x], __shfl_xor_sync(0xFFFFFFFFu, amax[x], y));
                    }
#pragma unroll
                    for (uint32_t x = 0; x < 16u; ++x) {
                        uint32_t w[4] = {raw[x].x, raw[x].y, raw[x].z, raw[x].w};
                        const float2 f = row_factors(x & 1u ? amax[x / 2] & 0xFFFF0000u : amax[x / 2] << 16);
                        const float back = __shfl_sync(0xFFFFFFFFu, f.y, (lane & 1u) << 4);   // of row 2 x + lane mod 2
                        if (lane >> 1 == x) c_row = p.scale_log2 * back;
#pragma unroll
                        for (int y = 0; y < 4; ++y) w[y] = pack_f16x2(__uint_as_float(w[y] << 16) * f.x, __uint_as_float(w[y] & 0xFFFF0000u) * f.x);
                        const uint32_t to = (r & 96u) + 2u * x + (lane >> 4), chunk = lane & 15u;
                        *reinterpret_cast<uint4*>(sh.q[q] + (chunk >> 3) * kAtomBytes + to * 128u + (((chunk & 7u) ^ (to & 7u)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0u) mbar_arrive(bar(kQFull + q));
                more = left > 0u;
                if (more) plan_next();
                for (uint32_t j = 0; j < steps && ok; ++j) {
                    // (not the K tile's barrier: while a group is still storing the rows of the segment before, that one may already be two steps on)
                    const uint32_t slot = (step0 + j) % kFactorSlots;
                    ok = mbar_wait(bar(kEFull + slot), (step0 + j) / kFactorSlots & 1u, failed);
                    const uint4 mk = sh.most[slot][0], mv = sh.most[slot][1];
                    const int ek = group_exponent(max(max(mk.x, mk.y), max(mk.z, mk.w))), e = group_exponent(max(max(mv.x, mv.y), max(mv.z, mv.w)));
                    const float c = fmaxf(c_row * __uint_as_float(static_cast<uint32_t>(127 + ek - kUp) << 23), kLeast), ef = static_cast<float>(e);
                    ok = ok && mbar_wait(bar(kSFull + q), s_phase, failed);
                    if (!ok) break;
                    s_phase ^= 1u;
                    tc_fence_after_sync();
                    uint32_t s[4][32];
#pragma unroll
                    for (int k = 0; k < 4; ++k) tmem_ld32(t_s + 32u * k, s[k]);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 4; ++k) reg_fence32(s[k]);
                    const uint32_t tok0 = (seg.first + j) * kStepTokens;
                    if (__any_sync(0xFFFFFFFFu, tok0 + kStepTokens > limit)) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
#pragma unroll
                            for (int x = 0; x < 32; ++x) {
                                if (tok0 + 32u * k + x >= limit) s[k][x] = 0xFF800000u;
                            }
                        }
                    }
                    float top[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        top[k] = fmaxf(__uint_as_float(s[k][0]), __uint_as_float(s[k][1]));
#pragma unroll
                        for (int x = 2; x < 32; x += 2) top[k] = fmaxf(top[k], fmaxf(__uint_as_float(s[k][x]), __uint_as_float(s[k][x + 1])));
                    }
                    const float most = fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), c, ef);
                    const bool over = most > m + kSlack;
                    if (__any_sync(0xFFFFFFFFu, over)) {
                        const float next = over ? most : m, f = ex2(m - next);
                        m = next;
                        l *= f;
                        if (j > 0u) {   // the product before this one is over: S came behind it
#pragma unroll 1
                            for (uint32_t k = 0; k < 8u; ++k) {
                                uint32_t o[16];
                                tmem_ld16(t_o + 16u * k, o);
                                tmem_wait_ld();
                                reg_fence16(o);
#pragma unroll
                                for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                                tmem_st16(t_o + 16u * k, o);
                            }
                            tmem_wait_st();
                        }
                    }
                    const float shift = ef - m;
                    float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
#pragma unroll
                        for (int x = 0; x < 16; ++x) {
                            uint32_t a = s[k][2 * x], b = s[k][2 * x + 1];
                            fma2(a, b, c, shift);
                            const float ea = ex2(__uint_as_float(a)), eb = ex2(__uint_as_float(b));
                            add2(l0, l1, ea, eb);
                            s[k][x] = pack_f16x2(ea, eb);   // (behind what it overwrites)
                        }
                        tmem_st16_of32(t_s + 16u * k, s[k]);
                        if (k & 1) {
                            tmem_wait_st();
                            tc_fence_before_sync();
                            __syncwarp();
                            if (lane == 0u) mbar_arrive(bar(kPFull + 2u * q + (k >> 1)));
                        }
                    }
                    l = fmaf(l0 + l1, __uint_as_float(static_cast<uint32_t>(127 - e) << 23), l);
                }
                step0 += seg.steps;
                const Segment done = seg;
                if (more) {
                    now = sh.plan[warp];
                    ask_rows(now.seg, now.n);
                } else {   // (assigned either way: nothing of the old rows stays in registers for it)
#pragma unroll
                    for (int x = 0; x < 16; ++x) raw[x] = make_uint4(0u, 0u, 0u, 0u);
                }
                ok = ok && mbar_wait(bar(kQEmpty + q), q_phase, failed);   // S is done with the rows
                q_phase ^= 1u;
                if (steps > 0u) {
                    ok = ok && mbar_wait(bar(kODone + q), o_phase, failed);
                    o_phase ^= 1u;
                    tc_fence_after_sync();
                }
                if (!ok) continue;
                const bool whole = done.steps == done.of, none = l == 0.0f;   // NaN is something
                const uint32_t h = done.head * p.group + row % p.group;
                const float factor = whole ? (none ? 0.0f : kDown / l) : kDown;
                // Blocks of V's NaN went into the product as 0, where NaN would meet the weights of 0 of rows that do not see it. A row sees the tokens in front of its limit.
                uint32_t nan_blocks = 0;
                if (steps > 0u) {
                    const uint32_t number = sh.plan[warp].number - (more ? 1u : 0u);   // (the plan is already the next segment's)
#pragma unroll
                    for (uint32_t w = 0; w < 4u; ++w) {
                        const uint4 from = sh.nan_from[number % kNanSlots][w];
                        nan_blocks |= (from.x < limit ? 1u : 0u) | (from.y < limit ? 2u : 0u) | (from.z < limit ? 4u : 0u) | (from.w < limit ? 8u : 0u);
                    }
                }
                const uint32_t at_row = exists ? (done.b * p.S + i) * p.H + h : 0xFFFFFFFFu;   // of out, in rows
                float* slot = slot_of(p.ws, gridDim.x, blockIdx.x, done.first == 0u ? 1u : 0u, kItemRows);
                // O by 64 columns: a thread writes its row's to shared memory, and the warp stores whole pieces of rows
#pragma unroll 1
                for (uint32_t c = 0; c < 2u; ++c) {
#pragma unroll
                    for (uint32_t k = 0; k < 2u; ++k) {
                        uint32_t o[32];
                        const float f = nan_blocks >> (2u * c + k) & 1u ? __uint_as_float(0x7FC00000u) : factor;
                        if (steps > 0u) {
                            tmem_ld32(t_o + 64u * c + 32u * k, o);
                            tmem_wait_ld();
                            reg_fence32(o);
                        } else {
#pragma unroll
                            for (int x = 0; x < 32; ++x) o[x] = 0u;
                        }
#pragma unroll
                        for (uint32_t x = 0; x < 8u; ++x) {
                            float4 v = make_float4(__uint_as_float(o[4 * x]) * f, __uint_as_float(o[4 * x + 1]) * f, __uint_as_float(o[4 * x + 2]) * f, __uint_as_float(o[4 * x + 3]) * f);
                            if (none) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            *reinterpret_cast<float4*>(mine + lane * 256u + (((8u * k + x) ^ (lane & 15u)) << 4)) = v;
                        }
                    }
                    if (c == 1u && steps > 0u) {
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0u) mbar_arrive(bar(kOFree + q));
                    }
                    __syncwarp();
                    if (whole) {
#pragma unroll 4
                        for (uint32_t x = 0; x < 8u; ++x) {   // four rows of 64 bf16 at a time
                            const uint32_t from = 4u * x + (lane >> 3), piece = lane & 7u, to = __shfl_sync(0xFFFFFFFFu, at_row, from);
                            const float4 u = *reinterpret_cast<const float4*>(mine + from * 256u + (((2u * piece) ^ (from & 15u)) << 4)), v = *reinterpret_cast<const float4*>(mine + from * 256u + (((2u * piece + 1u) ^ (from & 15u)) << 4));
                            if (to != 0xFFFFFFFFu)
                                *reinterpret_cast<uint4*>(p.out + static_cast<size_t>(to) * 128u + 64u * c + 8u * piece) = make_uint4(pack_bf16x2(u.x, u.y), pack_bf16x2(u.z, u.w), pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
                        }
                    } else {
#pragma unroll 4
                        for (uint32_t x = 0; x < 16u; ++x) {   // two rows of 64 f32 at a time
                            const uint32_t from = 2u * x + (lane >> 4), piece = lane & 15u;
                            *reinterpret_cast<float4*>(slot + (q * kTileRows + (r & 96u) + from) * 128u + 64u * c + 4u * piece) = *reinterpret_cast<const float4*>(mine + from * 256u + ((piece ^ (from & 15u)) << 4));
                        }
                    }
                    __syncwarp();
                }
                if (whole) {
                    if (exists && p.lse != nullptr) p.lse[(static_cast<size_t>(done.b) * p.H + h) * p.S + i] = none ? -INFINITY : (m + lg2(l)) * kLn2;
                } else if (limit != 0u) {
                    *reinterpret_cast<float2*>(slot + kItemRows * 128u + 2u * (q * kTileRows + r)) = make_float2(m, l);
                }
            }
        } else if (warp < 12u) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvertRegs));
            const uint32_t r = threadIdx.x & 127u, page = 1u << p.c.page_log2;
            uint32_t step = 0;   // so far
            bool ok = true;
            while (left > 0u && ok) {
                const Segment seg = next_segment(p, deal, at, left);
                if (lane == 0u) sh.nan_from[++sh.converting[warp & 3u] % kNanSlots][warp & 3u] = make_uint4(0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu);
                const uint32_t length = length_of(p.c, seg.b), n = count_of(p.counts, seg.b, p.S, length);
                // the token of this thread in step j: its page, looked up a step ahead of its bytes
                long long page_ahead = -1;
                auto look_up = [&](uint32_t j) {
                    const uint32_t t = (seg.first + j) * kStepTokens + r;
                    if (j < seg.steps && t < length) page_ahead = page_of(p.c, seg.b, t);
                };
                uint4 k[4], v[4];
                uint32_t ks = 0, vs = 0;
                bool lost = false, empty = true;
                auto fetch = [&](uint32_t j, bool values) {
                    const uint32_t t = (seg.first + j) * kStepTokens + r;
                    if (j >= seg.steps || t >= length || page_ahead < 0) return;
                    const uint8_t* rec = record_of(p.c, page_ahead, seg.head);
                    const uint32_t slot = t & (page - 1u);
                    if (values) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) v[x] = ld_v4(rec + 64u * (page + slot) + 16u * x);
                    } else {
#pragma unroll
                        for (int x = 0; x < 4; ++x) k[x] = ld_v4(rec + 64u * slot + 16u * x);
                        ks = ld_u32(rec + 128u * page + 4u * slot), vs = ld_u32(rec + 132u * page + 4u * slot);
                    }
                };
                look_up(0u);
                empty = seg.first * kStepTokens + r >= length, lost = page_ahead < 0;
                fetch(0u, false);
                fetch(0u, true);
                look_up(1u);
                for (uint32_t j = 0; j < seg.steps; ++j, ++step) {
                    const uint32_t st = step % kStages, parity = (step / kStages + 1u) & 1u, slot = step % kFactorSlots;
                    // A token behind the length must not bring NaN into P V; one that is lost makes the rows that see it NaN by its scores
                    const uint32_t top_k = empty || lost ? 0u : largest_byte(ks), met_k = __reduce_max_sync(0xFFFFFFFFu, top_k == 255u ? 0u : top_k);
                    uint32_t top_v = empty || lost ? 0u : largest_byte(vs), met_v = __reduce_max_sync(0xFFFFFFFFu, top_v);
                    if (met_v == 255u) {   // NaN in V: the first token of each block is noted, and its scale becomes 0
                        const uint32_t nan = empty || lost ? 0u : nan_bytes(vs);
                        note_nan(sh.nan_from[sh.converting[warp & 3u] % kNanSlots][warp & 3u], nan, (seg.first + j) * kStepTokens + (r & 96u));
                        vs &= ~nan;
                        top_v = empty || lost ? 0u : largest_byte(vs), met_v = __reduce_max_sync(0xFFFFFFFFu, top_v);
                    }
                    if (lane == 0u) reinterpret_cast<uint32_t*>(&sh.most[slot][0])[warp & 3u] = met_k, reinterpret_cast<uint32_t*>(&sh.most[slot][1])[warp & 3u] = met_v;
                    // (also where a wait has run out in one of the four warps: they leave together)
                    ok = named_bar_all(1u, 128u, ok);
                    if (!ok) break;
                    if (lane == 0u) mbar_arrive(bar(kEFull + slot));
                    const uint4 mk = sh.most[slot][0], mv = sh.most[slot][1];
                    ValueFactors fk = value_factors(ks, top_k, group_exponent(max(max(mk.x, mk.y), max(mk.z, mk.w))));
                    ValueFactors fv = value_factors(vs, top_v, group_exponent(max(max(mv.x, mv.y), max(mv.z, mv.w))));
                    if (empty || lost) {
                        fk.r01 = fk.r23 = empty ? 0u : 0x7E007E00u, fv.r01 = fv.r23 = 0u;   // (the codes are whatever they were: finite)
                    }
                    ok = mbar_wait(bar(kKEmpty + st), parity, failed);
                    if (ok) {
                        store_row(sh.k[st], r, k, fk);
                        fence_proxy_async_smem();
                        mbar_arrive(bar(kKFull + st));
                    }
                    empty = j + 1u >= seg.steps || (seg.first + j + 1u) * kStepTokens + r >= length, lost = page_ahead < 0;
                    fetch(j + 1u, false);
                    ok = ok && mbar_wait(bar(kVEmpty + st), parity, failed);
                    if (ok) {
                        store_row(sh.v[st], r, v, fv);
                        fence_proxy_async_smem();
                        mbar_arrive(bar(kVFull + st));
                    }
                    fetch(j + 1u, true);
                    look_up(j + 2u);
                }
            }
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
            if (warp < 14u) {
                // All of this runs on values that are the same in the warp's 32 lanes. The compiler has to see that (they come out of votes and reductions, which have uniform
                // results): the products' operands then stay in uniform registers and take few instructions to issue. A warp per tile: the two take turns with the tensor cores,
                // and neither's waits hold the other's products up.
                auto uniform = [](uint32_t x) { return __reduce_max_sync(0xFFFFFFFFu, x); };
                const uint32_t q = uniform(warp - 12u), t_s = uniform(tmem) + kColS + 128u * q, t_o = uniform(tmem) + kColO + 128u * q;
                constexpr uint32_t id_s = idesc_16bit(false, 128, 128, 0, 0), id_o = idesc_16bit(false, 128, 128, 0, 1);
                const uint64_t d_k = make_smem_desc(smem_u32(sh.q[0]), 16, 1024, kSwizzle128B), d_v = make_smem_desc(smem_u32(sh.v[0]), kAtomBytes, 1024, kSwizzle128B);
                const uint32_t k_hi = static_cast<uint32_t>(d_k >> 32), v_hi = static_cast<uint32_t>(d_v >> 32);
                const uint32_t q_lo = uniform(static_cast<uint32_t>(d_k)) + (q * kTileBytes >> 4), k_lo = uniform(static_cast<uint32_t>(d_k)) + (2u * kTileBytes >> 4), v_lo = uniform(static_cast<uint32_t>(d_v));
                static_assert(offsetof(Shared, k) == 2u * kTileBytes, "K behind Q");
                uint32_t step = 0, q_phase = 0, turn = q ^ 1u, p_phase = 0, o_phase = 1;   // (tile 0 goes first)
                bool ok = true;
                auto wait = [&](uint32_t b, uint32_t parity) {
                    ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait(b, parity, failed));
                    return ok;
                };
                auto commit = [&](uint32_t b) {
                    if (elect_one_sync()) tc_commit(b);
                };
                auto scores = [&](uint32_t st) {
                    if (elect_one_sync()) {
                        const uint32_t b = k_lo + (st * kTileBytes >> 4);
#pragma unroll
                        for (uint32_t x = 0; x < 8u; ++x) {
                            const uint32_t off = ((x >> 2) * kAtomBytes + (x & 3u) * 32u) >> 4;
                            mma_f16_ss(t_s, q_lo + off, k_hi, b + off, k_hi, id_s, x > 0u ? 1u : 0u);
                        }
                        tc_commit(bar(kSFull + q));
                    }
                };
                while (uniform(left) > 0u && ok) {
                    const Segment seg = next_segment(p, deal, at, left);
                    const uint32_t length = length_of(p.c, seg.b), n = count_of(p.counts, seg.b, p.S, length);
                    const uint32_t steps = uniform(tile_steps(p, seg, q, length, n)), seg_steps = uniform(seg.steps);
                    if (!wait(bar(kQFull + q), q_phase)) break;
                    q_phase ^= 1u;
                    if (!wait(bar(kKFull + step % kStages), step / kStages & 1u)) break;
                    tc_fence_after_sync();
                    if (steps > 0u) {
                        scores(step % kStages);   // overwrites P of the step before, behind its products
                        if (!wait(bar(kOFree + q), o_phase)) break;
                        o_phase ^= 1u;
                    }
                    commit(bar(kKEmpty + step % kStages));
                    if (seg_steps == 1u) commit(bar(kQEmpty + q));
                    for (uint32_t j = 0; j < seg_steps; ++j, ++step) {
                        const uint32_t st = step % kStages, next = (step + 1u) % kStages;
                        const bool more = j + 1u < seg_steps;
                        if (!wait(bar(kVFull + st), step / kStages & 1u)) break;
                        // The tiles take turns, so that one's products run under the other's softmax: without, both do the same at the same time
                        if (!wait(bar(kTurn + q), turn)) break;
                        turn ^= 1u;
                        if (j < steps) {
#pragma unroll
                            for (uint32_t h = 0; h < 2u; ++h) {
                                if (!wait(bar(kPFull + 2u * q + h), p_phase)) break;
                                tc_fence_after_sync();
                                if (elect_one_sync()) {
                                    const uint32_t b = v_lo + ((st * kTileBytes + h * kHalf * 128u) >> 4);
#pragma unroll
                                    for (uint32_t x = 0; x < 4u; ++x) mma_f16_ts(t_o, t_s + 32u * h + 8u * x, b + (x * 2048u >> 4), v_hi, id_o, (j > 0u || h + x > 0u) ? 1u : 0u);
                                    if (h == 1u && j + 1u == steps) tc_commit(bar(kODone + q));
                                }
                            }
                            p_phase ^= 1u;
                        }
                        if (!ok) break;
                        commit(bar(kVEmpty + st));
                        if (more) {
                            if (!wait(bar(kKFull + next), (step + 1u) / kStages & 1u)) break;
                            tc_fence_after_sync();
                            if (j + 1u < steps) scores(next);
                            commit(bar(kKEmpty + next));
                        }
                        if (lane == 0u) mbar_arrive(bar(kTurn + (q ^ 1u)));
                        if (j + 2u == seg_steps) commit(bar(kQEmpty + q));
                    }
                }
                if (!ok) {   // whatever was issued has to be over before the tensor memory goes back
                    commit(bar(kDrained + q));
                    (void)mbar_wait(bar(kDrained + q), 0u, &sh.not_drained);
                }
                __syncwarp();
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 0u && sh.failed != 0u) atomicOr(p.status, 1u);
    if (warp == 12u) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512u);
    }
}

}  // namespace

uint32_t kv4_prefill_grid() { return static_cast<uint32_t>(current_sm_count()); }
uint32_t kv4_prefill_rows() { return kItemRows; }

cudaError_t launch_kv4_prefill(const Kv4AttendParams& p, uint32_t row_tiles, cudaStream_t stream) {
    constexpr size_t smem = sizeof(Shared) + 1024u;
    static_assert(smem <= 227u * 1024u, "shared memory of a CTA");
    static std::atomic<bool> set[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_relaxed)) {
        e = cudaFuncSetAttribute(kv4_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_relaxed);
    }
    return kv4_launch(kv4_prefill_kernel, dim3(kv4_prefill_grid()), kThreads, smem, stream, p, row_tiles);
}

}  // namespace b200mx
