// Attention of many query rows over the 8-bit cache: prompts and chunks of them, on the tcgen05 tensor cores.
//
//   S = Q K'^T,  P = 2^(c S + e - m),  O += P V',  l += sum P 2^-e,  out = O / l
//
// K' and V' are the codes as f16, exactly; c = scale * log2(e) * K's scale * what was taken out of Q, e the exponent of V's scale, both one for 16 tokens, m a running reference per row.
// Q is f16 with a power of two per row taken out, exact down to 2^-30 of the row's largest.
//
// A CTA has 256 query rows of one KV head (rows of the sequence and of the head's group packed, whatever the group's size) as two tiles of 128 and goes over the tokens
// 80 at a time, five blocks: that is what makes a tile's O (128 columns), scores (80) and weights (40) fit half of tensor memory side by side, so that the next step's scores are computed
// while the softmax works on this step's. Per step one warp brings the codes (cp.async.bulk), four warps turn them into f16 in shared memory, once for both tiles, a thread a tile issues
// the products, S from shared memory, P V with P from tensor memory, and two groups of four warps do the softmax, one tile each, a thread a row. m moves only when a row's maximum
// exceeds it by 2^(kUp + kSlack), so O is hardly ever rescaled.
//
// Bound by a tile's chain of scores, softmax and product: a step takes 2780 clocks, of which the products of both tiles are 1280, the exponentials of both 1280 (they meet: two warps of a scheduler do
// them at the same time, which takes 1600), loads from tensor memory 250, the maximum 400, waits and stores 500. 4096 rows of 32 heads over 8192 tokens: 455 us among other calls (425 in a row), 0.91
// PFLOP/s, 0.56 of what a matrix product measures; a change of item is 9000 clocks, of which a CTA of 4 ragged chunks of 333 rows (50.4 us) has one or two to its 16 steps.
// Slower: steps of 128 tokens with P over S (514 us in place of 464 then), of 64 (500), a quarter and three eighths of the exponentials by a polynomial (470 and 485 in place of 461), locks or turns between the two
// groups at the exponentials (489 and more), K's and V's conversion by four warps each (504), query rows brought by the issuing warps (427 and 451 in place of 431, chunks 51.5 and 55 in place of 50.6),
// O stored 64 columns at a time (507) or exchanged between four lanes first (441).
//
// Steps are dealt out to one CTA per SM as kv4_schedule.cuh says; items that several CTAs worked on go through f32 partials and the combine kernel.
#include "kv4_schedule.cuh"
#include "kv8.cuh"
#include "ptx_sm100.cuh"

#include <atomic>
#include <cstddef>

namespace b200mx {

namespace {

using namespace kv8;
using namespace sm100;

constexpr uint32_t kTileRows = 128, kItemRows = 256, kStep = 80, kBlocks = kStep / kBlockTokens, kStages = 3, kRawStages = 2;
constexpr uint32_t kExtra = 5;   // what a CTA's change to another item costs, in steps (4 ragged chunks of 333 rows, 24 heads: 52.4, 50.6, 50.6 us with 3, 4, 5; 8 x 512 rows over 600 tokens 82.0, 82.4, 79.9)
// Slots of the steps' scales. Those of step j are written when its codes have come, for which those of step j - 2 must have been taken: behind the scores of step j - 5 (three stages of K)
// and so behind the softmax's reads of the scores of step j - 6
constexpr uint32_t kScaleSlots = 8;
// Slots of the segments. Segment n is published, and its first token with NaN in V noted, when the codes of a step of segment n - 3 at least have been taken, behind the products of one of
// segment n - 6, and so behind the end of segment n - 7
constexpr uint32_t kSegmentSlots = 8;
constexpr uint32_t kQAtom = 128u * 128u, kTileBytes = 2u * kQAtom;   // 128 rows x 64 elements with 128-byte swizzle; two of them a tile of query rows
constexpr uint32_t kAtomBytes = kStep * 128u, kStepBytes = 2u * kAtomBytes;   // the same of a step's K or V
constexpr uint32_t kThreads = 512;
// Warps 0-3 and 4-7: softmax of tile 0 and 1; 8-11: codes to f16; 12 and 13: products of tile 0 and 1; 14: copies; 15: scales. The pools of setmaxnreg come out of the launch's 128
// registers a thread.
constexpr uint32_t kIssueWarp = 12, kCopyWarp = 14;
constexpr int kSoftmaxRegs = 184, kConvertRegs = 72, kIssueRegs = 72;
static_assert(8 * kSoftmaxRegs + 4 * kConvertRegs + 4 * kIssueRegs <= 16 * 128, "register shares");
constexpr uint32_t kColP = 80, kColO = 128, kColTile = 256;   // of a tile's 256 columns: S, P, O
constexpr float kUpF = 6.0f, kSlack = 8.0f;   // (f16 has more room above 1 than a weight needs)
constexpr float kLeast = 1e-37f;   // times a masked score it is still -inf
constexpr float kLn2 = 0.69314718055994531f;

// barriers; kPFull by 2 q + half
enum Bar : uint32_t {
    kKFull = 0, kKEmpty = kKFull + kStages, kVFull = kKEmpty + kStages, kVEmpty = kVFull + kStages,   // by stage
    kRawFull = kVEmpty + kStages, kRawEmpty = kRawFull + kRawStages,
    kSFull = kRawEmpty + kRawStages, kSFree = kSFull + 2, kPFull = kSFree + 2, kPFree = kPFull + 2, kOFree = kPFree + 2, kQFull = kOFree + 2, kQEmpty = kQFull + 2, kDrained = kQEmpty + 2,   // by tile
    kScales = kDrained + 2, kSegment = kScales + kScaleSlots, kBars = kSegment + kSegmentSlots
};

struct Shared {
    uint8_t q[2][kTileBytes], k[kStages][kStepBytes], v[kStages][kStepBytes];
    uint8_t raw_k[kRawStages][kBlocks][kVCodes], raw_v[kRawStages][kBlocks][kMeta - kVCodes];   // a step's codes as they come
    uint4 meta[kRawStages][kBlocks];   // and its scales and masks
    uint32_t plain[kScaleSlots];       // whether every token of a step has numbers
    alignas(16) float scales[kScaleSlots][3][8];   // of a step's blocks: scale of K, exponent e of V's, 2^-e
    uint32_t wide[kScaleSlots];        // whether a step is (kv4.cuh)
    uint32_t nan_from[kSegmentSlots];  // of a segment: the first token that has NaN in its V, all ones where none has
    unsigned long long bars[kBars];
    Sums part[kThreads / 32];
    struct Plan {
        Segment seg;
        uint32_t length, n, more;      // more: whether the CTA has a segment behind this one. (One without steps: it has none at all)
        uint32_t steps[2];             // of the two tiles: those that their last live rows see
    } plan[kSegmentSlots];
    uint32_t tmem, failed, not_drained, to_next;   // to_next: from four columns of a part to the next four
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
__device__ __forceinline__ uint32_t tile_steps(const Kv8AttendParams& p, const Segment& s, uint32_t q, uint32_t length, uint32_t n) {
    const uint32_t r0 = s.row0 + q * kTileRows;
    if (r0 >= n * p.group) return 0u;
    const uint32_t last = (min(r0 + kTileRows, n * p.group) - 1u) / p.group;
    const uint32_t of = ((p.causal ? length - n + last + 1u : length) + kStep - 1u) / kStep;
    return of <= s.first ? 0u : min(s.steps, of - s.first);
}

// the larger of three
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// waits for two barriers; where both are there already, in the time that one takes
__device__ __forceinline__ bool mbar_wait2(uint32_t a, uint32_t a_parity, uint32_t b, uint32_t b_parity, volatile uint32_t* abort_flag) {
    uint32_t first, second;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%2], %3;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 q, [%4], %5;\n\t"
        "selp.u32 %0, 1, 0, p;\n\tselp.u32 %1, 1, 0, q;\n\t}"
        : "=r"(first), "=r"(second)
        : "r"(a), "r"(a_parity), "r"(b), "r"(b_parity)
        : "memory");
    return (first != 0u || mbar_wait(a, a_parity, abort_flag)) && (second != 0u || mbar_wait(b, b_parity, abort_flag));
}
// eight codes as f16
__device__ __forceinline__ uint4 to_f16(uint32_t lo, uint32_t hi) { return make_uint4(e4m3x2_lo(lo), e4m3x2_hi(lo), e4m3x2_lo(hi), e4m3x2_hi(hi)); }
__device__ __forceinline__ uint4* piece_at(uint8_t* tile, uint32_t row, uint32_t piece) {   // 8 elements of a row of a tile
    return reinterpret_cast<uint4*>(tile + (piece >> 3) * kAtomBytes + row * 128u + (((piece & 7u) ^ (row & 7u)) << 4));
}

struct RowSums {
    float m, l;
};
// A wide step (kv4.cuh) of a row, 16 tokens at a time: brings m to where the step has it, O and l with it, adds the weights up for themselves and leaves them to the product. All lanes. seen: tokens of
// the step that the row sees; product: the barrier of the step before's, 0 where there is none
__device__ __forceinline__ RowSums wide_step(Shared& sh, uint32_t slot, uint32_t t_s, float c_row, int seen, uint32_t product, uint32_t p_phase, uint32_t s_free, uint32_t p_full, RowSums now) {
    const uint32_t t_p = t_s + kColP, t_o = t_s + kColO;
    float most = -INFINITY, m = now.m, l = now.l;
#pragma unroll 1
    for (uint32_t k = 0; k < 2u * kBlocks; ++k) {   // the largest, then the weights
        const uint32_t b = k % kBlocks;
        if (k == kBlocks) {
            most -= kUpF;
            const float next = most > m + kSlack ? most : m, f = ex2(m - next), fl = sum_factor(l, m - next);
            m = next;
            l *= fl;
            if (product != 0u) {
                (void)mbar_wait(product, p_phase, &sh.failed);
                __syncwarp();
                tc_fence_after_sync();
                if (__any_sync(0xFFFFFFFFu, f != 1.0f)) {
#pragma unroll 1
                    for (uint32_t x = 0; x < 8u; ++x) {
                        uint32_t o[16];
                        tmem_ld16(t_o + 16u * x, o);
                        tmem_wait_ld();
                        reg_fence16(o);
#pragma unroll
                        for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
                        tmem_st16(t_o + 16u * x, o);
                    }
                }
            }
        }
        uint32_t x[16];
        tmem_ld16(t_s + 16u * b, x);
        tmem_wait_ld();
        reg_fence16(x);
        const float c = fmaxf(c_row * sh.scales[slot][0][b], kLeast), shift = sh.scales[slot][1][b], up = static_cast<float>(kWide) - m;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int z = 0; z < 16; ++z) x[z] = z < seen - static_cast<int>(16u * b) ? x[z] : 0xFF800000u;
        if (k < kBlocks) {
#pragma unroll
            for (int z = 0; z < 16; ++z) top = fmaxf(top, __uint_as_float(x[z]));
            most = fmaxf(most, fmaf(top, c, shift));
        } else {
#pragma unroll
            for (int z = 0; z < 8; ++z) {
                const float u = __uint_as_float(x[2 * z]), v = __uint_as_float(x[2 * z + 1]);
                sum += ex2_wide(fmaf(u, c, up)) + ex2_wide(fmaf(v, c, up));
                x[z] = pack_f16x2(ex2(fmaf(u, c, shift - m)), ex2(fmaf(v, c, shift - m)));
            }
            l = fmaf(sum, kWideDown, l);
            tmem_st8(t_p + 8u * b, x);
        }
    }
    tmem_wait_st();
    tc_fence_before_sync();
    __syncwarp();
    if ((threadIdx.x & 31u) == 0u) mbar_arrive(s_free), mbar_arrive(p_full);
    return {m, l};
}

__global__ void __launch_bounds__(kThreads, 1) kv8_prefill_kernel(const __grid_constant__ Kv8AttendParams p, uint32_t row_tiles) {
    extern __shared__ uint8_t smem_raw[];
    Shared& sh = *reinterpret_cast<Shared*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023u) & ~static_cast<uintptr_t>(1023u));
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t bars = smem_u32(sh.bars);
    auto bar = [&](uint32_t i) { return bars + 8u * i; };
    if (threadIdx.x == 0u) {
        for (uint32_t i = 0; i < kStages; ++i) mbar_init(bar(kKFull + i), 128u), mbar_init(bar(kVFull + i), 128u), mbar_init(bar(kKEmpty + i), 2u), mbar_init(bar(kVEmpty + i), 2u);
        for (uint32_t i = 0; i < kRawStages; ++i) mbar_init(bar(kRawFull + i), 1u), mbar_init(bar(kRawEmpty + i), 4u);
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(bar(kSFull + i), 1u), mbar_init(bar(kSFree + i), 4u), mbar_init(bar(kPFull + i), 4u), mbar_init(bar(kPFree + i), 1u), mbar_init(bar(kOFree + i), 4u);
            mbar_init(bar(kQFull + i), 4u), mbar_init(bar(kQEmpty + i), 1u), mbar_init(bar(kDrained + i), 1u);
        }
        for (uint32_t i = 0; i < kScaleSlots; ++i) mbar_init(bar(kScales + i), 1u);
        for (uint32_t i = 0; i < kSegmentSlots; ++i) mbar_init(bar(kSegment + i), 1u);
        fence_mbar_init();
        sh.failed = sh.not_drained = 0u;
        sh.to_next = few_parts(p.c, row_tiles, gridDim.x) ? 4u * kItemRows : 4u;
    }
    if (warp == kIssueWarp) tmem_alloc(smem_u32(&sh.tmem), 512u);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, sh.tmem, 0);
    pdl_launch();
    pdl_wait();
    const DealOf<kStep, kExtra> deal{kItemRows, row_tiles};
    const uint32_t all = sum_steps(p, deal, 0u, sh.part).all;
    const uint32_t n_work = workers(all, gridDim.x);
    volatile uint32_t* failed = &sh.failed;
    if (blockIdx.x >= n_work) {
        if (threadIdx.x == 0u) begin_nothing(p, deal);
        clear_empty_entries(p, deal);
    }
    if (blockIdx.x < n_work) {
        const uint32_t begin = run_begin(all, n_work, blockIdx.x);
        const uint32_t end = run_begin(all, n_work, blockIdx.x + 1u);
        uint32_t number = 0;   // of the role's segment
        // the next segment, once the copying warp has published it; all lanes. False: a wait has run out
        const auto next_plan = [&](Shared::Plan& x) {
            const uint32_t slot = number % kSegmentSlots;
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(bar(kSegment + slot), number / kSegmentSlots & 1u, failed))) return false;
            x = sh.plan[slot];
            ++number;
            return true;
        };
        if (warp < 8u) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
            const uint32_t q = warp >> 2, r = threadIdx.x & 127u, lanes = (warp & 3u) << 21;   // 32 TMEM lanes per warp, in bits 16 and up
            const uint32_t t_s = tmem + lanes + kColTile * q, t_p = t_s + kColP, t_o = t_s + kColO;
            uint32_t s_phase = 0, p_phase = 0, q_phase = 0, step0 = 0;   // step0: steps in front of the segment
            bool ok = true;
            // The query rows, fetched into L2 when the segment is published: asked for when that segment's last weights are written, and made f16 in their place, a thread its row's,
            // in the middle of storing its O: what is left of that the next scores' product runs beside.
            auto ask_rows = [&](const Segment& seg, uint32_t n) {
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(bar(kQEmpty + q), q_phase ^ 1u, failed))) return false;
                q_phase ^= 1u;
                const uint32_t row = seg.row0 + q * kTileRows + r, i = row / p.group, chunk = lane & 15u;
                const uint8_t* src = p.q.data + seg.b * p.q.stride_b + i * p.q.stride_s + (seg.head * p.group + row - i * p.group) * p.q.stride_h;
                const unsigned long long mine = i < n ? reinterpret_cast<unsigned long long>(src) : 0ull;
#pragma unroll 4
                for (uint32_t x = 0; x < 16u; ++x) {   // two rows at a time, a lane 16 bytes
                    const uint32_t from = 2u * x + (lane >> 4), to = (r & 96u) + from;
                    const unsigned long long at_row = __shfl_sync(0xFFFFFFFFu, mine, from);
                    cp_async_16(smem_u32(sh.q[q] + (chunk >> 3) * kQAtom + to * 128u + (((chunk & 7u) ^ (to & 7u)) << 4)),
                                at_row != 0ull ? reinterpret_cast<const uint8_t*>(at_row) + 16u * chunk : p.q.data, at_row != 0ull ? 16u : 0u);
                }
                return true;
            };
            // what the thread's row was multiplied by, taken out
            auto take_rows = [&]() {
                cp_async_wait_all();
                __syncwarp();
                uint4* const place = reinterpret_cast<uint4*>(sh.q[q] + r * 128u);
                uint4 v[16];
#pragma unroll
                for (uint32_t x = 0; x < 16u; ++x) v[x] = place[(x >> 3) * (kQAtom / 16u) + ((x & 7u) ^ (r & 7u))];
                uint32_t top = 0;   // sizes as bf16 bits
#pragma unroll
                for (uint32_t x = 0; x < 16u; ++x) top = __vmaxu2(top, __vmaxu2(__vmaxu2(v[x].x & 0x7FFF7FFFu, v[x].y & 0x7FFF7FFFu), __vmaxu2(v[x].z & 0x7FFF7FFFu, v[x].w & 0x7FFF7FFFu)));
                const float2 f = row_factors(max(top << 16, top & 0xFFFF0000u));
#pragma unroll
                for (uint32_t x = 0; x < 16u; ++x) {
                    uint32_t w[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
#pragma unroll
                    for (int y = 0; y < 4; ++y) w[y] = pack_f16x2(__uint_as_float(w[y] << 16) * f.x, __uint_as_float(w[y] & 0xFFFF0000u) * f.x);
                    place[(x >> 3) * (kQAtom / 16u) + ((x & 7u) ^ (r & 7u))] = make_uint4(w[0], w[1], w[2], w[3]);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0u) mbar_arrive(bar(kQFull + q));
                return p.scale_log2 * f.y;
            };
            // the next segment's number and rows; where its plan stands
            auto ask_next = [&]() {
                const uint32_t slot = number % kSegmentSlots;
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(bar(kSegment + slot), number / kSegmentSlots & 1u, failed))) return false;
                ++number;
                return sh.plan[slot].seg.steps > 0u && ask_rows(sh.plan[slot].seg, sh.plan[slot].n);
            };
            float c_row = 0.0f;
            const auto rescale = [&](float f) {   // O
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
            };
            Shared::Plan now;
            ok = ask_next();
            if (ok) c_row = take_rows();
            for (bool more = true; more && ok;) {
                const uint32_t nan_slot = (number - 1u) % kSegmentSlots;
                now = sh.plan[nan_slot];
                const Segment seg = now.seg;
                const uint32_t length = now.length, n = now.n;
                more = now.more != 0u;
                const uint32_t steps = q != 0u ? now.steps[1] : now.steps[0], row = seg.row0 + q * kTileRows + r, i = row / p.group;
                const bool exists = row < p.S * p.group;
                const uint32_t limit = !exists || i >= n ? 0u : p.causal ? length - n + i + 1u : length;
                float m = kLowest, l = 0.0f;
                uint32_t j = 0;
                // the step's scales and scores; false: it is a wide one, or a wait has run out
                const auto is_near_step = [&]() {
                    // (not the K tile's barrier: while a group is still storing the rows of the segment before, that one may already be two steps on)
                    const uint32_t slot = (step0 + j) % kScaleSlots;
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait2(bar(kScales + slot), (step0 + j) / kScaleSlots & 1u, bar(kSFull + q), s_phase, failed));
                    s_phase ^= 1u;
                    return ok && sh.wide[slot] == 0u;
                };
                for (; j < steps && ok; ++j) {
                    if (!is_near_step()) break;
                    const uint32_t slot = (step0 + j) % kScaleSlots;
                    tc_fence_after_sync();
                    uint32_t s[kStep];
                    tmem_ld32(t_s, *reinterpret_cast<uint32_t(*)[32]>(s));
                    tmem_ld32(t_s + 32u, *reinterpret_cast<uint32_t(*)[32]>(s + 32));
                    tmem_ld16(t_s + 64u, *reinterpret_cast<uint32_t(*)[16]>(s + 64));
                    float c[kBlocks], shift[kBlocks], back[kBlocks];
#pragma unroll
                    for (int k = 0; k < static_cast<int>(kBlocks); ++k) c[k] = fmaxf(c_row * sh.scales[slot][0][k], kLeast), shift[k] = sh.scales[slot][1][k], back[k] = sh.scales[slot][2][k];
                    tmem_wait_ld();
                    reg_fence32(*reinterpret_cast<uint32_t(*)[32]>(s)), reg_fence32(*reinterpret_cast<uint32_t(*)[32]>(s + 32)), reg_fence16(*reinterpret_cast<uint32_t(*)[16]>(s + 64));
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0u) mbar_arrive(bar(kSFree + q));   // the next scores may overwrite these
                    const int seen = static_cast<int>(limit) - static_cast<int>((seg.first + j) * kStep);
                    if (__any_sync(0xFFFFFFFFu, seen < static_cast<int>(kStep))) {
#pragma unroll
                        for (int y = 0; y < static_cast<int>(kStep); ++y) {
                            if (y >= seen) s[y] = 0xFF800000u;
                        }
                    }
                    float tops[kBlocks];
#pragma unroll
                    for (int k = 0; k < static_cast<int>(kBlocks); ++k) {
                        const uint32_t* y = s + 16 * k;
                        float top = max3(__uint_as_float(y[0]), __uint_as_float(y[1]), __uint_as_float(y[2]));
#pragma unroll
                        for (int z = 3; z < 15; z += 2) top = max3(top, __uint_as_float(y[z]), __uint_as_float(y[z + 1]));
                        tops[k] = fmaf(fmaxf(top, __uint_as_float(y[15])), c[k], shift[k]);
                    }
                    const float most = max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[4]) - kUpF;
                    const bool over = most > m + kSlack;
                    // once the product of the step before is over, O may be rescaled and P overwritten
                    bool waited = j == 0u;
                    const auto wait_product = [&]() {
                        if (!waited) {
                            ok = __all_sync(0xFFFFFFFFu, mbar_wait(bar(kPFree + q), p_phase, failed));
                            p_phase ^= 1u;
                            tc_fence_after_sync();
                        }
                        waited = true;
                    };
                    if (__any_sync(0xFFFFFFFFu, over)) {
                        wait_product();
                        const float next = over ? most : m, f = ex2(m - next);
                        m = next;
                        l *= f;
                        if (j > 0u) rescale(f);
                    }
#pragma unroll
                    for (int k = 0; k < static_cast<int>(kBlocks); ++k) {
                        const float down = shift[k] - m;
                        float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
                        for (int z = 0; z < 8; ++z) {
                            uint32_t a = s[16 * k + 2 * z], b = s[16 * k + 2 * z + 1];
                            fma2(a, b, c[k], down);
                            const float ea = ex2(__uint_as_float(a)), eb = ex2(__uint_as_float(b));
                            add2(l0, l1, ea, eb);
                            s[16 * k + z] = pack_f16x2(ea, eb);   // (behind what it overwrites)
                        }
                        l = fmaf(l0 + l1, back[k], l);
                        if (k == 3) {   // (four blocks at once, beside the last one's exponentials: a prompt of 4096 rows 427 us, 431 with all at the end, 453 with three)
                            wait_product();
#pragma unroll
                            for (int x = 0; x < 4; ++x) tmem_st8(t_p + 8u * x, s + 16 * x);
                        }
                    }
#pragma unroll
                    for (int k = 4; k < static_cast<int>(kBlocks); ++k) tmem_st8(t_p + 8u * k, s + 16 * k);
                    tmem_wait_st();
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0u) mbar_arrive(bar(kPFull + q));
                }
                // From the first wide step on all of them are. (Among the other steps' instructions, or as a call from there, this took 3 to 5 % of prompts that have none: 4096 rows over 8192 tokens 452 us without
                // it, 457 so, 464 with the scales waited for in front of the scores)
                for (bool here = true; j < steps && ok; ++j) {
                    if (!here) (void)is_near_step();
                    here = false;
                    if (!ok) break;
                    tc_fence_after_sync();
                    const RowSums x = wide_step(sh, (step0 + j) % kScaleSlots, t_s, c_row, static_cast<int>(limit) - static_cast<int>((seg.first + j) * kStep), j > 0u ? bar(kPFree + q) : 0u, p_phase, bar(kSFree + q),
                                                bar(kPFull + q), {m, l});
                    m = x.m, l = x.l;
                    p_phase ^= j > 0u;
                }
                step0 += seg.steps;
                if (!ok) break;
                if (more) {
                    ok = ask_next();
                    if (ok) c_row = take_rows();
                }
                if (steps > 0u) {
                    ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait(bar(kPFree + q), p_phase, failed));
                    p_phase ^= 1u;
                    tc_fence_after_sync();
                }
                if (!ok) break;
                const bool whole = seg.steps == seg.of, none = l == 0.0f;   // NaN is something
                const uint32_t h = seg.head * p.group + row % p.group;
                float factor = none ? 0.0f : whole ? 1.0f / l : 1.0f;
                // NaN of V went into the product as 0, where it would meet the weights of 0 of rows that do not see it. A row sees the tokens in front of its limit.
                if (steps > 0u && sh.nan_from[nan_slot] < limit) factor = __uint_as_float(0x7FC00000u);
                __nv_bfloat16* out = p.out + ((static_cast<size_t>(seg.b) * p.S + i) * p.H + h) * 128u;
                float* slot = slot_of(p.ws, gridDim.x, blockIdx.x, seg.first == 0u ? 1u : 0u, kItemRows);
                const uint32_t to_next = sh.to_next;
                // few parts: by four columns, then rows, so that a warp's stores are whole lines (a row a thread is 32 lines each); else by rows
                float* part = slot + (q * kTileRows + r) * (to_next == 4u ? 128u : 4u);
#pragma unroll 1
                for (uint32_t c = 0; c < 4u; ++c) {   // 32 columns at a time, a thread its row's
                    uint32_t o[32];
                    if (steps > 0u) {
                        tmem_ld32(t_o + 32u * c, o);
                        tmem_wait_ld();
                        reg_fence32(o);
                        if (c == 3u) {
                            tc_fence_before_sync();
                            __syncwarp();
                            if (lane == 0u) mbar_arrive(bar(kOFree + q));
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = steps == 0u || none ? 0u : __float_as_uint(__uint_as_float(o[x]) * factor);
                    if (whole) {
                        if (exists) {
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                uint32_t w[4];
#pragma unroll
                                for (int y = 0; y < 4; ++y) w[y] = pack_bf16x2(__uint_as_float(o[8 * x + 2 * y]), __uint_as_float(o[8 * x + 2 * y + 1]));
                                *reinterpret_cast<uint4*>(out + 32u * c + 8 * x) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    } else if (limit != 0u) {
#pragma unroll
                        for (int x = 0; x < 8; ++x) *reinterpret_cast<uint4*>(part + (8u * c + x) * to_next) = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
                    }
                }
                if (whole) {
                    if (exists && p.lse != nullptr) p.lse[(static_cast<size_t>(seg.b) * p.H + h) * p.S + i] = none ? -INFINITY : (m + lg2(l)) * kLn2;
                } else if (limit != 0u) {
                    *reinterpret_cast<float2*>(slot + kItemRows * 128u + 2u * (q * kTileRows + r)) = make_float2(m, l);
                }
            }
            if (!ok) cp_async_wait_all();   // (what was asked for has to have come before the CTA ends)
        } else if (warp < kIssueWarp) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvertRegs));
            // Block by block, 16 bytes of K and of V a thread: 16 elements of one token, 8 elements of both tokens of a pair
            const uint32_t t = threadIdx.x & 127u, k_row = t >> 3, k_piece = (t & 7u) ^ k_swap(k_row), v_row = 2u * (t >> 4), v_piece = (t & 15u) ^ v_swap(t >> 4);
            // (of a row's eight lanes the upper four store their second half first, so that the eight meet different banks)
            const uint32_t up = k_piece >> 2;
            uint4 *const k_first = piece_at(sh.k[0], k_row, 2u * k_piece + up), *const k_second = piece_at(sh.k[0], k_row, 2u * k_piece + (up ^ 1u));
            uint4 *const v_first = piece_at(sh.v[0], v_row, v_piece), *const v_second = piece_at(sh.v[0], v_row + 1u, v_piece);
            constexpr uint32_t kBlockOfTile = kBlockTokens * 128u / 16u;   // from a block's place in a tile to the next one's, in pieces
            uint32_t step = 0;   // so far
            Shared::Plan now;
            now.more = 1u;
            bool ok = true;
            while (now.more != 0u && ok) {
                if (!next_plan(now)) break;
                const Segment seg = now.seg;
                const uint32_t length = now.length;
                for (uint32_t j = 0; j < seg.steps; ++j, ++step) {
                    const uint32_t st = step % kStages, raw = step % kRawStages, slot = step % kScaleSlots, parity = (step / kStages + 1u) & 1u, to = st * (kStepBytes / 16u);
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait2(bar(kScales + slot), step / kScaleSlots & 1u, bar(kKEmpty + st), parity, failed));
                    if (!ok) break;
                    const uint8_t *k_codes = sh.raw_k[raw][0] + 16u * t, *v_codes = sh.raw_v[raw][0] + 16u * t;
                    const bool plain = sh.plain[slot] != 0u;
                    // tokens of a block below the length, and whether they have numbers in K and V: codes of others may be anything
                    const auto live = [&](uint32_t x) {
                        const uint32_t t0 = (seg.first + j) * kStep + x * kBlockTokens;
                        return t0 >= length ? 0u : 0xFFFFu >> (16u - min(length - t0, 16u));
                    };
                    uint4 codes[kBlocks];
                    if (plain) {
#pragma unroll
                        for (uint32_t x = 0; x < kBlocks; ++x) codes[x] = *reinterpret_cast<const uint4*>(k_codes + x * kVCodes);
#pragma unroll
                        for (uint32_t x = 0; x < kBlocks; ++x) {
                            const uint4 w = codes[x];
                            const uint32_t a = up ? w.z : w.x, b = up ? w.w : w.y, c = up ? w.x : w.z, d = up ? w.y : w.w;
                            k_first[to + x * kBlockOfTile] = to_f16(a, b);
                            k_second[to + x * kBlockOfTile] = to_f16(c, d);
                        }
                    } else {
#pragma unroll 1
                        for (uint32_t x = 0; x < kBlocks; ++x) {
                            const uint4 w = *reinterpret_cast<const uint4*>(k_codes + x * kVCodes);
                            const uint32_t here = live(x), masks = here != 0u ? sh.meta[raw][x].z : 0u;
                            uint4 first = up ? to_f16(w.z, w.w) : to_f16(w.x, w.y), second = up ? to_f16(w.x, w.y) : to_f16(w.z, w.w);
                            if (!(here >> k_row & 1u)) first = second = make_uint4(0u, 0u, 0u, 0u);
                            else if (masks >> k_row & 1u) first = second = make_uint4(0x7E007E00u, 0x7E007E00u, 0x7E007E00u, 0x7E007E00u);
                            k_first[to + x * kBlockOfTile] = first;
                            k_second[to + x * kBlockOfTile] = second;
                        }
                    }
                    fence_proxy_async_smem();
                    mbar_arrive(bar(kKFull + st));
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait(bar(kVEmpty + st), parity, failed));
                    if (!ok) break;
                    if (plain) {
#pragma unroll
                        for (uint32_t x = 0; x < kBlocks; ++x) codes[x] = *reinterpret_cast<const uint4*>(v_codes + x * kVCodes);
#pragma unroll
                        for (uint32_t x = 0; x < kBlocks; ++x) {
                            const uint4 w = codes[x];
                            v_first[to + x * kBlockOfTile] = to_f16(__byte_perm(w.x, w.y, 0x6420), __byte_perm(w.z, w.w, 0x6420));
                            v_second[to + x * kBlockOfTile] = to_f16(__byte_perm(w.x, w.y, 0x7531), __byte_perm(w.z, w.w, 0x7531));
                        }
                    } else {
#pragma unroll 1
                        for (uint32_t x = 0; x < kBlocks; ++x) {
                            uint4 w = *reinterpret_cast<const uint4*>(v_codes + x * kVCodes);
                            const uint32_t here = live(x), good = here != 0u ? here & ~(sh.meta[raw][x].z >> 16) : 0u;
                            const uint32_t keep = (good >> v_row & 1u ? 0x00FF00FFu : 0u) | (good >> (v_row + 1u) & 1u ? 0xFF00FF00u : 0u);
                            w.x &= keep, w.y &= keep, w.z &= keep, w.w &= keep;
                            v_first[to + x * kBlockOfTile] = to_f16(__byte_perm(w.x, w.y, 0x6420), __byte_perm(w.z, w.w, 0x6420));
                            v_second[to + x * kBlockOfTile] = to_f16(__byte_perm(w.x, w.y, 0x7531), __byte_perm(w.z, w.w, 0x7531));
                        }
                    }
                    fence_proxy_async_smem();
                    mbar_arrive(bar(kVFull + st));
                    __syncwarp();
                    if (lane == 0u) mbar_arrive(bar(kRawEmpty + raw));
                }
            }
            clear_empty_entries(p, deal, true, t, 128u);   // (while the others are still at the last steps)
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
            if (warp < kCopyWarp) {
                // All of this runs on values that are the same in the warp's 32 lanes. The compiler has to see that (they come out of votes and reductions, which have uniform
                // results): the products' operands then stay in uniform registers and take few instructions to issue. A warp per tile: neither's waits hold the other's products up.
                auto uniform = [](uint32_t x) { return __reduce_max_sync(0xFFFFFFFFu, x); };
                const uint32_t q = uniform(warp - kIssueWarp), t_s = uniform(tmem) + kColTile * q, t_p = t_s + kColP, t_o = t_s + kColO;
                constexpr uint32_t id_s = idesc_16bit(false, 128, kStep, 0, 0), id_o = idesc_16bit(false, 128, 128, 0, 1);
                const uint64_t d_k = make_smem_desc(smem_u32(sh.q[0]), 16, 1024, kSwizzle128B), d_v = make_smem_desc(smem_u32(sh.v[0]), kAtomBytes, 1024, kSwizzle128B);
                const uint32_t k_hi = static_cast<uint32_t>(d_k >> 32), v_hi = static_cast<uint32_t>(d_v >> 32);
                const uint32_t q_lo = uniform(static_cast<uint32_t>(d_k)) + (q * kTileBytes >> 4), k_lo = uniform(static_cast<uint32_t>(d_k)) + (2u * kTileBytes >> 4), v_lo = uniform(static_cast<uint32_t>(d_v));
                static_assert(offsetof(Shared, k) == 2u * kTileBytes, "K behind Q");
                uint32_t step = 0, q_phase = 0, p_phase = 0, o_phase = 1, s_phase = 1;
                bool ok = true;
                auto wait = [&](uint32_t b, uint32_t parity) {
                    ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait(b, parity, failed));
                    return ok;
                };
                auto commit = [&](uint32_t b) {
                    if (elect_one_sync()) tc_commit(b);
                };
                // the scores of a step that this tile takes part in, or not; the step's K is done with then, and behind the tile's last scores its query rows
                auto scores = [&](uint32_t at_step, bool taken, bool last) {
                    const uint32_t st = at_step % kStages;
                    if (!wait(bar(kKFull + st), at_step / kStages & 1u)) return;
                    if (taken) {
                        if (!wait(bar(kSFree + q), s_phase)) return;
                        s_phase ^= 1u;
                        tc_fence_after_sync();
                        if (elect_one_sync()) {
                            const uint32_t b = k_lo + (st * kStepBytes >> 4);
#pragma unroll
                            for (uint32_t x = 0; x < 8u; ++x) mma_f16_ss(t_s, q_lo + (((x >> 2) * kQAtom + (x & 3u) * 32u) >> 4), k_hi, b + (((x >> 2) * kAtomBytes + (x & 3u) * 32u) >> 4), k_hi, id_s, x > 0u ? 1u : 0u);
                            tc_commit(bar(kSFull + q));
                        }
                    }
                    commit(bar(kKEmpty + st));
                    if (last) commit(bar(kQEmpty + q));
                };
                Shared::Plan now;
                now.more = 1u;
                while (uniform(now.more) != 0u && ok) {
                    if (!next_plan(now) || uniform(now.seg.steps) == 0u) break;
                    const uint32_t steps = uniform(q != 0u ? now.steps[1] : now.steps[0]), seg_steps = uniform(now.seg.steps);
                    if (!wait(bar(kQFull + q), q_phase)) break;
                    q_phase ^= 1u;
                    scores(step, steps > 0u, steps <= 1u);
                    for (uint32_t j = 0; j < seg_steps && ok; ++j, ++step) {
                        const uint32_t st = step % kStages;
                        if (j + 1u < seg_steps) scores(step + 1u, j + 1u < steps, j + 2u == steps);
                        if (!ok || !wait(bar(kVFull + st), step / kStages & 1u)) break;
                        if (j < steps) {
                            if (j == 0u) {   // O of the segment before has been taken
                                if (!wait(bar(kOFree + q), o_phase)) break;
                                o_phase ^= 1u;
                            }
                            if (!wait(bar(kPFull + q), p_phase)) break;
                            p_phase ^= 1u;
                            tc_fence_after_sync();
                            if (elect_one_sync()) {
                                const uint32_t b = v_lo + (st * kStepBytes >> 4);
#pragma unroll
                                for (uint32_t x = 0; x < kBlocks; ++x) mma_f16_ts(t_o, t_p + 8u * x, b + (x * 2048u >> 4), v_hi, id_o, (j > 0u || x > 0u) ? 1u : 0u);
                                tc_commit(bar(kPFree + q));
                            }
                        }
                        commit(bar(kVEmpty + st));
                    }
                }
                if (!ok) {   // whatever was issued has to be over before the tensor memory goes back
                    commit(bar(kDrained + q));
                    (void)mbar_wait(bar(kDrained + q), 0u, &sh.not_drained);
                }
                __syncwarp();
            } else if (warp == kCopyWarp) {
                // The segments, for all roles, and the copies of a step: lane x brings block x
                uint32_t step = 0, left = end - begin, pos = begin;
                Place at = find_step(p, deal, begin);
                bool ok = true, have = false;
                Segment seg;
                // the first segment that has steps; those behind it begin an item, and have some if the run is longer than what a beginning counts as
                while (left > 0u && !have) {
                    pos = end - left;
                    seg = next_segment(p, deal, at, left);
                    have = seg.steps > 0u;
                }
                if (lane == 0u) {
                    begin_nothing(p, deal);
                    if (!have) {
                        sh.plan[0].seg.steps = sh.plan[0].more = 0u;
                        mbar_arrive(bar(kSegment));
                    }
                }
                while (have && ok) {
                    const uint32_t length = length_of(p.c, seg.b), n = count_of(p.counts, seg.b, p.S, length), segment_pos = pos;
                    have = left > kExtra;
                    if (lane == 0u) {
                        Shared::Plan& x = sh.plan[number % kSegmentSlots];
                        x.seg = seg, x.length = length, x.n = n, x.more = have;
                        for (uint32_t q = 0; q < 2u; ++q) x.steps[q] = tile_steps(p, seg, q, length, n);
                        mbar_arrive(bar(kSegment + number % kSegmentSlots));
                    }
                    ++number;
                    long long page = -1;   // of the lane's block in the next step
                    auto look_up = [&](uint32_t j) {
                        const uint32_t t = (seg.first + j) * kStep + lane * kBlockTokens;
                        if (lane < kBlocks && j < seg.steps && t < length) page = page_of(p.c, seg.b, t);
                    };
                    look_up(0u);
                    for (uint32_t j = 0; j < seg.steps; ++j, ++step) {
                        const uint32_t t = (seg.first + j) * kStep + lane * kBlockTokens, raw = step % kRawStages;
                        const bool live = lane < kBlocks && t < length, here = live && page >= 0;
                        const uint8_t* block = here ? block_of(p.c, page, seg.head, t) : nullptr;
                        const uint32_t blocks = static_cast<uint32_t>(__popc(__ballot_sync(0xFFFFFFFFu, here)));
                        ok = __all_sync(0xFFFFFFFFu, mbar_wait(bar(kRawEmpty + raw), (step / kRawStages + 1u) & 1u, failed));
                        if (!ok) break;
                        if (live && !here) sh.meta[raw][lane] = make_uint4(0x3F800000u, 0x3F800000u, 0xFFFFFFFFu, 0u);   // a page that the pool does not have: no numbers
                        __syncwarp();
                        if (lane == 0u) mbar_arrive_expect_tx(bar(kRawFull + raw), blocks * (kMeta + 16u));
                        __syncwarp();
                        if (here) {
                            bulk_load(smem_u32(&sh.meta[raw][lane]), block + kMeta, 16u, bar(kRawFull + raw));
                            bulk_load(smem_u32(sh.raw_k[raw][lane]), block, kVCodes, bar(kRawFull + raw));
                            bulk_load(smem_u32(sh.raw_v[raw][lane]), block + kVCodes, kMeta - kVCodes, bar(kRawFull + raw));
                        }
                        look_up(j + 1u);
                        if (j == 0u) {   // (what is not needed for the first copies)
                            if (lane == 0u) begin_item(p, deal, seg, segment_pos, all, n_work);
                            for (uint32_t r = lane; r < kItemRows && number > 1u; r += 32u) {
                                const uint32_t row = seg.row0 + r, i = row / p.group, h = seg.head * p.group + row - i * p.group;
                                const uint8_t* src = p.q.data + seg.b * p.q.stride_b + i * p.q.stride_s + h * p.q.stride_h;
                                if (i < n) asm volatile("prefetch.global.L2 [%0];\n\tprefetch.global.L2 [%0 + 128];" ::"l"(src));
                            }
                        }
                    }
                    if (have && ok) {
                        pos = end - left;
                        seg = next_segment(p, deal, at, left);
                    }
                }
                // after a failure: copies that are under way land before the CTA's shared memory is another's. (step: the one whose copies were not asked for)
                if (!ok) {
                    for (uint32_t i = 1; i <= kRawStages && i <= step; ++i) (void)mbar_wait(bar(kRawFull + (step - i) % kRawStages), (step - i) / kRawStages & 1u, &sh.not_drained, 20000000LL);
                }
                __syncwarp();
            } else {
                // The scales of a step, a lane a block: as the softmax wants them, and whether the step's tokens are all there and have numbers
                uint32_t step = 0;
                Shared::Plan now;
                now.more = 1u;
                bool ok = true;
                while (now.more != 0u && ok) {
                    if (!next_plan(now)) break;
                    const Segment seg = now.seg;
                    uint32_t* nan_from = &sh.nan_from[(number - 1u) % kSegmentSlots];
                    if (lane == 0u) *nan_from = 0xFFFFFFFFu;
                    int e_first = 0;   // of the segment's first block
                    bool wide = false;
                    const uint32_t length = now.length;
                    for (uint32_t j = 0; j < seg.steps; ++j, ++step) {
                        const uint32_t raw = step % kRawStages, slot = step % kScaleSlots, t0 = (seg.first + j) * kStep + lane * kBlockTokens;
                        const uint32_t live = lane >= kBlocks || t0 >= length ? 0u : 0xFFFFu >> (16u - min(length - t0, 16u));   // (behind the length there are no scales or masks)
                        ok = __all_sync(0xFFFFFFFFu, mbar_wait(bar(kRawFull + raw), step / kRawStages & 1u, failed));
                        if (!ok) break;
                        const uint4 meta = live != 0u ? sh.meta[raw][lane] : make_uint4(0x3F800000u, 0x3F800000u, 0u, 0u);
                        const int e = exponent_of(meta.y);
                        if (j == 0u) e_first = __shfl_sync(0xFFFFFFFFu, e, 0);
                        wide |= __any_sync(0xFFFFFFFFu, live != 0u && !is_near(e, e_first));
                        const bool plain = !__any_sync(0xFFFFFFFFu, lane < kBlocks && (live != 0xFFFFu || meta.z != 0u));
                        if (lane < kBlocks) {
                            float* of = sh.scales[slot][0] + lane;
                            of[0] = __uint_as_float(meta.x), of[8] = static_cast<float>(e), of[16] = power_of(-e);
                        }
                        uint32_t first = 0xFFFFFFFFu;
                        if (!plain) {
                            const uint32_t no_value = meta.z >> 16 & live;
                            first = __reduce_min_sync(0xFFFFFFFFu, no_value != 0u ? t0 + static_cast<uint32_t>(__ffs(static_cast<int>(no_value))) - 1u : 0xFFFFFFFFu);
                        }
                        __syncwarp();
                        if (lane == 0u) {
                            sh.plain[slot] = plain, sh.wide[slot] = wide;
                            if (first < *nan_from) *nan_from = first;
                            mbar_arrive(bar(kScales + slot));
                        }
                    }
                }
                __syncwarp();
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 0u && sh.failed != 0u) atomicOr(p.status, 1u);
    if (warp == kIssueWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512u);
    }
}

}  // namespace

uint32_t kv8_prefill_grid() { return static_cast<uint32_t>(current_sm_count()); }
uint32_t kv8_prefill_rows() { return kItemRows; }

cudaError_t launch_kv8_prefill(const Kv8AttendParams& p, uint32_t row_tiles, cudaStream_t stream) {
    constexpr size_t smem = sizeof(Shared) + 1024u;
    static_assert(smem <= 227u * 1024u, "shared memory of a CTA");
    static std::atomic<bool> set[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_relaxed)) {
        e = cudaFuncSetAttribute(kv8_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_relaxed);
    }
    return kv4_launch(kv8_prefill_kernel, dim3(kv8_prefill_grid()), kThreads, smem, stream, p, row_tiles);
}

}  // namespace b200mx
