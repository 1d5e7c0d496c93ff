// Eviction from the 4-bit cache by accumulated attention weight, one cluster of CTAs per (sequence, KV head), each CTA a run of consecutive tokens.
//
// A key is the weight's bits made to order as unsigned integers, NaN on top. The key of the last token that stays is found 11, 11 and 10 bits at a time from the top: a
// histogram of the keys that agree with the bits found so far, added up over the cluster through distributed shared memory, and a scan of its bins from above. Tokens
// above that key stay, and of those equal to it the earliest. Their places follow from ballots and counts in token order; the CTA then copies the 136 bytes of each
// token of its run that stays, 8 lanes a token.
//
// The keys stay in registers (8 a thread) where the runs are short enough; else they are read again from L2 for every pass.
#include "kv4.cuh"

#include <cooperative_groups.h>

#include <atomic>

namespace b200mx {

namespace {

using namespace kv4;
namespace cg = cooperative_groups;

constexpr unsigned kThreads = 1024, kWarps = kThreads / 32, kHeld = 8, kBins = 2048, kMostCtas = 8;

__device__ __forceinline__ uint32_t order_key(float w) {
    const uint32_t b = __float_as_uint(w);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
    if (b == 0x80000000u) return 0x80000000u;   // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Shared {
    uint32_t bins[3][kBins];          // of the three passes
    uint32_t sums[kWarps], equals[kWarps];
    uint32_t digit, rest;
    uint32_t above, equal;            // of this CTA's run: for the CTAs behind it
};

template <bool kInRegisters>
__global__ void __launch_bounds__(kThreads) kv4_evict_kernel(const __grid_constant__ Kv4EvictParams p) {
    __shared__ Shared sh;
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t n_ctas = cluster.num_blocks(), rank = cluster.block_rank(), lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    for (uint32_t i = threadIdx.x; i < 3u * kBins; i += kThreads) (&sh.bins[0][0])[i] = 0u;
    pdl_launch();
    pdl_wait();
    const uint32_t bh = blockIdx.x / n_ctas, b = bh / p.from.HK, head = bh % p.from.HK;
    const uint32_t L = length_of(p.from, b), keep = p.keep;
    const float* w = p.weights + static_cast<size_t>(bh) * p.weights_width;
    int32_t* kept = p.kept + static_cast<size_t>(bh) * keep;
    if (bh % p.from.HK == 0u && rank == 0u && threadIdx.x == 0u) p.into.lengths[b] = static_cast<int32_t>(min(L, keep));
    const bool all = L <= keep;
    // this CTA's tokens t0 .. t1 - 1, in rounds of a token per thread; tokens first .. last - 1 compete for `places`
    const uint32_t run = (L + n_ctas - 1u) / n_ctas, t0 = min(L, rank * run), t1 = min(L, t0 + run), rounds = (t1 - t0 + kThreads - 1u) / kThreads;
    const uint32_t last = all ? 0u : L - p.recent, places = all ? 0u : keep - p.first - p.recent;
    uint32_t held[kHeld];
    auto key_at = [&](uint32_t t) { return t < t1 && t >= p.first && t < last ? order_key(ld_f32(w + t)) : 0u; };
    if (kInRegisters) {
#pragma unroll
        for (uint32_t k = 0; k < kHeld; ++k) held[k] = k < rounds ? key_at(t0 + k * kThreads + threadIdx.x) : 0u;
    }
    // calls f(token, key) for the thread's tokens of the run that compete
    auto each = [&](auto f) {
        if (kInRegisters) {
#pragma unroll
            for (uint32_t k = 0; k < kHeld; ++k) {
                const uint32_t t = t0 + k * kThreads + threadIdx.x;
                if (t < t1 && t >= p.first && t < last) f(held[k]);
            }
        } else {
            for (uint32_t t = t0 + threadIdx.x; t < t1; t += kThreads) {
                if (t >= p.first && t < last) f(order_key(ld_f32(w + t)));
            }
        }
    };
    uint32_t found = 0, rest = places;   // the bits found, and how many of the keys that agree with them stay
    __syncthreads();
    if (places > 0u) {   // (the same in the whole cluster)
        constexpr int kShift[3] = {21, 10, 0};
        constexpr uint32_t kMask[3] = {2047u, 2047u, 1023u};
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            each([&](uint32_t key) {
                if (pass == 0 || (key >> kShift[pass == 0 ? 0 : pass - 1]) == found) atomicAdd(&sh.bins[pass][(key >> kShift[pass]) & kMask[pass]], 1u);
            });
            if (n_ctas > 1u) cluster.sync();
            else __syncthreads();
            // thread i has the bins 2047 - 2 i and 2046 - 2 i of the whole cluster
            const uint32_t hi_bin = kBins - 1u - 2u * threadIdx.x;
            uint32_t hi = 0, lo = 0;
            for (uint32_t c = 0; c < n_ctas; ++c) {
                const uint2 two = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(&sh.bins[pass][hi_bin - 1u], c));
                lo += two.x, hi += two.y;
            }
            uint32_t s = hi + lo;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t a = __shfl_up_sync(0xFFFFFFFFu, s, o);
                if (lane >= static_cast<unsigned>(o)) s += a;
            }
            if (lane == 31u) sh.sums[warp] = s;
            __syncthreads();
            uint32_t before = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? sh.sums[lane] : 0u) + s - hi - lo;   // keys in bins above
            if (before < rest && before + hi + lo >= rest) {   // one thread of the CTA
                const bool upper = before + hi >= rest;
                sh.digit = upper ? hi_bin : hi_bin - 1u;
                sh.rest = rest - before - (upper ? 0u : hi);
            }
            __syncthreads();
            found = (found << (pass == 2 ? 10 : 11)) | sh.digit;
            rest = sh.rest;
        }
    }
    // how many of the run stay for certain, and how many are equal to the key found
    uint32_t above = 0, equal = 0;
    for (uint32_t k = 0; k < rounds; ++k) {
        const uint32_t t = t0 + k * kThreads + threadIdx.x;
        if (t < t1 && (all || t < p.first || t >= last)) ++above;
    }
    if (places > 0u) each([&](uint32_t key) { above += key > found, equal += key == found; });
    const uint32_t above_w = __reduce_add_sync(0xFFFFFFFFu, above), equal_w = __reduce_add_sync(0xFFFFFFFFu, equal);
    if (lane == 0u) sh.sums[warp] = above_w, sh.equals[warp] = equal_w;
    __syncthreads();
    if (warp == 0u) {
        const uint32_t a = __reduce_add_sync(0xFFFFFFFFu, sh.sums[lane]), e = __reduce_add_sync(0xFFFFFFFFu, sh.equals[lane]);
        if (lane == 0u) sh.above = a, sh.equal = e;
    }
    if (n_ctas > 1u) cluster.sync();
    else __syncthreads();
    uint32_t place = 0, ties = 0;   // tokens of the runs in front that stay; those equal to the key
    for (uint32_t c = 0; c < rank; ++c) place += *cluster.map_shared_rank(&sh.above, c), ties += *cluster.map_shared_rank(&sh.equal, c);
    if (n_ctas > 1u) cluster.sync();   // (nobody looks at another CTA's shared memory behind it)
    place += min(ties, rest);
    const uint32_t first_place = place;
    // places, a round of 1024 tokens at a time
    for (uint32_t k = 0; k < rounds; ++k) {
        const uint32_t t = t0 + k * kThreads + threadIdx.x;
        const bool certain = t < t1 && (all || t < p.first || t >= last);
        uint32_t key = 0;
        if (kInRegisters) {
#pragma unroll
            for (uint32_t x = 0; x < kHeld; ++x) key = x == k ? held[x] : key;
        } else {
            key = key_at(t);
        }
        const bool competes = places > 0u && t < t1 && t >= p.first && t < last;
        const unsigned eq = __ballot_sync(0xFFFFFFFFu, competes && key == found), sure = __ballot_sync(0xFFFFFFFFu, certain || (competes && key > found));
        if (lane == 0u) sh.sums[warp] = __popc(sure), sh.equals[warp] = __popc(eq);
        __syncthreads();
        const uint32_t below = (1u << lane) - 1u;
        const uint32_t s = sh.sums[lane], e = sh.equals[lane];
        const uint32_t ties_before = ties + __reduce_add_sync(0xFFFFFFFFu, lane < warp ? e : 0u) + __popc(eq & below), all_ties = ties + __reduce_add_sync(0xFFFFFFFFu, e);
        const uint32_t sure_before = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? s : 0u) + __popc(sure & below), all_sure = __reduce_add_sync(0xFFFFFFFFu, s);
        const uint32_t at = place + sure_before + min(ties_before, rest) - min(ties, rest);
        if ((sure >> lane & 1u) || ((eq >> lane & 1u) && ties_before < rest)) kept[at] = static_cast<int32_t>(t);
        place += all_sure + min(all_ties, rest) - min(ties, rest);
        ties = all_ties;
        __syncthreads();
    }
    if (rank + 1u == n_ctas) {
        for (uint32_t j = min(L, keep) + threadIdx.x; j < keep; j += kThreads) kept[j] = -1;
    }
    // the tokens of the run that stay: lanes 0-3 of eight their K codes, 4-7 their V codes, 0 and 4 the scales too
    const unsigned part = threadIdx.x & 7u;
    const uint32_t page = 1u << p.from.page_log2, codes_at = part < 4u ? 0u : 64u * page, scales_at = part < 4u ? 128u * page : 132u * page;
    constexpr uint32_t kRows = 4;   // tokens of eight lanes on their way at once
    for (uint32_t j0 = first_place + (threadIdx.x >> 3); j0 < place; j0 += kRows * (kThreads / 8u)) {
        uint32_t t[kRows];
        long long from[kRows], to[kRows];
        uint4 codes[kRows];
        uint32_t sc[kRows];
#pragma unroll
        for (uint32_t k = 0; k < kRows; ++k) {
            const uint32_t j = j0 + k * (kThreads / 8u);
            t[k] = j < place ? static_cast<uint32_t>(ld_i32(kept + j)) : 0u;
        }
#pragma unroll
        for (uint32_t k = 0; k < kRows; ++k) {
            const uint32_t j = j0 + k * (kThreads / 8u);
            from[k] = to[k] = -1;
            if (j < place) from[k] = page_of(p.from, b, t[k]), to[k] = page_of(p.into, b, j);
        }
#pragma unroll
        for (uint32_t k = 0; k < kRows; ++k) {
            codes[k] = make_uint4(0u, 0u, 0u, 0u), sc[k] = 0xFFFFFFFFu;   // what a page outside the pool holds: NaN
            if (from[k] >= 0) {
                const uint8_t* in = record_of(p.from, from[k], head);
                const uint32_t s = t[k] & (page - 1u);
                codes[k] = ld_v4(in + codes_at + 64u * s + 16u * (part & 3u));
                if ((part & 3u) == 0u) sc[k] = ld_u32(in + scales_at + 4u * s);
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kRows; ++k) {
            const uint32_t j = j0 + k * (kThreads / 8u), d = j & (page - 1u);
            if (j < place && p.weights_out != nullptr && part == 0u) p.weights_out[static_cast<size_t>(bh) * p.weights_out_width + j] = ld_f32(w + t[k]);
            if (to[k] < 0) continue;
            uint8_t* out = record_of(p.into, to[k], head);
            *reinterpret_cast<uint4*>(out + codes_at + 64u * d + 16u * (part & 3u)) = codes[k];
            if ((part & 3u) == 0u) *reinterpret_cast<uint32_t*>(out + scales_at + 4u * d) = sc[k];
        }
    }
}

}  // namespace

cudaError_t launch_kv4_evict(const Kv4EvictParams& p, cudaStream_t stream) {
    // CTAs of a (sequence, head): as many as fill the machine, or as the longest sequence needs to keep its keys in registers
    const uint64_t tokens = static_cast<uint64_t>(p.from.table_width) << p.from.page_log2;
    const uint32_t items = p.from.B * p.from.HK, sms = static_cast<uint32_t>(current_sm_count());
    uint32_t ctas = 1;
    while (ctas < kMostCtas && (items * ctas * 2u <= sms + sms / 4u || tokens > static_cast<uint64_t>(ctas) * kHeld * kThreads)) ctas *= 2u;
    while (ctas > 1u && tokens < static_cast<uint64_t>(ctas) * 256u) ctas /= 2u;   // (no runs of less than 256 tokens)
    const bool held = tokens <= static_cast<uint64_t>(ctas) * kHeld * kThreads;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(items * ctas, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, held ? kv4_evict_kernel<true> : kv4_evict_kernel<false>, p);
}

}  // namespace b200mx
