// Eviction from the 4-bit cache by accumulated attention weight, one cluster of CTAs per (sequence, KV head), each CTA a run of consecutive tokens.
//
// A key is the weight's bits made to order as unsigned integers, NaN on top. The key of the last token that stays is found 8 bits at a time from the top: a
// histogram of the keys that agree with the bits found so far, added up over the cluster through distributed shared memory, and a scan of its bins from above. Tokens
// above that key stay, and of those equal to it the earliest. Their places follow from ballots and counts in token order; a second
// kernel copies the 136 bytes of each token that stays.
//
// The selection is bound by latency: the loads, four dependent rounds of histogram, barriers and scan (37 % of the issue slots with one CTA a head), and where a head has several CTAs an exchange of
// the cluster in each (1 to 2 us). The keys stay in registers (16 a thread) where
// the runs are short enough; else they are read again from L2 for every pass. 512 threads, so that two CTAs share an SM: with 1024, one a SM, 24 clusters of 8 took two rounds.
// 16 x 8 heads of 4096 tokens to 1024: selection 15 us, copy 12; 3 x 8 heads of 50001 tokens to 6250: 22 and 11.
#include "kv4.cuh"

#include <cooperative_groups.h>

#include <atomic>

namespace b200mx {

namespace {

using namespace kv4;
namespace cg = cooperative_groups;

constexpr unsigned kThreads = 512, kWarps = kThreads / 32, kHeld = 16, kBins = 256, kMostCtas = 8;
constexpr int kPasses = 4;

__device__ __forceinline__ uint32_t order_key(float w) {
    const uint32_t b = __float_as_uint(w);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
    if (b == 0x80000000u) return 0x80000000u;   // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Shared {
    uint32_t bins[kPasses][kBins];
    uint32_t counts[kHeld * kWarps];   // per round and warp: tokens that stay for certain in the upper half, tokens equal to the key found in the lower
    uint32_t sums[kWarps];
    uint32_t digit, rest;
    uint32_t above, equal;             // of this CTA's run: for the CTAs behind it
};

template <bool kInRegisters>
__global__ void __launch_bounds__(kThreads, 2) kv4_select_kernel(const __grid_constant__ Kv4EvictParams p) {
    __shared__ Shared sh;
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t n_ctas = cluster.num_blocks(), rank = cluster.block_rank(), lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    for (uint32_t i = threadIdx.x; i < kPasses * kBins; i += kThreads) (&sh.bins[0][0])[i] = 0u;
    pdl_launch();
    pdl_wait();
    const uint32_t bh = blockIdx.x / n_ctas, b = bh / p.from.HK;
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
#pragma unroll
        for (int pass = 0; pass < kPasses; ++pass) {
            const int shift = 24 - 8 * pass;
            each([&](uint32_t key) {
                if (pass == 0 || (key >> (shift + 8)) == found) atomicAdd(&sh.bins[pass][(key >> shift) & 255u], 1u);
            });
            if (n_ctas > 1u) cluster.sync();
            else __syncthreads();
            // thread i < 256 has bin 255 - i of the whole cluster
            uint32_t mine = 0, s = 0;
            if (threadIdx.x < kBins) {
                uint32_t parts[kMostCtas];   // all on their way at once
#pragma unroll
                for (uint32_t c = 0; c < kMostCtas; ++c) parts[c] = c < n_ctas ? *cluster.map_shared_rank(&sh.bins[pass][kBins - 1u - threadIdx.x], c) : 0u;
#pragma unroll
                for (uint32_t c = 0; c < kMostCtas; ++c) mine += parts[c];
                s = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t a = __shfl_up_sync(0xFFFFFFFFu, s, o);
                    if (lane >= static_cast<unsigned>(o)) s += a;
                }
                if (lane == 31u) sh.sums[warp] = s;
            }
            __syncthreads();
            const uint32_t before = __reduce_add_sync(0xFFFFFFFFu, lane < warp && lane < kBins / 32u ? sh.sums[lane] : 0u) + s - mine;   // keys in bins above
            if (threadIdx.x < kBins && before < rest && before + mine >= rest) sh.digit = kBins - 1u - threadIdx.x, sh.rest = rest - before;   // one thread
            __syncthreads();
            found = (found << 8) | sh.digit;
            rest = sh.rest;
        }
    }
    // how many of the run stay for certain, and how many are equal to the key found
    auto certain_at = [&](uint32_t t) { return t < t1 && (all || t < p.first || t >= last); };
    uint32_t both = 0, equal = 0;
    for (uint32_t k = 0; k < rounds; ++k) both += certain_at(t0 + k * kThreads + threadIdx.x);
    if (places > 0u) each([&](uint32_t key) { both += key > found, equal += key == found; });
    both = __reduce_add_sync(0xFFFFFFFFu, both), equal = __reduce_add_sync(0xFFFFFFFFu, equal);
    if (threadIdx.x == 0u) sh.above = sh.equal = 0u;
    __syncthreads();
    if (lane == 0u) atomicAdd(&sh.above, both), atomicAdd(&sh.equal, equal);
    if (n_ctas > 1u) cluster.sync();
    else __syncthreads();
    uint32_t place = 0, ties = 0;   // tokens of the runs in front that stay for certain; those equal to the key
#pragma unroll
    for (uint32_t c = 0; c + 1u < kMostCtas; ++c) {
        if (c < rank) place += *cluster.map_shared_rank(&sh.above, c), ties += *cluster.map_shared_rank(&sh.equal, c);
    }
    // places, kHeld rounds of a token per thread at a time: ballots per round and warp, and one scan over their counts
    for (uint32_t k0 = 0; k0 < rounds; k0 += kHeld) {
        uint32_t equals = 0, stays = 0;   // this thread's token of round k0 + k in bit k
#pragma unroll
        for (uint32_t k = 0; k < kHeld; ++k) {
            if (k0 + k >= rounds) {
                if (lane == 0u) sh.counts[k * kWarps + warp] = 0u;
                continue;
            }
            const uint32_t t = t0 + (k0 + k) * kThreads + threadIdx.x;
            const uint32_t key = kInRegisters ? held[k] : key_at(t);
            const bool competes = places > 0u && t < t1 && t >= p.first && t < last, eq = competes && key == found, sure = certain_at(t) || (competes && key > found);
            equals |= static_cast<uint32_t>(eq) << k, stays |= static_cast<uint32_t>(sure) << k;
            const uint32_t n_eq = __popc(__ballot_sync(0xFFFFFFFFu, eq)), n_sure = __popc(__ballot_sync(0xFFFFFFFFu, sure));
            if (lane == 0u) sh.counts[k * kWarps + warp] = n_sure << 16 | n_eq;
        }
        __syncthreads();
        uint32_t mine = 0, s = 0;
        if (threadIdx.x < kHeld * kWarps) {   // (counts of a run of kHeld rounds stay below 2^16)
            s = mine = sh.counts[threadIdx.x];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t a = __shfl_up_sync(0xFFFFFFFFu, s, o);
                if (lane >= static_cast<unsigned>(o)) s += a;
            }
            if (lane == 31u) sh.sums[warp] = s;
        }
        __syncthreads();
        const uint32_t sums = lane < kHeld * kWarps / 32u ? sh.sums[lane] : 0u, total = __reduce_add_sync(0xFFFFFFFFu, sums), front = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? sums : 0u);
        if (threadIdx.x < kHeld * kWarps) sh.counts[threadIdx.x] = front + s - mine;
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < kHeld; ++k) {
            if (k0 + k >= rounds) break;
            const uint32_t eq = __ballot_sync(0xFFFFFFFFu, equals >> k & 1u), sure = __ballot_sync(0xFFFFFFFFu, stays >> k & 1u), below = (1u << lane) - 1u;
            const uint32_t before = sh.counts[k * kWarps + warp], ties_before = ties + (before & 0xFFFFu) + __popc(eq & below);
            if ((stays >> k & 1u) || ((equals >> k & 1u) && ties_before < rest))
                kept[place + (before >> 16) + __popc(sure & below) + min(ties_before, rest)] = static_cast<int32_t>(t0 + (k0 + k) * kThreads + threadIdx.x);
        }
        place += total >> 16, ties += total & 0xFFFFu;
        __syncthreads();
    }
    if (rank + 1u == n_ctas) {
        for (uint32_t j = min(L, keep) + threadIdx.x; j < keep; j += kThreads) kept[j] = -1;
    }
    if (n_ctas > 1u) cluster.sync();   // (nobody looks at another CTA's shared memory behind it)
}

// Copies the tokens that stay: lanes 0-3 of eight a token's K codes, 4-7 its V codes, 0 and 4 the scales too. A kernel of its own: the selection's clusters leave half of the
// SMs idle where there are few of them, and the copy lives on as many tokens as possible being on their way.
constexpr uint32_t kMoveRows = 2;   // tokens of eight lanes on their way at once
__global__ void __launch_bounds__(256) kv4_move_kernel(const __grid_constant__ Kv4EvictParams p) {
    pdl_launch();
    pdl_wait();
    const unsigned part = threadIdx.x & 7u;
    const uint32_t page = 1u << p.from.page_log2, codes_at = part < 4u ? 0u : 64u * page, scales_at = part < 4u ? 128u * page : 132u * page;
    for (uint32_t bh = blockIdx.y; bh < p.from.B * p.from.HK; bh += gridDim.y) {
        const uint32_t b = bh / p.from.HK, head = bh - b * p.from.HK, n_kept = min(length_of(p.from, b), p.keep), j0 = blockIdx.x * (32u * kMoveRows) + (threadIdx.x >> 3);
        const float* w = p.weights + static_cast<size_t>(bh) * p.weights_width;
        const int32_t* kept = p.kept + static_cast<size_t>(bh) * p.keep;
        uint32_t t[kMoveRows], sc[kMoveRows];
        long long from[kMoveRows], to[kMoveRows];
        uint4 codes[kMoveRows];
        float weight[kMoveRows];
#pragma unroll
        for (uint32_t k = 0; k < kMoveRows; ++k) {
            const uint32_t j = j0 + 32u * k;
            t[k] = j < n_kept ? static_cast<uint32_t>(ld_i32(kept + j)) : 0u;
            to[k] = j < n_kept ? page_of(p.into, b, j) : -1;
        }
#pragma unroll
        for (uint32_t k = 0; k < kMoveRows; ++k) from[k] = j0 + 32u * k < n_kept ? page_of(p.from, b, t[k]) : -1;
#pragma unroll
        for (uint32_t k = 0; k < kMoveRows; ++k) {
            const uint32_t j = j0 + 32u * k;
            weight[k] = j < n_kept && p.weights_out != nullptr && part == 0u ? ld_f32(w + t[k]) : 0.0f;
            codes[k] = make_uint4(0u, 0u, 0u, 0u), sc[k] = 0xFFFFFFFFu;   // what a page outside the pool holds: NaN
            if (from[k] >= 0) {
                const uint8_t* in = record_of(p.from, from[k], head);
                const uint32_t s = t[k] & (page - 1u);
                codes[k] = ld_v4(in + codes_at + 64u * s + 16u * (part & 3u));
                if ((part & 3u) == 0u) sc[k] = ld_u32(in + scales_at + 4u * s);
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kMoveRows; ++k) {
            const uint32_t j = j0 + 32u * k, d = j & (page - 1u);
            if (j < n_kept && p.weights_out != nullptr && part == 0u) p.weights_out[static_cast<size_t>(bh) * p.weights_out_width + j] = weight[k];
            if (to[k] < 0) continue;
            uint8_t* out = record_of(p.into, to[k], head);
            *reinterpret_cast<uint4*>(out + codes_at + 64u * d + 16u * (part & 3u)) = codes[k];
            if ((part & 3u) == 0u) *reinterpret_cast<uint32_t*>(out + scales_at + 4u * d) = sc[k];
        }
    }
}

}  // namespace

cudaError_t launch_kv4_evict(const Kv4EvictParams& p, cudaStream_t stream) {
    // CTAs of a (sequence, head): as many as there are SMs for (8 items of 16384 tokens: 23.1 us with 8, 27.9 with the 2 that hold the keys; 128 items of 4096 tokens: 44.0 with 1,
    // 46.0 with 2), or as the longest sequence needs to keep its keys in registers (256 items of 16384 tokens: 166 us with 2, 174 with 1 that reads them again)
    const uint64_t tokens = static_cast<uint64_t>(p.from.table_width) << p.from.page_log2;
    const uint32_t items = p.from.B * p.from.HK, sms = static_cast<uint32_t>(current_sm_count());
    uint32_t ctas = 1;
    while (ctas < kMostCtas && (items * ctas * 2u <= sms || tokens > static_cast<uint64_t>(ctas) * kHeld * kThreads)) ctas *= 2u;
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, held ? kv4_select_kernel<true> : kv4_select_kernel<false>, p);
    if (e != cudaSuccess) return e;
    return kv4_launch(kv4_move_kernel, dim3((p.keep + 32u * kMoveRows - 1u) / (32u * kMoveRows), items < 65535u ? items : 65535u), 256u, 0, stream, p);
}

}  // namespace b200mx
