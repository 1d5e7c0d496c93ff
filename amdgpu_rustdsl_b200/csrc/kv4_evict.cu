// Eviction from the 4-bit cache by accumulated attention weight.
//
// Selection, one CTA per (sequence, KV head): the weight of the last token that stays is found by its bits, eight at a time from the top (a histogram of the keys
// that agree with the digits found so far); a key is the weight's bits made to order as unsigned integers, NaN on top. Tokens above that weight stay, and of those
// equal to it the earliest. Each thread has a run of consecutive tokens, so one scan over the threads gives the places of all. Then a copy of the 136 bytes of each
// token that stays, 8 lanes a token.
#include "kv4.cuh"

namespace b200mx {

namespace {

using namespace kv4;

constexpr unsigned kSelectThreads = 1024;

__device__ __forceinline__ uint32_t order_key(float w) {
    const uint32_t b = __float_as_uint(w);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
    if (b == 0x80000000u) return 0x80000000u;   // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// exclusive sums over the CTA's threads of x and y; total in every thread
__device__ __forceinline__ uint2 scan_pair(uint2 x, uint2* part, uint2& total) {
    const unsigned lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint2 s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xFFFFFFFFu, s.x, o), b = __shfl_up_sync(0xFFFFFFFFu, s.y, o);
        if (lane >= static_cast<unsigned>(o)) s.x += a, s.y += b;
    }
    if (lane == 31u) part[warp] = s;
    __syncthreads();
    uint2 before = make_uint2(0u, 0u);
    total = make_uint2(0u, 0u);
    for (unsigned w = 0; w < kSelectThreads / 32u; ++w) {
        if (w < warp) before.x += part[w].x, before.y += part[w].y;
        total.x += part[w].x, total.y += part[w].y;
    }
    __syncthreads();
    return make_uint2(before.x + s.x - x.x, before.y + s.y - x.y);
}

__global__ void __launch_bounds__(kSelectThreads) kv4_select_kernel(const __grid_constant__ Kv4EvictParams p) {
    __shared__ uint32_t bins[256];
    __shared__ uint2 part[kSelectThreads / 32u];
    __shared__ uint32_t found_digit, found_rest;
    pdl_launch();
    pdl_wait();
    const uint32_t b = blockIdx.x / p.from.HK, head = blockIdx.x % p.from.HK;
    const uint32_t L = length_of(p.from, b), keep = p.keep;
    const float* w = p.weights + static_cast<size_t>(blockIdx.x) * p.weights_width;
    int32_t* kept = p.kept + static_cast<size_t>(blockIdx.x) * keep;
    if (head == 0u && threadIdx.x == 0u) p.into.lengths[b] = static_cast<int32_t>(min(L, keep));
    if (L <= keep) {
        for (uint32_t j = threadIdx.x; j < keep; j += kSelectThreads) kept[j] = j < L ? static_cast<int32_t>(j) : -1;
        return;
    }
    // tokens first .. last - 1 compete for `places`
    const uint32_t last = L - p.recent;
    const uint32_t places = keep - p.first - p.recent;
    uint32_t prefix = 0, rest = places;   // rest: how many of the keys that agree with the prefix stay
    if (places > 0u) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (unsigned i = threadIdx.x; i < 256u; i += kSelectThreads) bins[i] = 0;
            __syncthreads();
            for (uint32_t t = p.first + threadIdx.x; t < last; t += kSelectThreads) {
                const uint32_t key = order_key(ld_f32(w + t));
                if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&bins[(key >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (threadIdx.x == 0u) {
                uint32_t above = 0;
                int d = 255;
                for (; d > 0; --d) {
                    if (above + bins[d] >= rest) break;
                    above += bins[d];
                }
                found_digit = static_cast<uint32_t>(d);
                found_rest = rest - above;
            }
            __syncthreads();
            prefix = (prefix << 8) | found_digit;
            rest = found_rest;
            __syncthreads();
        }
    }
    // a run of consecutive tokens per thread: how many are above the weight found, how many equal it
    const uint32_t run = (L + kSelectThreads - 1u) / kSelectThreads, t0 = min(L, threadIdx.x * run), t1 = min(L, t0 + run);
    uint2 mine = make_uint2(0u, 0u), total;
    for (uint32_t t = t0; t < t1; ++t) {
        if (t < p.first || t >= last) {
            ++mine.x;
        } else if (places > 0u) {
            const uint32_t key = order_key(ld_f32(w + t));
            mine.x += key > prefix;
            mine.y += key == prefix;
        }
    }
    const uint2 before = scan_pair(mine, part, total);
    uint32_t equal = before.y, j = before.x + min(before.y, rest);
    if (places == 0u) rest = 0u;
    for (uint32_t t = t0; t < t1; ++t) {
        bool stay = t < p.first || t >= last;
        if (!stay && places > 0u) {
            const uint32_t key = order_key(ld_f32(w + t));
            stay = key > prefix || (key == prefix && equal < rest);
            equal += key == prefix;
        }
        if (stay) kept[j++] = static_cast<int32_t>(t);
    }
}

__global__ void __launch_bounds__(256) kv4_move_kernel(const __grid_constant__ Kv4EvictParams p) {
    pdl_launch();
    pdl_wait();
    const unsigned long long n = static_cast<unsigned long long>(p.from.B) * p.from.HK * p.keep;
    const unsigned part = threadIdx.x & 7u;
    for (unsigned long long i = blockIdx.x * 32ull + (threadIdx.x >> 3); i < n; i += gridDim.x * 32ull) {
        const int32_t t = ld_i32(p.kept + i);
        if (t < 0) continue;
        const uint32_t j = static_cast<uint32_t>(i % p.keep);
        const unsigned long long bh = i / p.keep;
        const uint32_t b = static_cast<uint32_t>(bh / p.from.HK), head = static_cast<uint32_t>(bh % p.from.HK), page = 1u << p.from.page_log2;
        if (p.weights_out != nullptr && part == 0u) p.weights_out[bh * p.weights_out_width + j] = ld_f32(p.weights + bh * p.weights_width + static_cast<uint32_t>(t));
        const long long from = page_of(p.from, b, static_cast<uint32_t>(t)), to = page_of(p.into, b, j);
        if (to < 0) continue;
        const uint32_t s = static_cast<uint32_t>(t) & (page - 1u), d = j & (page - 1u);
        uint8_t* out = record_of(p.into, to, head);
        // lanes 0-3: K codes, 4-7: V codes; lanes 0 and 4 the scales too
        const uint32_t base = part < 4u ? 0u : 64u * page, scales = part < 4u ? 128u * page : 132u * page;
        uint4 codes = make_uint4(0u, 0u, 0u, 0u);
        uint32_t sc = 0xFFFFFFFFu;   // what a page outside the pool holds: NaN
        if (from >= 0) {
            const uint8_t* in = record_of(p.from, from, head);
            codes = ld_v4(in + base + 64u * s + 16u * (part & 3u));
            if ((part & 3u) == 0u) sc = ld_u32(in + scales + 4u * s);
        }
        *reinterpret_cast<uint4*>(out + base + 64u * d + 16u * (part & 3u)) = codes;
        if ((part & 3u) == 0u) *reinterpret_cast<uint32_t*>(out + scales + 4u * d) = sc;
    }
}

}  // namespace

cudaError_t launch_kv4_evict(const Kv4EvictParams& p, cudaStream_t stream) {
    cudaError_t e = kv4_launch(kv4_select_kernel, dim3(p.from.B * p.from.HK), kSelectThreads, 0, stream, p);
    if (e != cudaSuccess) return e;
    const unsigned long long blocks = (1ull * p.from.B * p.from.HK * p.keep + 31ull) / 32ull, cap = 8ull * static_cast<unsigned long long>(current_sm_count());
    return kv4_launch(kv4_move_kernel, dim3(static_cast<unsigned>(blocks < cap ? blocks : cap)), 256u, 0, stream, p);
}

}  // namespace b200mx
