// Page tables, lengths, positions and slot maps from the numbers of new tokens (include/fmha_pages_abi.h).
//
// Of a take every CTA goes over all sequences' lengths and counts for itself, two sums over them (pages needed in front of a sequence, tokens granted in front of it), and then writes its share
// of the maps and of the table; what all of them read, the lengths and the stack's height, is written by the one that is done last. So a call is one launch in which nothing waits for
// another CTA: a decode step is one CTA and a few trips to memory, the maps of whole prompts get as many CTAs as keep memory busy. A cut is one CTA. Bound by these trips and the launch: on the device, taken and cut
// back, 256 x 1 tokens 9.2 us (a cut of nothing 2.2), 256 x 8 11.3, 64 prompts to 2048 tokens 13.0 for 1.6 MB of maps, four of a thread's rows in flight.
#include "../../include/fmha_pages_abi.h"
#include "cache_args.cuh"

namespace b200mx {

namespace {

constexpr uint32_t kThreads = 512, kWarps = kThreads / 32, kMostRange = 1024;   // sequences of a CTA
constexpr uint32_t kTogether = 4;                                               // rows of the maps, or entries of the table, of a thread at a time
constexpr uint32_t kParts = 4;                                                  // of a warp, whose entries stay in registers

struct PagesParams {
    int32_t *free, *table, *lengths;
    uint32_t pages, pool_pages, B, page_log2, table_width;
    const int32_t* asked;   // counts, or what to keep
    int32_t *granted, *starts;
    void* positions;
    long long* slots;
    uint32_t S;
    bool positions_64;
};

// cached nowhere on the SM: other CTAs write it in the same launch
__device__ __forceinline__ int ld_now(const int32_t* p) {
    int v;
    asm volatile("ld.global.cg.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t length_at(const PagesParams& p, uint32_t b) {
    const long long cap = static_cast<long long>(p.table_width) << p.page_log2, n = ld_now(p.lengths + b);
    return static_cast<uint32_t>(n < 0 ? 0 : (n > cap ? cap : n));
}
__device__ __forceinline__ uint32_t asked_at(const PagesParams& p, uint32_t b) { return static_cast<uint32_t>(max(ld_now(p.asked + b), 0)); }
__device__ __forceinline__ uint32_t pages_of(const PagesParams& p, uint32_t tokens) { return static_cast<uint32_t>((tokens + (1ull << p.page_log2) - 1u) >> p.page_log2); }
__device__ __forceinline__ uint32_t height(const PagesParams& p) { return min(static_cast<uint32_t>(max(ld_now(p.free), 0)), p.pages); }

// sum of the threads in front, and of all
template <typename T>
__device__ __forceinline__ T sum_in_front(T x, T* part, T& all) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    T s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T a = __shfl_up_sync(0xFFFFFFFFu, s, o);
        if (lane >= static_cast<uint32_t>(o)) s += a;
    }
    if (lane == 31u) part[warp] = s;
    __syncthreads();
    T before = 0;
    all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
        const T a = part[w];
        if (w < warp) before += a;
        all += a;
    }
    __syncthreads();
    return before + s - x;
}

struct Range {
    uint32_t begin, end;
};
__device__ __forceinline__ uint32_t share(uint32_t n, uint32_t g) { return static_cast<uint32_t>(static_cast<unsigned long long>(n) * g / gridDim.x); }
// the sequences whose table and counts a CTA writes; its rows of the maps lie in these and the one behind
__device__ __forceinline__ Range own_range(const PagesParams& p) { return {share(p.B, blockIdx.x), share(p.B, blockIdx.x + 1u)}; }

// Whether this CTA is the last one, behind everything that the others wrote. All threads.
__device__ __forceinline__ bool is_last(const PagesParams& p, uint32_t* flag) {
    if (gridDim.x == 1u) {
        __syncthreads();
        return true;
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0u) {
        const bool last = atomicAdd(reinterpret_cast<uint32_t*>(p.free) + 1, 1u) == gridDim.x - 1u;
        if (last) p.free[1] = 0;
        *flag = last;
        __threadfence();
    }
    __syncthreads();
    return *flag != 0u;
}

// f(sequence's place in the range, its page, its pages) for the pages of a range's sequences, a warp or, with few of them, several a sequence; `pages` of a place
template <typename Count, typename F>
__device__ __forceinline__ void for_pages(uint32_t n, Count pages, F f) {
    const uint32_t warps = n >= kWarps || n == 0u ? 1u : kWarps / n, warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    if (warp / warps >= kWarps / warps) return;   // (warps that are left over)
    for (uint32_t x = warp / warps; x < n; x += kWarps / warps) {
        const uint32_t of = pages(x);
        for (uint32_t k = (warp % warps) * 32u + lane; k < of; k += warps * 32u) f(x, k);
    }
}

__global__ void __launch_bounds__(kThreads) pages_take_kernel(const __grid_constant__ PagesParams p) {
    __shared__ unsigned long long part64[kWarps];
    __shared__ uint32_t part32[kWarps];
    __shared__ uint32_t sm_length[kMostRange + 2], sm_granted[kMostRange + 2], sm_before[kMostRange + 2];
    __shared__ uint32_t last_flag;
    kv4::pdl_launch();
    kv4::pdl_wait();
    const uint32_t per = (p.B + kThreads - 1u) / kThreads, b0 = min(threadIdx.x * per, p.B), b1 = min(b0 + per, p.B), n_free = height(p);
    const unsigned long long cap = static_cast<unsigned long long>(p.table_width) << p.page_log2;
    // (a thread's first sequence stays in registers)
    const uint32_t length0 = b0 < b1 ? length_at(p, b0) : 0u, asked0 = b0 < b1 ? asked_at(p, b0) : 0u;
    const auto look = [&](uint32_t b, uint32_t& length, uint32_t& asked, bool& fits) {
        length = b == b0 ? length0 : length_at(p, b), asked = b == b0 ? asked0 : asked_at(p, b);
        fits = static_cast<unsigned long long>(length) + asked <= cap;
        return fits ? pages_of(p, length + asked) - pages_of(p, length) : 0u;
    };
    uint32_t length, asked;
    bool fits;
    unsigned long long mine = 0, all;
    for (uint32_t b = b0; b < b1; ++b) mine += look(b, length, asked, fits);
    const unsigned long long in_front = sum_in_front(mine, part64, all);
    uint32_t tokens = 0, all_tokens;
    unsigned long long upto = in_front;
    for (uint32_t b = b0; b < b1; ++b) {
        const uint32_t need = look(b, length, asked, fits);
        upto += need;
        if (fits && (need == 0u || upto <= n_free)) tokens += asked;
    }
    uint32_t start = sum_in_front(tokens, part32, all_tokens);
    const Range range = own_range(p);
    const uint32_t known = min(range.end + 1u, p.B);   // (the maps' rows may begin the sequence behind)
    const bool alone = gridDim.x == 1u;
    upto = in_front;
    uint32_t taken = 0;
    for (uint32_t b = b0; b < b1; ++b) {
        const uint32_t need = look(b, length, asked, fits);
        upto += need;
        const bool ok = fits && (need == 0u || upto <= n_free);
        const uint32_t granted = ok ? asked : 0u;
        if (ok && need != 0u) taken = static_cast<uint32_t>(upto);   // (ascending)
        if (b >= range.begin && b < known) {
            sm_length[b - range.begin] = length, sm_granted[b - range.begin] = granted, sm_before[b - range.begin] = static_cast<uint32_t>(min(upto - need, 0xFFFFFFFFull));
            if (b < range.end) {
                p.granted[b] = static_cast<int32_t>(granted);
                if (alone) p.lengths[b] = static_cast<int32_t>(length + granted);   // (each thread has read its own)
                if (p.starts != nullptr) p.starts[b] = static_cast<int32_t>(start);
            }
        }
        start += granted;
    }
    if (p.starts != nullptr && blockIdx.x == gridDim.x - 1u && threadIdx.x == 0u) p.starts[p.B] = static_cast<int32_t>(all_tokens);
    __syncthreads();
    const int32_t* stack = p.free + 4;
    for_pages(
        range.end - range.begin,
        [&](uint32_t x) { return sm_granted[x] == 0u ? 0u : pages_of(p, sm_length[x] + sm_granted[x]) - pages_of(p, sm_length[x]); },
        [&](uint32_t x, uint32_t k) { p.table[static_cast<size_t>(range.begin + x) * p.table_width + pages_of(p, sm_length[x]) + k] = ld_now(stack + (n_free - 1u - sm_before[x] - k)); });
    if (p.positions != nullptr || p.slots != nullptr) {
        const uint32_t rows = p.B * p.S, end = share(rows, blockIdx.x + 1u);
        for (uint32_t r0 = share(rows, blockIdx.x) + threadIdx.x; r0 < end; r0 += kTogether * kThreads) {
            int position[kTogether], page[kTogether];
#pragma unroll
            for (uint32_t k = 0; k < kTogether; ++k) {   // rows whose pages are on their way together
                const uint32_t r = r0 + k * kThreads, b = r / p.S, i = r - b * p.S, x = b - range.begin;
                position[k] = page[k] = -1;
                if (r >= end || i >= sm_granted[x]) continue;
                const uint32_t t = sm_length[x] + i;
                position[k] = static_cast<int>(t);
                if (p.slots == nullptr) continue;
                const uint32_t at = t >> p.page_log2, had = pages_of(p, sm_length[x]);
                page[k] = ld_now(at < had ? p.table + static_cast<size_t>(b) * p.table_width + at : stack + (n_free - 1u - sm_before[x] - (at - had)));
            }
#pragma unroll
            for (uint32_t k = 0; k < kTogether; ++k) {
                const uint32_t r = r0 + k * kThreads;
                if (r >= end) break;
                if (p.positions != nullptr) {
                    if (p.positions_64) static_cast<long long*>(p.positions)[r] = position[k];
                    else static_cast<int32_t*>(p.positions)[r] = position[k];
                }
                if (p.slots != nullptr) p.slots[r] = page[k] < 0 ? -1ll : (static_cast<long long>(page[k]) << p.page_log2) + (static_cast<uint32_t>(position[k]) & ((1u << p.page_log2) - 1u));
            }
        }
    }
    if (!is_last(p, &last_flag)) return;
    if (!alone) {
        for (uint32_t b = threadIdx.x; b < p.B; b += kThreads) p.lengths[b] = static_cast<int32_t>(length_at(p, b) + ld_now(p.granted + b));
    }
    const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, taken);
    if ((threadIdx.x & 31u) == 0u) part32[threadIdx.x >> 5] = most;
    __syncthreads();
    if (threadIdx.x == 0u) {
        uint32_t n = 0;
        for (uint32_t w = 0; w < kWarps; ++w) n = max(n, part32[w]);
        p.free[0] = static_cast<int32_t>(n_free - n);
    }
}

// One CTA, from the last sequences to the first, a thread's one at a time. What goes back is counted first, since entries that name no page do not: a sequence's one page by its thread, more by warps.
__global__ void __launch_bounds__(kThreads) pages_cut_kernel(const __grid_constant__ PagesParams p) {
    __shared__ unsigned long long part64[kWarps], sm_to[kThreads];   // sm_to: height at which a sequence's last page goes back
    __shared__ uint32_t sm_kept[kThreads], sm_many[kThreads], sm_count[kThreads];
    kv4::pdl_launch();
    kv4::pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, n_free = height(p);
    const auto names_page = [&](int entry) { return entry >= 0 && static_cast<uint32_t>(entry) < p.pool_pages; };
    unsigned long long given = 0;   // pages of the sequences behind
    for (uint32_t end = p.B, n; end > 0u; end -= n) {
        n = min(end, kThreads);
        const uint32_t first = end - n, x = threadIdx.x, b = first + x;
        uint32_t kept = 0, many = 0, count = 0;
        bool one = false;
        int entry = -1;
        if (x < n) {
            const uint32_t length = length_at(p, b), keep = min(length, asked_at(p, b)), had = pages_of(p, length);
            kept = pages_of(p, keep);
            one = had - kept == 1u, many = one ? 0u : had - kept;
            if (one) entry = ld_now(p.table + static_cast<size_t>(b) * p.table_width + kept);
            p.lengths[b] = static_cast<int32_t>(keep);   // (each thread has read its own)
            count = names_page(entry);
        }
        sm_kept[x] = kept, sm_many[x] = many;
        // Sequences of more than one page are cut up into parts, a warp's every kWarps-th; a part's entries are looked at kTogether of a lane at a time. Where a warp has kParts parts of one such look at most,
        // all of them are under way together and stay in registers until they are written (64 sequences of up to 128 pages taken and cut: 13.0 us of the device, 14.7 in the loop)
        const uint32_t parts_log2 = n >= kWarps ? 0u : 31u - static_cast<uint32_t>(__clz(static_cast<int>(kWarps / n))), parts = 1u << parts_log2;
        const bool any = __syncthreads_or(many != 0u) != 0, few = any && n * parts <= kParts * kWarps && __syncthreads_or(many > 32u * kTogether * parts) == 0;
        struct Part {
            int32_t* row;
            uint32_t of, y;
        };
        const auto part_of = [&](uint32_t u) {
            const uint32_t y = u < n * parts ? u >> parts_log2 : 0u, part = u - y * parts, of = u < n * parts ? sm_many[y] : 0u;
            const auto at = [&](uint32_t k) { return static_cast<uint32_t>(static_cast<unsigned long long>(of) * k >> parts_log2); };
            return Part{p.table + static_cast<size_t>(first + y) * p.table_width + sm_kept[y] + at(part), at(part + 1u) - at(part), y};
        };
        const auto look = [&](const Part& part, uint32_t k0, int (&e)[kTogether]) {
#pragma unroll
            for (uint32_t k = 0; k < kTogether; ++k) e[k] = k0 + 32u * k + lane < part.of ? ld_now(part.row + k0 + 32u * k + lane) : -1;
        };
        const auto pages_in = [&](const int (&e)[kTogether]) {
            uint32_t pages = 0;
#pragma unroll
            for (uint32_t k = 0; k < kTogether; ++k) pages += static_cast<uint32_t>(__popc(__ballot_sync(0xFFFFFFFFu, names_page(e[k]))));
            return pages;
        };
        // entries go back from the height `above` down
        const auto give_back = [&](const Part& part, uint32_t k0, const int (&e)[kTogether], unsigned long long& above) {
#pragma unroll
            for (uint32_t k = 0; k < kTogether; ++k) {
                const uint32_t pages = __ballot_sync(0xFFFFFFFFu, names_page(e[k]));
                const unsigned long long at = above - 1u - static_cast<uint32_t>(__popc(pages & ((1u << lane) - 1u)));
                if (names_page(e[k]) && at < p.pages) p.free[4u + at] = e[k];
                if (k0 + 32u * k + lane < part.of) part.row[k0 + 32u * k + lane] = -1;
                above -= static_cast<uint32_t>(__popc(pages));
            }
        };
        const auto height_of = [&](const Part& part, uint32_t u) {   // behind the parts behind
            unsigned long long above = sm_to[part.y];
            for (uint32_t k = u; k < (part.y + 1u) * parts; ++k) above += sm_count[k];
            return above;
        };
        int held[kParts][kTogether];
        if (few) {
#pragma unroll
            for (uint32_t i = 0; i < kParts; ++i) look(part_of(warp + i * kWarps), 0u, held[i]);
#pragma unroll
            for (uint32_t i = 0; i < kParts; ++i) {
                const uint32_t pages = pages_in(held[i]);
                if (lane == 0u && warp + i * kWarps < n * parts) sm_count[warp + i * kWarps] = pages;
            }
        } else if (any) {
            for (uint32_t u = warp; u < n * parts; u += kWarps) {
                const Part part = part_of(u);
                uint32_t pages = 0;
                for (uint32_t k0 = 0; k0 < part.of; k0 += 32u * kTogether) {
                    int e[kTogether];
                    look(part, k0, e);
                    pages += pages_in(e);
                }
                if (lane == 0u) sm_count[u] = pages;
            }
        }
        if (any) {
            __syncthreads();
            for (uint32_t k = 0; k < parts && many != 0u; ++k) count += sm_count[x * parts + k];
        }
        unsigned long long all;
        const unsigned long long in_front = sum_in_front<unsigned long long>(count, part64, all), to = n_free + given + (all - in_front - count);
        if (one) {
            if (count != 0u && to < p.pages) p.free[4u + to] = entry;
            p.table[static_cast<size_t>(b) * p.table_width + kept] = -1;
        }
        if (any) {
            sm_to[x] = to;
            __syncthreads();
        }
        if (few) {
#pragma unroll
            for (uint32_t i = 0; i < kParts; ++i) {
                const uint32_t u = warp + i * kWarps;
                if (u >= n * parts) break;
                const Part part = part_of(u);
                unsigned long long above = height_of(part, u);
                give_back(part, 0u, held[i], above);
            }
        } else if (any) {
            for (uint32_t u = warp; u < n * parts; u += kWarps) {
                const Part part = part_of(u);
                unsigned long long above = height_of(part, u);
                for (uint32_t k0 = 0; k0 < part.of; k0 += 32u * kTogether) {
                    int e[kTogether];
                    look(part, k0, e);
                    give_back(part, k0, e, above);
                }
            }
        }
        given += all;
        __syncthreads();   // (the tables are the next sequences')
    }
    if (threadIdx.x == 0u) p.free[0] = static_cast<int32_t>(min(n_free + given, static_cast<unsigned long long>(p.pages)));
}

}  // namespace
}  // namespace b200mx

namespace {

using b200mx::PagesParams;

int params_of(const fmha_pages* p, const char* name, PagesParams& r, char* err, size_t cap) {
    if (p == nullptr || p->free == nullptr || p->table == nullptr || p->lengths == nullptr) return refuse(err, cap, "%s: the stack of free pages, table and lengths must be given", name);
    if (p->page != 16u && p->page != 32u && p->page != 64u && p->page != 128u) return refuse(err, cap, "%s: pages hold 16, 32, 64 or 128 tokens, not %u", name, p->page);
    if (p->B == 0u || p->pages == 0u || p->table_width == 0u) return refuse(err, cap, "%s: no sequences, pages or table columns", name);
    if (p->pages > 0x7FFFFFF0u || p->B > kMostRows || static_cast<uint64_t>(p->table_width) * p->page > 0x7FFFFFFFull) return refuse(err, cap, "%s: more than 2^31 pages or tokens of a sequence, or 2^30 sequences", name);
    r.free = p->free, r.table = p->table, r.lengths = p->lengths;
    r.pages = p->pages, r.pool_pages = p->pool_pages != 0u ? p->pool_pages : 0x80000000u, r.B = p->B, r.table_width = p->table_width;
    r.page_log2 = p->page == 16u ? 4u : p->page == 32u ? 5u : p->page == 64u ? 6u : 7u;
    return 0;
}

struct Span {
    const void* at;
    uint64_t bytes;
    const char* name;
};
// the first `outputs` of them share no memory with any other
int check_apart(const Span* s, int n, int outputs, const char* name, char* err, size_t cap) {
    for (int i = 0; i < outputs; ++i) {
        for (int j = i + 1; j < n; ++j) {
            if (s[i].at != nullptr && s[j].at != nullptr && overlap(s[i].at, s[i].bytes, s[j].at, s[j].bytes)) return refuse(err, cap, "%s: %s must not share memory with %s", name, s[i].name, s[j].name);
        }
    }
    return 0;
}

// CTAs: a share of the sequences has to fit one's tables; rows of the maps are worth one per 2048, and as many as there is memory to keep busy
uint32_t grid_of(uint32_t B, uint64_t rows) {
    const uint64_t by_range = (static_cast<uint64_t>(B) + b200mx::kMostRange - 1u) / b200mx::kMostRange, by_rows = (rows + 2047u) / 2048u, most = 2u * static_cast<uint64_t>(b200mx::current_sm_count());
    const uint64_t wanted = by_rows < most ? by_rows : most;
    return static_cast<uint32_t>(wanted > by_range ? wanted : by_range);
}

}  // namespace

extern "C" {

int fmha_pages_take(const fmha_pages* pages, const int32_t* counts, int32_t* granted, void* positions, int positions_64, int64_t* slots, int32_t* starts, uint32_t S, void* stream, char* err, size_t cap) {
    PagesParams p = {};
    if (int r = params_of(pages, "take", p, err, cap)) return r;
    if (counts == nullptr || granted == nullptr) return refuse(err, cap, "take: counts and granted must be given");
    if (S == 0u) positions = nullptr, slots = nullptr;
    const bool maps = positions != nullptr || slots != nullptr;
    if (maps && static_cast<uint64_t>(p.B) * S > kMostRows) return refuse(err, cap, "take: more than 2^30 rows");
    // (a page's tokens for each free page, and what fits the pages that the sequences have)
    if (starts != nullptr && (static_cast<uint64_t>(p.pages) + p.B) << p.page_log2 > 0x7FFFFFFFull) return refuse(err, cap, "take: starts of up to 2^31 tokens and more");
    const uint64_t rows = maps ? static_cast<uint64_t>(p.B) * S : 0u;
    const Span s[] = {{granted, 4ull * p.B, "granted"}, {positions, (positions_64 ? 8u : 4u) * rows, "positions"}, {slots, 8u * rows, "slots"}, {starts, 4ull * (p.B + 1ull), "starts"}, {counts, 4ull * p.B, "counts"},
                      {p.free, 4ull * (p.pages + 4ull), "the stack"}, {p.table, 4ull * p.B * p.table_width, "the table"}, {p.lengths, 4ull * p.B, "the lengths"}};
    if (int r = check_apart(s, 8, 7, "take", err, cap)) return r;
    p.asked = counts, p.granted = granted, p.positions = positions, p.positions_64 = positions_64 != 0, p.slots = reinterpret_cast<long long*>(slots), p.starts = starts, p.S = S;
    return done(b200mx::kv4_launch(b200mx::pages_take_kernel, dim3(grid_of(p.B, rows)), b200mx::kThreads, 0, static_cast<cudaStream_t>(stream), p), err, cap);
}

int fmha_pages_cut(const fmha_pages* pages, const int32_t* keep, void* stream, char* err, size_t cap) {
    PagesParams p = {};
    if (int r = params_of(pages, "cut", p, err, cap)) return r;
    if (keep == nullptr) return refuse(err, cap, "cut: keep must be given");
    const Span s[] = {{p.free, 4ull * (p.pages + 4ull), "the stack"}, {p.table, 4ull * p.B * p.table_width, "the table"}, {p.lengths, 4ull * p.B, "the lengths"}, {keep, 4ull * p.B, "keep"}};
    if (int r = check_apart(s, 4, 3, "cut", err, cap)) return r;
    p.asked = keep;
    return done(b200mx::kv4_launch(b200mx::pages_cut_kernel, dim3(1), b200mx::kThreads, 0, static_cast<cudaStream_t>(stream), p), err, cap);
}

}  // extern "C"
