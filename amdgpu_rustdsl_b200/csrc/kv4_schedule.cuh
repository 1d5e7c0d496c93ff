// How the attention kernels of the 4-bit cache share their work, worked out on the device from the lengths.
//
// An entry is a sequence and one of its row tiles (`rows` query rows of a KV head); an item is an entry and a KV head, heads fastest. An item has as many steps as there
// are tiles of 128 tokens that its rows see. All steps of all items, in order, are dealt out in equal runs to the CTAs.
#pragma once
#include "kv4.cuh"

namespace b200mx {
namespace kv4 {

constexpr uint32_t kStepTokens = 128;

// (steps of kTokens: what the text above says of 128 tokens holds for them. kExtra: what it costs a CTA to begin an item, in steps: an item is dealt out as that many more, which lie in front
// of its steps and are not carried out. A CTA's run may then hold nothing else of an item)
template <uint32_t kTokens, uint32_t kExtra = 0>
struct DealOf {
    uint32_t rows, row_tiles;   // of an item, of a sequence
};
using Deal = DealOf<kStepTokens>;

template <uint32_t kTokens, uint32_t kExtra>
__device__ __forceinline__ uint32_t steps_of(const Kv4AttendParams& p, const DealOf<kTokens, kExtra>& d, uint32_t entry) {
    const uint32_t b = entry / d.row_tiles, row0 = (entry - b * d.row_tiles) * d.rows, length = length_of(p.c, b), n = count_of(p.counts, b, p.S, length);
    if (row0 >= n * p.group) return 0u;
    const uint32_t last = (min(row0 + d.rows, n * p.group) - 1u) / p.group;
    return ((p.causal ? length - n + last + 1u : length) + kTokens - 1u) / kTokens + kExtra;
}

struct Sums {
    uint32_t below, all;
};
// Steps of the entries below `upto`, and of all, times the heads (the host has checked that they stay below 2^32). All threads of the CTA; `part` has an element per warp.
template <uint32_t kTokens, uint32_t kExtra>
__device__ __forceinline__ Sums sum_steps(const Kv4AttendParams& p, const DealOf<kTokens, kExtra>& d, uint32_t upto, Sums* part) {
    uint32_t below = 0, all = 0;
    for (uint32_t e = threadIdx.x; e < p.c.B * d.row_tiles; e += blockDim.x) {
        const uint32_t t = steps_of(p, d, e);
        all += t;
        if (e < upto) below += t;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        below += __shfl_xor_sync(0xFFFFFFFFu, below, o);
        all += __shfl_xor_sync(0xFFFFFFFFu, all, o);
    }
    if ((threadIdx.x & 31u) == 0u) part[threadIdx.x >> 5] = {below, all};
    __syncthreads();
    below = all = 0;
    for (unsigned w = 0; w < blockDim.x / 32u; ++w) below += part[w].below, all += part[w].all;
    __syncthreads();
    return {below * p.c.HK, all * p.c.HK};
}

// CTA w of n has the steps [run_begin(w), run_begin(w + 1)) of `all`; worker_at is the one that has a step
__device__ __forceinline__ uint32_t workers(uint32_t all, uint32_t grid) { return min(all, grid); }
__device__ __forceinline__ uint32_t run_begin(uint32_t all, uint32_t n, uint32_t w) { return static_cast<uint32_t>(1ull * all * w / n); }
__device__ __forceinline__ uint32_t worker_at(uint32_t all, uint32_t n, uint32_t step) { return static_cast<uint32_t>(((step + 1ull) * n - 1ull) / all); }

// The entry that step `pos` belongs to and the step's number within it, for all lanes of a warp
struct Place {
    uint32_t entry;
    uint32_t in;   // step within the entry's items
};
template <uint32_t kTokens, uint32_t kExtra>
__device__ __forceinline__ Place find_step(const Kv4AttendParams& p, const DealOf<kTokens, kExtra>& d, uint32_t pos) {
    const unsigned lane = threadIdx.x & 31u;
    const uint32_t entries = p.c.B * d.row_tiles;
    uint32_t before = 0;
    for (uint32_t e0 = 0; e0 < entries; e0 += 32u) {
        const uint32_t t = e0 + lane < entries ? steps_of(p, d, e0 + lane) * p.c.HK : 0u;
        uint32_t s = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t a = __shfl_up_sync(0xFFFFFFFFu, s, o);
            if (lane >= static_cast<unsigned>(o)) s += a;
        }
        const unsigned hit = __ballot_sync(0xFFFFFFFFu, before + s > pos);
        if (hit != 0u) {
            const int at = __ffs(hit) - 1;
            return {e0 + static_cast<uint32_t>(at), pos - (before + __shfl_sync(0xFFFFFFFFu, s - t, at))};
        }
        before += __shfl_sync(0xFFFFFFFFu, s, 31);
    }
    return {entries, 0u};
}

// A run of steps of one item
struct Segment {
    uint32_t b, head, row0;         // the item
    uint32_t first, steps, of;      // steps first .. first + steps - 1 of `of`
    uint32_t before;                // of what the item is dealt out as, the part in front of the run
};
// The segment at the head of a CTA's run of `left` steps; moves on behind it
template <uint32_t kTokens, uint32_t kExtra>
__device__ __forceinline__ Segment next_segment(const Kv4AttendParams& p, const DealOf<kTokens, kExtra>& d, Place& at, uint32_t& left) {
    uint32_t of = steps_of(p, d, at.entry);
    while (at.in >= of * p.c.HK) {   // also where an entry has none
        at.in -= of * p.c.HK;
        of = steps_of(p, d, ++at.entry);
    }
    Segment s;
    s.b = at.entry / d.row_tiles, s.row0 = (at.entry - s.b * d.row_tiles) * d.rows;
    s.head = at.in / of, s.before = at.in - s.head * of, s.of = of - kExtra;
    const uint32_t dealt = min(of - s.before, left);
    s.first = max(s.before, kExtra) - kExtra, s.steps = max(s.before + dealt, kExtra) - kExtra - s.first;
    at.in += dealt;
    left -= dealt;
    return s;
}

// The workspace of a launch of `grid` CTAs: entries that say which CTAs worked on an item, one per item, or where there are more items than a quarter of the CTAs one per CTA for the item that it
// began and others went on with; behind room for `grid` of them the CTAs' partials: two slots (0: an item that an earlier CTA began, 1: one that a later CTA goes on with), each
// `rows` x 128 f32 of O in front of `rows` pairs of M (base 2) and l
struct Begun {
    uint32_t item, first, last, unused;   // the first and the last CTA that have a part; the same: there is nothing to put together
};
// (4 items of 74 parts each: 28 us with the item's entries, 36 with an entry and a row of idle CTAs for each of the 296 CTAs; 192 items of up to 7 parts among 592 CTAs: 72.6 and 69.7)
__host__ __device__ __forceinline__ bool begun_by_item(const Kv4View& c, uint32_t row_tiles, uint32_t grid) { return 4ull * c.B * c.HK * row_tiles <= grid; }
__host__ __device__ __forceinline__ uint32_t begun_entries(const Kv4View& c, uint32_t row_tiles, uint32_t grid) { return begun_by_item(c, row_tiles, grid) ? c.B * c.HK * row_tiles : grid; }
// Whether an item's parts are few, so that a warp goes over them one behind the other. (6 parts alike, 9 parts of 256 rows 60 us so and 54 with warps that share them)
__host__ __device__ __forceinline__ bool few_parts(const Kv4View& c, uint32_t row_tiles, uint32_t grid) { return grid / begun_entries(c, row_tiles, grid) <= 6u; }
__device__ __forceinline__ Begun* begun_at(float* ws, uint32_t x) { return reinterpret_cast<Begun*>(ws) + x; }
// by one thread of a CTA: at its start, and for each segment
template <uint32_t kTokens, uint32_t kExtra>
__device__ __forceinline__ void begin_nothing(const Kv4AttendParams& p, const DealOf<kTokens, kExtra>& d) {
    if (!begun_by_item(p.c, d.row_tiles, gridDim.x)) *begun_at(p.ws, blockIdx.x) = {0u, blockIdx.x, blockIdx.x, 0u};
}
template <uint32_t kTokens, uint32_t kExtra>
__device__ __forceinline__ void begin_item(const Kv4AttendParams& p, const DealOf<kTokens, kExtra>& d, const Segment& s, uint32_t pos, uint32_t all, uint32_t n_work) {
    if (s.first != 0u || s.steps == 0u) return;
    const uint32_t item = (s.b * d.row_tiles + s.row0 / d.rows) * p.c.HK + s.head, last = s.steps == s.of ? blockIdx.x : worker_at(all, n_work, pos - s.before + s.of + kExtra - 1u);
    const bool by_item = begun_by_item(p.c, d.row_tiles, gridDim.x);
    if (by_item || last != blockIdx.x) *begun_at(p.ws, by_item ? item : blockIdx.x) = {item, blockIdx.x, last, 0u};
}
__device__ __forceinline__ float* slot_of(float* ws, uint32_t grid, uint32_t w, uint32_t slot, uint32_t rows) { return ws + 4u * grid + (static_cast<size_t>(w) * 2u + slot) * rows * 130u; }
constexpr float kLowest = -1e30f;   // M of a row that has seen nothing

// Sequences' row tiles that no CTA has steps of: their rows see nothing. `threads` threads of every CTA of the grid; with few entries several CTAs share one's rows (4 tiles of 256 rows, 8 heads, by
// a CTA each: 15 us, longer than those CTAs' own work). `entries`: whether the workspace has entries
template <uint32_t kTokens, uint32_t kExtra>
__device__ __forceinline__ void clear_empty_entries(const Kv4AttendParams& p, const DealOf<kTokens, kExtra>& d, bool entries, uint32_t thread, uint32_t threads) {
    const uint32_t n = p.c.B * d.row_tiles, share = n < gridDim.x ? gridDim.x / n : 1u, part = blockIdx.x % share;
    for (uint32_t e = blockIdx.x / share; e < n; e += gridDim.x / share) {
        if (steps_of(p, d, e) != 0u) continue;
        if (part == 0u && entries && begun_by_item(p.c, d.row_tiles, gridDim.x)) {
            for (uint32_t h = thread; h < p.c.HK; h += threads) *begun_at(p.ws, e * p.c.HK + h) = {0u, 0u, 0u, 0u};
        }
        const uint32_t b = e / d.row_tiles, row0 = (e - b * d.row_tiles) * d.rows, rows = min(d.rows, p.S * p.group - row0), all = rows * p.c.HK;
        const uint32_t begin = static_cast<uint32_t>(static_cast<unsigned long long>(all) * part / share), end = static_cast<uint32_t>(static_cast<unsigned long long>(all) * (part + 1u) / share);
        for (uint32_t y = begin + (thread >> 4); y < end; y += threads >> 4) {   // 16 threads a row (rows and heads together are 2^30 at most)
            const uint32_t piece = thread & 15u, row = row0 + y % rows, head = y / rows, i = row / p.group, h = head * p.group + row % p.group;
            *reinterpret_cast<uint4*>(p.out + ((static_cast<size_t>(b) * p.S + i) * p.H + h) * 128u + 8u * piece) = make_uint4(0u, 0u, 0u, 0u);
            if (piece == 0u && p.lse != nullptr) p.lse[(static_cast<size_t>(b) * p.H + h) * p.S + i] = -INFINITY;
        }
    }
}
template <uint32_t kTokens, uint32_t kExtra>
__device__ __forceinline__ void clear_empty_entries(const Kv4AttendParams& p, const DealOf<kTokens, kExtra>& d, bool entries = true) {
    clear_empty_entries(p, d, entries, threadIdx.x, blockDim.x);
}

}  // namespace kv4

inline uint64_t kv4_partial_bytes(uint32_t grid, uint32_t rows) { return static_cast<uint64_t>(grid) * (16u + 2u * rows * 130u * 4u); }

}  // namespace b200mx
