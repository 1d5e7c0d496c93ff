// How the attention kernels of the 4-bit cache share their work, worked out on the device from the lengths.
//
// An entry is a sequence and one of its row tiles (`rows` query rows of a KV head); an item is an entry and a KV head, heads fastest. An item has as many steps as there
// are tiles of 128 tokens that its rows see. All steps of all items, in order, are dealt out in equal runs to the CTAs.
#pragma once
#include "kv4.cuh"

namespace b200mx {
namespace kv4 {

constexpr uint32_t kStepTokens = 128;

struct Deal {
    uint32_t rows, row_tiles;   // of an item, of a sequence
};

__device__ __forceinline__ uint32_t steps_of(const Kv4AttendParams& p, const Deal& d, uint32_t entry) {
    const uint32_t b = entry / d.row_tiles, row0 = (entry - b * d.row_tiles) * d.rows, length = length_of(p.c, b), n = count_of(p.counts, b, p.S, length);
    if (row0 >= n * p.group) return 0u;
    const uint32_t last = (min(row0 + d.rows, n * p.group) - 1u) / p.group;
    return ((p.causal ? length - n + last + 1u : length) + kStepTokens - 1u) / kStepTokens;
}

struct Sums {
    uint32_t below, all;
};
// Steps of the entries below `upto`, and of all, times the heads (the host has checked that they stay below 2^32). All threads of the CTA; `part` has an element per warp.
__device__ __forceinline__ Sums sum_steps(const Kv4AttendParams& p, const Deal& d, uint32_t upto, Sums* part) {
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
__device__ __forceinline__ Place find_step(const Kv4AttendParams& p, const Deal& d, uint32_t pos) {
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
};
// The segment at the head of a CTA's run of `left` steps; moves on behind it
__device__ __forceinline__ Segment next_segment(const Kv4AttendParams& p, const Deal& d, Place& at, uint32_t& left) {
    uint32_t of = steps_of(p, d, at.entry);
    while (at.in >= of * p.c.HK) {   // also where an entry has none
        at.in -= of * p.c.HK;
        of = steps_of(p, d, ++at.entry);
    }
    Segment s;
    s.b = at.entry / d.row_tiles, s.row0 = (at.entry - s.b * d.row_tiles) * d.rows;
    s.head = at.in / of, s.first = at.in - s.head * of, s.of = of;
    s.steps = min(of - s.first, left);
    at.in += s.steps;
    left -= s.steps;
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
__device__ __forceinline__ Begun* begun_at(float* ws, uint32_t x) { return reinterpret_cast<Begun*>(ws) + x; }
// by one thread of a CTA: at its start, and for each segment
__device__ __forceinline__ void begin_nothing(const Kv4AttendParams& p, const Deal& d) {
    if (!begun_by_item(p.c, d.row_tiles, gridDim.x)) *begun_at(p.ws, blockIdx.x) = {0u, blockIdx.x, blockIdx.x, 0u};
}
__device__ __forceinline__ void begin_item(const Kv4AttendParams& p, const Deal& d, const Segment& s, uint32_t pos, uint32_t all, uint32_t n_work) {
    if (s.first != 0u) return;
    const uint32_t item = (s.b * d.row_tiles + s.row0 / d.rows) * p.c.HK + s.head, last = s.steps == s.of ? blockIdx.x : worker_at(all, n_work, pos + s.of - 1u);
    const bool by_item = begun_by_item(p.c, d.row_tiles, gridDim.x);
    if (by_item || last != blockIdx.x) *begun_at(p.ws, by_item ? item : blockIdx.x) = {item, blockIdx.x, last, 0u};
}
__device__ __forceinline__ float* slot_of(float* ws, uint32_t grid, uint32_t w, uint32_t slot, uint32_t rows) { return ws + 4u * grid + (static_cast<size_t>(w) * 2u + slot) * rows * 130u; }
constexpr float kLowest = -1e30f;   // M of a row that has seen nothing

// Sequences' row tiles that no CTA has steps of: their rows see nothing. All threads of the grid.
__device__ __forceinline__ void clear_empty_entries(const Kv4AttendParams& p, const Deal& d) {
    for (uint32_t e = blockIdx.x; e < p.c.B * d.row_tiles; e += gridDim.x) {
        if (steps_of(p, d, e) != 0u) continue;
        if (begun_by_item(p.c, d.row_tiles, gridDim.x)) {
            for (uint32_t h = threadIdx.x; h < p.c.HK; h += blockDim.x) *begun_at(p.ws, e * p.c.HK + h) = {0u, 0u, 0u, 0u};
        }
        const uint32_t b = e / d.row_tiles, row0 = (e - b * d.row_tiles) * d.rows, rows = min(d.rows, p.S * p.group - row0);
        for (uint32_t x = threadIdx.x; x < rows * p.c.HK * 16u; x += blockDim.x) {
            const uint32_t part = x & 15u, row = row0 + (x >> 4) % rows, head = (x >> 4) / rows, i = row / p.group, h = head * p.group + row % p.group;
            *reinterpret_cast<uint4*>(p.out + ((static_cast<size_t>(b) * p.S + i) * p.H + h) * 128u + 8u * part) = make_uint4(0u, 0u, 0u, 0u);
            if (part == 0u && p.lse != nullptr) p.lse[(static_cast<size_t>(b) * p.H + h) * p.S + i] = -INFINITY;
        }
    }
}

}  // namespace kv4

inline uint64_t kv4_partial_bytes(uint32_t grid, uint32_t rows) { return static_cast<uint64_t>(grid) * (16u + 2u * rows * 130u * 4u); }

}  // namespace b200mx
