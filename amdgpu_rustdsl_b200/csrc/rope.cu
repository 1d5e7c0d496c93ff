// Rotary positions (include/fmha_rope_abi.h): pairs of a row's elements are turned by position * frequency.
//
// A CTA has one to four tokens. Its threads first work out the tokens' sines and cosines, one pair each, into shared memory: the phase is position * frequency in 64-bit integers, whole
// turns fall out at the top, and the quarter turn is taken off before the rest becomes f32. Then a thread keeps those of the pairs that it has in every head and goes over the token's
// heads, 16 bytes of both halves of a head (or of neighbours) at a time, four heads in flight.
// Bound by bytes: each row once in and once out; with one token a sequence by the launch and one trip to memory. 4 x 4096 tokens of 40 heads of 128, bf16: 57.5 to 59.7 us by box for 336 MB, 5.6 to 5.8 TB/s,
// 0.86 to 0.89 of the copy rate (16-bit elements in arrays of their own went through local memory: 108).
#include "../../include/fmha_rope_abi.h"
#include "cache_args.cuh"

#include <cuda_fp16.h>

namespace b200mx {

namespace {

constexpr uint32_t kMostTokens = 4, kMostPairs = FMHA_ROPE_MAX_HEAD_DIM / 2;

struct Rows {
    const uint8_t* in;
    uint8_t* out;
    long long in_b, in_s, in_h, out_b, out_s, out_h;   // bytes
};

struct RopeParams {
    Rows x, y;
    const unsigned long long* turns;
    const void* positions;
    long long positions_b, positions_s;
    uint32_t S, tokens, heads_x, heads, head_dim, n;
    uint32_t per_cta;      // tokens
    uint32_t rotate, items;   // pieces of a row that are turned, and with those that are only copied
    bool positions_64, backward, interleaved;
    float factor;
};

// cos and sin of 2 pi phase / 2^64, the phase without whole turns
__device__ __forceinline__ float2 turn(unsigned long long phase) {
    const unsigned long long quarter = (phase + (1ull << 61)) >> 62;             // nearest quarter turn
    const long long rest = static_cast<long long>(phase - (quarter << 62));      // within an eighth of a turn of it
    float s, c;
    sincospif(__ll2float_rn(rest) * 1.0842021724855044e-19f, &s, &c);            // 2^-63
    if (quarter & 1ull) {
        const float t = s;
        s = c, c = -t;
    }
    return quarter & 2ull ? make_float2(-c, -s) : make_float2(c, s);
}

// N elements of T in words. (Arrays of 16-bit elements would be kept in local memory.)
template <typename T, int N>
struct Piece {
    static constexpr int kBytes = sizeof(T) * N, kWords = kBytes >= 4 ? kBytes / 4 : 1;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const uint8_t* p) {   // (volatile: behind the wait for the grid before)
        if constexpr (kBytes == 16) asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
        if constexpr (kBytes == 8) asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
        if constexpr (kBytes == 4) asm volatile("ld.global.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
        if constexpr (kBytes == 2) asm volatile("{\n\t.reg .b16 h;\n\tld.global.b16 h, [%1];\n\tmov.b32 %0, {h, h};\n\t}" : "=r"(w[0]) : "l"(p));
    }
    __device__ __forceinline__ void store(uint8_t* p) const {
        if constexpr (kBytes == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        if constexpr (kBytes == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
        if constexpr (kBytes == 2) *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
    }
};
// a word's two elements, and back
template <typename T> __device__ __forceinline__ float2 unpack(uint32_t w);
template <> __device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
template <> __device__ __forceinline__ float2 unpack<__half>(uint32_t w) { return kv4::f16x2_to_f32(w); }
template <typename T> __device__ __forceinline__ uint32_t pack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float lo, float hi) { return kv4::pack_bf16x2(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack<__half>(float lo, float hi) { return kv4::pack_f16x2(lo, hi); }

__device__ __forceinline__ float2 turn_pair(float u, float v, float2 t) { return make_float2(fmaf(u, t.x, -(v * t.y)), fmaf(u, t.y, v * t.x)); }

// the pairs of a piece, or of a piece and its partner
template <typename T, int N, bool kNeighbours>
__device__ __forceinline__ void turn_piece(Piece<T, N>& a, Piece<T, N>& c, const float2* t) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < (kNeighbours ? N / 2 : N); ++i) {
            uint32_t &u = kNeighbours ? a.w[2 * i] : a.w[i], &v = kNeighbours ? a.w[2 * i + 1] : c.w[i];
            const float2 r = turn_pair(__uint_as_float(u), __uint_as_float(v), t[i]);
            u = __float_as_uint(r.x), v = __float_as_uint(r.y);
        }
    } else if constexpr (N == 1) {
        const float2 r = turn_pair(unpack<T>(a.w[0]).x, unpack<T>(c.w[0]).x, t[0]);
        a.w[0] = pack<T>(r.x, 0.0f), c.w[0] = pack<T>(r.y, 0.0f);
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float2 u = unpack<T>(a.w[i]);
            if constexpr (kNeighbours) {
                const float2 r = turn_pair(u.x, u.y, t[i]);
                a.w[i] = pack<T>(r.x, r.y);
            } else {
                const float2 v = unpack<T>(c.w[i]), r = turn_pair(u.x, v.x, t[2 * i]), q = turn_pair(u.y, v.y, t[2 * i + 1]);
                a.w[i] = pack<T>(r.x, q.x), c.w[i] = pack<T>(r.y, q.y);
            }
        }
    }
}

// heads of a thread at a time: ten loads of a piece and its partner, or eight of a piece alone
template <bool kNeighbours>
constexpr uint32_t kFlightOf = kNeighbours ? 8u : 5u;

// N elements of T at a time. N = 1 takes both layouts, a pair's elements one by one.
template <typename T, int N, bool kNeighbours, uint32_t kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == 128 ? 5 : 3) rope_kernel(const __grid_constant__ RopeParams p) {
    __shared__ float2 table[kMostTokens * kMostPairs];
    kv4::pdl_launch();
    kv4::pdl_wait();
    const uint32_t token0 = blockIdx.x * p.per_cta, tokens = min(p.per_cta, p.tokens - token0);
    // groups of `items` threads: one item each, tokens and heads dealt out to the groups
    const uint32_t groups = p.items < kThreads ? kThreads / p.items : 1u, group = p.items < kThreads ? threadIdx.x / p.items : 0u;
    const uint32_t sharing = groups / p.per_cta;   // groups that share a token, of each CTA along the grid's second dimension
    const uint32_t mine = group % p.per_cta, stride = gridDim.y * sharing;
    const bool active = group < sharing * p.per_cta && mine < tokens;
    const uint32_t token = token0 + (active ? mine : 0u), b = token / p.S, s = token - b * p.S;
    const uint32_t first = blockIdx.y * sharing + group / p.per_cta;
    constexpr uint32_t kFlight = kFlightOf<kNeighbours>;
    constexpr bool kScalar = N == 1;
    constexpr uint32_t kPairs = kScalar ? 1 : kNeighbours ? N / 2 : N;
    const uint32_t item0 = p.items < kThreads ? threadIdx.x - group * p.items : threadIdx.x, item_step = p.items < kThreads ? p.items : kThreads;
    const uint8_t *in_x = p.x.in + b * p.x.in_b + s * p.x.in_s, *in_y = p.y.in + b * p.y.in_b + s * p.y.in_s;
    uint8_t *out_x = p.x.out + b * p.x.out_b + s * p.x.out_s, *out_y = p.y.out + b * p.y.out_b + s * p.y.out_s;
    // byte offsets within a row of an item's elements, and of their partners
    const auto turned = [&](uint32_t item) { return item < p.rotate; };
    const auto offset = [&](uint32_t item) {
        return (turned(item) ? (kScalar && p.interleaved ? 2u * item : item * N) : 2u * p.n + (item - p.rotate) * N) * static_cast<uint32_t>(sizeof(T));
    };
    const uint32_t partner = (kScalar && p.interleaved ? 1u : p.n) * static_cast<uint32_t>(sizeof(T));
    Piece<T, N> a[kFlight], c[kFlight];
    const auto fetch = [&](uint32_t item, uint32_t h0) {
#pragma unroll
        for (uint32_t k = 0; k < kFlight; ++k) {
            const uint32_t h = h0 + k * stride;
            if (h >= p.heads) continue;
            const uint8_t* src = (h < p.heads_x ? in_x + h * p.x.in_h : in_y + (h - p.heads_x) * p.y.in_h) + offset(item);
            a[k].load(src);
            if (!kNeighbours && turned(item)) c[k].load(src + partner);
        }
    };
    if (active && item0 < p.items) fetch(item0, first);   // under way while the sines are worked out
    for (uint32_t k = threadIdx.x; k < tokens * p.n; k += kThreads) {
        const uint32_t at_token = token0 + k / p.n, i = k % p.n, at_b = at_token / p.S, at_s = at_token - at_b * p.S;
        const long long at = at_b * p.positions_b + at_s * p.positions_s;
        long long position;
        if (p.positions_64) asm volatile("ld.global.s64 %0, [%1];" : "=l"(position) : "l"(static_cast<const long long*>(p.positions) + at));
        else position = kv4::ld_i32(static_cast<const int32_t*>(p.positions) + at);
        unsigned long long turns;
        asm volatile("ld.global.u64 %0, [%1];" : "=l"(turns) : "l"(p.turns + i));
        float2 t = turn(static_cast<unsigned long long>(position) * turns);
        t.x *= p.factor, t.y *= p.backward ? -p.factor : p.factor;
        table[k] = t;
    }
    __syncthreads();
    if (!active) return;
    for (uint32_t item = item0; item < p.items; item += item_step) {
        float2 t[kPairs];
#pragma unroll
        for (uint32_t i = 0; i < kPairs; ++i) t[i] = turned(item) ? table[mine * p.n + item * kPairs + i] : make_float2(1.0f, 0.0f);
        for (uint32_t h0 = first; h0 < p.heads; h0 += kFlight * stride) {
            if (item != item0 || h0 != first) fetch(item, h0);
#pragma unroll
            for (uint32_t k = 0; k < kFlight; ++k) {
                const uint32_t h = h0 + k * stride;
                if (h >= p.heads) continue;
                uint8_t* dst = (h < p.heads_x ? out_x + h * p.x.out_h : out_y + (h - p.heads_x) * p.y.out_h) + offset(item);
                if (turned(item)) {
                    turn_piece<T, N, kNeighbours>(a[k], c[k], t);
                    if (!kNeighbours) c[k].store(dst + partner);
                }
                a[k].store(dst);
            }
        }
    }
}

template <typename T, int N, bool kNeighbours>
cudaError_t launch(RopeParams p, bool copies, cudaStream_t stream) {
    p.rotate = N == 1 ? p.n : kNeighbours ? 2u * p.n / N : p.n / N;
    p.items = p.rotate + (copies ? (p.head_dim - 2u * p.n) / N : 0u);
    const uint32_t sms = static_cast<uint32_t>(current_sm_count());
    // Threads a CTA and, with many tokens, tokens a CTA: what gives the most threads the most heads in their rounds of loads; then the fewest rounds, the smaller CTA. With few tokens one
    // each, their heads dealt out over up to four CTAs. (4 x 4096 tokens of 40 heads of 128, bf16 halves: 128 threads, 2 tokens 57.6 us, 256 and 4 62.2, 256 and 3 with one head less
    // in flight 65.5. 3 x 1337 of 24 heads of 96, f32 neighbours, 40 turned: 256 and 3 16.4, 128 and 1 32.5)
    uint32_t threads = 256u, best = 0u;
    p.per_cta = 1u;
    if (p.tokens >= 16u * sms) {
        for (uint32_t n = 128u; n <= 256u; n += 128u) {
            const uint32_t groups = p.items < n ? n / p.items : 1u;
            for (uint32_t t = 1; t <= kMostTokens && t <= groups; ++t) {
                const uint32_t at_once = groups / t * kFlightOf<kNeighbours>, rounds = (p.heads + at_once - 1u) / at_once;
                const uint32_t busy = static_cast<uint32_t>(static_cast<uint64_t>(t) * p.heads * (p.items < n ? p.items : n) * 1024u / (static_cast<uint64_t>(rounds) * kFlightOf<kNeighbours> * n));
                const uint32_t score = 16u * (busy < 1024u ? busy : 1024u) + 16u - (rounds < 15u ? rounds : 15u);
                if (score > best) best = score, threads = n, p.per_cta = t;
            }
        }
    }
    const uint32_t groups = p.items < threads ? threads / p.items : 1u, ctas = (p.tokens + p.per_cta - 1u) / p.per_cta, sharing = groups / p.per_cta;
    uint32_t split = 1;
    while (split < 4u && 2u * split * ctas <= 2u * sms && 2u * split * sharing <= p.heads) split *= 2u;
    if (threads == 128u) return kv4_launch(rope_kernel<T, N, kNeighbours, 128u>, dim3(ctas, split), 128u, 0, stream, p);
    return kv4_launch(rope_kernel<T, N, kNeighbours, 256u>, dim3(ctas, split), 256u, 0, stream, p);
}

template <typename T, int N>
cudaError_t launch_layout(const RopeParams& p, bool copies, cudaStream_t stream) {
    if constexpr (N == 1) return launch<T, 1, false>(p, copies, stream);
    else return p.interleaved ? launch<T, N, true>(p, copies, stream) : launch<T, N, false>(p, copies, stream);
}
// `unit`: the most elements that all rows and parts of rows are multiples of
template <typename T>
cudaError_t launch_type(const RopeParams& p, uint32_t unit, bool copies, cudaStream_t stream) {
    if constexpr (sizeof(T) == 2) {
        if (unit >= 8u) return launch_layout<T, 8>(p, copies, stream);
    }
    if (unit >= 4u) return launch_layout<T, 4>(p, copies, stream);
    if (unit >= 2u) return launch_layout<T, 2>(p, copies, stream);
    return launch_layout<T, 1>(p, copies, stream);
}

}  // namespace
}  // namespace b200mx

namespace {

using b200mx::RopeParams;
using b200mx::Rows;

struct Extent {
    uint64_t begin, end;   // bytes
};
Extent extent_of(const fmha_rope_rows& r, const fmha_rope_args& a, uint32_t heads, uint64_t size) {
    const uint64_t begin = reinterpret_cast<uintptr_t>(r.data);
    return {begin, begin + size * ((a.B - 1u) * static_cast<uint64_t>(r.stride_b) + (a.S - 1u) * static_cast<uint64_t>(r.stride_s) + (heads - 1u) * static_cast<uint64_t>(r.stride_h) + a.head_dim)};
}

// Whether two rows of places have an element in common: count * stride, summed over the dimensions, comes within a row's length of `distance` for some counts of their ranges, in elements. From the longest stride
// down, only counts that the shorter ones can make up for are looked at: one or two a dimension in layouts that are nested as usual. Layouts that take more steps than kMostLooks count as overlapping.
struct Dimension {
    int64_t stride, least, most;   // counts
};
constexpr uint32_t kMostLooks = 1u << 16;
struct Places {
    int64_t row;    // elements of a row - 1
    bool itself;    // the places of one tensor, against themselves: counts of 0 throughout are no meeting
    int n;
    uint32_t looks;
    Dimension d[6];
    void add(int64_t stride, int64_t least, int64_t most) {
        if (least == most || (stride == 0 && !itself)) return;
        for (int i = 0; i < n && !itself; ++i) {
            if (d[i].stride != stride) continue;
            d[i].least += least, d[i].most += most;
            return;
        }
        int at = n++;
        for (; at > 0 && d[at - 1].stride < stride; --at) d[at] = d[at - 1];
        d[at] = {stride, least, most};
    }
    bool meet(int64_t distance, int from = 0, bool moved = false) {
        if (from == n) return (moved || !itself) && distance <= row && -distance <= row;
        if (++looks > kMostLooks) return true;
        int64_t low = -row, high = row;   // what the dimensions behind reach
        for (int i = from + 1; i < n; ++i) low += d[i].stride * d[i].least, high += d[i].stride * d[i].most;
        const Dimension& x = d[from];
        int64_t begin = x.least, end = x.most;
        if (x.stride != 0) {
            const auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0 ? 1 : 0); };
            const int64_t first = -floor_div(high - distance, x.stride), last = floor_div(distance - low, x.stride);
            begin = begin > first ? begin : first, end = end < last ? end : last;
        }
        for (int64_t k = begin; k <= end; ++k) {
            if (meet(distance - k * x.stride, from + 1, moved || k != 0)) return true;
        }
        return false;
    }
};
// whether each dimension's stride, from the shortest on, is as long as what lies within it: the usual layouts, known without the search (0.2 us of a call's host time)
bool nested(Dimension (&d)[3], int n, uint64_t inner) {
    for (int i = 0; i < n; ++i) {
        for (int k = i + 1; k < n; ++k) {
            if (d[k].stride < d[i].stride) {
                const Dimension t = d[i];
                d[i] = d[k], d[k] = t;
            }
        }
        if (d[i].most == 0) continue;
        if (static_cast<uint64_t>(d[i].stride) < inner) return false;
        inner += static_cast<uint64_t>(d[i].stride) * static_cast<uint64_t>(d[i].most);
    }
    return true;
}
// whether no element stands twice
bool distinct(const fmha_rope_rows& r, const fmha_rope_args& a, uint32_t heads) {
    Dimension d[3] = {{r.stride_b, 0, a.B - 1ll}, {r.stride_s, 0, a.S - 1ll}, {r.stride_h, 0, heads - 1ll}};
    if (nested(d, 3, a.head_dim)) return true;
    Places x = {};
    x.row = a.head_dim - 1, x.itself = true;
    for (const Dimension& y : d) x.add(y.stride, -y.most, y.most);
    return !x.meet(0);
}
// whether two tensors have no element in common
bool apart(const fmha_rope_rows& r, uint32_t r_heads, const fmha_rope_rows& q, uint32_t q_heads, const fmha_rope_args& a, uint64_t size) {
    const Extent x = extent_of(r, a, r_heads, size), y = extent_of(q, a, q_heads, size);
    if (x.end <= y.begin || y.end <= x.begin) return true;
    const int64_t distance = static_cast<int64_t>(y.begin - x.begin) / static_cast<int64_t>(size);
    if (r.stride_b == q.stride_b && r.stride_s == q.stride_s) {   // a token's heads of both as one row
        const uint64_t r_row = (r_heads - 1ull) * static_cast<uint64_t>(r.stride_h) + a.head_dim, q_row = (q_heads - 1ull) * static_cast<uint64_t>(q.stride_h) + a.head_dim;
        const uint64_t ahead = static_cast<uint64_t>(distance < 0 ? -distance : distance);
        Dimension d[3] = {{r.stride_b, 0, a.B - 1ll}, {r.stride_s, 0, a.S - 1ll}, {}};
        if (ahead >= (distance < 0 ? q_row : r_row) && nested(d, 2, ahead + (distance < 0 ? r_row : q_row))) return true;
    }
    Places z = {};
    z.row = a.head_dim - 1;
    z.add(r.stride_b, 0, a.B - 1ll), z.add(r.stride_s, 0, a.S - 1ll), z.add(r.stride_h, 0, r_heads - 1ll);
    z.add(q.stride_b, 1ll - a.B, 0), z.add(q.stride_s, 1ll - a.S, 0), z.add(q.stride_h, 1ll - q_heads, 0);
    return !z.meet(distance);
}

int check_rows(const fmha_rope_rows& r, const fmha_rope_args& a, uint32_t heads, uint64_t size, const char* name, char* err, size_t cap) {
    if (r.data == nullptr) return refuse(err, cap, "rope: %s must be given", name);
    if (reinterpret_cast<uintptr_t>(r.data) % size != 0) return refuse(err, cap, "rope: %s must be aligned as its elements are", name);
    if (r.stride_b < 0 || r.stride_s < 0 || r.stride_h < 0) return refuse(err, cap, "rope: %s has negative strides", name);
    const int64_t most = 1ll << 56;
    const auto fits = [&](int64_t stride, uint64_t n) { return n <= 1u || static_cast<uint64_t>(stride) <= static_cast<uint64_t>(most) / n; };
    if (!fits(r.stride_b, a.B) || !fits(r.stride_s, a.S) || !fits(r.stride_h, heads)) return refuse(err, cap, "rope: %s is larger than any memory", name);
    return 0;
}

// strides that dimensions of one element have are of no matter
void clear_strides(fmha_rope_rows& r, const fmha_rope_args& a, uint32_t heads) {
    if (a.B == 1u) r.stride_b = 0;
    if (a.S == 1u) r.stride_s = 0;
    if (heads <= 1u) r.stride_h = 0;
}

}  // namespace

extern "C" int fmha_rope_rotate(const fmha_rope_args* args, void* stream, char* err, size_t cap) {
    if (args == nullptr) return refuse(err, cap, "rope: no arguments");
    fmha_rope_args a = *args;
    if (a.type > FMHA_ROPE_F32) return refuse(err, cap, "rope: type must be bf16, f16 or f32");
    if (a.head_dim == 0u || a.head_dim > FMHA_ROPE_MAX_HEAD_DIM || a.rotary < 2u || a.rotary % 2u != 0u || a.rotary > a.head_dim)
        return refuse(err, cap, "rope: heads have up to %u elements, of which an even number is turned (%u of %u)", FMHA_ROPE_MAX_HEAD_DIM, a.rotary, a.head_dim);
    if (!(a.factor > 0.0f) || a.factor > 3.0e38f) return refuse(err, cap, "rope: factor must be a positive number");
    if (a.heads_x == 0u) return refuse(err, cap, "rope: x has no heads");
    if (a.turns == nullptr || (reinterpret_cast<uintptr_t>(a.turns) & 7u) != 0) return refuse(err, cap, "rope: turns must be given and aligned");
    if (a.B == 0u || a.S == 0u) return 0;
    const uint64_t size = a.type == FMHA_ROPE_F32 ? 4u : 2u;
    if (a.positions == nullptr || reinterpret_cast<uintptr_t>(a.positions) % (a.positions_64 ? 8u : 4u) != 0) return refuse(err, cap, "rope: positions must be given and aligned");
    if (static_cast<uint64_t>(a.B) * a.S > kMostRows || static_cast<uint64_t>(a.heads_x) + a.heads_y > kMostRows || static_cast<uint64_t>(a.B) * a.S * (static_cast<uint64_t>(a.heads_x) + a.heads_y) > (1ull << 40))
        return refuse(err, cap, "rope: more than 2^30 tokens, or 2^40 rows");
    clear_strides(a.x, a, a.heads_x), clear_strides(a.x_out, a, a.heads_x), clear_strides(a.y, a, a.heads_y), clear_strides(a.y_out, a, a.heads_y);
    if (int r = check_rows(a.x, a, a.heads_x, size, "x", err, cap)) return r;
    if (int r = check_rows(a.x_out, a, a.heads_x, size, "x_out", err, cap)) return r;
    const auto same = [](const fmha_rope_rows& r, const fmha_rope_rows& q) { return r.data == q.data && r.stride_b == q.stride_b && r.stride_s == q.stride_s && r.stride_h == q.stride_h; };
    if (!distinct(a.x_out, a, a.heads_x)) return refuse(err, cap, "rope: elements of x_out share memory");
    if (!same(a.x, a.x_out) && !apart(a.x, a.heads_x, a.x_out, a.heads_x, a, size)) return refuse(err, cap, "rope: x_out must be x or share no memory with it");
    bool copies = !same(a.x, a.x_out);
    if (a.heads_y != 0u) {
        if (int r = check_rows(a.y, a, a.heads_y, size, "y", err, cap)) return r;
        if (int r = check_rows(a.y_out, a, a.heads_y, size, "y_out", err, cap)) return r;
        if (!distinct(a.y_out, a, a.heads_y)) return refuse(err, cap, "rope: elements of y_out share memory");
        if (!same(a.y, a.y_out) && !apart(a.y, a.heads_y, a.y_out, a.heads_y, a, size)) return refuse(err, cap, "rope: y_out must be y or share no memory with it");
        if (!apart(a.x_out, a.heads_x, a.y_out, a.heads_y, a, size) || !apart(a.x_out, a.heads_x, a.y, a.heads_y, a, size) || !apart(a.x, a.heads_x, a.y_out, a.heads_y, a, size))
            return refuse(err, cap, "rope: an output must not share memory with the other input or output");
        copies |= !same(a.y, a.y_out);
    }
    RopeParams p = {};
    const auto rows = [&](const fmha_rope_rows& in, const fmha_rope_rows& out) {
        const long long z = static_cast<long long>(size);
        return Rows{static_cast<const uint8_t*>(in.data), static_cast<uint8_t*>(out.data), z * in.stride_b, z * in.stride_s, z * in.stride_h, z * out.stride_b, z * out.stride_s, z * out.stride_h};
    };
    p.x = rows(a.x, a.x_out);
    p.y = a.heads_y != 0u ? rows(a.y, a.y_out) : p.x;
    p.turns = reinterpret_cast<const unsigned long long*>(a.turns);
    p.positions = a.positions, p.positions_b = a.positions_stride_b, p.positions_s = a.positions_stride_s, p.positions_64 = a.positions_64 != 0u;
    p.S = a.S, p.tokens = a.B * a.S, p.heads_x = a.heads_x, p.heads = a.heads_x + a.heads_y, p.head_dim = a.head_dim, p.n = a.rotary / 2u;
    p.backward = a.backward != 0u, p.interleaved = a.interleaved != 0u, p.factor = a.factor;
    // the widest access that everything is a multiple of
    uint32_t unit = 16u / static_cast<uint32_t>(size);
    const auto limit = [&](uint64_t bytes) {
        while (unit > 1u && bytes % (unit * size) != 0u) unit /= 2u;
    };
    for (const fmha_rope_rows* r : {&a.x, &a.x_out, &a.y, &a.y_out}) {
        if (r == &a.y && a.heads_y == 0u) break;
        limit(reinterpret_cast<uintptr_t>(r->data)), limit(size * r->stride_b), limit(size * r->stride_s), limit(size * r->stride_h);
    }
    limit(size * (p.interleaved ? 2u * p.n : p.n));
    if (copies) limit(size * (p.head_dim - 2u * p.n));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return done(a.type == FMHA_ROPE_BF16 ? b200mx::launch_type<__nv_bfloat16>(p, unit, copies, st) : a.type == FMHA_ROPE_F16 ? b200mx::launch_type<__half>(p, unit, copies, st)
                                                                                                                      : b200mx::launch_type<float>(p, unit, copies, st),
                err, cap);
}
