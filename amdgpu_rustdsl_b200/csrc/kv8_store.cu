// Tokens into and out of the 8-bit cache: kv8_append rounds bf16 rows to e4m3 with one power of two per block of 16 tokens of a head, K and V for themselves, and writes them to
// their pages; kv8_read gives the values back in bf16.
//
//   scale = 2^max(ceil(log2(amax / 448)), -90),   code = e4m3_rne_sat(x / scale),   value = code * scale;   a block that had tokens keeps a larger scale, or its codes move to the new one
//
// A warp has a block's K or its V: 16 tokens of 128 elements are 8 loads of 16 bytes a lane (half a warp a token), all in flight together, and stay in registers between the largest
// element and the rounding. Where there is one block the chain length -> page -> block -> store is what takes the time (64 x 1 tokens of 8 heads: append 3.7 us, read 2.4 of the device), where there
// are many the chain's few rounds of warps and bytes: 8 ragged prompts of up to 1337 tokens of 8 heads, append 7.6 us for 22 MB, read 8.8 for 51 MB (5.8 TB/s, 0.89 of the copy rate).
#include "kv8.cuh"

namespace b200mx {

namespace {

using namespace kv8;

struct StoreParams {
    Kv4View c;
    Kv4Rows k, v;
    uint32_t S;
    int last;
    const int32_t* counts;
};

constexpr uint32_t kThreads = 256, kWarps = kThreads / 32;

// The scale's exponent field for a largest element given as bf16 bits: the carry out of the mantissa is there if it exceeds 1.75
__device__ __forceinline__ uint32_t scale_field(uint32_t amax) {
    const int field = static_cast<int>(((amax << 16) + 0x1FFFFFu) >> 23) - 8;
    return static_cast<uint32_t>(min(max(field, 37), 246));
}

// bytes of the even and the odd token of a pair of V
__device__ __forceinline__ uint32_t pair_bytes(bool even, bool odd) { return (even ? 0x00FF00FFu : 0u) | (odd ? 0xFF00FF00u : 0u); }

// codes times a power of two (f16, twice), rounded again
__device__ __forceinline__ uint32_t shrink(uint32_t codes, uint32_t factor) { return e4m3x4_of_f16(mul_f16x2(e4m3x2_lo(codes), factor), mul_f16x2(e4m3x2_hi(codes), factor)); }

// kCtas: that an SM is to have room for. Many blocks take 4 (8 ragged prompts of up to 1337 tokens, read back after: 18.0 us in place of 19.6 with 2, whose next launch finds less room to begin in); few
// are quicker with 2 and the registers to have all loads in flight (64 x 1 tokens: 3.7 us of the device in place of 4.3)
template <int kCtas>
__global__ void __launch_bounds__(kThreads, kCtas) kv8_append_kernel(const __grid_constant__ StoreParams p) {
    pdl_launch();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, piece = lane & 15u, odd = lane >> 4;
    const uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5), part = unit / p.c.HK, head = unit - part * p.c.HK, nth = part >> 1;
    const bool is_v = part & 1u;
    for (uint32_t b = blockIdx.y; b < p.c.B; b += gridDim.y) {
        const uint32_t L = length_of(p.c, b), n = count_of(p.counts, b, p.S, L), t0 = L - n, base = (t0 / kBlockTokens + nth) * kBlockTokens;   // (the block's first token)
        if (base >= L || n == 0u) continue;
        const long long page = page_of(p.c, b, base);
        const Kv4Rows& rows = is_v ? p.v : p.k;
        const uint8_t* src = rows.data + b * rows.stride_b + head * rows.stride_h + 16u * piece;
        uint4 raw[8];
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) {
            const uint32_t t = base + 2u * i + odd;
            raw[i] = t >= t0 && t < L ? ld_v4(src + static_cast<long long>(t - t0) * rows.stride_s) : make_uint4(0u, 0u, 0u, 0u);
        }
        if (page < 0) continue;
        uint8_t* block = block_of(p.c, page, head, base);
        const uint32_t old = base < t0 ? t0 - base : 0u;   // tokens that are there already
        uint32_t had = 0, had_mask = 0;
        if (old != 0u) had = ld_u32(block + kMeta + (is_v ? kVScale : 0u)) >> 23, had_mask = (ld_u32(block + kMeta + kMasks) >> (is_v ? 16 : 0)) & ((1u << old) - 1u);
        uint32_t amax = 0, mask = had_mask;
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) {
            const uint4 x = raw[i];
            uint32_t m = __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu), __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
            m = max(m & 0xFFFFu, m >> 16);
            const uint32_t broken = __ballot_sync(0xFFFFFFFFu, m >= 0x7F80u);
            if (broken != 0u) {
                mask |= (broken & 0xFFFFu ? 1u << (2u * i) : 0u) | (broken >> 16 ? 2u << (2u * i) : 0u);
                if (odd ? broken >> 16 : broken & 0xFFFFu) raw[i] = make_uint4(0u, 0u, 0u, 0u), m = 0u;
            }
            amax = max(amax, m);
        }
        const uint32_t field = max(scale_field(__reduce_max_sync(0xFFFFFFFFu, amax)), had);
        const float inv = __uint_as_float((254u - field) << 23);
        const bool grows = old != 0u && field > had;
        const uint32_t shift = field - had, factor = !grows ? 0u : (shift < 15u ? (15u - shift) << 10 : shift < 25u ? 1u << (24u - shift) : 0u) * 0x10001u;   // 2^-shift in f16
        uint8_t* codes = block + (is_v ? kVCodes : 0u);
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
            float f[8];
#pragma unroll
            for (int x = 0; x < 4; ++x) f[2 * x] = __uint_as_float(w[x] << 16) * inv, f[2 * x + 1] = __uint_as_float(w[x] & 0xFFFF0000u) * inv;
            uint2 c = make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
            const uint32_t t = 2u * i + odd;   // of the block
            if (!is_v) {
                uint2* to = reinterpret_cast<uint2*>(codes + 128u * t + 16u * ((piece >> 1) ^ k_swap(t)) + 8u * (piece & 1u));
                if (t < old) {
                    if (!grows) continue;
                    c = make_uint2(shrink(ld_u32(to), factor), shrink(ld_u32(reinterpret_cast<uint32_t*>(to) + 1), factor));
                } else if (base + t >= L) {
                    continue;
                }
                *to = c;
            } else {
                // the lanes of a pair's even token take elements 0 to 3 of both, those of the odd one 4 to 7
                const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, odd ? c.x : c.y, 16), even_word = odd ? got : c.x, odd_word = odd ? c.y : got;
                c = make_uint2(__byte_perm(even_word, odd_word, 0x5140), __byte_perm(even_word, odd_word, 0x7362));
                const uint32_t first = 2u * i;
                if (base + first >= L) continue;
                uint2* to = reinterpret_cast<uint2*>(codes + 256u * i + 16u * (piece ^ v_swap(i)) + 8u * odd);
                if (first < old) {   // a pair with one or two older tokens
                    if (!grows && first + 1u < old) continue;
                    uint2 was = make_uint2(ld_u32(to), ld_u32(reinterpret_cast<uint32_t*>(to) + 1));
                    if (grows) was = make_uint2(shrink(was.x, factor), shrink(was.y, factor));
                    const uint32_t keep = pair_bytes(true, first + 1u < old);
                    c = make_uint2((was.x & keep) | (c.x & ~keep), (was.y & keep) | (c.y & ~keep));
                }
                *to = c;
            }
        }
        if (lane == 0u) {
            *reinterpret_cast<uint32_t*>(block + kMeta + (is_v ? kVScale : 0u)) = field << 23;
            *reinterpret_cast<uint16_t*>(block + kMeta + kMasks + (is_v ? 2u : 0u)) = static_cast<uint16_t>(mask);
        }
    }
}

// two codes as f16 times the block's scale (twice in `scale`), in bf16
__device__ __forceinline__ uint32_t value_pair(uint32_t two, unsigned long long scale) {
    const float2 x = f16x2_to_f32(two);
    unsigned long long y;
    float lo, hi;
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(x.x), "f"(x.y));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(y), "l"(scale));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(y));
    return pack_bf16x2(lo, hi);
}

// A warp has a block's K or its V as kv8_append does, of which it gives back the rows that are asked for; half a warp a row
__global__ void __launch_bounds__(kThreads, 4) kv8_read_kernel(const __grid_constant__ StoreParams p) {
    pdl_launch();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, piece = lane & 15u, odd = lane >> 4;
    const uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5), part = unit / p.c.HK, head = unit - part * p.c.HK, nth = part >> 1;
    const bool is_v = part & 1u;
    for (uint32_t b = blockIdx.y; b < p.c.B; b += gridDim.y) {
        const uint32_t L = length_of(p.c, b), n = p.last ? count_of(p.counts, b, p.S, L) : min(p.S, L), t0 = p.last ? L - n : 0u, base = (t0 / kBlockTokens + nth) * kBlockTokens;
        if (base >= t0 + p.S) continue;
        const uint32_t stop = t0 + n;   // rows from there on stand for nothing
        const long long page = base < stop ? page_of(p.c, b, base) : -1;
        uint4 codes[4];   // V: of a pair of tokens, 8 elements; K: of two tokens, 8 elements each
        uint32_t scale_bits = 0, mask = base < stop ? 0xFFFFu : 0u;   // (tokens of a page that the pool does not have are without numbers)
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) codes[i] = make_uint4(0u, 0u, 0u, 0u);
        if (page >= 0) {
            const uint8_t* block = block_of(p.c, page, head, base);
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                if (is_v) {
                    const uint32_t pair = 2u * i + odd;
                    codes[i] = ld_v4(block + kVCodes + 256u * pair + 16u * (piece ^ v_swap(pair)));
                } else {
                    const uint32_t t = 4u * i + odd;
                    const uint2 x = ld_v2(block + 128u * t + 16u * ((piece >> 1) ^ k_swap(t)) + 8u * (piece & 1u)), y = ld_v2(block + 128u * (t + 2u) + 16u * ((piece >> 1) ^ k_swap(t + 2u)) + 8u * (piece & 1u));
                    codes[i] = make_uint4(x.x, x.y, y.x, y.y);
                }
            }
            const uint4 meta = ld_v4(block + kMeta);
            scale_bits = is_v ? meta.y : meta.x, mask = is_v ? meta.z >> 16 : meta.z;
        }
        const Kv4Rows& rows = is_v ? p.v : p.k;
        uint8_t* to = rows.data + b * rows.stride_b + head * rows.stride_h + 16u * piece;
        unsigned long long scale;
        asm("mov.b64 %0, {%1, %1};" : "=l"(scale) : "r"(scale_bits));
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) {
            const uint4 c = codes[i >> 1];
            // K: tokens 2 i and 2 i + 1 in the two halves of the warp; V: those of the pair i - i % 2 and the next, one after the other
            const uint32_t t = is_v ? 4u * (i >> 1) + 2u * odd + (i & 1u) : 2u * i + odd, pick = i & 1u ? 0x7531u : 0x6420u;
            const uint32_t w0 = is_v ? __byte_perm(c.x, c.y, pick) : i & 1u ? c.z : c.x, w1 = is_v ? __byte_perm(c.z, c.w, pick) : i & 1u ? c.w : c.y;
            if (base + t < t0 || base + t >= t0 + p.S) continue;
            const bool live = base + t < stop;
            uint4 out = make_uint4(value_pair(e4m3x2_lo(w0), scale), value_pair(e4m3x2_hi(w0), scale), value_pair(e4m3x2_lo(w1), scale), value_pair(e4m3x2_hi(w1), scale));
            if (mask >> t & 1u) out = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
            if (!live) out = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(to + static_cast<long long>(base + t - t0) * rows.stride_s) = out;
        }
    }
}

uint32_t grid_y(const Kv4View& c) { return c.B < 65535u ? c.B : 65535u; }

}  // namespace

cudaError_t launch_kv8_append(const Kv4View& c, const Kv4Rows& k, const Kv4Rows& v, uint32_t S, const int32_t* counts, cudaStream_t stream) {
    const uint32_t blocks = (S + 2u * kBlockTokens - 2u) / kBlockTokens, units = blocks * c.HK * 2u;   // blocks that S tokens may fall into
    const dim3 grid((units + kWarps - 1u) / kWarps, grid_y(c));
    const StoreParams p{c, k, v, S, 1, counts};
    return static_cast<uint64_t>(grid.x) * grid.y <= 2u * current_sm_count() ? kv4_launch(kv8_append_kernel<2>, grid, kThreads, 0, stream, p) : kv4_launch(kv8_append_kernel<4>, grid, kThreads, 0, stream, p);
}
cudaError_t launch_kv8_read(const Kv4View& c, const Kv4Rows& k, const Kv4Rows& v, uint32_t S, bool last, const int32_t* counts, cudaStream_t stream) {
    const uint32_t units = (S + 2u * kBlockTokens - 2u) / kBlockTokens * c.HK * 2u;
    return kv4_launch(kv8_read_kernel, dim3((units + kWarps - 1u) / kWarps, grid_y(c)), kThreads, 0, stream, StoreParams{c, k, v, S, last ? 1 : 0, counts});
}

}  // namespace b200mx
