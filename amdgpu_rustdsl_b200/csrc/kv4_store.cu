// Tokens into and out of the 4-bit cache: kv4_append rounds bf16 rows to MXFP4 and writes them to their pages, kv4_read gives the values back in bf16.
//
//   E = clamp(floor(log2 amax) - 2 + 127, 1, 252) over 32 elements,   code = e2m1_rne_sat(x * 2^(127 - E)),   value = code * 2^(E - 127)
//
// A row of one token and KV head, its K and its V, is the work of 16 lanes: a lane holds 8 consecutive elements (16 bytes of bf16), four lanes a block. Both directions
// are bound by bytes (512 of bf16 and 136 of the cache per row) as long as enough of them are on the way and few instructions go into finding them: K and V share
// what the row needs, the sequence is the grid's second dimension, and a lane works on kRows rows at once.
// 8 prompts of up to 1337 tokens: 21 us to append and read back, 3.1 TB/s over both and two launches; the instruction stream is the next limit (70 and
// 80 % of the issue slots, at 3.7 and 4.5 TB/s over 16 prompts).
#include "kv4.cuh"

namespace b200mx {

namespace {

using namespace kv4;

// Rows of a lane. With one, 8 prompts of up to 1337 tokens take 24.5 us to append and read back, with two 22.8, with four 22.8 as well (all before the arithmetic was packed); the tokens that an eviction keeps
// (16 sequences, 8 heads, 1024 each) are read fastest with two; calls of few rows do not tell.
constexpr int kRows = 2;

struct StoreParams {
    Kv4View c;
    Kv4Rows k, v;
    uint32_t S;
    int last;
    const int32_t* counts;
    uint32_t rows;       // of a sequence: S * HK, heads fastest
    uint32_t hk_log2;    // 32: HK is no power of two
};

__device__ __forceinline__ uint2 row_and_head(const StoreParams& p, uint32_t r) {   // (row of the sequence, head)
    const uint32_t i = p.hk_log2 < 32u ? r >> p.hk_log2 : r / p.c.HK;
    return make_uint2(i, r - i * p.c.HK);
}

// One row: 16 bytes of bf16 per lane to codes and scales at `record` (null: nowhere)
__device__ __forceinline__ void append_row(const uint4 raw, uint8_t* record, uint32_t page, uint32_t slot, bool is_v) {
    const unsigned part = threadIdx.x & 15u, blk = part >> 2, tig = part & 3u;
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    // the block's largest magnitude, as bf16 bits (ordered as integers; Inf and NaN come out on top)
    uint32_t amax = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu), __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
    amax = __vmaxu2(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
    amax = __vmaxu2(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
    const uint32_t field = max(amax >> 23, amax >> 7 & 255u);
    const bool broken = field == 255u;
    const uint32_t e = broken ? 255u : (field < 3u ? 1u : field - 2u);
    // x * 2^(127 - E) in bf16, exact up to what rounds to a code of 0 anyway; 127 - E lies in [-125, 126]
    const uint32_t up = ((254u - e) << 7) * 0x10001u;
    uint32_t code[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = mul_bf16x2(w[i], up);
        code[i] = f32x2_to_e2m1x2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
    }
    // elements 32 blk + 8 tig ..: bytes 0, 1 belong to group g = 2 tig, bytes 2, 3 to group 2 tig + 1; a group's bytes 2 blk, 2 blk + 1. Lanes of an even and an
    // odd block swap halves, so that each holds a word of one group: lane (blk, tig) word 4 tig + 2 (blk & 1) + (blk >> 1)
    uint32_t word = __byte_perm(__byte_perm(code[0], code[1], 0x0040), __byte_perm(code[2], code[3], 0x0040), 0x5410);
    if (broken) word = 0u;
    word = __byte_perm(word, __shfl_xor_sync(0xFFFFFFFFu, word, 4), blk & 1u ? 0x3276 : 0x5410);
    if (record != nullptr) {
        uint8_t* codes = record + (is_v ? 64u * page : 0u) + 64u * slot;
        *reinterpret_cast<uint32_t*>(codes + 4u * (4u * tig + 2u * (blk & 1u) + (blk >> 1))) = word;
        if (tig == 0u) record[(is_v ? 132u : 128u) * page + 4u * slot + blk] = static_cast<uint8_t>(e);
    }
}

__global__ void __launch_bounds__(256) kv4_append_kernel(const __grid_constant__ StoreParams p) {
    pdl_launch();
    pdl_wait();
    const unsigned part = threadIdx.x & 15u;
    const uint32_t page = 1u << p.c.page_log2, first = blockIdx.x * (16u * kRows) + (threadIdx.x >> 4);
    for (uint32_t b = blockIdx.y; b < p.c.B; b += gridDim.y) {
        const uint32_t L = length_of(p.c, b), n = count_of(p.counts, b, p.S, L), rows = n * p.c.HK;
        const uint8_t *k_rows = p.k.data + b * p.k.stride_b, *v_rows = p.v.data + b * p.v.stride_b;
        uint4 raw[kRows][2];
        uint2 at[kRows];
        long long id[kRows];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const uint32_t r = first + 16u * k;
            raw[k][0] = raw[k][1] = make_uint4(0u, 0u, 0u, 0u);
            at[k] = row_and_head(p, r);
            if (r < rows) {
                raw[k][0] = ld_v4(k_rows + at[k].x * p.k.stride_s + at[k].y * p.k.stride_h + 16u * part);
                raw[k][1] = ld_v4(v_rows + at[k].x * p.v.stride_s + at[k].y * p.v.stride_h + 16u * part);
            }
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) id[k] = first + 16u * k < rows ? page_of(p.c, b, L - n + at[k].x) : -1;
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            uint8_t* record = id[k] >= 0 ? record_of(p.c, id[k], at[k].y) : nullptr;
            const uint32_t slot = (L - n + at[k].x) & (page - 1u);
            append_row(raw[k][0], record, page, slot, false);
            append_row(raw[k][1], record, page, slot, true);
        }
    }
}

// a pair of codes as f16 times the block's factor (twice in `scale`), in bf16
__device__ __forceinline__ uint32_t value_pair(uint32_t two, unsigned long long scale) {
    const float2 x = f16x2_to_f32(two);
    unsigned long long y;
    float lo, hi;
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(x.x), "f"(x.y));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(y), "l"(scale));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(y));
    return pack_bf16x2(lo, hi);
}
// 8 elements of a row
__device__ __forceinline__ uint4 values_of(uint32_t word, float scale) {
    unsigned long long both;
    asm("mov.b64 %0, {%1, %1};" : "=l"(both) : "f"(scale));
    return make_uint4(value_pair(e2m1x2_to_f16x2<0>(word), both), value_pair(e2m1x2_to_f16x2<1>(word), both), value_pair(e2m1x2_to_f16x2<2>(word), both), value_pair(e2m1x2_to_f16x2<3>(word), both));
}

__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ StoreParams p) {
    pdl_launch();
    pdl_wait();
    const unsigned part = threadIdx.x & 15u, blk = part >> 2, tig = part & 3u;
    const uint32_t page = 1u << p.c.page_log2, first = blockIdx.x * (16u * kRows) + (threadIdx.x >> 4);
    for (uint32_t b = blockIdx.y; b < p.c.B; b += gridDim.y) {
        const uint32_t L = length_of(p.c, b), n = p.last ? count_of(p.counts, b, p.S, L) : min(p.S, L), t0 = p.last ? L - n : 0u, rows = n * p.c.HK;
        uint8_t *k_rows = p.k.data + b * p.k.stride_b, *v_rows = p.v.data + b * p.v.stride_b;
        uint32_t word[kRows][2], sc[kRows][2];
        uint2 at[kRows];
        long long id[kRows];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            at[k] = row_and_head(p, first + 16u * k);
            id[k] = first + 16u * k < rows ? page_of(p.c, b, t0 + at[k].x) : -1;
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            word[k][0] = word[k][1] = sc[k][0] = sc[k][1] = 0u;
            if (id[k] >= 0) {
                const uint32_t slot = (t0 + at[k].x) & (page - 1u);
                const uint8_t *record = record_of(p.c, id[k], at[k].y), *codes = record + 64u * slot + 4u * (4u * tig + 2u * (blk & 1u) + (blk >> 1)), *scales = record + 128u * page + 4u * slot;
                word[k][0] = ld_u32(codes), word[k][1] = ld_u32(codes + 64u * page);
                sc[k][0] = ld_u32(scales), sc[k][1] = ld_u32(scales + 4u * page);
            }
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const uint32_t r = first + 16u * k;
#pragma unroll
            for (int x = 0; x < 2; ++x) word[k][x] = __byte_perm(word[k][x], __shfl_xor_sync(0xFFFFFFFFu, word[k][x], 4), blk & 1u ? 0x3276 : 0x5410);   // (as in append_row)
            if (r >= p.rows) continue;
            const bool lost = id[k] < 0 && r < rows;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                // zeros (of codes of 0) for a row that stands for no token
                const uint4 out = lost ? make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu) : values_of(word[k][x], scale_f32(sc[k][x], static_cast<int>(blk)));
                uint8_t* to = x ? v_rows + at[k].x * p.v.stride_s + at[k].y * p.v.stride_h : k_rows + at[k].x * p.k.stride_s + at[k].y * p.k.stride_h;
                *reinterpret_cast<uint4*>(to + 16u * part) = out;
            }
        }
    }
}

StoreParams params_of(const Kv4View& c, const Kv4Rows& k, const Kv4Rows& v, uint32_t S, bool last, const int32_t* counts) {
    uint32_t log2 = 0;
    while (log2 < 31u && (1u << log2) < c.HK) ++log2;
    return {c, k, v, S, last ? 1 : 0, counts, S * c.HK, (1u << log2) == c.HK ? log2 : 32u};
}
dim3 grid_of(const StoreParams& p) {
    return dim3((p.rows + 16u * kRows - 1u) / (16u * kRows), p.c.B < 65535u ? p.c.B : 65535u);
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4View& c, const Kv4Rows& k, const Kv4Rows& v, uint32_t S, const int32_t* counts, cudaStream_t stream) {
    const StoreParams p = params_of(c, k, v, S, true, counts);
    return kv4_launch(kv4_append_kernel, grid_of(p), 256u, 0, stream, p);
}
cudaError_t launch_kv4_read(const Kv4View& c, const Kv4Rows& k, const Kv4Rows& v, uint32_t S, bool last, const int32_t* counts, cudaStream_t stream) {
    const StoreParams p = params_of(c, k, v, S, last, counts);
    return kv4_launch(kv4_read_kernel, grid_of(p), 256u, 0, stream, p);
}

}  // namespace b200mx
