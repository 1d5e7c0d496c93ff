// The 8-bit key/value cache's format and the pieces its kernels share (include/fmha_kv8_abi.h has the layout). Views, schedule and partials are the 4-bit cache's.
#pragma once
#include "../../include/fmha_kv8_abi.h"
#include "kv4.cuh"

namespace b200mx {

// (the fields that make the weights of the 4-bit cache's tokens stay empty)
using Kv8AttendParams = Kv4AttendParams;

cudaError_t launch_kv8_append(const Kv4View& c, const Kv4Rows& k, const Kv4Rows& v, uint32_t S, const int32_t* counts, cudaStream_t stream);
cudaError_t launch_kv8_read(const Kv4View& c, const Kv4Rows& k, const Kv4Rows& v, uint32_t S, bool last, const int32_t* counts, cudaStream_t stream);
uint64_t kv8_attend_workspace(const Kv4View& c, uint32_t S, uint32_t H);
cudaError_t launch_kv8_attend(const Kv8AttendParams& p, cudaStream_t stream);
// kv8_prefill.cu: one CTA per SM, items of kv8_prefill_rows() query rows, partials in p.ws as the decode kernels leave them
uint32_t kv8_prefill_grid();
uint32_t kv8_prefill_rows();
cudaError_t launch_kv8_prefill(const Kv8AttendParams& p, uint32_t row_tiles, cudaStream_t stream);

#ifdef __CUDACC__
namespace kv8 {

using namespace kv4;

constexpr uint32_t kBlockTokens = FMHA_KV8_BLOCK_TOKENS, kBlockBytes = FMHA_KV8_BLOCK_BYTES;
constexpr uint32_t kVCodes = 2048, kMeta = 4096, kVScale = 4, kMasks = 8;   // within a block; scales and masks behind kMeta

// the block that holds token t, on the page that page_of() gave
__device__ __forceinline__ uint8_t* block_of(const Kv4View& c, long long page, uint32_t head, uint32_t t) {
    const uint32_t in = (t & ((1u << c.page_log2) - 1u)) / kBlockTokens, blocks = 1u << (c.page_log2 - 4u);
    return c.pool + static_cast<uint64_t>(page) * c.page_bytes + (static_cast<uint64_t>(head) * blocks + in) * kBlockBytes;
}
// 16-byte pieces change places within a row so that the eight lanes of a shared-memory access meet eight groups of banks
__device__ __forceinline__ uint32_t k_swap(uint32_t t) { return t & 7u; }
__device__ __forceinline__ uint32_t v_swap(uint32_t pair) { return (pair & 1u) | ((pair & 2u) << 1); }

__device__ __forceinline__ uint2 ld_v2(const void* p) {
    uint2 v;
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
// two e4m3 codes of a word, the lower or the upper half, as f16
__device__ __forceinline__ uint32_t e4m3x2_lo(uint32_t w) {
    uint32_t r;
    asm("{.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;}" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2_hi(uint32_t w) {
    uint32_t r;
    asm("{.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;}" : "=r"(r) : "r"(w));
    return r;
}
// four f32 to codes in the bytes of a word
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint32_t r;
    asm("{.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};}" : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}
// two pairs of f16 to codes
__device__ __forceinline__ uint32_t e4m3x4_of_f16(uint32_t lo, uint32_t hi) {
    uint32_t r;
    asm("{.reg .b16 a, b;\n\tcvt.rn.satfinite.e4m3x2.f16x2 a, %1;\n\tcvt.rn.satfinite.e4m3x2.f16x2 b, %2;\n\tmov.b32 %0, {a, b};}" : "=r"(r) : "r"(lo), "r"(hi));
    return r;
}
// A scale's exponent, and 2 to minus that, from its bits. (Scales are powers of two from 2^-90 to 2^119: sums of weights up to 2^14 times 2^90 stay within f32.)
__device__ __forceinline__ int exponent_of(uint32_t scale) { return min(max(static_cast<int>(scale >> 23) - 127, -90), 119); }
__device__ __forceinline__ float power_of(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

}  // namespace kv8
#endif

}  // namespace b200mx
