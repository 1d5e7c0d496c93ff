// The 4-bit key/value cache's format and the pieces its kernels share (include/fmha_kv4_abi.h has the layout).
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../../include/fmha_kv4_abi.h"

namespace b200mx {

struct Kv4View {
    uint8_t* pool;
    const int32_t* table;
    int32_t* lengths;
    uint64_t pages, page_bytes;   // page_bytes = HK * 136 << page_log2
    uint32_t B, HK, page_log2, table_width;
};

struct Kv4Rows {
    uint8_t* data;
    long long stride_b, stride_s, stride_h;   // bytes
};

struct Kv4AttendParams {
    Kv4View c;
    Kv4Rows q;
    __nv_bfloat16* out;
    const int32_t* counts;
    float* lse;
    float* weights;
    const float* weights_in;
    float* ws;
    float* scores;      // null, or [B][HK][tokens of the table][rows of a KV head, even]: what the weights are made of
    unsigned long long weights_width;
    uint32_t S, H, group, causal;
    float scale_log2;   // scale * log2(e)
    uint32_t* status;
};

struct Kv4EvictParams {
    Kv4View from, into;
    const float* weights;
    int32_t* kept;
    float* weights_out;
    unsigned long long weights_width, weights_out_width;
    uint32_t keep, recent, first;
};

int current_sm_count();   // host_api.cu
cudaError_t launch_kv4_append(const Kv4View& c, const Kv4Rows& k, const Kv4Rows& v, uint32_t S, const int32_t* counts, cudaStream_t stream);
cudaError_t launch_kv4_read(const Kv4View& c, const Kv4Rows& k, const Kv4Rows& v, uint32_t S, bool last, const int32_t* counts, cudaStream_t stream);
uint64_t kv4_attend_workspace(const Kv4View& c, uint32_t S, uint32_t H, bool weights, bool lse);
cudaError_t launch_kv4_attend(const Kv4AttendParams& p, cudaStream_t stream);
// kv4_weigh.cu: the attention weights, from p.lse and, if there, p.scores
cudaError_t launch_kv4_weigh(const Kv4AttendParams& p, cudaStream_t stream);
// kv4_prefill.cu: one CTA per SM, items of kv4_prefill_rows() query rows, partials in p.ws as the decode kernels leave them
uint32_t kv4_prefill_grid();
uint32_t kv4_prefill_rows();
cudaError_t launch_kv4_prefill(const Kv4AttendParams& p, uint32_t row_tiles, cudaStream_t stream);
cudaError_t launch_kv4_evict(const Kv4EvictParams& p, cudaStream_t stream);

// Every kernel of the cache goes out with programmatic dependent launch: all of its threads pass pdl_wait() in front of their first global access and before they
// end (a grid that ended without it would let the grid behind it start on data of the grid before).
template <typename... Params, typename... Args>
cudaError_t kv4_launch(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

#ifdef __CUDACC__
namespace kv4 {

__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Loads that stay behind the wait (volatile) and are not of the non-coherent kind
__device__ __forceinline__ int ld_i32(const int32_t* p) {
    int v;
    asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ float ld_f32(const float* p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ld_u32(const void* p) {
    uint32_t v;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 ld_v4(const void* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ uint32_t length_of(const Kv4View& c, uint32_t b) {
    const long long cap = static_cast<long long>(c.table_width) << c.page_log2;
    const long long n = ld_i32(c.lengths + b);
    return static_cast<uint32_t>(n < 0 ? 0 : (n > cap ? cap : n));
}
// rows of a sequence that stand for tokens
__device__ __forceinline__ uint32_t count_of(const int32_t* counts, uint32_t b, uint32_t S, uint32_t length) {
    const uint32_t most = S < length ? S : length;
    if (counts == nullptr) return most;
    const int n = ld_i32(counts + b);
    return n < 0 ? 0u : (static_cast<uint32_t>(n) > most ? most : static_cast<uint32_t>(n));
}
// the page that holds token t of sequence b, or -1 where the table names none of the pool
__device__ __forceinline__ long long page_of(const Kv4View& c, uint32_t b, uint32_t t) {
    const int id = ld_i32(c.table + static_cast<size_t>(b) * c.table_width + (t >> c.page_log2));
    return id >= 0 && static_cast<uint64_t>(id) < c.pages ? id : -1;
}
__device__ __forceinline__ uint8_t* record_of(const Kv4View& c, long long page, uint32_t head) {
    return c.pool + static_cast<uint64_t>(page) * c.page_bytes + (static_cast<uint64_t>(head) * FMHA_KV4_TOKEN_BYTES << c.page_log2);
}

// the two e2m1 codes of byte i of w (low nibble first) as f16
template <int kByte>
__device__ __forceinline__ uint32_t e2m1x2_to_f16x2(uint32_t w) {
    uint32_t r;
    if (kByte == 0) asm("{.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;}" : "=r"(r) : "r"(w));
    if (kByte == 1) asm("{.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;}" : "=r"(r) : "r"(w));
    if (kByte == 2) asm("{.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, c;}" : "=r"(r) : "r"(w));
    if (kByte == 3) asm("{.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, d;}" : "=r"(r) : "r"(w));
    return r;
}
// a byte of two e2m1 codes, the first in the low nibble
__device__ __forceinline__ uint32_t f32x2_to_e2m1x2(float lo, float hi) {
    uint32_t r;
    asm("{.reg .b8 a;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %1, %2;\n\tcvt.u32.u8 %0, a;}" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 2^(scale - 127); 0 for scale 0, infinity for 255 (times a code of 0, which such blocks hold: NaN)
__device__ __forceinline__ float scale_f32(uint32_t word, int byte) { return __uint_as_float(((word >> (8 * byte)) & 0xFFu) << 23); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 f16x2_to_f32(uint32_t h) {
    float2 f;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Softmax of rows that multiply V in f16. V's factors of a group of tokens that are worked on together are taken relative to 2^e, e the exponent of the group's largest, kept
// within what f32 sums of 2^(s - M) bear (they lie between 2^-kHighE and 2^(8 - kLowE) a token when M follows s + e). The factors go in times 2^kUp, which the division
// by the sums takes out again: f16 has more room below 1 than above, and factors are exact down to 2^-34 of the group's largest.
constexpr int kLowE = -100, kHighE = 124, kUp = 10;
constexpr float kDown = 1.0f / (1 << kUp);
// 0xFF in the place of the scale bytes that stand for NaN
__device__ __forceinline__ uint32_t nan_bytes(uint32_t word) { return __vcmpeq4(word, 0xFFFFFFFFu); }
// the largest of a token's four scale bytes
__device__ __forceinline__ uint32_t largest_byte(uint32_t word) { return max(max(word & 0xFFu, (word >> 8) & 0xFFu), max((word >> 16) & 0xFFu, word >> 24)); }
__device__ __forceinline__ int group_exponent(uint32_t largest) { return min(max(static_cast<int>(largest) - 127, kLowE), kHighE); }
// A query row in f16: the factor that brings its largest element (f32 bits of its size) to the exponent 14, and what undoes it. Rows of zeros or with Inf or NaN keep 1.
__device__ __forceinline__ float2 row_factors(uint32_t largest) {
    int field = static_cast<int>(largest >> 23);
    if (field == 255 || largest == 0u) field = 141;
    if (field < 15) field = 15;   // both stay normal
    return make_float2(__uint_as_float(static_cast<uint32_t>(268 - field) << 23), __uint_as_float(static_cast<uint32_t>(field - 14) << 23));
}
struct ValueFactors {
    uint32_t r01, r23;   // 2^(E - 127 - e + kUp) of the blocks, f16 (E <= 252 leaves them below its largest); NaN for 255
};
__device__ __forceinline__ ValueFactors value_factors(uint32_t word, uint32_t largest, int e) {
    const int e0 = word & 0xFFu, e1 = (word >> 8) & 0xFFu, e2 = (word >> 16) & 0xFFu, e3 = word >> 24, up = kUp - e;
    float r0 = __uint_as_float(static_cast<uint32_t>(max(e0 + up, 0)) << 23), r1 = __uint_as_float(static_cast<uint32_t>(max(e1 + up, 0)) << 23);
    float r2 = __uint_as_float(static_cast<uint32_t>(max(e2 + up, 0)) << 23), r3 = __uint_as_float(static_cast<uint32_t>(max(e3 + up, 0)) << 23);
    if (largest == 255u) {
        const float nan = __uint_as_float(0x7FC00000u);
        r0 = e0 == 255 ? nan : r0, r1 = e1 == 255 ? nan : r1, r2 = e2 == 255 ? nan : r2, r3 = e3 == 255 ? nan : r3;
    }
    return {pack_f16x2(r0, r1), pack_f16x2(r2, r3)};
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
// D (f32 16 x 8) = A (bf16 16 x 16) B (bf16 16 x 8) + C; mma_f16: the same of f16
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

}  // namespace kv4
#endif

}  // namespace b200mx
