// Tokens into and out of the 4-bit cache: kv4_append rounds bf16 rows to MXFP4 and writes them to their pages, kv4_read gives the values back in bf16.
//
//   E = clamp(floor(log2 amax) - 2 + 127, 1, 252) over 32 elements,   code = e2m1_rne_sat(x * 2^(127 - E)),   value = code * 2^(E - 127)
//
// A token's row of one KV head (K or V) is the work of 16 lanes: a lane holds 8 consecutive elements (16 bytes of bf16), four lanes a block. Both directions are
// bound by bytes (256 of bf16 and 68 of the cache per row).
#include "kv4.cuh"

namespace b200mx {

namespace {

using namespace kv4;

struct StoreParams {
    Kv4View c;
    Kv4Rows k, v;
    uint32_t S;
    int last;
    const int32_t* counts;
};

// Row r of the launch: (b, i, head) with the heads fastest, K rows in front of the V rows
struct RowOf {
    uint32_t b, i, head;
    bool is_v;
};
__device__ __forceinline__ RowOf row_of(const StoreParams& p, unsigned long long r) {
    RowOf o;
    const unsigned long long half = static_cast<unsigned long long>(p.c.B) * p.S * p.c.HK;
    o.is_v = r >= half;
    if (o.is_v) r -= half;
    o.head = static_cast<uint32_t>(r % p.c.HK);
    r /= p.c.HK;
    o.i = static_cast<uint32_t>(r % p.S);
    o.b = static_cast<uint32_t>(r / p.S);
    return o;
}
__device__ __forceinline__ uint8_t* row_address(const Kv4Rows& x, const RowOf& o) {
    return x.data + o.b * x.stride_b + o.i * x.stride_s + o.head * x.stride_h;
}

__global__ void __launch_bounds__(256) kv4_append_kernel(const __grid_constant__ StoreParams p) {
    pdl_launch();
    pdl_wait();
    const unsigned long long rows = 2ull * p.c.B * p.S * p.c.HK, step = gridDim.x * 16ull;
    const unsigned lane = threadIdx.x & 31u, part = lane & 15u, blk = part >> 2, tig = part & 3u;
    // whole warps stay in the loop together (shuffles): the bound is the warp's first row
    for (unsigned long long r0 = blockIdx.x * 16ull + (threadIdx.x >> 5) * 2u; r0 < rows; r0 += step) {
        const unsigned long long r = r0 + (lane >> 4);
        bool live = r < rows;
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        uint8_t* record = nullptr;
        uint32_t slot = 0;
        bool is_v = false;
        if (live) {
            const RowOf o = row_of(p, r);
            const uint32_t L = length_of(p.c, o.b), n = count_of(p.counts, o.b, p.S, L);
            live = o.i < n;
            if (live) {
                const uint32_t t = L - n + o.i;
                const long long page = page_of(p.c, o.b, t);
                live = page >= 0;
                if (live) {
                    raw = ld_v4(row_address(o.is_v ? p.v : p.k, o) + 16u * part);
                    record = record_of(p.c, page, o.head);
                    slot = t & ((1u << p.c.page_log2) - 1u);
                    is_v = o.is_v;
                }
            }
        }
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        // the block's largest magnitude, as the bits of an f32 (ordered as integers; Inf and NaN come out on top)
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = max(amax, max((w[i] << 16) & 0x7FFFFFFFu, w[i] & 0x7FFF0000u));
        amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
        const uint32_t field = amax >> 23;
        const bool broken = field == 255u;
        const uint32_t e = broken ? 255u : (field < 3u ? 1u : field - 2u);
        // x * 2^(127 - E), exact up to what rounds to a code of 0 anyway; 127 - E lies in [-125, 126]
        const float up = broken ? 0.0f : __uint_as_float((254u - e) << 23);
        uint32_t code[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) code[i] = broken ? 0u : f32x2_to_e2m1x2(__fmul_rn(__uint_as_float(w[i] << 16), up), __fmul_rn(__uint_as_float(w[i] & 0xFFFF0000u), up));
        // elements 32 blk + 8 tig ..: bytes 0, 1 belong to group g = 2 tig, bytes 2, 3 to group 2 tig + 1; a group's bytes 2 blk, 2 blk + 1. Lanes of an even and an
        // odd block swap halves, so that each holds a word of one group: lane (blk, tig) word 4 tig + 2 (blk & 1) + (blk >> 1)
        const uint32_t lo = code[0] | (code[1] << 8), hi = code[2] | (code[3] << 8);
        const bool odd = blk & 1u;
        const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, odd ? lo : hi, 4);
        const uint32_t word = odd ? (got | (hi << 16)) : (lo | (got << 16));
        // the row's four scale bytes
        uint32_t scales = e << (8u * blk);
        scales |= __shfl_xor_sync(0xFFFFFFFFu, scales, 4);
        scales |= __shfl_xor_sync(0xFFFFFFFFu, scales, 8);
        if (live) {
            const uint32_t page = 1u << p.c.page_log2;
            uint8_t* codes = record + (is_v ? 64u * page : 0u) + 64u * slot;
            *reinterpret_cast<uint32_t*>(codes + 4u * (4u * tig + 2u * (blk & 1u) + (blk >> 1))) = word;
            if (part == 0u) *reinterpret_cast<uint32_t*>(record + (is_v ? 132u : 128u) * page + 4u * slot) = scales;
        }
    }
}

__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ StoreParams p) {
    pdl_launch();
    pdl_wait();
    const unsigned long long rows = 2ull * p.c.B * p.S * p.c.HK, step = gridDim.x * 16ull;
    const unsigned part = threadIdx.x & 15u, blk = part >> 2, tig = part & 3u;
    for (unsigned long long r = blockIdx.x * 16ull + (threadIdx.x >> 4); r < rows; r += step) {
        const RowOf o = row_of(p, r);
        const uint32_t L = length_of(p.c, o.b), n = p.last ? count_of(p.counts, o.b, p.S, L) : min(p.S, L);
        uint4 out = make_uint4(0u, 0u, 0u, 0u);
        if (o.i < n) {
            const uint32_t t = p.last ? L - n + o.i : o.i, page = 1u << p.c.page_log2, slot = t & (page - 1u);
            const long long id = page_of(p.c, o.b, t);
            if (id >= 0) {
                const uint8_t* record = record_of(p.c, id, o.head);
                const uint8_t* codes = record + (o.is_v ? 64u * page : 0u) + 64u * slot;
                // the two groups' bytes of this lane's block
                const uint8_t* two = codes + 16u * tig + 2u * blk;
                const uint32_t word = *reinterpret_cast<const volatile uint16_t*>(two) | (static_cast<uint32_t>(*reinterpret_cast<const volatile uint16_t*>(two + 8)) << 16);
                const float scale = scale_f32(ld_u32(record + (o.is_v ? 132u : 128u) * page + 4u * slot), static_cast<int>(blk));
                const float2 a = f16x2_to_f32(e2m1x2_to_f16x2<0>(word)), b = f16x2_to_f32(e2m1x2_to_f16x2<1>(word));
                const float2 c = f16x2_to_f32(e2m1x2_to_f16x2<2>(word)), d = f16x2_to_f32(e2m1x2_to_f16x2<3>(word));
                out = make_uint4(pack_bf16x2(a.x * scale, a.y * scale), pack_bf16x2(b.x * scale, b.y * scale), pack_bf16x2(c.x * scale, c.y * scale),
                                 pack_bf16x2(d.x * scale, d.y * scale));
            } else {
                out = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
            }
        }
        *reinterpret_cast<uint4*>(row_address(o.is_v ? p.v : p.k, o) + 16u * part) = out;
    }
}

unsigned store_grid(const Kv4View& c, uint32_t S) {
    const unsigned long long blocks = (2ull * c.B * S * c.HK + 15ull) / 16ull, cap = 8ull * static_cast<unsigned long long>(current_sm_count());
    return static_cast<unsigned>(blocks < cap ? blocks : cap);
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4View& c, const Kv4Rows& k, const Kv4Rows& v, uint32_t S, const int32_t* counts, cudaStream_t stream) {
    return kv4_launch(kv4_append_kernel, dim3(store_grid(c, S)), 256u, 0, stream, StoreParams{c, k, v, S, 1, counts});
}
cudaError_t launch_kv4_read(const Kv4View& c, const Kv4Rows& k, const Kv4Rows& v, uint32_t S, bool last, const int32_t* counts, cudaStream_t stream) {
    return kv4_launch(kv4_read_kernel, dim3(store_grid(c, S)), 256u, 0, stream, StoreParams{c, k, v, S, last ? 1 : 0, counts});
}

}  // namespace b200mx
