// The attention weights that the cached tokens received: w[t] = sum of 2^(s - lse) over the query rows and the heads of a KV head's group, once the rows' log-sum-exps are
// known. The sums run over the rows in order, a token's all in one warp: the same bits every time.
//
// With up to 8 rows the attention kernel has left the scores (a token's all in one 8- to 32-byte piece), and a thread adds up a token's. With more rows S^T = K Q^T is computed
// again, a warp for 32 tokens whose K it converts once (to bf16, which a code times its factor is exactly), against blocks of 64 rows that all warps of the CTA use. The rows
// come as they are, by asynchronous copies into the operand's layout, a block ahead. That is bound by the matrix instructions (8 per 16 tokens and 8 rows): 400 rows
// over four ragged sequences of up to 4001 tokens, 8 heads, 32 us where the instructions' rate gives about 15 and two uneven rounds of CTAs twice that; 46 us before the rows
// were copied as they are, 35 with CTAs of half the tokens.
#include "kv4.cuh"
#include "ptx_sm100.cuh"

namespace b200mx {

namespace {

using namespace kv4;

constexpr uint32_t kWarps = 8, kThreads = 32 * kWarps, kUnit = 32, kTile = kWarps * kUnit, kBlock = 64;   // kBlock: rows at a time
static_assert(kBlock == 8 * kWarps, "a warp brings 8 rows");
constexpr float kLog2e = 1.44269504088896341f;

__device__ __forceinline__ void store_weight(const Kv4AttendParams& p, uint32_t bh, uint32_t t, uint32_t length, uint32_t n, float v) {
    const size_t at = static_cast<size_t>(bh) * p.weights_width + t;
    const bool old = p.weights_in != nullptr && (!p.causal || t < length - n);   // new tokens bring no weight along
    p.weights[at] = (old ? ld_f32(p.weights_in + at) : 0.0f) + v;
}

template <int kRows>   // rows of a KV head, even
__global__ void __launch_bounds__(256) kv4_add_scores_kernel(const __grid_constant__ Kv4AttendParams p, uint32_t blocks) {
    pdl_launch();
    pdl_wait();
    const uint32_t bh = blockIdx.x / blocks, head = bh % p.c.HK, b = bh / p.c.HK, t = (blockIdx.x - bh * blocks) * 256u + threadIdx.x;
    const uint32_t length = length_of(p.c, b);
    if (t >= length) return;
    const uint32_t n = count_of(p.counts, b, p.S, length), rows = n * p.group;
    const float* s = p.scores + (static_cast<size_t>(bh) * (static_cast<size_t>(p.c.table_width) << p.c.page_log2) + t) * kRows;
    float2 two[kRows / 2];
#pragma unroll
    for (int r = 0; r < kRows / 2; ++r) {
        two[r] = make_float2(-INFINITY, -INFINITY);
        if (2u * r < rows) asm volatile("ld.global.v2.f32 {%0, %1}, [%2];" : "=f"(two[r].x), "=f"(two[r].y) : "l"(s + 2 * r));
    }
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (static_cast<uint32_t>(r) >= rows) break;
        const uint32_t i = r / p.group, h = head * p.group + r % p.group;
        const float lse = ld_f32(p.lse + (static_cast<size_t>(b) * p.H + h) * p.S + i) * kLog2e, score = r & 1 ? two[r / 2].y : two[r / 2].x;
        const bool sees = !p.causal || t < length - n + i + 1u;
        sum += sees ? ex2(score - lse) : 0.0f;
    }
    store_weight(p, bh, t, length, n, sum);
}

struct Shared {
    uint4 q[2][kBlock / 8][4][32];   // [buffer][group of 8 rows][block of elements][lane]: the operand's elements
    float lse[2][kBlock];
    uint32_t limit[2][kBlock];
};

// two elements in f16, times f, in bf16
__device__ __forceinline__ uint32_t times(uint32_t two, float f) {
    const float2 x = f16x2_to_f32(two);
    return pack_bf16x2(x.x * f, x.y * f);
}

__global__ void __launch_bounds__(kThreads) kv4_weigh_kernel(const __grid_constant__ Kv4AttendParams p, uint32_t tiles) {
    __shared__ Shared sh;
    pdl_launch();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, gid = lane >> 2, tig = lane & 3u;
    const uint32_t bh = blockIdx.x / tiles, head = bh % p.c.HK, b = bh / p.c.HK, tile0 = (blockIdx.x - bh * tiles) * kTile, tok0 = tile0 + warp * kUnit;
    const uint32_t length = length_of(p.c, b), n = count_of(p.counts, b, p.S, length), page = 1u << p.c.page_log2, rows = n * p.group;
    if (tile0 >= length) return;   // (the same for the CTA)
    // rows that see none of the tile are left out: with a causal mask the first that sees a token of it is token tile0 itself
    const uint32_t first = p.causal && tile0 > length - n ? (tile0 - (length - n)) * p.group / kBlock * kBlock : 0u;
    // a warp brings 8 rows: lane (gid, tig) the elements 32 blk + 8 tig .. + 7 of row gid. Rows behind the last become zeros that see nothing.
    auto bring = [&](uint32_t row0, uint32_t into) {
        if (row0 >= rows) return;
        const uint32_t r = 8u * warp + gid, row = row0 + r, i = row / p.group, h = head * p.group + row - i * p.group;
        const bool live = row < rows;
        const uint8_t* from = live ? p.q.data + b * p.q.stride_b + i * p.q.stride_s + h * p.q.stride_h + 16u * tig : p.q.data;
#pragma unroll
        for (uint32_t blk = 0; blk < 4u; ++blk) sm100::cp_async_16(sm100::smem_u32(&sh.q[into][warp][blk][lane]), from + (live ? 64u * blk : 0u), live ? 16u : 0u);
        if (tig == 0u) {
            sm100::cp_async_4(sm100::smem_u32(&sh.lse[into][r]), live ? p.lse + (static_cast<size_t>(b) * p.H + h) * p.S + i : p.lse, live ? 4u : 0u);
            sh.limit[into][r] = !live ? 0u : p.causal ? length - n + i + 1u : length;
        }
    };
    bring(first, 0u);
    // A lane's share of the K operand, 16 tokens at a time: the elements 32 blk + 8 tig .. + 7 of the tokens gid and gid + 8
    uint32_t k[2][4][8];
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t t = tok0 + 16u * gr + 8u * half + gid;
            uint4 codes = make_uint4(0u, 0u, 0u, 0u);
            uint32_t scales = 0xFFFFFFFFu;   // a page outside the pool: NaN
            const long long id = t < length ? page_of(p.c, b, t) : -1;
            if (id >= 0) {
                const uint8_t* rec = record_of(p.c, id, head);
                codes = ld_v4(rec + 64u * (t & (page - 1u)) + 16u * tig), scales = ld_u32(rec + 128u * page + 4u * (t & (page - 1u)));
            }
#pragma unroll
            for (int blk = 0; blk < 4; ++blk) {
                const uint32_t w0 = blk < 2 ? codes.x : codes.y, w1 = blk < 2 ? codes.z : codes.w, scale = scales >> (8 * blk) & 0xFFu;
                const float f = scale == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(scale << 23);
                k[gr][blk][half] = times(blk & 1 ? e2m1x2_to_f16x2<2>(w0) : e2m1x2_to_f16x2<0>(w0), f);
                k[gr][blk][2 + half] = times(blk & 1 ? e2m1x2_to_f16x2<3>(w0) : e2m1x2_to_f16x2<1>(w0), f);
                k[gr][blk][4 + half] = times(blk & 1 ? e2m1x2_to_f16x2<2>(w1) : e2m1x2_to_f16x2<0>(w1), f);
                k[gr][blk][6 + half] = times(blk & 1 ? e2m1x2_to_f16x2<3>(w1) : e2m1x2_to_f16x2<1>(w1), f);
            }
        }
    }
    float sum[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
    uint32_t from = 0;
    for (uint32_t row0 = first; row0 < rows; row0 += kBlock, from ^= 1u) {
        sm100::cp_async_wait_all();
        __syncthreads();   // the block is there, and all are done with the one before
        bring(row0 + kBlock, from ^ 1u);
        if (tok0 >= length) continue;
        const uint32_t groups = min(kBlock, rows - row0 + 7u) / 8u;
        for (uint32_t g = 0; g < groups; ++g) {
            float d[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int blk = 0; blk < 4; ++blk) {
                const uint4 q = sh.q[from][g][blk][lane];
#pragma unroll
                for (int gr = 0; gr < 2; ++gr) {
                    mma_bf16(d[gr], k[gr][blk][0], k[gr][blk][1], k[gr][blk][2], k[gr][blk][3], q.x, q.y, d[gr]);
                    mma_bf16(d[gr], k[gr][blk][4], k[gr][blk][5], k[gr][blk][6], k[gr][blk][7], q.z, q.w, d[gr]);
                }
            }
            float2 lse = *reinterpret_cast<const float2*>(&sh.lse[from][8u * g + 2u * tig]);
            const uint2 limit = *reinterpret_cast<const uint2*>(&sh.limit[from][8u * g + 2u * tig]);
            lse.x *= kLog2e, lse.y *= kLog2e;
#pragma unroll
            for (int gr = 0; gr < 2; ++gr) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t t = tok0 + 16u * gr + 8u * (i >> 1) + gid;
                    const float w = ex2(fmaf(d[gr][i], p.scale_log2, -(i & 1 ? lse.y : lse.x)));
                    if (t < (i & 1 ? limit.y : limit.x)) sum[gr][i >> 1] += w;
                }
            }
        }
    }
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float v = sum[gr][half];
            v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
            v += __shfl_xor_sync(0xFFFFFFFFu, v, 2);
            const uint32_t t = tok0 + 16u * gr + 8u * half + gid;
            if (tig == 0u && t < length) store_weight(p, bh, t, length, n, v);
        }
    }
}

}  // namespace

cudaError_t launch_kv4_weigh(const Kv4AttendParams& p, cudaStream_t stream) {
    const uint64_t tokens = static_cast<uint64_t>(p.c.table_width) << p.c.page_log2;
    const uint32_t items = p.c.B * p.c.HK, rows = p.S * p.group;
    if (p.scores != nullptr) {
        const uint32_t blocks = static_cast<uint32_t>((tokens + 255u) / 256u);
        return kv4_launch(rows <= 2u ? kv4_add_scores_kernel<2> : rows <= 4u ? kv4_add_scores_kernel<4> : rows <= 6u ? kv4_add_scores_kernel<6> : kv4_add_scores_kernel<8>, dim3(blocks * items), 256u, 0, stream, p, blocks);
    }
    const uint32_t tiles = static_cast<uint32_t>((tokens + kTile - 1u) / kTile);
    return kv4_launch(kv4_weigh_kernel, dim3(tiles * items), kThreads, 0, stream, p, tiles);
}

}  // namespace b200mx
