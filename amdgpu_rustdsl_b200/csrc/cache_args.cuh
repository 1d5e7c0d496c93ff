// Checks of arguments that the C entries around the caches share: refusals with a message, views of caches and rows.
#pragma once
#include "kv4.cuh"

#include <cstdarg>
#include <cstdio>

namespace b200mx {
uint32_t* device_status_word();   // host_api.cu
}

namespace {

using b200mx::Kv4Rows;
using b200mx::Kv4View;

[[maybe_unused]] int refuse(char* err, size_t cap, const char* format, ...) {
    if (err != nullptr && cap > 0) {
        va_list args;
        va_start(args, format);
        std::vsnprintf(err, cap, format, args);
        va_end(args);
    }
    return 6;   // FMHA_MXFP8_E_ARG
}
[[maybe_unused]] int done(cudaError_t e, char* err, size_t cap) {
    if (e == cudaSuccess) return 0;
    (void)refuse(err, cap, "launch failed: %s", cudaGetErrorString(e));
    return -static_cast<int>(e);
}

[[maybe_unused]] bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// whether two ranges of bytes have any in common
[[maybe_unused]] bool overlap(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
    const uint64_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + b_bytes && y < x + a_bytes;
}

// kernels keep row numbers in 32 bits and grids in 31
constexpr uint64_t kMostRows = 1ull << 30;

// token_bytes: of a token and KV head
[[maybe_unused]] int view_of(const fmha_kv4_cache* c, const char* name, Kv4View& v, char* err, size_t cap, uint32_t token_bytes = FMHA_KV4_TOKEN_BYTES) {
    if (c == nullptr || c->pool == nullptr || c->table == nullptr || c->lengths == nullptr) return refuse(err, cap, "%s: pool, table and lengths must be given", name);
    if (c->page != 16u && c->page != 32u && c->page != 64u && c->page != 128u) return refuse(err, cap, "%s: pages hold 16, 32, 64 or 128 tokens, not %u", name, c->page);
    if (c->B == 0u || c->HK == 0u || c->pages == 0u || c->table_width == 0u) return refuse(err, cap, "%s: no sequences, heads, pages or table columns", name);
    if (!aligned16(c->pool)) return refuse(err, cap, "%s: the pool must be 16-byte aligned", name);
    if (c->pages > 0x7FFFFFFFull || static_cast<uint64_t>(c->B) * c->HK > kMostRows || static_cast<uint64_t>(c->table_width) * c->page > 0x7FFFFFFFull)
        return refuse(err, cap, "%s: more than 2^31 pages or tokens of a sequence, or 2^30 sequences x heads", name);
    if (static_cast<uint64_t>(c->HK) * token_bytes * c->page > 0xFFFFFFFFull) return refuse(err, cap, "%s: pages of 4 GiB and more", name);   // (the decode kernel holds their size in 32 bits)
    v.pool = static_cast<uint8_t*>(c->pool);
    v.table = c->table;
    v.lengths = c->lengths;
    v.pages = c->pages;
    v.page_bytes = static_cast<uint64_t>(c->HK) * token_bytes * c->page;
    v.B = c->B, v.HK = c->HK, v.table_width = c->table_width;
    v.page_log2 = c->page == 16u ? 4u : c->page == 32u ? 5u : c->page == 64u ? 6u : 7u;
    return 0;
}

[[maybe_unused]] int rows_of(const fmha_kv4_rows* x, uint32_t S, const char* name, Kv4Rows& r, char* err, size_t cap) {
    if (x == nullptr || (x->data == nullptr && S != 0u)) return refuse(err, cap, "%s must be given", name);   // (no rows have no address)
    if (!aligned16(x->data) || ((x->stride_b | x->stride_s | x->stride_h) & 7) != 0) return refuse(err, cap, "%s: pointer and strides must be multiples of 16 bytes", name);
    r.data = static_cast<uint8_t*>(x->data);
    r.stride_b = 2 * x->stride_b, r.stride_s = 2 * x->stride_s, r.stride_h = 2 * x->stride_h;
    return 0;
}

}  // namespace
