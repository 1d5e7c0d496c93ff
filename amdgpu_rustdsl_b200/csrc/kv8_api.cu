// C ABI of the operators around the 8-bit cache (include/fmha_kv8_abi.h): checks of the arguments and launches.
#include "cache_args.cuh"
#include "kv8.cuh"

namespace {

constexpr uint32_t kTokenBytes = FMHA_KV8_BLOCK_BYTES / FMHA_KV8_BLOCK_TOKENS;

int too_many_rows(const Kv4View& c, uint32_t S, const char* name, char* err, size_t cap) {
    return static_cast<uint64_t>(c.B) * S * c.HK > kMostRows ? refuse(err, cap, "%s: more than 2^30 rows", name) : 0;
}

}  // namespace

extern "C" {

int fmha_kv8_append(const fmha_kv8_cache* cache, const fmha_kv4_rows* k, const fmha_kv4_rows* v, uint32_t S, const int32_t* counts, void* stream, char* err, size_t cap) {
    Kv4View c;
    Kv4Rows rk, rv;
    if (int r = view_of(cache, "append", c, err, cap, kTokenBytes)) return r;
    if (int r = rows_of(k, S, "append: k", rk, err, cap)) return r;
    if (int r = rows_of(v, S, "append: v", rv, err, cap)) return r;
    if (S == 0u) return 0;
    if (int r = too_many_rows(c, S, "append", err, cap)) return r;
    return done(b200mx::launch_kv8_append(c, rk, rv, S, counts, static_cast<cudaStream_t>(stream)), err, cap);
}

int fmha_kv8_read(const fmha_kv8_cache* cache, const fmha_kv4_rows* k, const fmha_kv4_rows* v, uint32_t S, int last, const int32_t* counts, void* stream, char* err, size_t cap) {
    Kv4View c;
    Kv4Rows rk, rv;
    if (int r = view_of(cache, "read", c, err, cap, kTokenBytes)) return r;
    if (int r = rows_of(k, S, "read: k", rk, err, cap)) return r;
    if (int r = rows_of(v, S, "read: v", rv, err, cap)) return r;
    if (!last && counts != nullptr) return refuse(err, cap, "read: counts go with the newest tokens only");
    if (S == 0u) return 0;
    if (int r = too_many_rows(c, S, "read", err, cap)) return r;
    return done(b200mx::launch_kv8_read(c, rk, rv, S, last != 0, counts, static_cast<cudaStream_t>(stream)), err, cap);
}

uint64_t fmha_kv8_attend_workspace(const fmha_kv8_cache* cache, const fmha_kv8_attend_args* a) {
    Kv4View c;
    if (a == nullptr || view_of(cache, "", c, nullptr, 0, kTokenBytes) != 0 || a->H == 0u || a->H % c.HK != 0u) return 0;
    return b200mx::kv8_attend_workspace(c, a->S, a->H);
}

int fmha_kv8_attend(const fmha_kv8_cache* cache, const fmha_kv8_attend_args* a, void* stream, char* err, size_t cap) {
    b200mx::Kv8AttendParams p = {};
    if (a == nullptr) return refuse(err, cap, "attend: no arguments");
    if (int r = view_of(cache, "attend", p.c, err, cap, kTokenBytes)) return r;
    if (int r = rows_of(&a->q, a->S, "attend: q", p.q, err, cap)) return r;
    if (a->H == 0u || a->H % p.c.HK != 0u || a->H / p.c.HK > 16u) return refuse(err, cap, "attend: H must be 1 to 16 times the KV heads (H %u, HK %u)", a->H, p.c.HK);
    if ((a->out == nullptr && a->S != 0u) || !aligned16(a->out)) return refuse(err, cap, "attend: out must be given and 16-byte aligned");
    if (a->S == 0u) return 0;
    if (static_cast<uint64_t>(p.c.B) * a->S * a->H > kMostRows) return refuse(err, cap, "attend: more than 2^30 query rows");
    // the kernels deal out steps of 80 tokens and 256 rows at least, counted in 32 bits
    const uint64_t tokens = static_cast<uint64_t>(p.c.table_width) << p.c.page_log2, row_tiles = (static_cast<uint64_t>(a->S) * (a->H / p.c.HK) + 255u) / 256u;
    if (((tokens + 79u) / 80u + 5u) * p.c.B * p.c.HK > 0xFFFFFFFFull / row_tiles) return refuse(err, cap, "attend: more than 2^32 steps of 80 tokens and 256 query rows");
    if (!(a->scale > 0.0f) || a->scale > 2.3e38f) return refuse(err, cap, "attend: scale must be a positive number");
    if (a->workspace == nullptr || !aligned16(a->workspace) || a->workspace_bytes < fmha_kv8_attend_workspace(cache, a))
        return refuse(err, cap, "attend: the workspace must be 16-byte aligned and hold fmha_kv8_attend_workspace() bytes");
    if (a->out == a->q.data) {   // a row's elements are read before it is written, by whoever writes it
        const int64_t row = 128, rows = row * a->H, all = rows * a->S;
        if ((a->H > 1u && a->q.stride_h != row) || (a->S > 1u && a->q.stride_s != rows) || (p.c.B > 1u && a->q.stride_b != all)) return refuse(err, cap, "attend: out may be q only where q is packed as out is");
    }
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.counts = a->counts;
    p.lse = a->lse;
    p.ws = static_cast<float*>(a->workspace);
    p.S = a->S, p.H = a->H, p.group = a->H / p.c.HK, p.causal = a->causal != 0u;
    p.scale_log2 = a->scale * 1.44269504088896341f;
    p.status = b200mx::device_status_word();
    if (p.status == nullptr) return -static_cast<int>(cudaErrorInvalidSymbol);
    return done(b200mx::launch_kv8_attend(p, static_cast<cudaStream_t>(stream)), err, cap);
}

}  // extern "C"
