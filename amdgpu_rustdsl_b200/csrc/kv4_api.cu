// C ABI of the operators around the 4-bit cache (include/fmha_kv4_abi.h): checks of the arguments and launches.
#include "cache_args.cuh"

extern "C" {

int fmha_kv4_append(const fmha_kv4_cache* cache, const fmha_kv4_rows* k, const fmha_kv4_rows* v, uint32_t S, const int32_t* counts, void* stream, char* err, size_t cap) {
    Kv4View c;
    Kv4Rows rk, rv;
    if (int r = view_of(cache, "append", c, err, cap)) return r;
    if (int r = rows_of(k, S, "append: k", rk, err, cap)) return r;
    if (int r = rows_of(v, S, "append: v", rv, err, cap)) return r;
    if (S == 0u) return 0;
    if (static_cast<uint64_t>(c.B) * S * c.HK > kMostRows) return refuse(err, cap, "append: more than 2^30 rows");
    return done(b200mx::launch_kv4_append(c, rk, rv, S, counts, static_cast<cudaStream_t>(stream)), err, cap);
}

int fmha_kv4_read(const fmha_kv4_cache* cache, const fmha_kv4_rows* k, const fmha_kv4_rows* v, uint32_t S, int last, const int32_t* counts, void* stream, char* err, size_t cap) {
    Kv4View c;
    Kv4Rows rk, rv;
    if (int r = view_of(cache, "read", c, err, cap)) return r;
    if (int r = rows_of(k, S, "read: k", rk, err, cap)) return r;
    if (int r = rows_of(v, S, "read: v", rv, err, cap)) return r;
    if (!last && counts != nullptr) return refuse(err, cap, "read: counts go with the newest tokens only");
    if (S == 0u) return 0;
    if (static_cast<uint64_t>(c.B) * S * c.HK > kMostRows) return refuse(err, cap, "read: more than 2^30 rows");
    return done(b200mx::launch_kv4_read(c, rk, rv, S, last != 0, counts, static_cast<cudaStream_t>(stream)), err, cap);
}

uint64_t fmha_kv4_attend_workspace(const fmha_kv4_cache* cache, const fmha_kv4_attend_args* a) {
    Kv4View c;
    if (a == nullptr || view_of(cache, "", c, nullptr, 0) != 0 || a->H == 0u || a->H % c.HK != 0u) return 0;
    return b200mx::kv4_attend_workspace(c, a->S, a->H, a->weights != nullptr, a->lse != nullptr);
}

int fmha_kv4_attend(const fmha_kv4_cache* cache, const fmha_kv4_attend_args* a, void* stream, char* err, size_t cap) {
    b200mx::Kv4AttendParams p = {};
    if (a == nullptr) return refuse(err, cap, "attend: no arguments");
    if (int r = view_of(cache, "attend", p.c, err, cap)) return r;
    if (int r = rows_of(&a->q, a->S, "attend: q", p.q, err, cap)) return r;
    if (a->H == 0u || a->H % p.c.HK != 0u || a->H / p.c.HK > 16u) return refuse(err, cap, "attend: H must be 1 to 16 times the KV heads (H %u, HK %u)", a->H, p.c.HK);
    if ((a->out == nullptr && a->S != 0u) || !aligned16(a->out)) return refuse(err, cap, "attend: out must be given and 16-byte aligned");
    if (a->S == 0u && (a->weights == nullptr || a->weights == a->weights_in)) return 0;
    if (static_cast<uint64_t>(p.c.B) * a->S * a->H > kMostRows) return refuse(err, cap, "attend: more than 2^30 query rows");
    const uint64_t tokens = static_cast<uint64_t>(p.c.table_width) << p.c.page_log2;
    // the kernels deal out steps of 128 tokens and 256 rows at most, counted in 32 bits
    const uint64_t row_tiles = a->S == 0u ? 1u : (static_cast<uint64_t>(a->S) * (a->H / p.c.HK) + 255u) / 256u;
    if (((tokens + 127u) / 128u) * p.c.B * p.c.HK > 0xFFFFFFFFull / row_tiles) return refuse(err, cap, "attend: more than 2^32 steps of 128 tokens and 256 query rows");
    if (a->weights != nullptr && a->weights_width < tokens) return refuse(err, cap, "attend: weights must have room for the %llu tokens of the table", static_cast<unsigned long long>(tokens));
    const uint64_t weights_bytes = 4u * static_cast<uint64_t>(p.c.B) * p.c.HK * a->weights_width;
    if (a->weights != nullptr && a->weights_in != nullptr && a->weights_in != a->weights && overlap(a->weights, weights_bytes, a->weights_in, weights_bytes))
        return refuse(err, cap, "attend: weights_in must be weights or share no memory with it");
    if (a->weights == nullptr && a->weights_in != nullptr) return refuse(err, cap, "attend: weights_in without weights");
    if (a->weights != nullptr && static_cast<uint64_t>(p.c.B) * p.c.HK * ((tokens + 127u) / 128u) > kMostRows) return refuse(err, cap, "attend: more than 2^37 cached tokens x heads with weights");
    if (!(a->scale > 0.0f) || a->scale > 2.3e38f) return refuse(err, cap, "attend: scale must be a positive number");
    if (a->workspace == nullptr || !aligned16(a->workspace) || a->workspace_bytes < fmha_kv4_attend_workspace(cache, a))
        return refuse(err, cap, "attend: the workspace must be 16-byte aligned and hold fmha_kv4_attend_workspace() bytes");
    if (a->out == a->q.data && a->S != 0u) {   // a row's elements are read before it is written, by whoever writes it; the weights of many rows go by the queries again
        const int64_t row = 128, rows = row * a->H, all = rows * a->S;
        if ((a->H > 1u && a->q.stride_h != row) || (a->S > 1u && a->q.stride_s != rows) || (p.c.B > 1u && a->q.stride_b != all)) return refuse(err, cap, "attend: out may be q only where q is packed as out is");
        if (a->weights != nullptr && a->S * (a->H / p.c.HK) > 8u) return refuse(err, cap, "attend: out may not be q where the weights of more than 8 rows of a KV head are asked for");
    }
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.counts = a->counts;
    p.lse = a->lse;
    p.weights = a->weights, p.weights_in = a->weights_in, p.weights_width = a->weights_width;
    p.ws = static_cast<float*>(a->workspace);
    p.S = a->S, p.H = a->H, p.group = a->H / p.c.HK, p.causal = a->causal != 0u;
    p.scale_log2 = a->scale * 1.44269504088896341f;
    p.status = b200mx::device_status_word();
    if (p.status == nullptr) return -static_cast<int>(cudaErrorInvalidSymbol);
    return done(a->S == 0u ? b200mx::launch_kv4_weigh(p, static_cast<cudaStream_t>(stream)) : b200mx::launch_kv4_attend(p, static_cast<cudaStream_t>(stream)), err, cap);
}

int fmha_kv4_evict(const fmha_kv4_cache* cache, const fmha_kv4_cache* into, const fmha_kv4_evict_args* a, void* stream, char* err, size_t cap) {
    b200mx::Kv4EvictParams p = {};
    if (a == nullptr) return refuse(err, cap, "evict: no arguments");
    if (int r = view_of(cache, "evict", p.from, err, cap)) return r;
    if (int r = view_of(into, "evict: into", p.into, err, cap)) return r;
    if (p.from.B != p.into.B || p.from.HK != p.into.HK || p.from.page_log2 != p.into.page_log2) return refuse(err, cap, "evict: into must have the cache's sequences, heads and page size");
    if (p.from.lengths == p.into.lengths || p.from.table == p.into.table) return refuse(err, cap, "evict: into needs a table and lengths of its own");
    if (a->weights == nullptr || a->kept == nullptr) return refuse(err, cap, "evict: weights and kept must be given");
    const uint64_t tokens = static_cast<uint64_t>(p.from.table_width) << p.from.page_log2, room = static_cast<uint64_t>(p.into.table_width) << p.into.page_log2;
    if (a->weights_width < tokens) return refuse(err, cap, "evict: weights must cover the %llu tokens of the table", static_cast<unsigned long long>(tokens));
    if (a->keep == 0u || a->keep > room) return refuse(err, cap, "evict: keep must be 1 to the %llu tokens that into has room for", static_cast<unsigned long long>(room));
    if (static_cast<uint64_t>(a->recent) + a->first > a->keep) return refuse(err, cap, "evict: first + recent must not exceed keep");
    if (a->weights_out != nullptr && a->weights_out_width < a->keep) return refuse(err, cap, "evict: weights_out must have room for keep tokens");
    const uint64_t heads = static_cast<uint64_t>(p.from.B) * p.from.HK;
    if (a->weights_out != nullptr && overlap(a->weights, 4u * heads * a->weights_width, a->weights_out, 4u * heads * a->weights_out_width))
        return refuse(err, cap, "evict: weights_out must not share memory with weights");
    p.weights = a->weights, p.kept = a->kept, p.weights_out = a->weights_out;
    p.weights_width = a->weights_width, p.weights_out_width = a->weights_out_width;
    p.keep = a->keep, p.recent = a->recent, p.first = a->first;
    return done(b200mx::launch_kv4_evict(p, static_cast<cudaStream_t>(stream)), err, cap);
}

}  // extern "C"
