// capi_serving.cpp - the C ABI of the operators that serve several prompts
// (include/vla_simd_hip.h, "decoders with several sequences"): device forms only,
// which validate on the host and launch on the caller's stream.

#include "vla_simd_hip.h"

#include "kv4.h"
#include "runtime.h"
#include "serving.h"

#include <cmath>

using namespace vla::hip;

namespace {

hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

Kv4Args cache_args(void* cache, int32_t n_pages, int32_t page_size, const int32_t* table, int32_t ld_table, int32_t n_seqs,
                   int32_t n_kv, int32_t head_dim, int32_t dtype) {
    Kv4Args a{};
    a.cache = static_cast<uint8_t*>(cache);
    a.n_pages = n_pages;
    a.page_size = page_size;
    a.table = table;
    a.ld_table = ld_table;
    a.n_seqs = n_seqs;
    a.n_kv = n_kv;
    a.head_dim = head_dim;
    a.dtype = dtype;
    return a;
}

bool page_shape_ok(int32_t n_kv, int32_t head_dim, int32_t page_size) {
    return n_kv > 0 && n_kv <= 1024 && kv4_head_dim_ok(head_dim) && page_size > 0 && page_size % 32 == 0 && page_size <= kKv4MaxPage;
}

}  // namespace

extern "C" {

VLA_API int32_t vla_qk_norm_rope_dev(void* q_out, int64_t ldqo, void* k_out, int64_t ldko, const void* q, int64_t ldq,
                                     const void* k, int64_t ldk, const float* q_weight, const float* k_weight, float eps,
                                     const int32_t* pos, int64_t ld_pos, const int32_t* sections, int32_t n_axes, float base,
                                     int32_t seq, int32_t n_q, int32_t n_kv, int32_t head_dim, int32_t dtype, void* stream) {
    return guarded("vla_qk_norm_rope_dev", [&] {
        RopeHeadsArgs a{};
        a.q_out = q_out;
        a.ldqo = ldqo;
        a.k_out = k_out;
        a.ldko = ldko;
        a.q = q;
        a.ldq = ldq;
        a.k = k;
        a.ldk = ldk;
        a.wq = q_weight;
        a.wk = k_weight;
        a.eps = eps;
        a.pos = pos;
        a.ld_pos = ld_pos;
        a.n_axes = n_axes;
        VLA_REQUIRE(n_axes >= 1 && n_axes <= kMaxAxes && sections, "1 to 8 axes, a section each");
        int64_t end = 0;
        for (int i = 0; i < n_axes; i++) {
            VLA_REQUIRE(sections[i] >= 0 && sections[i] <= 256, "a section holds 0 to head_dim / 2 pairs");
            end += sections[i];
            a.ends[i] = (int)end;
        }
        VLA_REQUIRE(base > 0.0f && std::isfinite(base), "base must be positive");
        a.log2_base = std::log2((double)base);
        a.seq = seq;
        a.n_q = n_q;
        a.n_kv = n_kv;
        a.head_dim = head_dim;
        a.dtype = dtype;
        launch_qk_norm_rope(a, as_stream(stream));
    });
}

VLA_API int32_t vla_packed_attention_dev(void* out, int64_t ldo, const void* Q, int64_t ldq, const void* K, int64_t ldk,
                                         const void* V, int64_t ldv, const int32_t* q_start, const int32_t* k_start,
                                         int32_t n_seqs, int32_t total_q, int32_t total_k, int32_t n_q, int32_t n_kv,
                                         int32_t head_dim, float scale, int32_t causal, int32_t dtype, void* stream) {
    return guarded("vla_packed_attention_dev", [&] {
        PackedAttnArgs a{};
        a.out = out;
        a.ldo = ldo;
        a.Q = Q;
        a.ldq = ldq;
        a.K = K;
        a.ldk = ldk;
        a.V = V;
        a.ldv = ldv;
        a.q_start = q_start;
        a.k_start = k_start ? k_start : q_start;
        a.n_seqs = n_seqs;
        a.total_q = total_q;
        a.total_k = total_k;
        a.n_q = n_q;
        a.n_kv = n_kv;
        a.head_dim = head_dim;
        a.scale = scale;
        a.causal = causal != 0;
        a.dtype = dtype;
        launch_packed_attention(a, as_stream(stream));
    });
}

VLA_API int64_t vla_kv4_page_bytes(int32_t n_kv, int32_t head_dim, int32_t page_size) {
    return page_shape_ok(n_kv, head_dim, page_size) ? (int64_t)kv4_page_bytes(n_kv, head_dim, page_size) : -1;
}

VLA_API int64_t vla_kv4_offset(int32_t n_kv, int32_t head_dim, int32_t page_size, int32_t n_pages, const int32_t* table_row,
                               int32_t ld_table, int64_t token, int32_t part, int32_t head, int32_t block) {
    if (!page_shape_ok(n_kv, head_dim, page_size) || !table_row || token < 0 || part < 0 || part > 3 || head < 0 || head >= n_kv ||
        block < 0 || block >= head_dim / kKv4Block)
        return -1;
    const int page = kv4_page(table_row, ld_table, n_pages, token / page_size);
    if (page < 0) return -1;
    const int64_t slot = token % page_size;
    const int64_t nc = (int64_t)kv4_code_bytes(n_kv, head_dim, page_size), ns = (int64_t)kv4_scale_bytes(n_kv, head_dim, page_size);
    const int64_t base = (int64_t)page * 2 * (nc + ns);
    if (part < 2) return base + part * nc + ((int64_t)head * page_size + slot) * (head_dim / 2) + block * (kKv4Block / 2);
    return base + 2 * nc + (part - 2) * ns + ((int64_t)head * (head_dim / kKv4Block) + block) * page_size + slot;
}

VLA_API int32_t vla_kv4_append_dev(void* cache, int32_t n_pages, int32_t page_size, const void* K, int64_t ldk, const void* V,
                                   int64_t ldv, const int32_t* table, int32_t ld_table, const int32_t* lens, const int32_t* start,
                                   int32_t n_seqs, int32_t total, int32_t n_kv, int32_t head_dim, int32_t dtype, void* stream) {
    return guarded("vla_kv4_append_dev", [&] {
        Kv4Args a = cache_args(cache, n_pages, page_size, table, ld_table, n_seqs, n_kv, head_dim, dtype);
        a.K = const_cast<void*>(K);
        a.ldk = ldk;
        a.V = const_cast<void*>(V);
        a.ldv = ldv;
        a.lens = lens;
        a.start = start;
        a.total = total;
        launch_kv4_append(a, as_stream(stream));
    });
}

VLA_API int32_t vla_kv4_gather_dev(void* K, int64_t ldk, void* V, int64_t ldv, const void* cache, int32_t n_pages, int32_t page_size,
                                   const int32_t* table, int32_t ld_table, const int32_t* start, const int32_t* first, int32_t n_seqs,
                                   int32_t total, int32_t n_kv, int32_t head_dim, int32_t dtype, void* stream) {
    return guarded("vla_kv4_gather_dev", [&] {
        Kv4Args a = cache_args(const_cast<void*>(cache), n_pages, page_size, table, ld_table, n_seqs, n_kv, head_dim, dtype);
        a.K = K;
        a.ldk = ldk;
        a.V = V;
        a.ldv = ldv;
        a.start = start;
        a.first = first;
        a.total = total;
        launch_kv4_gather(a, as_stream(stream));
    });
}

VLA_API int64_t vla_kv4_attention_work_bytes(int32_t total_q, int32_t n_seqs, int32_t max_new, int32_t max_len, int32_t n_q,
                                             int32_t n_kv, int32_t head_dim) {
    return (int64_t)kv4_attention_work_bytes(total_q, n_seqs, max_new, max_len, n_q, n_kv, head_dim);
}

VLA_API int32_t vla_kv4_attention_dev(void* out, int64_t ldo, const void* Q, int64_t ldq, const void* cache, int32_t n_pages,
                                      int32_t page_size, const int32_t* table, int32_t ld_table, const int32_t* lens,
                                      const int32_t* q_start, int32_t n_seqs, int32_t total_q, int32_t max_new, int32_t max_len,
                                      int32_t n_q, int32_t n_kv, int32_t head_dim, float scale, int32_t dtype, void* work,
                                      int64_t work_bytes, void* stream) {
    return guarded("vla_kv4_attention_dev", [&] {
        Kv4Args a = cache_args(const_cast<void*>(cache), n_pages, page_size, table, ld_table, n_seqs, n_kv, head_dim, dtype);
        a.lens = lens;
        a.start = q_start;
        a.total = total_q;
        a.out = out;
        a.ldo = ldo;
        a.Q = Q;
        a.ldq = ldq;
        a.n_q = n_q;
        a.max_new = max_new;
        a.max_len = max_len;
        a.scale = scale;
        a.work = static_cast<float*>(work);
        a.work_bytes = work_bytes > 0 ? (size_t)work_bytes : 0;
        launch_kv4_attention(a, as_stream(stream));
    });
}

VLA_API int32_t vla_draft_tree_dev(int32_t* pos, uint32_t* see, int32_t ld_see, const int32_t* parent, const int32_t* lens,
                                   const int32_t* start, int32_t n_seqs, int32_t total, void* stream) {
    return guarded("vla_draft_tree_dev", [&] {
        DraftTreeArgs a{};
        a.pos = pos;
        a.see = see;
        a.ld_see = ld_see;
        a.parent = parent;
        a.lens = lens;
        a.start = start;
        a.n_seqs = n_seqs;
        a.total = total;
        launch_draft_tree(a, as_stream(stream));
    });
}

VLA_API int32_t vla_rope_freqs(double* freqs, double* magnitude, int32_t rot_dim, double base, int32_t scaling, double factor,
                               double trained, double low, double high) {
    return guarded("vla_rope_freqs", [&] {
        VLA_REQUIRE(freqs && rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= 1 << 20, "rope_freqs: rot_dim must be even, from 2 to 2^20");
        VLA_REQUIRE(base > 0.0 && std::isfinite(base), "rope_freqs: base must be positive");
        VLA_REQUIRE(scaling >= VLA_ROPE_PLAIN && scaling <= VLA_ROPE_PARTS, "rope_freqs: unknown scaling");
        VLA_REQUIRE(scaling == VLA_ROPE_PLAIN || (factor >= 1.0 && std::isfinite(factor)), "rope_freqs: factor must be at least 1");
        VLA_REQUIRE(scaling != VLA_ROPE_BASE || rot_dim > 2, "rope_freqs: a scaled base needs more than one pair");
        VLA_REQUIRE(scaling != VLA_ROPE_PARTS || (trained > 0.0 && std::isfinite(trained) && low >= 0.0 && high > low && std::isfinite(high)),
                    "rope_freqs: parts need a trained length and 0 <= low < high");
        const double b = scaling == VLA_ROPE_BASE ? base * std::pow(factor, (double)rot_dim / (rot_dim - 2)) : base;
        for (int i = 0; i < rot_dim / 2; i++) {
            double f = std::pow(b, -2.0 * i / rot_dim);
            if (scaling == VLA_ROPE_LINEAR) f /= factor;
            if (scaling == VLA_ROPE_PARTS) {
                const double turns = trained * f / (2.0 * M_PI), ramp = (turns - low) / (high - low);
                const double keep = ramp < 0.0 ? 0.0 : ramp > 1.0 ? 1.0 : ramp;
                f = f / factor + (f - f / factor) * keep;
            }
            freqs[i] = f;
        }
        if (magnitude) *magnitude = scaling == VLA_ROPE_PARTS ? 0.1 * std::log(factor) + 1.0 : 1.0;
    });
}

VLA_API int32_t vla_rope_kv4_append_dev(void* q_out, int64_t ldqo, void* k_out, int64_t ldko, void* cache, int32_t n_pages,
                                        int32_t page_size, const void* q, int64_t ldq, const void* K, int64_t ldk, const void* V,
                                        int64_t ldv, const float* q_weight, const float* k_weight, float eps, const int32_t* pos,
                                        const double* freqs, int32_t rot_dim, double magnitude, int32_t interleaved,
                                        const int32_t* table, int32_t ld_table, const int32_t* lens, const int32_t* start,
                                        int32_t n_seqs, int32_t total, int32_t n_q, int32_t n_kv, int32_t head_dim, int32_t dtype,
                                        void* stream) {
    return guarded("vla_rope_kv4_append_dev", [&] {
        RopeAppendArgs a{};
        // without a cache no token has a page
        a.kv = cache_args(cache, cache ? n_pages : 0, cache ? page_size : kKv4Block, cache ? table : nullptr, cache ? ld_table : 0, n_seqs,
                          n_kv, head_dim, dtype);
        a.kv.K = const_cast<void*>(K);
        a.kv.ldk = ldk;
        a.kv.V = const_cast<void*>(V);
        a.kv.ldv = ldv;
        a.kv.lens = lens;
        a.kv.start = start;
        a.kv.total = total;
        a.q = q;
        a.ldq = ldq;
        a.q_out = q_out;
        a.ldqo = ldqo;
        a.k_out = k_out;
        a.ldko = ldko;
        a.wq = q_weight;
        a.wk = k_weight;
        a.eps = eps;
        a.pos = pos;
        a.freqs = freqs;
        a.rot = rot_dim;
        a.magnitude = magnitude;
        a.interleaved = interleaved != 0;
        a.n_q = n_q;
        launch_rope_kv4_append(a, as_stream(stream));
    });
}

VLA_API int64_t vla_kv4_tree_attention_work_bytes(int32_t total_q, int32_t n_seqs, int32_t max_new, int32_t max_len, int32_t n_q,
                                                  int32_t n_kv, int32_t head_dim) {
    return (int64_t)kv4_tree_attention_work_bytes(total_q, n_seqs, max_new, max_len, n_q, n_kv, head_dim);
}

VLA_API int32_t vla_kv4_tree_attention_dev(void* out, int64_t ldo, const void* Q, int64_t ldq, const void* cache, int32_t n_pages,
                                           int32_t page_size, const int32_t* table, int32_t ld_table, const int32_t* lens,
                                           const int32_t* q_start, const uint32_t* see, int32_t ld_see, int32_t n_seqs,
                                           int32_t total_q, int32_t max_new, int32_t max_len, int32_t n_q, int32_t n_kv,
                                           int32_t head_dim, float scale, int32_t dtype, void* work, int64_t work_bytes,
                                           void* stream) {
    return guarded("vla_kv4_tree_attention_dev", [&] {
        Kv4TreeArgs t{};
        Kv4Args& a = t.kv;
        a = cache_args(const_cast<void*>(cache), n_pages, page_size, table, ld_table, n_seqs, n_kv, head_dim, dtype);
        a.lens = lens;
        a.start = q_start;
        a.total = total_q;
        a.out = out;
        a.ldo = ldo;
        a.Q = Q;
        a.ldq = ldq;
        a.n_q = n_q;
        a.max_new = max_new;
        a.max_len = max_len;
        a.scale = scale;
        a.work = static_cast<float*>(work);
        a.work_bytes = work_bytes > 0 ? (size_t)work_bytes : 0;
        t.see = see;
        t.ld_see = ld_see;
        launch_kv4_tree_attention(t, as_stream(stream));
    });
}

VLA_API int32_t vla_verify_drafts_dev(int32_t* path, int32_t* count, int32_t* token, const void* p, int64_t ldp, const void* q,
                                      int64_t ldq, const int32_t* tokens, const int32_t* parent, const int32_t* start, const float* u,
                                      const float* u_next, int32_t n_seqs, int32_t total, int32_t vocab, int32_t dtype, void* stream) {
    return guarded("vla_verify_drafts_dev", [&] {
        VerifyArgs a{};
        a.path = path;
        a.count = count;
        a.token = token;
        a.p = p;
        a.ldp = ldp;
        a.q = q;
        a.ldq = ldq;
        a.tokens = tokens;
        a.parent = parent;
        a.start = start;
        a.u = u;
        a.u_next = u_next;
        a.n_seqs = n_seqs;
        a.total = total;
        a.vocab = vocab;
        a.dtype = dtype;
        launch_verify_drafts(a, as_stream(stream));
    });
}

VLA_API int32_t vla_kv4_keep_dev(void* cache, int32_t n_pages, int32_t page_size, const int32_t* table, int32_t ld_table,
                                 const int32_t* lens, const int32_t* start, const int32_t* path, const int32_t* count,
                                 int32_t* new_lens, int32_t n_seqs, int32_t total, int32_t n_kv, int32_t head_dim, void* stream) {
    return guarded("vla_kv4_keep_dev", [&] {
        Kv4KeepArgs a{};
        a.kv = cache_args(cache, n_pages, page_size, table, ld_table, n_seqs, n_kv, head_dim, kF32);
        a.kv.lens = lens;
        a.kv.start = start;
        a.kv.total = total;
        a.path = path;
        a.count = count;
        a.new_lens = new_lens;
        launch_kv4_keep(a, as_stream(stream));
    });
}

}  // extern "C"
