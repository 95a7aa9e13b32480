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

}  // extern "C"
