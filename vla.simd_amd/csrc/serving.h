// serving.h - the operators of a decoder that serves several prompts: their
// launchers, and the device helpers that their kernels share. Values are
// fp32, bf16 or fp16 (vla_dtype); every sum and statistic is held in fp32 or more (angles, and the
// norm's squares where they leave fp32's range, in 64 bits), and a result is rounded to its type once.
#pragma once

#include "common.h"

namespace vla {
namespace hip {

// vla_dtype (include/vla_simd_hip.h)
enum : int { kF32 = 0, kBf16 = 1, kF16 = 2 };
inline int dtype_size(int dtype) { return dtype == kF32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == kF32 || dtype == kBf16 || dtype == kF16; }

constexpr int kMaxAxes = 8;

// rope_heads.hip
struct RopeHeadsArgs {
    void* q_out; int64_t ldqo;
    void* k_out; int64_t ldko;
    const void* q; int64_t ldq;
    const void* k; int64_t ldk;
    const float* wq;     // [head_dim] or null: no norm
    const float* wk;
    float eps;
    const int32_t* pos;  // [n_axes] rows of ld_pos
    int64_t ld_pos;
    int ends[kMaxAxes];  // first pair behind each axis' section, host values
    int n_axes;
    double log2_base;
    int seq, n_q, n_kv, head_dim, dtype;
    int tokens_per_block;  // set by the launcher
};
void launch_qk_norm_rope(RopeHeadsArgs a, hipStream_t st);

// packed_attn.hip
struct PackedAttnArgs {
    void* out; int64_t ldo;
    const void* Q; int64_t ldq;
    const void* K; int64_t ldk;
    const void* V; int64_t ldv;
    const int32_t* q_start;  // [n_seqs + 1]
    const int32_t* k_start;  // [n_seqs + 1]
    int n_seqs, total_q, total_k, n_q, n_kv, head_dim;
    float scale;
    int causal, dtype;
    float lift;  // set by the launcher
};
void launch_packed_attention(PackedAttnArgs a, hipStream_t st);

// kv4.hip: the paged cache of 4-bit values (layout in kv4.h)
struct Kv4Args {
    uint8_t* cache;
    int n_pages, page_size, n_kv, head_dim;
    const int32_t* table;  // [n_seqs] rows of ld_table
    int ld_table;
    const int32_t* lens;   // [n_seqs] tokens cached, the new ones included
    const int32_t* start;  // [n_seqs + 1] first packed row of each sequence; null: one row each
    const int32_t* first;  // gather: [n_seqs] first token, null: 0
    int n_seqs, total;     // packed rows
    void* K; int64_t ldk;
    void* V; int64_t ldv;
    int dtype;
    // attention only
    void* out; int64_t ldo;
    const void* Q; int64_t ldq;
    int n_q, max_new, max_len;
    float scale;
    float* work;
    size_t work_bytes;
};
void launch_kv4_append(const Kv4Args& a, hipStream_t st);
void launch_kv4_gather(const Kv4Args& a, hipStream_t st);
void launch_kv4_attention(const Kv4Args& a, hipStream_t st);
size_t kv4_attention_work_bytes(int total_q, int n_seqs, int max_new, int max_len, int n_q, int n_kv, int head_dim);

// kv4_tree.hip: the attention of drafted tokens (Kv4Args as for launch_kv4_attention)
struct Kv4TreeArgs {
    Kv4Args kv;
    const uint32_t* see;  // [total] rows of ld_see words: bit t of a row's words, it sees new token t
    int ld_see;
};
void launch_kv4_tree_attention(const Kv4TreeArgs& a, hipStream_t st);
size_t kv4_tree_attention_work_bytes(int total_q, int n_seqs, int max_new, int max_len, int n_q, int n_kv, int head_dim);

// rope_append.hip: norms and rotation of packed rows, keys and values into the cache
struct RopeAppendArgs {
    Kv4Args kv;          // K, V: the rows; cache null: only rotated
    const void* q; int64_t ldq;
    void* q_out; int64_t ldqo;
    void* k_out; int64_t ldko;  // null: not wanted
    const float* wq;     // [head_dim] or null: no norm
    const float* wk;
    float eps;
    const int32_t* pos;  // [total] or null: a token's number in its sequence
    const double* freqs; // [rot / 2] angles per position
    int rot;             // values of a head that turn
    double magnitude;
    int interleaved;
    int n_q;
    int tokens_per_block;  // set by the launcher
};
void launch_rope_kv4_append(RopeAppendArgs a, hipStream_t st);

// draft.hip
struct DraftTreeArgs {
    int32_t* pos;        // [total]
    uint32_t* see;       // [total] rows of ld_see words
    int ld_see;
    const int32_t* parent;  // [total], in its sequence; null: the row before
    const int32_t* lens;
    const int32_t* start;
    int n_seqs, total;
};
void launch_draft_tree(const DraftTreeArgs& a, hipStream_t st);

struct VerifyArgs {
    int32_t* path;       // [total]
    int32_t* count;      // [n_seqs]
    int32_t* token;      // [n_seqs]
    const void* p; int64_t ldp;
    const void* q; int64_t ldq;  // null: drafted with certainty
    const int32_t* tokens;  // [total]
    const int32_t* parent;  // [total], in its sequence; null: the row before
    const int32_t* start;
    const float* u;      // [total]
    const float* u_next; // [n_seqs]
    int n_seqs, total, vocab, dtype;
};
void launch_verify_drafts(const VerifyArgs& a, hipStream_t st);

struct Kv4KeepArgs {
    Kv4Args kv;
    const int32_t* path;   // [total]
    const int32_t* count;  // [n_seqs]
    int32_t* new_lens;     // [n_seqs] or null
};
void launch_kv4_keep(const Kv4KeepArgs& a, hipStream_t st);

#ifdef __HIPCC__

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// N values of 16 or fewer bytes, loaded and stored as one access
template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16_t x) { return (float)x; }
__device__ __forceinline__ float to_f32(f16_t x) { return (float)x; }

// The sequence of packed row `row`: the last s with start[s] <= row among
// starts clamped to [0, total], or n_seqs when the row lies behind them all.
// `start` may be LDS or global memory.
__device__ __forceinline__ int seq_of_row(const int32_t* start, int n_seqs, int row) {
    int lo = 0, hi = n_seqs;  // the first s in (lo, hi] with start[s] > row
    if (start[n_seqs] <= row) return n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

#endif

}  // namespace hip
}  // namespace vla
