// packed_attn.hip - attention over packed sequences of different lengths:
//   out[i] = sum_j softmax_j(scale * q[i] . k[j]) v[j]
// over the keys j of the query's own sequence that it sees: all of them, or with
// `causal` those with j <= i + (len_k - len_q), so that the last query sees the last
// key. A query that sees no key gets zeros; a key that it does not see
// counts for nothing, whatever it holds (infinities and NaN included).
//
// One pass over the keys with the running maximum m and sum l of the softmax; the
// weights stay in registers. Both products run on the matrix cores with fp32 sums:
//   S^T = K Q^T  (A: 32 keys, B: 32 queries) leaves in lane n + 32 h, for query n, the
//                scores of keys 8 (i / 4) + 4 h + i % 4, i = 0..15;
//   O^T = V^T P^T takes of that lane 8 weights per 16 keys: with the product's
//                inner index 8 h + j read as key 4 h + j (j < 4) and 8 + 4 h + j - 4, those
//                are the ones it holds, so no weight moves between lanes.
//                V^T's operand, 4 keys of one dim per half, is what a
//                transposed LDS read (ds_read_b64_tr_b16) of row-major V gives.
//
// 16-bit types: the weights are rounded to the operands' type for the second product
// (bf16: each by 2^-8 of itself at most; fp16: by 2^-11 of itself or 2^-34 of the row's largest,
// whichever is more); the sum l is of the unrounded ones. fp16 has few bits below 2^-14, and next to a key
// that takes nearly all, what is left of the output may be just the small weights: they are all taken 2^9
// times as large (lift, below).
// fp32 up to 128 columns: both products from three bf16 parts of each operand, as exact as
// fp32 products; past that on the fp32 matrix cores.
//
// The matrix cores bound long prompts with heads of 128: one causal prompt of 8192, 32 heads on 8, bf16,
// 516 us, 1065 TFLOP/s of the 1156 that a large library product reaches; 12 mixed up to 2048
// 210 us, 727 (beginnings and ends of blocks that see few keys). With heads of 64 the exponentials
// take as long as both products (a wave's 64 keys: 512 cycles each, 400 more of other vector
// work): 8 sequences of 1024 without a mask, 12 heads, fp16, 39.8 us, 650 TFLOP/s. Short calls are bound by latency: 32
// heads over 64 tokens 8.3 us.

#include "serving.h"
#include "wave.h"

#include <cmath>

namespace vla {
namespace hip {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef bf16_t v8bf __attribute__((ext_vector_type(8)));
typedef f16_t v8h __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;

template <class T>
struct Vec8;
template <>
struct Vec8<bf16_t> { typedef v8bf type; };
template <>
struct Vec8<f16_t> { typedef v8h type; };

__device__ __forceinline__ v16f mfma32(v8bf a, v8bf b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v16f mfma32(v8h a, v8h b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// max / sum of x over the lanes l and l ^ 32
__device__ __forceinline__ float halves_max(float x) {
    const unsigned u = __float_as_uint(x);
    const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
    const unsigned u = __float_as_uint(x);
    const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Sums of weights times values are divided at the end only, and must be in range before. The reference m of
// the weights follows the row's maximum when that has grown by 2^6, so weights reach 2^6 and a sum over n
// keys 2^6 n times the largest value.
// 16-bit types: weights are exp2(score - m + lift), which cancels in o / l. fp16: 9, for the small weights' sake;
// sums have room enough. bf16: -(6 + log2 n), so that no values overflow; the sum m - lift is rounded to 2^-19 or so
// of a weight, of which 8 bits are kept. What vanishes for it are weights below 2^-100 of the largest.
// fp32: such a rounding would show. A block whose values reach 2^90 (2^28 keys of them still add up) takes them and its
// sums 2^-34 as large from there on, exactly; others keep their small values. (All weights times a factor of
// one or 2^-34: 2% slower.) Past 128 columns the weights are 2^lift as large in the product, exactly (the same check of
// the values there: 7% slower).
float lift_of(const PackedAttnArgs& a) {
    if (a.dtype == kF16) return 9.0f;
    int log2_n = 0;
    while ((int64_t)1 << log2_n < a.total_k) log2_n++;
    return -(6.0f + (float)log2_n);
}
constexpr unsigned kLargeBits = 0x6c800000u;  // 2^90
constexpr float kLargeScale = 0x1p-34f;

// What a block works on: query rows [q0, q0 + nq) of the packed buffers, at
// offset `at` in their sequence, and its keys [k0, k0 + nk).
struct Job {
    int q0, nq, at, len_q, k0, nk;
};

__device__ __forceinline__ int clamp_row(int x, int total) { return x < 0 ? 0 : (x < total ? x : total); }

// The block's tile number -> its job; false for a number without a tile. Up to 64 sequences: tiles are
// counted, a sequence to a lane. More: sequence s has the numbers from q_start[s] / QT + s on, of
// which the next sequence's leave it at least as many as it has tiles, so that there is no sum over
// the sequences, only a search among increasing numbers, 64 at a time. (For few sequences the
// numbers without a tile cost more than the sum, as their blocks hold places when others are
// dealt: 8 sequences of 177, 15 heads of 64, 9.9 us for 8.8. For many the sum
// grows with their number in every block: 70 of 100 tokens, 32 heads of 128, 63.7 us for 59.5, 1000 of 30
// 1118 for 432, 8000 of 16 42.5 ms for 3.4.)
// Numbers run backwards, as queries late in a sequence see the most keys under a causal mask.
// (Counted by their depth over all sequences, the deepest first, 12 mixed prompts took 224 us for
// 212: neighbours no longer share keys.) Starts are read clamped to the buffers' rows, and a
// sequence that would end before it begins is empty, so that no offsets can lead out of the buffers.
// Every wave does the same search.
template <int QT>
__device__ __forceinline__ bool find_job(const PackedAttnArgs& a, int tile, Job& job) {
    const int lane = threadIdx.x & 63;
    int want = (int)(gridDim.x / a.n_q) - 1 - tile;
    int lo = 0, count = a.n_seqs;  // the sequence is one of [lo, lo + count)
    while (count > 64) {
        const int step = (count + 63) / 64, s = lo + lane * step;
        const bool in = lane * step < count && clamp_row(a.q_start[s], a.total_q) / QT + s <= want;
        const int k = __popcll(__ballot(in));
        const int first = lo + (k ? k - 1 : 0) * step;
        count = count - (first - lo) < step ? count - (first - lo) : step;
        lo = first;
    }
    const int s = lo + lane;
    int q0 = 0, n = 0, k0 = 0, nk = 0;  // of the lane's sequence
    if (lane < count) {
        q0 = clamp_row(a.q_start[s], a.total_q);
        n = clamp_row(a.q_start[s + 1], a.total_q) - q0;
        k0 = clamp_row(a.k_start[s], a.total_k);
        nk = clamp_row(a.k_start[s + 1], a.total_k) - k0;
    }
    int number = q0 / QT + s;  // of its first tile
    if (a.n_seqs <= 64) {
        const int tiles = n > 0 ? (n + QT - 1) / QT : 0;
        int incl = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d);
            if (lane >= d) incl += o;
        }
        number = incl - tiles;
        want = __builtin_amdgcn_readlane(incl, 63) - 1 - tile;
    }
    const int found = __popcll(__ballot(lane < count && number <= want));
    if (!found) return false;
    // the same in every lane: kept in scalar registers
    const int l = __builtin_amdgcn_readfirstlane(found - 1);
    const int start = __builtin_amdgcn_readlane(q0, l);
    job.len_q = __builtin_amdgcn_readlane(n, l);
    const int64_t at = (int64_t)(want - __builtin_amdgcn_readlane(number, l)) * QT;
    if (at < 0 || at >= job.len_q) return false;  // (below 0: starts out of order)
    job.at = (int)at;
    job.q0 = start + job.at;
    job.nq = job.len_q - job.at < QT ? job.len_q - job.at : QT;
    job.k0 = __builtin_amdgcn_readlane(k0, l);
    job.nk = __builtin_amdgcn_readlane(nk, l);
    if (job.nk < 0) job.nk = 0;
    return true;
}

// Blocks of one kv head share its rows, so where the heads divide over the 8
// XCDs (the hardware deals block i to XCD i % 8) each XCD's L2 gets heads of its own.
__device__ __forceinline__ void tile_and_head(const PackedAttnArgs& a, int& tile, int& h) {
    const int b = blockIdx.x;
    tile = b / a.n_q;
    const int r = b - tile * a.n_q;
    h = a.n_q % 8 == 0 ? (r & 7) * (a.n_q >> 3) + (r >> 3) : r;
}

// ---------------------------------------------------- 16-bit types ----

// waits for this wave's loads, those into LDS among them (vmcnt 0 alone)
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// LDS rows of HDP values in 16-byte chunks; chunk c of row r lies at c ^ swz(r).
// 16 rows' reads of one chunk (K) then fall on all 64 banks, and so do the 64-byte
// pieces of 4 neighbouring rows that a transposed read takes (V).
template <int HDP>
__device__ __forceinline__ int swz(int row) {
    return (HDP == 64 ? (row >> 1 & 1) << 2 : (row & 3) << 2) | (row >> 2 & 3);
}

// Rows in global memory from `first` on, `bytes` of them, read 16 bytes a lane straight into
// LDS at lds + 16 * lane, or into registers. Reads from `bytes` on (checked by the hardware)
// give zeros, writes there do nothing.
struct Rows {
    __amdgpu_buffer_rsrc_t rs;
    __device__ __forceinline__ Rows(const void* first, int64_t bytes)
        : rs(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(first), 0, bytes < 0x7fffffff ? (int)bytes : 0x7fffffff, 0x27000)) {}
    __device__ __forceinline__ void to_lds(void* lds, unsigned offset) const {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds, 16, offset, 0, 0, 0);
    }
    template <class V>
    __device__ __forceinline__ V load16(unsigned offset) const {
        return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(rs, offset, 0, 0));
    }
    template <class V>
    __device__ __forceinline__ void store8(V v, unsigned offset) const {
        typedef unsigned v2u __attribute__((ext_vector_type(2)));
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(v2u, v), rs, offset, 0, 0);
    }
    template <class V>
    __device__ __forceinline__ void store16(V v, unsigned offset) const {
        typedef unsigned v4u __attribute__((ext_vector_type(4)));
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, v), rs, offset, 0, 0);
    }
};
constexpr unsigned kNoRow = 0x80000000u;  // an offset behind every row

// HC: columns worked on, head_dim rounded up (zeros behind it); HDP: those of an LDS row, a
// power of two. QW: waves of 32 queries each. SPLIT 2: as many waves again take every other tile
// of keys for the same queries, joined at the end.
template <class T, int HDP, int HC, int KT, int SPLIT, int QW>
__global__ __launch_bounds__(64 * QW * SPLIT, HDP == 64 || HDP == 128 && QW == 4 ? 2 : 1) void packed_attn_16(PackedAttnArgs a) {
    typedef typename Vec8<T>::type v8;
    constexpr int QT = 32 * QW, NK = KT / 32;
    constexpr int NTH = 64 * QW;            // threads that share a tile of keys
    constexpr int CH = HDP / 8;             // chunks of a row
    constexpr int LOADS = KT * CH / NTH;    // chunks per thread of a K or V tile
    constexpr int DT = HC / 32, KS = HC / 16;
    constexpr int TILE = KT * HDP;
    constexpr unsigned kExp = __is_same(T, bf16_t) ? 0x7f80u : 0x7c00u;  // exponent bits: all set where not finite
    __shared__ __attribute__((aligned(16))) T K0[SPLIT * TILE], K1[SPLIT * TILE], V0[SPLIT * TILE], V1[SPLIT * TILE];

    int tile, head;
    tile_and_head(a, tile, head);
    Job job;
    if (!find_job<QT>(a, tile, job)) return;

    const int tid = threadIdx.x % NTH, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int part = SPLIT == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / NTH);
    const int n = lane & 31, hf = lane >> 5;
    const int hd = a.head_dim;
    const int kvh = __builtin_amdgcn_readfirstlane(head / (a.n_q / a.n_kv));
    const T* Kg = static_cast<const T*>(a.K) + (size_t)job.k0 * a.ldk + kvh * hd;
    const T* Vg = static_cast<const T*>(a.V) + (size_t)job.k0 * a.ldv + kvh * hd;

    const int qi = wave * 32 + n;  // in the tile
    const bool qok = qi < job.nq;
    // the sign goes to the queries, so that larger products are larger scores; 0 becomes the
    // smallest factor, which leaves scores at 0 and masked ones at -inf
    const float c2 = a.scale == 0.0f ? 1.17549435e-38f : fabsf(a.scale) * kLog2e;
    const Rows qrows(static_cast<const T*>(a.Q) + (size_t)job.q0 * a.ldq + head * hd, (int64_t)job.nq * a.ldq * (int)sizeof(T));
    v8 qv[KS];
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const int d = 16 * s + 8 * hf;
        qv[s] = qrows.load16<v8>(qok && d < hd ? (unsigned)(qi * (int)a.ldq + d) * (int)sizeof(T) : kNoRow);
        if (a.scale < 0.0f) qv[s] = -qv[s];
    }
    // keys [0, lim) are seen by the lane's query, [0, wave_all) by all of the wave's,
    // [wave_end, ..) by none of them
    const int off = job.nk - job.len_q + job.at + 1;
    auto limit = [&](int q) {
        const int e = a.causal ? q + off : job.nk;
        return e < 0 ? 0 : (e < job.nk ? e : job.nk);
    };
    const int lim = qok ? limit(qi) : 0;
    const int wq_last = wave * 32 + 31 < job.nq ? wave * 32 + 31 : job.nq - 1;
    const int wave_end = wave * 32 < job.nq ? limit(wq_last) : 0;
    const int wave_all = wave * 32 < job.nq ? limit(wave * 32) : 0;
    const int end = limit(job.nq - 1);
    // a turn is SPLIT tiles; turns [0, plain) are seen whole by every query
    const int turns = (end + SPLIT * KT - 1) / (SPLIT * KT), plain = limit(0) / (SPLIT * KT);

    typedef __attribute__((address_space(3))) v4s* trptr;
    // 16-byte piece e of a tile is chunk e % CH of row e / CH, which holds the row's chunk
    // (e % CH) ^ swz; its offset from the tile's first row is the same in every tile
    unsigned ko[LOADS], vo[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        const int e = tid + NTH * i, row = e / CH, d = ((e % CH) ^ swz<HDP>(row)) * 8;
        const bool in = d < hd;  // behind head_dim: behind every row, zeros
        ko[i] = in ? (unsigned)(row * (int)a.ldk + d) * (int)sizeof(T) : kNoRow;
        vo[i] = in ? (unsigned)(row * (int)a.ldv + d) * (int)sizeof(T) : kNoRow;
    }
    auto issue = [&](int turn, T* kd, T* vd) {
        const int t = turn * SPLIT + part;
        // the rows from the tile's first to the last key: reads behind them give zeros
        const int64_t rows = end - t * KT > 0 ? end - t * KT : 0;
        const int64_t kb = rows * a.ldk * (int)sizeof(T), vb = rows * a.ldv * (int)sizeof(T);
        const Rows kt(Kg + (size_t)t * KT * a.ldk, kb), vt(Vg + (size_t)t * KT * a.ldv, vb);  // (no rows: nothing is read)
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            kt.to_lds(kd + part * TILE + (NTH * i + wave * 64) * 8, ko[i]);
            vt.to_lds(vd + part * TILE + (NTH * i + wave * 64) * 8, vo[i]);
        }
    };
    v16f o[DT] = {};
    float m = -INFINITY, l = 0.0f;  // the reference of the weights, in log2, and their sum
    int cleaned = 0x7fffffff;       // first key of the first tile with values taken out

    // one tile of keys; masked: some query of the block does not see all of the turn's. One
    // code for both, twice over for the two buffers: a block of a short prompt runs through it
    // once, and fetching it costs more than the branches (a first turn of 2.2 us against 1.4).
    auto step = [&](bool masked, int k0, const T* Kt, T* Vt) {
        if (masked) {
            // A value that is not finite must not meet a zero weight in the product.
            // Such values are taken out here and added at the end to the queries that see them.
            int bad = 0;
#pragma unroll 1
            for (int i = 0; i < LOADS; i++) {
                const uint4 w = *reinterpret_cast<const uint4*>(Vt + (tid + NTH * i) * 8);
                const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int x = 0; x < 4; x++) bad |= (u[x] & kExp) == kExp || (u[x] >> 16 & kExp) == kExp;
            }
            if (__syncthreads_or(bad)) {
                cleaned = cleaned < k0 - part * KT ? cleaned : k0 - part * KT;
                unsigned short* w = reinterpret_cast<unsigned short*>(Vt);
#pragma unroll 1
                for (int e = tid; e < TILE; e += NTH)
                    if ((w[e] & kExp) == kExp) w[e] = 0;
                __syncthreads();
            }
        }
        if (k0 >= wave_end) return;
        v16f s[NK] = {};
#pragma unroll
        for (int x = 0; x < KS; x++)
#pragma unroll
            for (int kt = 0; kt < NK; kt++) {
                const int row = 32 * kt + n;
                const v8 k = *reinterpret_cast<const v8*>(Kt + row * HDP + ((2 * x + hf) ^ swz<HDP>(row)) * 8);
                s[kt] = mfma32(k, qv[x], s[kt]);
            }
        // two rows' reads stay ahead of the products that take them
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * NK, 0);
#pragma unroll
        for (int x = 0; x < KS - 2; x++) {
            __builtin_amdgcn_sched_group_barrier(0x8, NK, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, NK, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 2 * NK, 0);
        if (k0 + KT > wave_all) {
            const int seen = lim - k0 - 4 * hf;
#pragma unroll
            for (int kt = 0; kt < NK; kt++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (32 * kt + 8 * (i >> 2) + (i & 3) >= seen) s[kt][i] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int kt = 0; kt < NK; kt++)
#pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[kt][i]);
        mx = halves_max(mx) * c2;
        if (__any(mx > m + 6.0f)) {
            const float mn = fmaxf(m, mx);
            const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
            m = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] *= alpha;
        }
        const float mu = (m == -INFINITY ? 0.0f : m) - a.lift;
        v8 p[NK][2];
#pragma unroll
        for (int kt = 0; kt < NK; kt++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], c2, -mu));
                l += x;
                p[kt][i >> 3][i & 7] = (T)x;
            }
        // 8 keys of dim 32 d + n: rows 4 hf + 0..3 and 8 + 4 hf + 0..3 of the 16 at kb
        auto vfrag = [&](int d, int kb) {
            const int r = kb + 4 * hf + (lane >> 2 & 3);
            const int col = 32 * d + (lane >> 4 & 1) * 16 + (lane & 3) * 4;
            const int c = col >> 3, in = col & 7;
            const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((trptr)(Vt + r * HDP + (c ^ swz<HDP>(r)) * 8 + in));
            const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((trptr)(Vt + (r + 8) * HDP + (c ^ swz<HDP>(r + 8)) * 8 + in));
            return __builtin_bit_cast(v8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        };
#pragma unroll
        for (int kt = 0; kt < NK; kt++)
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] = mfma32(vfrag(d, 32 * kt + 16 * x), p[kt][x], o[d]);
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 1);
#pragma unroll
        for (int x = 0; x < 2 * NK * DT - 4; x++) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 1);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 4, 1);
    };
    // turns alternate between the two buffers; the next one is loaded while this one is worked on
    auto turn = [&](int t, T* kc, T* vc, T* kn, T* vn) {
        if (t + 1 < turns) issue(t + 1, kn, vn);
        step(t >= plain, (t * SPLIT + part) * KT, kc + part * TILE, vc + part * TILE);
        wait_loads();
        __syncthreads();
    };

    if (turns) issue(0, K0, V0);
    wait_loads();
    __syncthreads();
    for (int t = 0; t < turns; t += 2) {
        turn(t, K0, V0, K1, V1);
        if (t + 1 < turns) turn(t + 1, K1, V1, K0, V0);
    }

    if constexpr (SPLIT == 2) {
        // Every wave of the second half leaves its state to the one with its queries, lane by
        // lane: 32 x HC floats, half of what K0 or K1 holds.
        static_assert(2 * 32 * HC * sizeof(float) <= sizeof(K0) && QW <= 4);
        float* x = reinterpret_cast<float*>(wave < 2 ? K0 : K1) + (wave & 1) * 32 * HC + lane;
        __shared__ float ml[QW][2][64];
        if (part == 1) {
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) x[(d * 16 + i) * 64] = o[d][i];
            ml[wave][0][lane] = m;
            ml[wave][1][lane] = l;
        }
        __syncthreads();
        if (part == 1) return;
        const float m1 = ml[wave][0][lane], l1 = ml[wave][1][lane];
        const float mn = fmaxf(m, m1), mu = mn == -INFINITY ? 0.0f : mn;
        const float f0 = __builtin_amdgcn_exp2f(m - mu), f1 = __builtin_amdgcn_exp2f(m1 - mu);
        l = l * f0 + l1 * f1;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] = o[d][i] * f0 + x[(d * 16 + i) * 64] * f1;
    }

#pragma unroll 1
    for (int j = cleaned; j < end; j++) {
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int col = 32 * d + 8 * (i >> 2) + 4 * hf + (i & 3);
                const float x = col < hd ? to_f32(Vg[(size_t)j * a.ldv + col]) : 0.0f;
                if (!(fabsf(x) < INFINITY) && j < lim) o[d][i] += x;
            }
    }

    l = halves_sum(l);
    const float inv = 1.0f / l;
    const Rows orows(static_cast<const T*>(a.out) + (size_t)job.q0 * a.ldo + head * hd, (int64_t)job.nq * a.ldo * (int)sizeof(T));
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int col = 32 * d + 8 * i + 4 * hf;
            Pack<T, 4> z;
#pragma unroll
            for (int r = 0; r < 4; r++) z.v[r] = (T)(l == 0.0f ? 0.0f : o[d][4 * i + r] * inv);
            orows.store8(z, qok && col < hd ? (unsigned)(qi * (int)a.ldo + col) * (int)sizeof(T) : kNoRow);
        }
}

// ---------------------------------------------- fp32 up to 128 columns ----
// Each operand as three bf16 parts, h + m + l = x to 2^-25 of it: h its upper 16 bits, m and l the
// rounded rests. Of the nine products six are formed, h h, h m, m h, m m, h l and l h; m l, l m
// and l l stay below 2^-22 of |x y|, a few roundings of an fp32 sum. Six bf16 products
// run at 2.6 times the rate of one on the fp32 matrix cores, and bf16 has fp32's range.
// Parts of what is not finite would not add up again: such rows of K are marked and
// their scores formed with fp32 products, such values of V are taken out and added at the
// end to the queries that see them.
// K and V rows go through registers, which split them, into LDS planes [3][KT][HDP] with the
// layout of the 16-bit kernel; the next tile's are loaded while this one is worked on.

struct Parts {
    v8bf h, m, l;
};
__device__ __forceinline__ Parts split8(const float* x) {
    Parts p;
    typedef unsigned v4u __attribute__((ext_vector_type(4)));
    v4u h;
    float r[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const unsigned a = __float_as_uint(x[2 * i]), b = __float_as_uint(x[2 * i + 1]);
        h[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        r[2 * i] = x[2 * i] - __uint_as_float(a & 0xffff0000u);
        r[2 * i + 1] = x[2 * i + 1] - __uint_as_float(b & 0xffff0000u);
    }
    p.h = __builtin_bit_cast(v8bf, h);
#pragma unroll
    for (int i = 0; i < 8; i++) p.m[i] = (bf16_t)r[i];
#pragma unroll
    for (int i = 0; i < 8; i++) p.l[i] = (bf16_t)(r[i] - (float)p.m[i]);
    return p;
}

// c + x y, the smaller products first
__device__ __forceinline__ v16f mfma_parts(const Parts& x, const Parts& y, v16f c) {
    c = mfma32(x.l, y.h, c);
    c = mfma32(x.h, y.l, c);
    c = mfma32(x.m, y.m, c);
    c = mfma32(x.m, y.h, c);
    c = mfma32(x.h, y.m, c);
    return mfma32(x.h, y.h, c);
}

// KP 2 and 4: so many waves share 32 queries and a tile's keys, joined at the end; the block has
// 64 queries then.
constexpr int parts_threads(int kp) { return kp == 4 ? 512 : 256; }

template <int HDP, int HC, int KT, int KP>
__global__ __launch_bounds__(parts_threads(KP), KP == 4 || KT * HC <= 4096 && HC <= 96 ? 2 : 1) void packed_attn_parts(PackedAttnArgs a) {
    constexpr int NTH = parts_threads(KP), QT = KP == 1 ? 128 : 64, NK = KT / 32 / KP;  // 32-key steps of a wave
    constexpr int CH = HDP / 8;             // 8-value pieces of a row
    constexpr int LOADS = KT * CH / NTH;    // pieces per thread of a K or V tile
    constexpr int DT = HC / 32, KS = HC / 16;
    constexpr int PLANE = KT * HDP;
    __shared__ __attribute__((aligned(16))) bf16_t Ks[3 * PLANE], Vs[3 * PLANE];
    __shared__ unsigned long long kbad[2][KT <= 64 ? 1 : 2];  // rows of the tile with values that are not finite
    __shared__ int vbad;                    // first key of the first tile with such values of V
    __shared__ int vlarge;                  // values of V have reached 2^90

    int tile, head;
    tile_and_head(a, tile, head);
    Job job;
    if (!find_job<QT>(a, tile, job)) return;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, hf = lane >> 5;
    const int hd = a.head_dim;
    const int kvh = __builtin_amdgcn_readfirstlane(head / (a.n_q / a.n_kv));
    const float* Kg = static_cast<const float*>(a.K) + (size_t)job.k0 * a.ldk + kvh * hd;
    const float* Vg = static_cast<const float*>(a.V) + (size_t)job.k0 * a.ldv + kvh * hd;

    const int off = job.nk - job.len_q + job.at + 1;
    auto limit = [&](int q) {
        const int e = a.causal ? q + off : job.nk;
        return e < 0 ? 0 : (e < job.nk ? e : job.nk);
    };
    const int qw = KP == 1 ? wave : wave & 1, kp = KP == 1 ? 0 : wave >> 1;
    const int kw = kp * 32 * NK;  // the wave's first key of a tile
    const int qi = qw * 32 + n;
    const bool qok = qi < job.nq;
    const int lim = qok ? limit(qi) : 0;
    const int wq_last = qw * 32 + 31 < job.nq ? qw * 32 + 31 : job.nq - 1;
    const int wave_end = qw * 32 < job.nq ? limit(wq_last) : 0;
    const int wave_all = qw * 32 < job.nq ? limit(qw * 32) : 0;
    const int end = limit(job.nq - 1);
    const int tiles = (end + KT - 1) / KT;

    unsigned ko[LOADS], vo[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        const int e = tid + NTH * i, row = e / CH, d = (e % CH) * 8;
        ko[i] = d < hd ? (unsigned)(row * (int)a.ldk + d) * 4u : kNoRow;
        vo[i] = d < hd ? (unsigned)(row * (int)a.ldv + d) * 4u : kNoRow;
    }
    float kr[LOADS][8], vr[LOADS][8];
    auto fetch = [&](int t) {
        const int64_t rows = end - t * KT;
        const Rows kt(Kg + (size_t)t * KT * a.ldk, rows * a.ldk * 4), vt(Vg + (size_t)t * KT * a.ldv, rows * a.ldv * 4);
#pragma unroll
        for (int i = 0; i < LOADS; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float4 k = kt.load16<float4>(ko[i] + 16 * h), v = vt.load16<float4>(vo[i] + 16 * h);
                kr[i][4 * h] = k.x, kr[i][4 * h + 1] = k.y, kr[i][4 * h + 2] = k.z, kr[i][4 * h + 3] = k.w;
                vr[i][4 * h] = v.x, vr[i][4 * h + 1] = v.y, vr[i][4 * h + 2] = v.z, vr[i][4 * h + 3] = v.w;
            }
    };
    auto top8 = [](const float* x) {  // bits of the largest magnitude, those of what is not finite above all others
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const unsigned u = __float_as_uint(x[i]) & 0x7fffffffu;
            top = u > top ? u : top;
        }
        return top;
    };
    auto put = [&](bf16_t* planes, int e, const float* x) {
        const Parts p = split8(x);
        const int row = e / CH, at = row * HDP + ((e % CH) ^ swz<HDP>(row)) * 8;
        *reinterpret_cast<v8bf*>(planes + at) = p.h;
        *reinterpret_cast<v8bf*>(planes + PLANE + at) = p.m;
        *reinterpret_cast<v8bf*>(planes + 2 * PLANE + at) = p.l;
    };
    bool large = false;  // V in LDS and o are 2^-34 as large
    auto land = [&](int t) {
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int e = tid + NTH * i;
            if (top8(kr[i]) >= 0x7f800000u) {
                atomicOr(&kbad[t & 1][e / CH >> 6], 1ull << (e / CH & 63));
#pragma unroll
                for (int x = 0; x < 8; x++) kr[i][x] = 0.0f;
            }
            if (__builtin_expect(top8(vr[i]) >= kLargeBits, 0)) {
                if (top8(vr[i]) >= 0x7f800000u) {
                    atomicMin(&vbad, t * KT);
#pragma unroll
                    for (int x = 0; x < 8; x++)
                        if (!(fabsf(vr[i][x]) < INFINITY)) vr[i][x] = 0.0f;
                }
                if (top8(vr[i]) >= kLargeBits) vlarge = 1;
            }
            put(Ks, e, kr[i]);
            if (large) {
#pragma unroll
                for (int x = 0; x < 8; x++) vr[i][x] *= kLargeScale;
            }
            put(Vs, e, vr[i]);
        }
    };

    if (tiles) fetch(0);
    const float c2 = a.scale == 0.0f ? 1.17549435e-38f : fabsf(a.scale) * kLog2e;  // as in the 16-bit kernel
    const Rows qrows(static_cast<const float*>(a.Q) + (size_t)job.q0 * a.ldq + head * hd, (int64_t)job.nq * a.ldq * 4);
    Parts qv[KS];
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const int d = 16 * s + 8 * hf;
        const unsigned o = qok && d < hd ? (unsigned)(qi * (int)a.ldq + d) * 4u : kNoRow;
        const float4 x = qrows.load16<float4>(o), y = qrows.load16<float4>(o + 16);
        float f[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        if (a.scale < 0.0f) {
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = -f[i];
        }
        qv[s] = split8(f);
    }
    if (tid == 0) {
        for (auto& w : kbad)
            for (auto& x : w) x = 0;
        vbad = 0x7fffffff;
        vlarge = 0;
    }

    v16f o[DT] = {};
    float m = -INFINITY, l = 0.0f;
    typedef __attribute__((address_space(3))) v4s* trptr;
    for (int t = 0; t < tiles; t++) {
        const int k0 = t * KT;
        __syncthreads();  // the previous tile is read
        land(t);
        __syncthreads();
        if (__builtin_expect(!large && __builtin_amdgcn_readfirstlane(vlarge), 0)) {  // the first such tile: its values again
            large = true;
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
#pragma unroll
                for (int x = 0; x < 8; x++) vr[i][x] *= kLargeScale;
                put(Vs, tid + NTH * i, vr[i]);
            }
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] *= kLargeScale;
            __syncthreads();
        }
        if (t + 1 < tiles) fetch(t + 1);
        const unsigned long long marked = kbad[t & 1][kw >> 6] >> (kw & 63);  // of the wave's keys on
        if (tid == 0)
            for (auto& x : kbad[(t + 1) & 1]) x = 0;
        if (k0 + kw >= wave_end) continue;
        v16f s[NK] = {};
#pragma unroll
        for (int x = 0; x < KS; x++)
#pragma unroll
            for (int kt = 0; kt < NK; kt++) {
                const int row = kw + 32 * kt + n, at = row * HDP + ((2 * x + hf) ^ swz<HDP>(row)) * 8;
                const Parts k{*reinterpret_cast<const v8bf*>(Ks + at), *reinterpret_cast<const v8bf*>(Ks + PLANE + at),
                              *reinterpret_cast<const v8bf*>(Ks + 2 * PLANE + at)};
                s[kt] = mfma_parts(k, qv[x], s[kt]);
            }
        if (marked) {
#pragma unroll 1
            for (int j = 0; j < 32 * NK; j++) {
                if (!(marked >> j & 1) || k0 + kw + j >= end) continue;
                unsigned at = 0;
                asm volatile("" : "+v"(at));  // (keeps all of this inside the branch)
                const Rows krow(Kg + (size_t)(k0 + kw + j) * a.ldk, (int64_t)hd * 4);
                float dot = 0.0f;
#pragma unroll 1
                for (int d = 8 * hf; d < hd; d += 16)
#pragma unroll
                    for (int e = 0; e < 8; e += 4) {
                        const float4 q = qrows.load16<float4>(qok ? (unsigned)(qi * (int)a.ldq + d + e) * 4u + at : kNoRow);
                        const float4 k = krow.load16<float4>((d + e) * 4u + at);
                        dot += q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
                    }
                dot = halves_sum(a.scale < 0.0f ? -dot : dot);
#pragma unroll
                for (int kt = 0; kt < NK; kt++)
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (32 * kt + 8 * (i >> 2) + 4 * hf + (i & 3) == j) s[kt][i] = dot;
            }
        }
        if (k0 + KT > wave_all) {
            const int seen = lim - k0 - kw - 4 * hf;
#pragma unroll
            for (int kt = 0; kt < NK; kt++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (32 * kt + 8 * (i >> 2) + (i & 3) >= seen) s[kt][i] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int kt = 0; kt < NK; kt++)
#pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[kt][i]);
        mx = halves_max(mx) * c2;
        if (__any(mx > m + 6.0f)) {  // as in the 16-bit kernel
            const float mn = fmaxf(m, mx);
            const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
            m = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] *= alpha;
        }
        const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int kt = 0; kt < NK; kt++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                float w[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][8 * x + i], c2, -mu));
                    l += w[i];
                }
                const Parts p = split8(w);
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const int r = kw + 32 * kt + 16 * x + 4 * hf + (lane >> 2 & 3);
                    const int col = 32 * d + (lane >> 4 & 1) * 16 + (lane & 3) * 4, c = col >> 3, in = col & 7;
                    const int a0 = r * HDP + (c ^ swz<HDP>(r)) * 8 + in, a1 = (r + 8) * HDP + (c ^ swz<HDP>(r + 8)) * 8 + in;
                    auto frag = [&](const bf16_t* plane) {
                        const v4s y0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((trptr)(plane + a0));
                        const v4s y1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((trptr)(plane + a1));
                        return __builtin_bit_cast(v8bf, __builtin_shufflevector(y0, y1, 0, 1, 2, 3, 4, 5, 6, 7));
                    };
                    o[d] = mfma_parts(Parts{frag(Vs), frag(Vs + PLANE), frag(Vs + 2 * PLANE)}, p, o[d]);
                }
            }
    }
    __syncthreads();
    if constexpr (KP > 1) {  // lane by lane, as the two halves of the 16-bit kernel
        static_assert((KP - 1) * 2 * 32 * HC * 4 <= (int)sizeof(Ks));
        float* x = reinterpret_cast<float*>(Ks) + qw * 32 * HC + lane;
        __shared__ float ml[KP][2][2][64];
        if (kp) {
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) x[(kp - 1) * 64 * HC + (d * 16 + i) * 64] = o[d][i];
        }
        ml[kp][qw][0][lane] = m;
        ml[kp][qw][1][lane] = l;
        __syncthreads();
        if (kp) return;
        float mn = m;
#pragma unroll
        for (int p = 1; p < KP; p++) mn = fmaxf(mn, ml[p][qw][0][lane]);
        const float mu = mn == -INFINITY ? 0.0f : mn, f0 = __builtin_amdgcn_exp2f(m - mu);
        l *= f0;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] *= f0;
#pragma unroll
        for (int p = 1; p < KP; p++) {
            const float f = __builtin_amdgcn_exp2f(ml[p][qw][0][lane] - mu);
            l += f * ml[p][qw][1][lane];
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] += f * x[(p - 1) * 64 * HC + (d * 16 + i) * 64];
        }
    }
    const int cleaned = vbad;
#pragma unroll 1
    for (int j = cleaned; j < end; j++) {
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int col = 32 * d + 8 * (i >> 2) + 4 * hf + (i & 3);
                const float x = col < hd ? Vg[(size_t)j * a.ldv + col] : 0.0f;
                if (!(fabsf(x) < INFINITY) && j < lim) o[d][i] += x;
            }
    }

    l = halves_sum(l);
    const float inv = 1.0f / (large ? l * kLargeScale : l);
    const Rows orows(static_cast<const float*>(a.out) + (size_t)job.q0 * a.ldo + head * hd, (int64_t)job.nq * a.ldo * 4);
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int col = 32 * d + 8 * i + 4 * hf;
            float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
            if (l != 0.0f) z = make_float4(o[d][4 * i] * inv, o[d][4 * i + 1] * inv, o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv);
            orows.store16(z, qok && col < hd ? (unsigned)(qi * (int)a.ldo + col) * 4u : kNoRow);
        }
}

// ---------------------------------------------- fp32 past 128 columns ----
// A wave owns 16 queries: v_mfma_f32_16x16x4_f32 leaves in lane n + 16 g, for query
// n, the scores of keys 4 g + r of 16, and takes weight r of the lane as key 4 g
// + r of its step r. The head dimension is walked as d = g * (HDP / 4) + s, so
// that a lane's K row comes in 16-byte reads.

__device__ __forceinline__ v4f mfma_f32(float a, float b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

template <int HDP>
__global__ __launch_bounds__(256) void packed_attn_f32(PackedAttnArgs a) {
    constexpr int KT = 32, QT = 64, SK = HDP + 4, QS = HDP / 4, DT = HDP / 16;
    constexpr int LOADS = KT * HDP / 4 / 256;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* Ks = reinterpret_cast<float*>(smem);  // [KT][SK]
    float* Vs = Ks + KT * SK;

    int tile, head;
    tile_and_head(a, tile, head);
    Job job;
    if (!find_job<QT>(a, tile, job)) return;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = lane & 15, g = lane >> 4;
    const int hd = a.head_dim;
    const int kvh = head / (a.n_q / a.n_kv);
    const float* Kg = static_cast<const float*>(a.K) + (size_t)job.k0 * a.ldk + kvh * hd;
    const float* Vg = static_cast<const float*>(a.V) + (size_t)job.k0 * a.ldv + kvh * hd;

    const int qi = wave * 16 + n;
    const bool qok = qi < job.nq;
    float qv[QS];
#pragma unroll
    for (int s = 0; s < QS; s += 4) {
        const int d = g * QS + s;
        float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
        if (qok && d < hd) z = *reinterpret_cast<const float4*>(static_cast<const float*>(a.Q) + (size_t)(job.q0 + qi) * a.ldq + head * hd + d);
        qv[s] = z.x;
        qv[s + 1] = z.y;
        qv[s + 2] = z.z;
        qv[s + 3] = z.w;
    }
    const int off = job.nk - job.len_q + job.at + 1;
    auto limit = [&](int q) {
        const int e = a.causal ? q + off : job.nk;
        return e < 0 ? 0 : (e < job.nk ? e : job.nk);
    };
    const int lim = qok ? limit(qi) : 0;
    const int wq_last = wave * 16 + 15 < job.nq ? wave * 16 + 15 : job.nq - 1;
    const int wave_end = wave * 16 < job.nq ? limit(wq_last) : 0;
    const int wave_all = wave * 16 < job.nq ? limit(wave * 16) : 0;
    const int end = limit(job.nq - 1);
    const int tiles = (end + KT - 1) / KT;

    float4 kr[LOADS], vr[LOADS];
    auto gload = [&](int t) {
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int e = tid + 256 * i, row = e / (HDP / 4), d = 4 * (e % (HDP / 4));
            int j = t * KT + row;
            if (j >= end) j = end - 1;
            kr[i] = vr[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (d < hd) {
                kr[i] = *reinterpret_cast<const float4*>(Kg + (size_t)j * a.ldk + d);
                vr[i] = *reinterpret_cast<const float4*>(Vg + (size_t)j * a.ldv + d);
            }
        }
    };
    auto lstore = [&]() {
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int e = tid + 256 * i, row = e / (HDP / 4), d = 4 * (e % (HDP / 4));
            *reinterpret_cast<float4*>(Ks + row * SK + d) = kr[i];
            *reinterpret_cast<float4*>(Vs + row * SK + d) = vr[i];
        }
    };

    v4f o[DT] = {};
    float m = -INFINITY, l = 0.0f;
    const float c2 = a.scale * kLog2e, ws = __builtin_amdgcn_exp2f(a.lift);
    if (tiles) gload(0);
    for (int t = 0; t < tiles; t++) {
        const int k0 = t * KT;
        __syncthreads();
        lstore();
        __syncthreads();
        if (t + 1 < tiles) gload(t + 1);
        bool rare = false;
        if (k0 + KT > limit(0)) {
            int bad = 0;
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                const int e = tid + 256 * i, row = e / (HDP / 4), d = 4 * (e % (HDP / 4));
                const uint4 w = *reinterpret_cast<const uint4*>(Vs + row * SK + d);
                const unsigned E = 0x7f800000u;
                bad |= (w.x & E) == E || (w.y & E) == E || (w.z & E) == E || (w.w & E) == E;
            }
            rare = __syncthreads_or(bad);
        }
        if (k0 < wave_end) {
            v4f s[KT / 16] = {};
#pragma unroll
            for (int kt = 0; kt < KT / 16; kt++)
#pragma unroll
                for (int x = 0; x < QS; x += 4) {
                    const float4 k = *reinterpret_cast<const float4*>(Ks + (16 * kt + n) * SK + g * QS + x);
                    s[kt] = mfma_f32(k.x, qv[x], s[kt]);
                    s[kt] = mfma_f32(k.y, qv[x + 1], s[kt]);
                    s[kt] = mfma_f32(k.z, qv[x + 2], s[kt]);
                    s[kt] = mfma_f32(k.w, qv[x + 3], s[kt]);
                }
            const bool full = k0 + KT <= wave_all;
            float mx = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < KT / 16; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float x = s[kt][r] * c2;
                    if (!full && k0 + 16 * kt + 4 * g + r >= lim) x = -INFINITY;
                    s[kt][r] = x;
                    mx = fmaxf(mx, x);
                }
            const float mn = fmaxf(m, rows_max(mx));
            const float mu = mn == -INFINITY ? 0.0f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m - mu);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int r = 0; r < 4; r++) o[d][r] *= alpha;
#pragma unroll
            for (int kt = 0; kt < KT / 16; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    s[kt][r] = __builtin_amdgcn_exp2f(s[kt][r] - mu);
                    l += s[kt][r];
                    s[kt][r] *= ws;
                }
            if (!rare) {
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int kt = 0; kt < KT / 16; kt++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            o[d] = mfma_f32(Vs[(16 * kt + 4 * g + r) * SK + 16 * d + n], s[kt][r], o[d]);
            } else {
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    v4f keep = o[d];
#pragma unroll 1
                    for (int q = 0; q < 16; q++) {
                        const int rl = __shfl(lim, q);
                        v4f acc = o[d];
#pragma unroll
                        for (int kt = 0; kt < KT / 16; kt++)
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const int j = 16 * kt + 4 * g + r;
                                const float v = k0 + j < rl ? Vs[j * SK + 16 * d + n] : 0.0f;
                                acc = mfma_f32(v, s[kt][r], acc);
                            }
#pragma unroll
                        for (int r = 0; r < 4; r++) keep[r] = n == q ? acc[r] : keep[r];
                    }
                    o[d] = keep;
                }
            }
        }
    }

    l = rows_sum(l);
    const float inv = 1.0f / (l * ws);
    if (!qok) return;
    float* dst = static_cast<float*>(a.out) + (size_t)(job.q0 + qi) * a.ldo + head * hd;
#pragma unroll
    for (int d = 0; d < DT; d++) {
        const int col = 16 * d + 4 * g;
        float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
        if (l != 0.0f) z = make_float4(o[d][0] * inv, o[d][1] * inv, o[d][2] * inv, o[d][3] * inv);
        if (col < hd) *reinterpret_cast<float4*>(dst + col) = z;
    }
}

// tile numbers of find_job: the most tiles that n_seqs sequences of total_q rows can have
int64_t max_tiles(const PackedAttnArgs& a, int qt) { return a.total_q / qt + (int64_t)a.n_seqs; }

template <class F>
void launch_tiles(F* kernel, const PackedAttnArgs& a, int qt, int threads, int lds, hipStream_t st) {
    if (lds > 65536)
        VLA_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    const int64_t blocks = max_tiles(a, qt) * a.n_q;
    VLA_REQUIRE(blocks * threads < (int64_t)1 << 32, "packed_attention: too many rows times heads for one call");
    kernel<<<(unsigned)blocks, threads, lds, st>>>(a);
    VLA_LAUNCH_CHECK();
}

template <class T, int HDP, int HC, int KT, int SPLIT, int QW>
void run_16_split(const PackedAttnArgs& a, hipStream_t st) {
    launch_tiles(&packed_attn_16<T, HDP, HC, KT, SPLIT, QW>, a, 32 * QW, 64 * QW * SPLIT, 0, st);
}
// Two halves of the keys per block, and blocks of 64 queries, where blocks of four waves would
// leave CUs idle or alone and the sequences have some length. (304 is of blocks as max_tiles counts them, up to one tile
// a sequence more than there are: some more than the 256 CUs for a few sequences.) Measured, us, four waves with 128
// queries | two halves | two halves with 64 (blocks of 128 named): 96 blocks of 256 keys 13.6 | 13.4 |
// 11.4, 160 of 512 18.5 | 17.2 | 14.5, 108 of 1024 (no mask, heads of 64) 17.1 | 15.4 | 12.4, 216 of 1024
// 18.2 | 16.6 | 16.7, 288 of 1024 (heads of 128) 28.4 | 25.1 | 30.1; one half is ahead where a block has but one tile, 32
// of 64 keys 8.3 | 10.5 | 9.7, and with more blocks, 324 of 1024 (heads of 64) 26.5 | 29.9 | 26.1, 1280 of 512 46.6 |
// 59.6 | 85.7, one prompt of 8192 528 | 560.
template <class T, int HDP, int HC>
void run_16_hc(const PackedAttnArgs& a, hipStream_t st) {
    const bool keys = a.total_k >= (int64_t)256 * a.n_seqs;
    if (keys && max_tiles(a, 64) * a.n_q <= 304) run_16_split<T, HDP, HC, 64, 2, 2>(a, st);
    else if (keys && max_tiles(a, 128) * a.n_q <= 304) run_16_split<T, HDP, HC, 64, 2, 4>(a, st);
    else run_16_split<T, HDP, HC, 64, 1, 4>(a, st);
}
template <class T>
void run_16(const PackedAttnArgs& a, hipStream_t st) {
    if (a.head_dim <= 32) run_16_hc<T, 64, 32>(a, st);
    else if (a.head_dim <= 64) run_16_hc<T, 64, 64>(a, st);
    else if (a.head_dim <= 96) run_16_hc<T, 128, 96>(a, st);
    else if (a.head_dim <= 128) run_16_hc<T, 128, 128>(a, st);
    else if (a.head_dim <= 192) run_16_split<T, 256, 192, 32, 1, 4>(a, st);
    else run_16_split<T, 256, 256, 32, 1, 4>(a, st);
}
// Two waves to 32 queries where the blocks of four times 32 would leave CUs idle, four where
// sequences have some length. Measured, us, one wave | two | four: 75 blocks of 512 keys (heads
// of 64) 33 | 26 | 21.5, 108 of 1024 (no mask) - | 45 | 36, 288 of 1024 61 | 60 | 49; 165 of mixed lengths up to
// 177 15.5 | 13.5 | 13.7, 285 of 177 17.0 | 17.6 | 24, 15 of 64 - | 8.6 | 10.4; heads of 128: 160 of 512 67 | 45,
// 544 of 2048 253 | 320. The fp32 matrix cores took 30, -, 88, 14.4, 21.8, 7.9 | 52, 361.
template <int HDP, int HC>
void run_parts(const PackedAttnArgs& a, hipStream_t st) {
    if constexpr (HDP == 64) {
        if (max_tiles(a, 64) * a.n_q <= 768 && a.total_k >= (int64_t)384 * a.n_seqs) {
            launch_tiles(&packed_attn_parts<64, HC, 128, 4>, a, 64, 512, 0, st);
            return;
        }
    }
    if (max_tiles(a, 128) * a.n_q <= 256) launch_tiles(&packed_attn_parts<HDP, HC, 64, 2>, a, 64, 256, 0, st);
    else launch_tiles(&packed_attn_parts<HDP, HC, HDP == 64 ? 64 : 32, 1>, a, 128, 256, 0, st);
}
void run_f32(const PackedAttnArgs& a, hipStream_t st) {
    if (a.head_dim <= 32) run_parts<64, 32>(a, st);
    else if (a.head_dim <= 64) run_parts<64, 64>(a, st);
    else if (a.head_dim <= 96) run_parts<128, 96>(a, st);
    else if (a.head_dim <= 128) run_parts<128, 128>(a, st);
    else launch_tiles(&packed_attn_f32<256>, a, 64, 256, 2 * 32 * (256 + 4) * 4, st);
}

}  // namespace

void launch_packed_attention(PackedAttnArgs a, hipStream_t st) {
    VLA_REQUIRE(dtype_ok(a.dtype), "packed_attention: dtype must be VLA_F32, VLA_BF16 or VLA_F16");
    VLA_REQUIRE(a.n_seqs >= 0 && a.total_q >= 0 && a.total_k >= 0 && a.n_q > 0 && a.n_kv > 0,
                "packed_attention: need n_seqs, total_q, total_k >= 0, n_q > 0, n_kv > 0");
    VLA_REQUIRE(a.n_seqs <= 1 << 28 && a.total_q <= 1 << 28 && a.total_k <= 1 << 28,
                "packed_attention: at most 2^28 sequences and rows");
    VLA_REQUIRE(a.n_q <= 65536 && a.n_q % a.n_kv == 0, "packed_attention: n_q must be a multiple of n_kv up to 65536");
    VLA_REQUIRE(a.head_dim > 0 && a.head_dim <= 256 && a.head_dim % 8 == 0,
                "packed_attention: head_dim must be a multiple of 8 in [8, 256]");
    VLA_REQUIRE(std::isfinite(a.scale), "packed_attention: scale must be finite");
    if (a.n_seqs == 0 || a.total_q == 0) return;
    VLA_REQUIRE(a.out && a.Q && a.q_start && a.k_start, "packed_attention: null buffer");
    VLA_REQUIRE(a.total_k == 0 || (a.K && a.V), "packed_attention: null keys or values");
    const int sz = dtype_size(a.dtype);
    VLA_REQUIRE(aligned(a.Q, 16) && aligned(a.K, 16) && aligned(a.V, 16) && aligned(a.out, 16) && a.ldq * sz % 16 == 0 &&
                    a.ldk * sz % 16 == 0 && a.ldv * sz % 16 == 0 && a.ldo * sz % 16 == 0,
                "packed_attention: rows must be 16-byte aligned");
    VLA_REQUIRE(a.ldq < 1 << 22 && a.ldk < 1 << 22 && a.ldv < 1 << 22 && a.ldo < 1 << 22,
                "packed_attention: row stride past 2^22 values");
    VLA_REQUIRE(a.ldq >= a.n_q * a.head_dim && a.ldo >= a.n_q * a.head_dim && a.ldk >= a.n_kv * a.head_dim &&
                    a.ldv >= a.n_kv * a.head_dim,
                "packed_attention: row stride shorter than heads * head_dim");
    a.lift = lift_of(a);
    if (a.dtype == kBf16) run_16<bf16_t>(a, st);
    else if (a.dtype == kF16) run_16<f16_t>(a, st);
    else run_f32(a, st);
}

}  // namespace hip
}  // namespace vla
