// kv4.hip - a paged cache of 4-bit keys and values: writing rows into it, reading
// tokens back as rows, and the attention of a sequence's newest tokens over it.
// The format and its rounding are in kv4.h.

#include "kv4.h"

#include "serving.h"
#include "wave.h"

#include <cmath>

namespace vla {
namespace hip {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef bf16_t v2bf __attribute__((ext_vector_type(2)));
typedef bf16_t v8bf __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;

// 2^e of a scale byte as the converters take it: they read the exponent bits
// alone, and give NaN for 255 (and 2^-127 for 0)
__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }

// ------------------------------------------------------ append, gather ----
// HBM bounds both: a value is 2 or 4 bytes on one side and 17/32 on the other. A
// lane owns EPL neighbouring values (16 bytes of the row type, 2 or 4 of codes), the
// 32 / EPL lanes of a block share its scale; a thread block takes neighbouring
// tokens of one head and part (K or V), whose codes lie together in a page.

constexpr int kStartsInLds = 1024;

struct Where {
    int seq, page, slot;
};

// Where packed row `row` lives in the cache: page -1 for a row behind the last
// sequence (seq -1 then), a position before the first token or a page that is not there.
__device__ __forceinline__ Where locate(const Kv4Args& a, const int32_t* start, int row, bool gather) {
    Where w{-1, -1, 0};
    const int s = seq_of_row(start, a.n_seqs, row);
    if (s >= a.n_seqs || row < start[s]) return w;
    w.seq = s;
    const int64_t i = (int64_t)row - start[s];
    const int64_t tok = gather ? (int64_t)(a.first ? a.first[s] : 0) + i
                               : (int64_t)a.lens[s] - ((int64_t)start[s + 1] - start[s]) + i;
    if (tok < 0) return w;
    const int64_t no = (uint64_t)tok / (unsigned)a.page_size;
    w.slot = (int)(tok - no * a.page_size);
    w.page = kv4_page(a.table + (size_t)s * a.ld_table, a.ld_table, a.n_pages, no);
    return w;
}

// The starts in LDS where they fit, so that the search of every row's
// sequence costs no chain of global reads.
__device__ __forceinline__ const int32_t* stage_starts(const Kv4Args& a, int32_t* lds) {
    if (a.n_seqs >= kStartsInLds) return a.start;
    for (int i = threadIdx.x; i <= a.n_seqs; i += blockDim.x) lds[i] = a.start[i];
    __syncthreads();
    return lds;
}

template <class T>
struct RowGeo {
    static constexpr int EPL = 16 / sizeof(T);      // values of a lane
    static constexpr int LPB = kKv4Block / EPL;     // lanes of a block
};

template <class T>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Args a) {
    constexpr int EPL = RowGeo<T>::EPL, LPB = RowGeo<T>::LPB;
    __shared__ int32_t starts[kStartsInLds];
    const int lanes = a.head_dim / EPL;  // of a token's head
    const int per = 256 / lanes;         // tokens of the block
    const int head = blockIdx.y >> 1, part = blockIdx.y & 1;
    const int tt = threadIdx.x / lanes, ln = threadIdx.x - tt * lanes;
    const int row = blockIdx.x * per + tt;
    const bool on = tt < per && row < a.total;
    const T* src = static_cast<const T*>(part ? a.V : a.K) + (size_t)(on ? row : 0) * (part ? a.ldv : a.ldk) + head * a.head_dim;
    Pack<T, EPL> x = {};
    if (on) x = *reinterpret_cast<const Pack<T, EPL>*>(src + ln * EPL);
    const int32_t* start = stage_starts(a, starts);

    float f[EPL];
    unsigned top = 0;  // bits of the largest magnitude: NaN above infinity above all numbers
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        f[i] = to_f32(x.v[i]);
        const unsigned u = __float_as_uint(f[i]) & 0x7fffffffu;
        top = u > top ? u : top;
    }
#pragma unroll
    for (int m = 1; m < LPB; m <<= 1) {
        const unsigned u = __shfl_xor(top, m);
        top = u > top ? u : top;
    }
    // 1.f * 2^(E - 127) <= 1.75 * 2^(e + 2), so e + 127 = E - 2, one more where 1.f > 1.75
    int byte = (int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x600000u);
    byte = byte < kKv4MinByte ? kKv4MinByte : byte;
    const bool bad = top >= 0x7f800000u;
    const float sc = scale_of(byte);
    unsigned codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, f[0], f[1], sc, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[2], f[3], sc, 1);
    if constexpr (EPL == 8) {
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[4], f[5], sc, 2);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[6], f[7], sc, 3);
    }
    if (bad) {
        codes = 0;
        byte = kKv4NanByte;
    }
    if (!on) return;
    const Where w = locate(a, start, row, false);
    if (w.page < 0) return;
    const size_t nc = kv4_code_bytes(a.n_kv, a.head_dim, a.page_size), ns = kv4_scale_bytes(a.n_kv, a.head_dim, a.page_size);
    uint8_t* pg = a.cache + (size_t)w.page * (2 * (nc + ns));
    uint8_t* cd = pg + part * nc + ((size_t)head * a.page_size + w.slot) * (a.head_dim / 2) + ln * (EPL / 2);
    if (EPL == 8) *reinterpret_cast<uint32_t*>(cd) = codes;
    else *reinterpret_cast<uint16_t*>(cd) = (uint16_t)codes;
    if (ln % LPB == 0)
        pg[2 * nc + part * ns + ((size_t)head * (a.head_dim / kKv4Block) + ln / LPB) * a.page_size + w.slot] = (uint8_t)byte;
}

template <class T>
__global__ __launch_bounds__(256) void kv4_gather_kernel(Kv4Args a) {
    constexpr int EPL = RowGeo<T>::EPL, LPB = RowGeo<T>::LPB;
    __shared__ int32_t starts[kStartsInLds];
    const int lanes = a.head_dim / EPL;
    const int per = 256 / lanes;
    const int head = blockIdx.y >> 1, part = blockIdx.y & 1;
    const int tt = threadIdx.x / lanes, ln = threadIdx.x - tt * lanes;
    const int row = blockIdx.x * per + tt;
    const int32_t* start = stage_starts(a, starts);
    if (tt >= per || row >= a.total) return;
    const Where w = locate(a, start, row, true);
    if (w.seq < 0) return;
    unsigned codes = 0, byte = kKv4NanByte;  // a page that is not there reads as NaN
    if (w.page >= 0) {
        const size_t nc = kv4_code_bytes(a.n_kv, a.head_dim, a.page_size), ns = kv4_scale_bytes(a.n_kv, a.head_dim, a.page_size);
        const uint8_t* pg = a.cache + (size_t)w.page * (2 * (nc + ns));
        const uint8_t* cd = pg + part * nc + ((size_t)head * a.page_size + w.slot) * (a.head_dim / 2) + ln * (EPL / 2);
        codes = EPL == 8 ? *reinterpret_cast<const uint32_t*>(cd) : *reinterpret_cast<const uint16_t*>(cd);
        byte = pg[2 * nc + part * ns + ((size_t)head * (a.head_dim / kKv4Block) + ln / LPB) * a.page_size + w.slot];
    }
    const float sc = scale_of(byte);
    Pack<T, EPL> x;
    auto put = [&](int i, v2f z) {
        x.v[2 * i] = (T)z[0];
        x.v[2 * i + 1] = (T)z[1];
    };
    put(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, sc, 0));
    put(1, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, sc, 1));
    if constexpr (EPL == 8) {
        put(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, sc, 2));
        put(3, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, sc, 3));
    }
    T* dst = static_cast<T*>(part ? a.V : a.K) + (size_t)row * (part ? a.ldv : a.ldk) + head * a.head_dim;
    *reinterpret_cast<Pack<T, EPL>*>(dst + ln * EPL) = x;
}

// ----------------------------------------------------------- attention ----
// out[i] = sum_j softmax_j(scale * q[i] . k[j]) v[j] for the n newest tokens of a
// sequence of len cached ones; token i sees keys j < len - n + i + 1.
//
// HBM bounds it: each cached token is read once for a handful of queries. A block
// works on one (sequence, kv head, run of keys); its rows are the queries that
// share those keys: 16 of them, the heads of a group for as many new tokens as fit.
// Its W waves take tiles of 32 keys in turn, each with a running maximum and
// sum of its own, joined through LDS at the end. Where sequences and heads are
// too few for the card, the keys are split further over blocks (gridDim.x) whose
// partial results a second kernel joins.
//
// Both products run on the bf16 matrix cores, where a cached value c * 2^e is exact:
//   S^T = K Q^T   one step takes 16 keys and 32 dims; lane c + 16 g holds dims of key c;
//   O^T = V^T P^T one step takes 32 keys and 16 dims; the lane's 8 keys are 4 g + r and
//                 16 + 4 g + r, those whose scores it holds, so weights stay put.
// Operands with more bits than bf16 are cut into parts of 8 bits, largest first,
// whose products add up in fp32: queries exactly (bf16 one part, fp16 two, fp32
// three), weights to 16 bits (24 for fp32 results).
//
// A lane reads VB (K) or VW (V) bytes-times-4 or bytes of a row at once, the most
// that NB = head_dim / 32 allows; which dim a step's row then stands for is only
// a renaming, undone where the results are written.

template <int NB>
struct Kv4Geo {
    static constexpr int VB = NB % 4 == 0 ? 4 : NB % 2 == 0 ? 2 : 1;  // dwords of a K load
    static constexpr int NL = NB / VB;
    static constexpr int VW = VB;                                     // bytes of a V load
    static constexpr int NT = 2 * NB;                                 // 16-dim tiles of O
};

__device__ __forceinline__ float upper_part(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// the upper halves of two floats, a in the low half
__device__ __forceinline__ unsigned pack_upper(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

struct U4 {
    unsigned u[4];
};

template <int SEL>
__device__ __forceinline__ unsigned bf16_of(unsigned codes, float scale) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
}

__device__ __forceinline__ v4f mfma16(const U4& a, const U4& b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

constexpr int kTile = 32;

struct Kv4Run {
    int chunk;         // keys of a split, a multiple of kTile
    int tok_tiles;     // row tiles over the new tokens, times head tiles in gridDim.y / n_kv
    int head_tiles;
    unsigned per_page; // tiles of a page, and 2^32 / per_page rounded up
    unsigned magic;
    int rows;          // total queries * n_q: rows of the partial results
};

// tile / per_page; exact while tile * per_page < 2^32
__device__ __forceinline__ unsigned page_no(const Kv4Run& r, unsigned tile) {
    return r.per_page == 1 ? tile : __umulhi(tile, r.magic);
}

template <class T, int NB, int PQ, int PP, int W>
__global__ __launch_bounds__(W * 64) void kv4_attn_kernel(Kv4Args a, Kv4Run run) {
    using G = Kv4Geo<NB>;
    constexpr int VB = G::VB, NL = G::NL, VW = G::VW, NT = G::NT, HD = 32 * NB;
    constexpr int MO = HD + 4;
    __shared__ __attribute__((aligned(16))) float so[W * 16 * MO];
    __shared__ float sml[W][2][16];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = lane & 15, g = lane >> 4;
    const int split = blockIdx.x, seq = blockIdx.z;
    const int kvh = blockIdx.y % a.n_kv, rt = blockIdx.y / a.n_kv;
    const int ht = rt % run.head_tiles;
    const int group = a.n_q / a.n_kv;
    const int heads = group < 16 ? group : 16;         // heads of a row tile
    const int toks = group < 16 ? 16 / group : 1;      // tokens of a row tile

    int q0 = seq, n = 1;
    if (a.start) {
        const int s0 = a.start[seq], s1 = a.start[seq + 1];
        q0 = s0 < 0 ? 0 : s0;
        n = (s1 < a.total ? s1 : a.total) - q0;
    }
    const int64_t cap = (int64_t)a.ld_table * a.page_size;
    int len = a.lens[seq];
    len = len < 0 ? 0 : ((int64_t)len > cap ? (int)cap : len);
    const int32_t* table = a.table + (size_t)seq * a.ld_table;
    const size_t nc = kv4_code_bytes(a.n_kv, HD, a.page_size), ns = kv4_scale_bytes(a.n_kv, HD, a.page_size);
    const size_t page_bytes = 2 * (nc + ns);
    const float c2 = a.scale * kLog2e;
    const int splits = gridDim.x;

    for (int tt = rt / run.head_tiles; tt * toks < n; tt += run.tok_tiles) {
        const int t0 = tt * toks;
        const int tn = n - t0 < toks ? n - t0 : toks;
        const int tok = t0 + c / heads, hh = ht * 16 + c % heads;  // this lane's row
        const bool rok = c < heads * tn && hh < group;
        const int head = kvh * group + hh;
        const int lim = rok ? (len - n + tok + 1 > 0 ? len - n + tok + 1 : 0) : 0;
        const int lim_lo = len - n + t0 + 1, lim_hi = len - n + t0 + tn;  // of the tile's rows
        int k_end = lim_hi < 0 ? 0 : lim_hi;
        const int k_begin = split * run.chunk;
        if (split + 1 < splits && k_begin + run.chunk < k_end) k_end = k_begin + run.chunk;

        U4 qv[PQ][NB];
#pragma unroll
        for (int u = 0; u < NL; u++)
#pragma unroll
            for (int i = 0; i < VB; i++) {
                float x[8] = {};
                if (rok) {
                    const T* src = static_cast<const T*>(a.Q) + (size_t)(q0 + tok) * a.ldq + head * HD + u * 32 * VB + g * 8 * VB + 8 * i;
#pragma unroll
                    for (int j = 0; j < 8; j += 16 / (int)sizeof(T)) {
                        const auto z = *reinterpret_cast<const Pack<T, 16 / sizeof(T)>*>(src + j);
#pragma unroll
                        for (int e = 0; e < 16 / (int)sizeof(T); e++) x[j + e] = to_f32(z.v[e]);
                    }
                }
#pragma unroll
                for (int p = 0; p < PQ; p++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        qv[p][u * VB + i].u[j] = pack_upper(x[2 * j], x[2 * j + 1]);
                        x[2 * j] -= upper_part(x[2 * j]);
                        x[2 * j + 1] -= upper_part(x[2 * j + 1]);
                    }
            }

        v4f o[NT] = {};
        float m = -INFINITY, l = 0.0f;
        for (int k0 = k_begin + wave * kTile; k0 < k_end; k0 += W * kTile) {
            const unsigned tile = (unsigned)k0 / kTile, pn = page_no(run, tile);
            const int slot = (int)(tile - pn * run.per_page) * kTile;
            const int page = kv4_page(table, a.ld_table, a.n_pages, pn);
            // a page that is not there: read the first one, make every score NaN
            const uint8_t* pg = a.cache + (size_t)(page < 0 ? 0 : page) * page_bytes;
            const uint8_t* kc = pg + ((size_t)kvh * a.page_size + slot) * (HD / 2);
            const uint8_t* vc = kc + nc;
            const uint8_t* ks = pg + 2 * nc + (size_t)kvh * NB * a.page_size + slot;
            const uint8_t* vs = ks + ns;

            unsigned kd[2][NB], kb[2][NL], vd[8][NL], vw[2][NL];
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int u = 0; u < NL; u++) {
                    const auto z = *reinterpret_cast<const Pack<unsigned, VB>*>(kc + (16 * s + c) * (HD / 2) + u * 16 * VB + g * 4 * VB);
#pragma unroll
                    for (int i = 0; i < VB; i++) kd[s][u * VB + i] = z.v[i];
                    kb[s][u] = ks[(u * VB + g * VB / 4) * a.page_size + 16 * s + c];
                }
#pragma unroll
            for (int u = 0; u < NL; u++) {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const uint8_t* p = vc + (16 * (k >> 2) + 4 * g + (k & 3)) * (HD / 2) + u * 16 * VW + c * VW;
                    vd[k][u] = VW == 4 ? *reinterpret_cast<const uint32_t*>(p) : VW == 2 ? *reinterpret_cast<const uint16_t*>(p) : *p;
                }
#pragma unroll
                for (int s = 0; s < 2; s++)
                    vw[s][u] = *reinterpret_cast<const uint32_t*>(vs + (u * VW + c * VW / 16) * a.page_size + 16 * s + 4 * g);
            }

            v4f s[2] = {};
#pragma unroll
            for (int sub = 0; sub < 2; sub++)
#pragma unroll
                for (int u = 0; u < NL; u++) {
                    const float sc = scale_of(kb[sub][u]);
#pragma unroll
                    for (int i = 0; i < VB; i++) {
                        const unsigned w = kd[sub][u * VB + i];
                        const U4 k{{bf16_of<0>(w, sc), bf16_of<1>(w, sc), bf16_of<2>(w, sc), bf16_of<3>(w, sc)}};
#pragma unroll
                        for (int p = PQ - 1; p >= 0; p--) s[sub] = mfma16(k, qv[p][u * VB + i], s[sub]);
                    }
                }
            const bool full = k0 + kTile <= lim_lo && k0 + kTile <= k_end;
            float mx = -INFINITY;
#pragma unroll
            for (int sub = 0; sub < 2; sub++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float x = s[sub][r] * c2;
                    if (page < 0) x = NAN;
                    if (!full && k0 + 16 * sub + 4 * g + r >= lim) x = -INFINITY;
                    s[sub][r] = x;
                    mx = fmaxf(mx, x);
                }
            const float mn = fmaxf(m, rows_max(mx));
            const float mu = mn == -INFINITY ? 0.0f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m - mu);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) o[t][r] *= alpha;
            float p[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                p[k] = __builtin_amdgcn_exp2f(s[k >> 2][k & 3] - mu);
                l += p[k];
            }
            U4 pb[PP];
#pragma unroll
            for (int q = 0; q < PP; q++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    pb[q].u[j] = pack_upper(p[2 * j], p[2 * j + 1]);
                    p[2 * j] -= upper_part(p[2 * j]);
                    p[2 * j + 1] -= upper_part(p[2 * j + 1]);
                }
            // V's operands of tile pair (u, b) for keys below `seen`
            auto vfrag = [&](int u, int b, int seen, U4& lo, U4& hi) {
                unsigned z[8];
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const unsigned byte = vw[k >> 2][u] >> (8 * (k & 3)) & 255u;
                    const bool in = k0 + 16 * (k >> 2) + 4 * g + (k & 3) < seen;
                    const float sc = in ? scale_of(byte) : 1.0f;
                    const unsigned w = in ? vd[k][u] : 0u;
                    z[k] = b == 0 ? bf16_of<0>(w, sc) : b == 1 ? bf16_of<1>(w, sc) : b == 2 ? bf16_of<2>(w, sc) : bf16_of<3>(w, sc);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    lo.u[j] = __builtin_amdgcn_perm(z[2 * j + 1], z[2 * j], 0x05040100u);
                    hi.u[j] = __builtin_amdgcn_perm(z[2 * j + 1], z[2 * j], 0x07060302u);
                }
            };
            // a key that some rows of the tile do not see and that is not finite must
            // not meet their zero weights: the product is then done row by row
            bool rare = false;
            if (!full && lim_lo < lim_hi) {
                int nan = 0;
#pragma unroll
                for (int u = 0; u < NL; u++)
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const int j = k0 + 16 * (k >> 2) + 4 * g + (k & 3);
                        nan |= j >= lim_lo && j < lim_hi && (vw[k >> 2][u] >> (8 * (k & 3)) & 255u) == kKv4NanByte;
                    }
                rare = __any(nan);
            }
            const int seen = full ? 0x7fffffff : k_end;
            if (!rare) {
#pragma unroll
                for (int u = 0; u < NL; u++)
#pragma unroll
                    for (int b = 0; b < VW; b++) {
                        U4 lo, hi;
                        vfrag(u, b, seen, lo, hi);
                        const int t = u * 2 * VW + 2 * b;
#pragma unroll
                        for (int q = PP - 1; q >= 0; q--) {
                            o[t] = mfma16(lo, pb[q], o[t]);
                            o[t + 1] = mfma16(hi, pb[q], o[t + 1]);
                        }
                    }
            } else {
#pragma unroll
                for (int u = 0; u < NL; u++)
#pragma unroll
                    for (int b = 0; b < VW; b++) {
                        const int t = u * 2 * VW + 2 * b;
                        v4f keep0 = o[t], keep1 = o[t + 1];
#pragma unroll 1
                        for (int row = 0; row < 16; row++) {
                            const int rl = __shfl(lim, row);
                            U4 lo, hi;
                            vfrag(u, b, rl < seen ? rl : seen, lo, hi);
                            v4f a0 = o[t], a1 = o[t + 1];
#pragma unroll
                            for (int q = PP - 1; q >= 0; q--) {
                                a0 = mfma16(lo, pb[q], a0);
                                a1 = mfma16(hi, pb[q], a1);
                            }
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                keep0[r] = c == row ? a0[r] : keep0[r];
                                keep1[r] = c == row ? a1[r] : keep1[r];
                            }
                        }
                        o[t] = keep0;
                        o[t + 1] = keep1;
                    }
            }
        }

        // join the waves: rows of LDS hold a row's dims in their own order
        l = rows_sum(l);
        if (g == 0) {
            sml[wave][0][c] = m;
            sml[wave][1][c] = l;
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int u = t / (2 * VW), e = t % (2 * VW);
#pragma unroll
            for (int r = 0; r < 4; r++) so[(wave * 16 + c) * MO + u * 32 * VW + (4 * g + r) * 2 * VW + e] = o[t][r];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * HD; i += W * 64) {
            const int r = i / HD, d = i % HD;
            const int rtok = t0 + r / heads, rhh = ht * 16 + r % heads;
            if (r >= heads * tn || rhh >= group) continue;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < W; w++) top = fmaxf(top, sml[w][0][r]);
            const float mu = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f, acc = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float f = __builtin_amdgcn_exp2f(sml[w][0][r] - mu);
                sum += f * sml[w][1][r];
                acc += f * so[(w * 16 + r) * MO + d];
            }
            const size_t tokrow = (size_t)(q0 + rtok);
            const int rhead = kvh * group + rhh;
            if (splits == 1) {
                static_cast<T*>(a.out)[tokrow * a.ldo + rhead * HD + d] = (T)(sum == 0.0f ? 0.0f : acc / sum);
            } else {
                const size_t rr = (size_t)split * run.rows + tokrow * a.n_q + rhead;
                float* po = a.work;
                float* pml = a.work + (size_t)splits * run.rows * HD;
                po[rr * HD + d] = acc;
                if (d == 0) {
                    pml[rr * 2] = top;
                    pml[rr * 2 + 1] = sum;
                }
            }
        }
        __syncthreads();
    }
}

// joins the splits: one block per row (query token and head)
template <class T>
__global__ __launch_bounds__(256) void kv4_join_kernel(Kv4Args a, int splits, int rows) {
    const int row = blockIdx.x, tok = row / a.n_q, head = row - tok * a.n_q;
    if (tok < (a.start ? a.start[0] : 0) || tok >= (a.start ? a.start[a.n_seqs] : a.n_seqs)) return;
    const float* pml = a.work + (size_t)splits * rows * a.head_dim;
    float top = -INFINITY;
    for (int s = 0; s < splits; s++) top = fmaxf(top, pml[((size_t)s * rows + row) * 2]);
    const float mu = top == -INFINITY ? 0.0f : top;
    for (int d = threadIdx.x; d < a.head_dim; d += blockDim.x) {
        float sum = 0.0f, acc = 0.0f;
        for (int s = 0; s < splits; s++) {
            const size_t rr = (size_t)s * rows + row;
            const float f = __builtin_amdgcn_exp2f(pml[rr * 2] - mu);
            sum += f * pml[rr * 2 + 1];
            acc += f * a.work[rr * a.head_dim + d];
        }
        static_cast<T*>(a.out)[(size_t)tok * a.ldo + head * a.head_dim + d] = (T)(sum == 0.0f ? 0.0f : acc / sum);
    }
}

int row_tiles(int max_new, int n_q, int n_kv, int* head_tiles) {
    const int group = n_q / n_kv;
    *head_tiles = group <= 16 ? 1 : (group + 15) / 16;
    const int toks = group <= 16 ? 16 / group : 1;
    return (max_new + toks - 1) / toks;
}

// Splits of the key axis: enough that every CU has two blocks, none shorter than
// 256 keys.
int split_count(int n_seqs, int max_new, int max_len, int n_q, int n_kv) {
    int ht;
    const int64_t blocks = (int64_t)row_tiles(max_new, n_q, n_kv, &ht) * ht * n_kv * n_seqs;
    const int64_t want = (512 + blocks - 1) / blocks, most = (max_len + 255) / 256;
    return (int)(want < most ? want : (most < 1 ? 1 : most));
}

template <class T, int PQ, int PP, int NB>
void run_attn_nb(const Kv4Args& a, const Kv4Run& r, int splits, hipStream_t st) {
    constexpr int W = NB >= 6 ? 2 : 4;  // the joined waves' rows stay within 64 KiB of LDS
    kv4_attn_kernel<T, NB, PQ, PP, W><<<dim3(splits, a.n_kv * r.tok_tiles * r.head_tiles, a.n_seqs), W * 64, 0, st>>>(a, r);
    VLA_LAUNCH_CHECK();
}

template <class T, int PQ, int PP>
void run_attn(const Kv4Args& a, const Kv4Run& r, int splits, hipStream_t st) {
    switch (a.head_dim / 32) {
    case 1: run_attn_nb<T, PQ, PP, 1>(a, r, splits, st); break;
    case 2: run_attn_nb<T, PQ, PP, 2>(a, r, splits, st); break;
    case 3: run_attn_nb<T, PQ, PP, 3>(a, r, splits, st); break;
    case 4: run_attn_nb<T, PQ, PP, 4>(a, r, splits, st); break;
    case 6: run_attn_nb<T, PQ, PP, 6>(a, r, splits, st); break;
    default: run_attn_nb<T, PQ, PP, 8>(a, r, splits, st); break;
    }
    if (splits == 1) return;
    kv4_join_kernel<T><<<r.rows, a.head_dim <= 64 ? 64 : 128, 0, st>>>(a, splits, r.rows);
    VLA_LAUNCH_CHECK();
}

bool head_dim_ok(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 192 || hd == 256; }

void check_cache(const Kv4Args& a, const char* who) {
    const std::string w(who);
    VLA_REQUIRE(dtype_ok(a.dtype), w + ": dtype must be VLA_F32, VLA_BF16 or VLA_F16");
    VLA_REQUIRE(a.n_seqs >= 0 && a.total >= 0 && a.n_kv > 0 && a.n_kv <= 1024, w + ": need n_seqs, rows >= 0 and 1 to 1024 kv heads");
    VLA_REQUIRE(head_dim_ok(a.head_dim), w + ": head_dim must be 32, 64, 96, 128, 192 or 256");
    VLA_REQUIRE(a.page_size > 0 && a.page_size % kTile == 0 && a.page_size <= kKv4MaxPage,
                w + ": page_size must be a multiple of 32 in [32, 2048]");
    VLA_REQUIRE(a.n_pages >= 0 && a.ld_table >= 0 && (int64_t)a.ld_table * a.page_size <= (int64_t)1 << 30,
                w + ": a sequence has at most 2^30 tokens");
}

void check_rows(const Kv4Args& a, const char* who) {
    const std::string w(who);
    const int sz = dtype_size(a.dtype);
    VLA_REQUIRE(a.n_pages > 0 && a.cache && aligned(a.cache, 16), w + ": the cache must hold a page and be 16-byte aligned");
    VLA_REQUIRE(a.table && a.ld_table > 0, w + ": page table missing");
    VLA_REQUIRE(a.K && a.V && a.start, w + ": null buffer");
    VLA_REQUIRE(a.ldk >= a.n_kv * a.head_dim && a.ldv >= a.n_kv * a.head_dim, w + ": row stride shorter than heads * head_dim");
    VLA_REQUIRE(aligned(a.K, 16) && aligned(a.V, 16) && a.ldk * sz % 16 == 0 && a.ldv * sz % 16 == 0,
                w + ": rows must be 16-byte aligned");
}

dim3 row_grid(const Kv4Args& a) {
    const int per = 256 / (a.head_dim * dtype_size(a.dtype) / 16);
    return dim3((a.total + per - 1) / per, 2 * a.n_kv);
}

}  // namespace

void launch_kv4_append(const Kv4Args& a, hipStream_t st) {
    check_cache(a, "kv4_append");
    if (a.n_seqs == 0 || a.total == 0) return;
    check_rows(a, "kv4_append");
    VLA_REQUIRE(a.lens, "kv4_append: lens missing");
    if (a.dtype == kF32) kv4_append_kernel<float><<<row_grid(a), 256, 0, st>>>(a);
    else if (a.dtype == kBf16) kv4_append_kernel<bf16_t><<<row_grid(a), 256, 0, st>>>(a);
    else kv4_append_kernel<f16_t><<<row_grid(a), 256, 0, st>>>(a);
    VLA_LAUNCH_CHECK();
}

void launch_kv4_gather(const Kv4Args& a, hipStream_t st) {
    check_cache(a, "kv4_gather");
    if (a.n_seqs == 0 || a.total == 0) return;
    check_rows(a, "kv4_gather");
    if (a.dtype == kF32) kv4_gather_kernel<float><<<row_grid(a), 256, 0, st>>>(a);
    else if (a.dtype == kBf16) kv4_gather_kernel<bf16_t><<<row_grid(a), 256, 0, st>>>(a);
    else kv4_gather_kernel<f16_t><<<row_grid(a), 256, 0, st>>>(a);
    VLA_LAUNCH_CHECK();
}

size_t kv4_attention_work_bytes(int total_q, int n_seqs, int max_new, int max_len, int n_q, int n_kv, int head_dim) {
    if (total_q <= 0 || n_seqs <= 0 || max_new <= 0 || max_len <= 0 || n_kv <= 0 || n_q <= 0 || n_q % n_kv || head_dim <= 0) return 0;
    const int splits = split_count(n_seqs, max_new, max_len, n_q, n_kv);
    return splits == 1 ? 0 : (size_t)splits * total_q * n_q * (head_dim + 2) * sizeof(float);
}

void launch_kv4_attention(const Kv4Args& a, hipStream_t st) {
    check_cache(a, "kv4_attention");
    VLA_REQUIRE(a.n_q > 0 && a.n_q % a.n_kv == 0, "kv4_attention: n_q must be a multiple of n_kv");
    VLA_REQUIRE(std::isfinite(a.scale), "kv4_attention: scale must be finite");
    VLA_REQUIRE(a.max_new >= 0 && a.max_len >= 0, "kv4_attention: max_new and max_len must not be negative");
    VLA_REQUIRE(a.start || a.total >= a.n_seqs, "kv4_attention: without q_start every sequence has one query row");
    if (a.n_seqs == 0 || a.total == 0) return;
    VLA_REQUIRE(a.max_new >= 1, "kv4_attention: max_new must be at least 1");
    VLA_REQUIRE(a.n_seqs <= 65535, "kv4_attention: at most 65535 sequences");
    VLA_REQUIRE(a.n_pages > 0 && a.cache && aligned(a.cache, 16), "kv4_attention: the cache must hold a page and be 16-byte aligned");
    VLA_REQUIRE(a.table && a.ld_table > 0 && a.lens, "kv4_attention: page table or lens missing");
    VLA_REQUIRE(a.out && a.Q, "kv4_attention: null buffer");
    const int sz = dtype_size(a.dtype);
    VLA_REQUIRE(a.ldq >= a.n_q * a.head_dim && a.ldo >= a.n_q * a.head_dim, "kv4_attention: row stride shorter than heads * head_dim");
    VLA_REQUIRE(aligned(a.Q, 16) && aligned(a.out, 16) && a.ldq * sz % 16 == 0 && a.ldo * sz % 16 == 0,
                "kv4_attention: rows must be 16-byte aligned");
    VLA_REQUIRE((int64_t)a.total * a.n_q < (int64_t)1 << 31, "kv4_attention: too many query rows times heads");
    Kv4Run r{};
    r.tok_tiles = row_tiles(a.max_new, a.n_q, a.n_kv, &r.head_tiles);
    const int64_t most = 65535 / ((int64_t)a.n_kv * r.head_tiles);  // gridDim.y; a block loops over the rest
    if (r.tok_tiles > most) r.tok_tiles = (int)(most < 1 ? 1 : most);
    VLA_REQUIRE((int64_t)a.n_kv * r.head_tiles <= 65535, "kv4_attention: too many heads");
    int splits = split_count(a.n_seqs, a.max_new, a.max_len, a.n_q, a.n_kv);
    if (!a.work || !aligned(a.work, 16) ||
        a.work_bytes < kv4_attention_work_bytes(a.total, a.n_seqs, a.max_new, a.max_len, a.n_q, a.n_kv, a.head_dim))
        splits = 1;
    r.chunk = ((a.max_len + splits - 1) / splits + kTile - 1) / kTile * kTile;
    if (r.chunk < kTile) r.chunk = kTile;
    r.per_page = a.page_size / kTile;
    r.magic = r.per_page == 1 ? 0 : (unsigned)((((uint64_t)1 << 32) + r.per_page - 1) / r.per_page);
    r.rows = a.total * a.n_q;
    if (a.dtype == kF32) run_attn<float, 3, 3>(a, r, splits, st);
    else if (a.dtype == kBf16) run_attn<bf16_t, 1, 2>(a, r, splits, st);
    else run_attn<f16_t, 2, 2>(a, r, splits, st);
}

}  // namespace hip
}  // namespace vla
