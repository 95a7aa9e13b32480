// kv4.hip - a paged cache of 4-bit keys and values: writing rows into it, reading
// tokens back as rows, and the attention of a sequence's newest tokens over it.
// The format and its rounding are in kv4.h.

#include "kv4_attn.h"

#include <cmath>

namespace vla {
namespace hip {
namespace {

// ------------------------------------------------------ append, gather ----
// HBM bounds both: a value is 2 or 4 bytes on one side and 17/32 on the other (20500 bf16 rows
// of 8 heads of 128, 106 MB each: append 25 us, 4.3 TB/s, gather 19 us, 5.6). A
// lane owns EPL neighbouring values (16 bytes of the row type, 2 or 4 of codes), the
// 32 / EPL lanes of a block share its scale; a thread block takes neighbouring
// tokens of one head and part (K or V), whose codes lie together in a page.

// R rows per thread, 256 / lanes apart: their loads are under way together.
template <class T, int R>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Args a) {
    constexpr int EPL = RowGeo<T>::EPL;
    __shared__ int32_t starts[kStartsInLds];
    __shared__ Where place[256];
    const int lanes = a.head_dim / EPL;  // of a token's head
    const int per = 256 / lanes;         // tokens of the block at once
    const int head = blockIdx.y >> 1, part = blockIdx.y & 1;
    const int tt = threadIdx.x / lanes, ln = threadIdx.x - tt * lanes;
    const int first = blockIdx.x * (R * per), row0 = first + tt;
    const T* src = static_cast<const T*>(part ? a.V : a.K) + head * a.head_dim + ln * EPL;
    const int64_t ld = part ? a.ldv : a.ldk;
    Pack<T, EPL> x[R];
    bool on[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int row = row0 + i * per;
        on[i] = tt < per && row < a.total;
        x[i] = Pack<T, EPL>{};
        if (on[i]) x[i] = *reinterpret_cast<const Pack<T, EPL>*>(src + row * ld);
    }
    locate_rows(a, first, R * per, false, starts, place);
#pragma unroll
    for (int i = 0; i < R; i++) {
        float f[EPL];
#pragma unroll
        for (int e = 0; e < EPL; e++) f[e] = to_f32(x[i].v[e]);
        const Kv4Lane z = quantize_lane(f);
        const Where w = place[tt + i * per];
        if (on[i] && w.page >= 0) store_lane<EPL>(a, w, part, head, ln, z);
    }
}

template <class T, int R>
__global__ __launch_bounds__(256) void kv4_gather_kernel(Kv4Args a) {
    constexpr int EPL = RowGeo<T>::EPL, LPB = RowGeo<T>::LPB;
    __shared__ int32_t starts[kStartsInLds];
    __shared__ Where place[256];
    const int lanes = a.head_dim / EPL;
    const int per = 256 / lanes;
    const int head = blockIdx.y >> 1, part = blockIdx.y & 1;
    const int tt = threadIdx.x / lanes, ln = threadIdx.x - tt * lanes;
    const int first = blockIdx.x * (R * per), row0 = first + tt;
    locate_rows(a, first, R * per, true, starts, place);
    if (tt >= per) return;
    const size_t nc = kv4_code_bytes(a.n_kv, a.head_dim, a.page_size), ns = kv4_scale_bytes(a.n_kv, a.head_dim, a.page_size);
    Where w[R];
    unsigned codes[R], byte[R];
#pragma unroll
    for (int i = 0; i < R; i++) w[i] = place[tt + i * per];
#pragma unroll
    for (int i = 0; i < R; i++) {
        codes[i] = 0;
        byte[i] = kKv4NanByte;  // a page that is not there reads as NaN
        if (w[i].page >= 0) {
            const uint8_t* pg = a.cache + (size_t)w[i].page * (2 * (nc + ns));
            const uint8_t* cd = pg + part * nc + ((size_t)head * a.page_size + w[i].slot) * (a.head_dim / 2) + ln * (EPL / 2);
            codes[i] = EPL == 8 ? *reinterpret_cast<const uint32_t*>(cd) : *reinterpret_cast<const uint16_t*>(cd);
            byte[i] = pg[2 * nc + part * ns + ((size_t)head * (a.head_dim / kKv4Block) + ln / LPB) * a.page_size + w[i].slot];
        }
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
        if (w[i].seq < 0) continue;
        const float sc = scale_of(byte[i]);
        Pack<T, EPL> x;
        auto put = [&](int e, v2f z) {
            x.v[2 * e] = (T)z[0];
            x.v[2 * e + 1] = (T)z[1];
        };
        put(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], sc, 0));
        put(1, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], sc, 1));
        if constexpr (EPL == 8) {
            put(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], sc, 2));
            put(3, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], sc, 3));
        }
        T* dst = static_cast<T*>(part ? a.V : a.K) + (row0 + i * per) * (part ? a.ldv : a.ldk) + head * a.head_dim;
        *reinterpret_cast<Pack<T, EPL>*>(dst + ln * EPL) = x;
    }
}

// ----------------------------------------------------------- attention ----
// out[i] = sum_j softmax_j(scale * q[i] . k[j]) v[j] for the n newest tokens of a
// sequence of len cached ones; token i sees keys j < len - n + i + 1.
//
// HBM bounds it: each cached token is read once for a handful of queries (bf16, 32 heads on 8 of
// 128: 64 sequences of 4096 in 49 us, 5.8 TB/s; 48 mixed up to 8192 in 42.6 us, 3.5 TB/s: 37 and
// 5 for the join, as runs are cut at sequences; 2 of 131072, fp16, 58 us, 4.9 TB/s). A block
// works on one kv head and on the 16 queries (a row tile) that share its keys: the heads of a
// group for as many new tokens as fit. Its W waves take tiles of 32 keys in turn, each with a
// running maximum and sum of its own, joined through LDS.
// The tiles of all sequences, one behind the other, are dealt to the blocks of a head in equal
// runs, whatever the sequences' lengths: as many blocks as the card holds at once then end
// together. A run may begin and end inside a sequence; such pieces are kept in the
// workspace and a second kernel joins them. The host does not see the lengths, so every block
// adds them up itself. Without a workspace, or with more sequences than that pays for, a
// block takes a whole sequence.
//
// Both products run on the bf16 matrix cores, where a cached value c * 2^e is exact:
//   S^T = K Q^T   one step takes 16 keys and 32 dims; lane c + 16 g holds dims of key c;
//   O^T = V^T P^T one step takes 32 keys and 16 dims; the lane's 8 keys are 4 g + r and
//                 16 + 4 g + r, those whose scores it holds, so weights stay put.
// Operands with more bits than bf16 are cut into parts of 8 bits, largest first,
// whose products add up in fp32: queries exactly (bf16 one part, fp16 two, fp32
// three), weights to 16 bits (24 for fp32 results).
//
// A lane reads vb dwords (K) or vb bytes (V) of a row at once, for the vb of its blocks that
// the load covers; which dim a step's row then stands for is only a renaming, undone where the
// results are written.


template <class T, int NB, int PQ, int PP, int W>
__global__ __launch_bounds__(W * 64, 2) void kv4_attn_kernel(Kv4Args a, Kv4Run run) {
    using G = Kv4Geo<NB>;
    constexpr int NL = G::NL, NT = G::NT, HD = 32 * NB;
    constexpr int MO = HD + 4;
    __shared__ __attribute__((aligned(16))) float so[W * 16 * MO];
    __shared__ float sml[W][2][16];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    // blocks of all heads over the same run are neighbours: they read neighbouring parts of its pages
    const int kvh = __builtin_amdgcn_readfirstlane(blockIdx.x % a.n_kv), rt = __builtin_amdgcn_readfirstlane(blockIdx.x / a.n_kv);
    const int block = blockIdx.y;
    const int ht = rt % run.head_tiles;
    const int group = a.n_q / a.n_kv;
    const int heads = group < 16 ? group : 16;         // heads of a row tile
    const int toks = group < 16 ? 16 / group : 1;      // tokens of a row tile
    const float c2 = a.scale * kLog2e;

    int per = 0, seq = block, first = 0, cached = 0;
    if (!run.runs) cached = uniform_entry(a.lens, seq);
    else if (!find_run(a, run.runs, block, per, seq, first, cached)) return;
    const int seq0 = seq;
    const int run_begin = block * per, run_end = run_begin + per;

    // the sequences of the run; [first, first + tiles) are a sequence's tiles among all
    for (int tiles = 0; seq < a.n_seqs && (first < run_end || !run.runs); seq++, first += tiles) {
    if (!run.runs && seq != block) break;
    int len;
    if (seq != seq0) cached = uniform_entry(a.lens, seq);
    tiles = seq_tiles(a, cached, len);
    int q0 = seq, n = 1;
    if (a.start) {
        const int s0 = uniform_entry(a.start, seq), s1 = uniform_entry(a.start, seq + 1);
        q0 = s0 < 0 ? 0 : s0;
        n = (s1 < a.total ? s1 : a.total) - q0;
    }
    // this block's tiles of the sequence, and the pieces that runs cut it into
    int t_begin = 0, t_end = tiles, pieces = 1, slot = 0;
    if (run.runs) {
        const int b0 = first / per, b1 = (first + tiles - 1) / per;
        if (n > run.tok_cap) {  // no room for its pieces: the first block takes all of it
            if (block != b0) continue;
        } else {
            pieces = b1 - b0 + 1;
            slot = block + seq;  // counts up with every cut between blocks or sequences
            t_begin = run_begin > first ? run_begin - first : 0;
            t_end = run_end - first < tiles ? run_end - first : tiles;
        }
        if (block == b0 && blockIdx.x == 0)
            for (int i = threadIdx.x; i < n; i += W * 64) run.info[q0 + i] = make_int4(b0 + seq, pieces, i, 0);
    }
    const int32_t* table = a.table + (size_t)seq * a.ld_table;

    for (int tt = rt / run.head_tiles; tt * toks < n; tt += run.tok_tiles) {
        const int t0 = tt * toks;
        const int tn = n - t0 < toks ? n - t0 : toks;
        const int tok = t0 + c / heads, hh = ht * 16 + c % heads;  // this lane's row
        const bool rok = c < heads * tn && hh < group;
        const int lim = rok ? (len - n + tok + 1 > 0 ? len - n + tok + 1 : 0) : 0;
        const int lim_lo = len - n + t0 + 1, lim_hi = len - n + t0 + tn;  // of the tile's rows
        const int k_begin = t_begin * kTile;
        int k_end = t_end * kTile;
        k_end = lim_hi < k_end ? (lim_hi < 0 ? 0 : lim_hi) : k_end;

        const int k_first = k_begin + wave * kTile;
        Kv4Tile<NB> ta;
        // (a load behind the last tile reads the first again: always as many loads, so that the waits
        // for one tile can count those of the next: 48 mixed up to 8192 46.1 us for 42.8, 2 of 131072 65 for 58)
        auto load = [&](Kv4Tile<NB>& t, int k) { t.load(a, run, table, kvh, c, g, k < k_end ? (unsigned)k / kTile : 0u); };
        load(ta, k_first);

        // (rows without a query read the first one's and take zeros, by a mask that the compiler
        // cannot make a branch of: around the loads it would wait for each by itself)
        U4 qv[PQ][NB];
        constexpr int QL = 8 * (int)sizeof(T) / 16;  // loads of 8 values
        typedef Pack<T, 16 / (int)sizeof(T)> QPack;
        QPack qx[NB][QL];
        const T* qrow = static_cast<const T*>(a.Q) + (size_t)(q0 + (rok ? tok : t0)) * a.ldq + (kvh * group + (rok ? hh : ht * 16)) * HD;
        unsigned keep = rok ? ~0u : 0u;
        asm volatile("" : "+v"(keep));
        each_load<NL>([&]<int u>() {
            constexpr int VB = G::vb(u), BS = G::bs(u);
#pragma unroll
            for (int i = 0; i < VB; i++)
#pragma unroll
                for (int j = 0; j < QL; j++)
                    qx[BS + i][j] = *reinterpret_cast<const QPack*>(qrow + BS * 32 + g * 8 * VB + 8 * i + j * (8 / QL));
        });
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = __uint_as_float(__float_as_uint(to_f32(qx[b][e / (8 / QL)].v[e % (8 / QL)])) & keep);
#pragma unroll
            for (int q = 0; q < PQ; q++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    qv[q][b].u[j] = pack_upper(x[2 * j], x[2 * j + 1]);
                    x[2 * j] -= upper_part(x[2 * j]);
                    x[2 * j + 1] -= upper_part(x[2 * j + 1]);
                }
        }

        v4f o[NT] = {};
        float m = -INFINITY, l = 0.0f;  // the reference of the weights, in log2, and their sum
        int cleaned = 0;
        auto step = [&](Kv4Tile<NB>& t, int k0) {
            v4f s[2] = {};
#pragma unroll
            for (int sub = 0; sub < 2; sub++)
                each_load<NL>([&]<int u>() {
                    constexpr int VB = G::vb(u), BS = G::bs(u);
                    const float sc = scale_of(t.kb[sub][u]);
#pragma unroll
                    for (int i = 0; i < VB; i++) {
                        const unsigned w = t.kd[sub][BS + i];
                        const U4 k{{bf16_of<0>(w, sc), bf16_of<1>(w, sc), bf16_of<2>(w, sc), bf16_of<3>(w, sc)}};
#pragma unroll
                        for (int p = PQ - 1; p >= 0; p--) s[sub] = mfma16(k, qv[p][BS + i], s[sub]);
                    }
                });
            float x[8];  // of keys k0 + 8 g + i
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = s[i >> 2][i & 3] * c2;
            const int kl = k0 + 8 * g;
            if (k0 + kTile > lim_lo || !t.there) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (!t.there) x[i] = NAN;
                    if (kl + i >= lim) x[i] = -INFINITY;
                    // What no row sees is taken out, it may be anything; and so is, of the keys
                    // that some rows see, blocks that may not be finite and must not meet the other rows'
                    // zero weights: they are put in as NaN at the end. (Code by code, so that the finite
                    // ones of a block at the end of fp32's range stay: 45 us for 43, 48 mixed up to 8192.)
#pragma unroll
                    for (int u = 0; u < NL; u++) {
                        const bool nan = kl + i >= lim_lo && t.vbyte(i, u) >= kKv4LargeByte;
                        if (nan || kl + i >= k_end) t.hide(i, u);
                        cleaned |= nan;
                    }
                }
            }
            float mx = x[0];
#pragma unroll
            for (int i = 1; i < 8; i++) mx = fmaxf(mx, x[i]);
            mx = rows_max(mx);
            // The reference only has to keep the weights in range: it follows the
            // maximum when a row's has grown by 2^6, so most tiles rescale nothing.
            if (__any(mx > m + 6.0f)) {
                const float mn = fmaxf(m, mx);
                const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
                m = mn;
                l *= alpha;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) o[t][r] *= alpha;
            }
            // Weights reach 2^6, and no sum over all keys may leave fp32's range: they are 2^-lift as large, in the
            // product alone where they have 24 bits, as their exponent's rounding to 2^-19 would show.
            const float mu = (m == -INFINITY ? 0.0f : m) + (PP == 3 ? 0.0f : run.lift);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = __builtin_amdgcn_exp2f(x[i] - mu);
                l += x[i];
                if (PP == 3) x[i] *= run.wscale;
            }
            U4 pb[PP];
#pragma unroll
            for (int q = 0; q < PP; q++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    pb[q].u[j] = pack_upper(x[2 * j], x[2 * j + 1]);
                    x[2 * j] -= upper_part(x[2 * j]);
                    x[2 * j + 1] -= upper_part(x[2 * j + 1]);
                }
            each_load<NL>([&]<int u>() {
                constexpr int VB = G::vb(u), BS = G::bs(u);
#pragma unroll
                for (int b = 0; b < VB; b++) {
                    U4 lo, hi;
                    t.vfrag(u, b, lo, hi);
                    const int d = 2 * (BS + b);
#pragma unroll
                    for (int q = PP - 1; q >= 0; q--) {
                        o[d] = mfma16(lo, pb[q], o[d]);
                        o[d + 1] = mfma16(hi, pb[q], o[d + 1]);
                    }
                }
            });
        };
        if constexpr (NB <= 4) {  // two tiles in turn: one is loaded while the other is worked on (three: 43.9 us, 59.7)
            Kv4Tile<NB> tb;
            for (int k0 = k_first; k0 < k_end;) {
                const int k1 = k0 + W * kTile;
                load(tb, k1);
                step(ta, k0);
                if (k1 >= k_end) break;
                k0 = k1 + W * kTile;
                load(ta, k0);
                step(tb, k1);
            }
        } else {  // (registers for one)
            for (int k0 = k_first; k0 < k_end; k0 += W * kTile) {
                if (k0 != k_first) load(ta, k0);
                step(ta, k0);
            }
        }
        if (__any(cleaned)) {
            const size_t nc = kv4_code_bytes(a.n_kv, HD, a.page_size), ns = kv4_scale_bytes(a.n_kv, HD, a.page_size);
            for (int j = lim_lo < 0 ? 0 : lim_lo; j < lim_hi; j++) {  // fewer keys than the tile has tokens
                const unsigned pn = page_no(run, (unsigned)j / kTile);
                const int page = uniform_page(table, a.ld_table, a.n_pages, pn);
                if (page < 0) continue;  // NaN through its scores
                const uint8_t* vs = a.cache + (size_t)page * (2 * (nc + ns)) + 2 * nc + ns + (size_t)kvh * NB * a.page_size + (j - pn * a.page_size);
                each_load<NL>([&]<int u>() {
                    constexpr int VB = G::vb(u), BS = G::bs(u);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const bool nan = vs[(size_t)(BS + (4 * g + r) * VB / 16) * a.page_size] >= kKv4LargeByte;
#pragma unroll
                        for (int e = 0; e < 2 * VB; e++)
                            if (nan && j < lim) o[2 * BS + e][r] = NAN;
                    }
                });
            }
        }

        // join the waves: rows of LDS hold a row's dims in their own order
        l = rows_sum(l);
        if (g == 0) {
            sml[wave][0][c] = m;
            sml[wave][1][c] = l;
        }
        each_load<NL>([&]<int u>() {
            constexpr int VB = G::vb(u), BS = G::bs(u);
#pragma unroll
            for (int e = 0; e < 2 * VB; e++)
#pragma unroll
                for (int r = 0; r < 4; r++) so[(wave * 16 + c) * MO + 32 * BS + (4 * g + r) * 2 * VB + e] = o[2 * BS + e][r];
        });
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
            const int rhead = kvh * group + rhh;
            if (pieces == 1) {
                static_cast<T*>(a.out)[(size_t)(q0 + rtok) * a.ldo + rhead * HD + d] = (T)(sum == 0.0f ? 0.0f : acc / (sum * run.wscale));
            } else {
                const size_t rr = ((size_t)slot * run.tok_cap + rtok) * a.n_q + rhead;
                run.o[rr * HD + d] = acc;
                if (d == 0) {
                    run.ml[rr * 2] = top;
                    run.ml[rr * 2 + 1] = sum;
                }
            }
        }
        __syncthreads();
    }
    }
}

int64_t row_tiles(int max_new, int n_q, int n_kv, int* head_tiles) {
    const int group = n_q / n_kv;
    *head_tiles = group <= 16 ? 1 : (group + 15) / 16;
    const int toks = group <= 16 ? 16 / group : 1;
    return ((int64_t)max_new + toks - 1) / toks;
}

// waves of a block: the joined waves' rows stay within 64 KiB of LDS
constexpr int attn_waves(int head_dim) { return head_dim >= 192 ? 2 : 4; }

// Blocks with work where each sequence has its own: of all row tiles that there can be, not of as many in every sequence.
int64_t row_blocks(const Kv4Run& r, int total_q, int n_seqs, int n_q, int n_kv) {
    const int toks = r.head_tiles == 1 ? 16 / (n_q / n_kv) : 1;
    const int64_t spread = (int64_t)r.tok_tiles * n_seqs, sum = total_q / toks + (int64_t)n_seqs;
    return (int64_t)n_kv * r.head_tiles * (spread < sum ? spread : sum);
}

// How a call runs, from sizes the host knows. Equal runs of tiles (and a second kernel) or a
// block per sequence: the latter costs 5 us and 0.7 us for every step of its waves (5.7 us for 1000
// keys, heads of 128) until its blocks take the card's bandwidth among them; the former 12 us and
// what the bytes take, more where runs are cut into pieces of several sequences. Measured, us,
// runs | sequences (32 heads on 8 of 128): 1 x 1000 keys 11.6 | 11.3, 1 x 2000 13.1 | 17.2, 4 x 1500
// 15.6 | 14.6, 4 x 2000 13.4 | 17.5, 16 x 2000 21.8 | 18.4, 16 x 4000 27.1 | 30.6, 64 mixed up to 2000
// 34.9 | 21.5, 48 mixed up to 8192 42.6 | 67.5; where the sequences' blocks fill the card only
// one much longer than the others is worth runs: 64 mixed up to 4000 37.8 | 35.3, 64 of 8192 108 | 104, 64
// mixed up to 16384 95 | 118.
// Runs: as many blocks as the card holds at once (two waves on a SIMD: 512 of 4 waves;
// 768 and 1024 of them took 40.5 and 46 us for the 48, 118 and 115 for the 64 of 8192), each with at
// least two rounds of its waves, 8 tiles for 4 waves (4: 1 x 2000 11.8 us, but 4 x 2000 16.9; 16: 14.4)
// and 4 for 2 (heads of 256: 1 x 1000 14.8 us, with 8 tiles 16.6).
// Blocks are counted by the row tiles that there are at most over all sequences, not by max_new in
// each: one chunk of 128 new tokens among 47 single ones, 48 x 16384 keys, 3527 us with runs for 512 blocks of such
// chunks, 563 now, 503 without runs (chunks of 50: 972, 262, 232; 8 x 65536, one of 50: 646, 288, 580).
// max_new is any bound, 2^31 - 1 where the caller knows none: no sequence has more than all rows.
Kv4Run plan(int total_q, int n_seqs, int max_new, int64_t max_len, int n_q, int n_kv, int head_dim) {
    Kv4Run r{};
    max_new = max_new < total_q ? max_new : total_q;
    const int64_t tiles_of_rows = row_tiles(max_new, n_q, n_kv, &r.head_tiles);
    const int64_t most = ((int64_t)1 << 23) / ((int64_t)n_kv * r.head_tiles);  // (a launch has less than 2^32 threads; a block loops over the rest)
    r.tok_tiles = (int)(tiles_of_rows < most ? tiles_of_rows : most);
    const int64_t blocks = row_blocks(r, total_q, n_seqs, n_q, n_kv);
    const int64_t card = attn_waves(head_dim) == 4 ? 512 : 1024;
    const int64_t steps = max_len / (kTile * attn_waves(head_dim));
    if (steps <= 64 && steps * (card - blocks) <= 12 * card) return r;
    const int64_t tiles = (max_len + kTile - 1) / kTile * n_seqs;
    int64_t runs = (card * n_seqs + blocks - 1) / blocks;
    const int64_t rounds = tiles / (2 * attn_waves(head_dim));
    runs = runs < rounds ? runs : rounds;
    runs = runs < kMaxPieces ? runs : kMaxPieces;
    r.runs = runs <= 1 ? 0 : (int)runs;
    r.tok_cap = max_new;
    r.slots = r.runs + n_seqs;
    if (plan_bytes(r, 0, n_q, head_dim) > (size_t)1 << 28) r.runs = 0;  // pieces of long chunks
    return r;
}

template <class T, int PQ, int PP, int NB>
void run_attn_nb(const Kv4Args& a, const Kv4Run& r, hipStream_t st) {
    constexpr int W = attn_waves(32 * NB);
    kv4_attn_kernel<T, NB, PQ, PP, W><<<dim3(a.n_kv * r.tok_tiles * r.head_tiles, r.runs ? r.runs : a.n_seqs), W * 64, 0, st>>>(a, r);
    VLA_LAUNCH_CHECK();
}

template <class T, int PQ, int PP>
void run_attn(const Kv4Args& a, const Kv4Run& r, hipStream_t st) {
    switch (a.head_dim / 32) {
    case 1: run_attn_nb<T, PQ, PP, 1>(a, r, st); break;
    case 2: run_attn_nb<T, PQ, PP, 2>(a, r, st); break;
    case 3: run_attn_nb<T, PQ, PP, 3>(a, r, st); break;
    case 4: run_attn_nb<T, PQ, PP, 4>(a, r, st); break;
    case 6: run_attn_nb<T, PQ, PP, 6>(a, r, st); break;
    default: run_attn_nb<T, PQ, PP, 8>(a, r, st); break;
    }
    if (!r.runs) return;
    if (r.runs > 8 * a.n_seqs) kv4_join_kernel<T, 256><<<a.total * a.n_q, 256, 0, st>>>(a, r);
    else kv4_join_kernel<T, 64><<<a.total * a.n_q, 64, 0, st>>>(a, r);
    VLA_LAUNCH_CHECK();
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

template <class T, int R>
void run_rows(const Kv4Args& a, bool gather, hipStream_t st) {
    const int per = R * (256 / (a.head_dim / RowGeo<T>::EPL));
    const dim3 grid((unsigned)(((int64_t)a.total + per - 1) / per), 2 * a.n_kv);
    if (gather) kv4_gather_kernel<T, R><<<grid, 256, 0, st>>>(a);
    else kv4_append_kernel<T, R><<<grid, 256, 0, st>>>(a);
    VLA_LAUNCH_CHECK();
}
// Rows per thread by the blocks that one each would take: more loads under way, and the search
// for a row's place paid once, against blocks for every CU. Append and gather together, us, 1 | 2
// | 4 rows: 1024 rows of 8 heads of 128 (1024 blocks) 8.3 | 8.3 | 9.9, 4000 rows 17.9 | 13.7 | 14.9,
// 20500 rows 66.9 | 49.1 | 46.4 (4.6 TB/s; 8 rows 48.0).
template <class T>
void run_rows(const Kv4Args& a, bool gather, hipStream_t st) {
    const int64_t blocks = (int64_t)a.total * (a.head_dim / RowGeo<T>::EPL) / 256 * 2 * a.n_kv;
    if (blocks >= 8192) run_rows<T, 4>(a, gather, st);
    else if (blocks >= 2048) run_rows<T, 2>(a, gather, st);
    else run_rows<T, 1>(a, gather, st);
}
void run_rows(const Kv4Args& a, bool gather, hipStream_t st) {
    if (a.dtype == kF32) run_rows<float>(a, gather, st);
    else if (a.dtype == kBf16) run_rows<bf16_t>(a, gather, st);
    else run_rows<f16_t>(a, gather, st);
}

}  // namespace

void launch_kv4_append(const Kv4Args& a, hipStream_t st) {
    check_cache(a, "kv4_append");
    if (a.n_seqs == 0 || a.total == 0) return;
    check_rows(a, "kv4_append");
    VLA_REQUIRE(a.lens, "kv4_append: lens missing");
    run_rows(a, false, st);
}

void launch_kv4_gather(const Kv4Args& a, hipStream_t st) {
    check_cache(a, "kv4_gather");
    if (a.n_seqs == 0 || a.total == 0) return;
    check_rows(a, "kv4_gather");
    run_rows(a, true, st);
}

size_t kv4_attention_work_bytes(int total_q, int n_seqs, int max_new, int max_len, int n_q, int n_kv, int head_dim) {
    if (total_q <= 0 || n_seqs <= 0 || max_new <= 0 || max_len <= 0 || n_kv <= 0 || n_q <= 0 || n_q % n_kv || head_dim <= 0) return 0;
    // sizes that the call refuses, or that it does not split
    if (!kv4_head_dim_ok(head_dim) || n_kv > 1024 || n_q > 65536 || n_seqs > kMaxSeqs || !joins(total_q, n_q)) return 0;
    return plan_bytes(plan(total_q, n_seqs, max_new, max_len, n_q, n_kv, head_dim), total_q, n_q, head_dim);
}

void launch_kv4_attention(const Kv4Args& a, hipStream_t st) {
    check_cache(a, "kv4_attention");
    VLA_REQUIRE(a.n_q > 0 && a.n_q <= 65536 && a.n_q % a.n_kv == 0, "kv4_attention: n_q must be a multiple of n_kv up to 65536");
    VLA_REQUIRE(std::isfinite(a.scale), "kv4_attention: scale must be finite");
    VLA_REQUIRE(a.max_new >= 0 && a.max_len >= 0, "kv4_attention: max_new and max_len must not be negative");
    VLA_REQUIRE(a.start || a.total >= a.n_seqs, "kv4_attention: without q_start every sequence has one query row");
    if (a.n_seqs == 0 || a.total == 0) return;
    VLA_REQUIRE(a.max_new >= 1, "kv4_attention: max_new must be at least 1");
    VLA_REQUIRE(a.n_seqs <= kMaxSeqs, "kv4_attention: at most 65535 sequences");
    VLA_REQUIRE(a.n_pages > 0 && a.cache && aligned(a.cache, 16), "kv4_attention: the cache must hold a page and be 16-byte aligned");
    VLA_REQUIRE(a.table && a.ld_table > 0 && a.lens, "kv4_attention: page table or lens missing");
    VLA_REQUIRE(a.out && a.Q, "kv4_attention: null buffer");
    const int sz = dtype_size(a.dtype);
    VLA_REQUIRE(a.ldq >= a.n_q * a.head_dim && a.ldo >= a.n_q * a.head_dim, "kv4_attention: row stride shorter than heads * head_dim");
    VLA_REQUIRE(aligned(a.Q, 16) && aligned(a.out, 16) && a.ldq * sz % 16 == 0 && a.ldo * sz % 16 == 0,
                "kv4_attention: rows must be 16-byte aligned");
    VLA_REQUIRE((int64_t)a.total * a.n_q < (int64_t)1 << 31, "kv4_attention: too many query rows times heads");
    Kv4Run r = plan(a.total, a.n_seqs, a.max_new, a.max_len, a.n_q, a.n_kv, a.head_dim);
    // (the tiles of all sequences are counted in 32 bits)
    const bool counts = (int64_t)a.n_seqs * ((int64_t)a.ld_table * a.page_size / kTile + 2) < (int64_t)1 << 30;
    if (!counts || !joins(a.total, a.n_q) || !a.work || !aligned(a.work, 16) || a.work_bytes < plan_bytes(r, a.total, a.n_q, a.head_dim)) r.runs = 0;
    if (r.runs) {
        r.info = reinterpret_cast<int4*>(a.work);
        char* ml = reinterpret_cast<char*>(a.work) + info_bytes(a.total);
        r.ml = reinterpret_cast<float*>(ml);
        r.o = reinterpret_cast<float*>(ml + ml_bytes(r, a.n_q));
    }
    r.per_page = a.page_size / kTile;
    r.magic = r.per_page == 1 ? 0 : (unsigned)((((uint64_t)1 << 32) + r.per_page - 1) / r.per_page);
    // Blocks without a row tile cost 2 to 6 ns of the launch each, so where max_new is far above most sequences' tokens, or
    // is not known, there are 2^16 blocks or twice as many as can have work; they take several row tiles then. (2000 single tokens
    // of 64 keys, max_new 2000: 15.1 ms without this, 0.41 now, 0.11 with max_new 1.)
    const int64_t busy = row_blocks(r, a.total, a.n_seqs, a.n_q, a.n_kv), grid = 2 * busy > 1 << 16 ? 2 * busy : 1 << 16;
    const int64_t most = grid / ((int64_t)a.n_kv * r.head_tiles * (r.runs ? r.runs : a.n_seqs));
    if (r.tok_tiles > most) r.tok_tiles = (int)(most < 1 ? 1 : most);
    int log2_n = 0;
    while (1 << log2_n < a.ld_table * a.page_size) log2_n++;
    r.lift = 6.0f + (float)log2_n;
    r.wscale = a.dtype == kF32 ? std::ldexp(1.0f, -6 - log2_n) : 1.0f;
    if (a.dtype == kF32) run_attn<float, 3, 3>(a, r, st);
    else if (a.dtype == kBf16) run_attn<bf16_t, 1, 2>(a, r, st);
    else run_attn<f16_t, 2, 2>(a, r, st);
}

}  // namespace hip
}  // namespace vla
