// kv4_tree.hip - attention of drafted tokens over the 4-bit cache: of a sequence's
// newest tokens each sees those that its bits name, of the others all.
//
// out[i] = sum_j softmax_j(scale * q[i] . k[j]) v[j] for the n newest tokens of a sequence of len
// cached ones, over j < len - n and over j = len - n + t where bit t of row i's words is set.
//
// As in the attention of a causal chunk a block works on one kv head, its waves take
// tiles of 32 keys in turn, and the tiles of all sequences may be dealt to the blocks in
// equal runs whose pieces a second kernel joins. A wave holds NQ row tiles of 16 queries (the heads
// of a group for some of the new tokens) against each tile of keys that it loads and converts.

#include "kv4_attn.h"

#include <cmath>

namespace vla {
namespace hip {
namespace {

template <class T, int NB, int PQ, int PP, int W, int NQ>
__global__ __launch_bounds__(W * 64, 2) void kv4_tree_kernel(Kv4TreeArgs ta, Kv4Run run) {
    using G = Kv4Geo<NB>;
    constexpr int NL = G::NL, NT = G::NT, HD = 32 * NB;
    constexpr int MO = HD + 4;
    const Kv4Args& a = ta.kv;
    __shared__ __attribute__((aligned(16))) float so[W * 16 * MO];
    __shared__ float sml[W][2][16];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int kvh = __builtin_amdgcn_readfirstlane(blockIdx.x % a.n_kv), rt = __builtin_amdgcn_readfirstlane(blockIdx.x / a.n_kv);
    const int block = blockIdx.y;
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
    const int s0 = uniform_entry(a.start, seq), s1 = uniform_entry(a.start, seq + 1);
    const int q0 = s0 < 0 ? 0 : s0;
    const int n = (s1 < a.total ? s1 : a.total) - q0;
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
    const int base = len - n;  // the first new token, before the first key where more are new than there are
    const int k_begin = t_begin * kTile, k_end = t_end * kTile < len ? t_end * kTile : len;
    const int subs = (n + toks - 1) / toks * run.head_tiles;  // row tiles of the sequence

    for (int r0 = rt * NQ; r0 < subs; r0 += run.tok_tiles * NQ) {
        int tok[NQ], hh[NQ], t0[NQ], h0[NQ];  // this lane's row of each row tile, and the row tile's first
        bool rok[NQ];
#pragma unroll
        for (int z = 0; z < NQ; z++) {
            h0[z] = (r0 + z) % run.head_tiles * 16;
            t0[z] = (r0 + z) / run.head_tiles * toks;
            tok[z] = t0[z] + c / heads;
            hh[z] = h0[z] + c % heads;
            rok[z] = c < heads * toks && tok[z] < n && hh[z] < group;
        }

        const int k_first = k_begin + wave * kTile;
        Kv4Tile<NB> t_a;
        // (a load behind the last tile reads the first again: always as many loads, so that the waits
        // for one tile can count those of the next)
        auto load = [&](Kv4Tile<NB>& t, int k) { t.load(a, run, table, kvh, c, g, k < k_end ? (unsigned)k / kTile : 0u); };
        load(t_a, k_first);

        // (rows without a query read the sequence's first one and take zeros, by a mask that the compiler
        // cannot make a branch of: around the loads it would wait for each by itself)
        U4 qv[NQ][PQ][NB];
        constexpr int QL = 8 * (int)sizeof(T) / 16;  // loads of 8 values
        typedef Pack<T, 16 / (int)sizeof(T)> QPack;
#pragma unroll
        for (int z = 0; z < NQ; z++) {
            QPack qx[NB][QL];
            const T* qrow = static_cast<const T*>(a.Q) + (size_t)(q0 + (rok[z] ? tok[z] : 0)) * a.ldq + (kvh * group + (rok[z] ? hh[z] : 0)) * HD;
            unsigned keep = rok[z] ? ~0u : 0u;
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
                        qv[z][q][b].u[j] = pack_upper(x[2 * j], x[2 * j + 1]);
                        x[2 * j] -= upper_part(x[2 * j]);
                        x[2 * j + 1] -= upper_part(x[2 * j + 1]);
                    }
            }
        }

        // bits of the keys key .. key + 7 that this lane's row of row tile z sees
        auto seen = [&](int z, int key) -> unsigned {
            const int t = key - base;
            const int have = n - t;
            const uint32_t* words = ta.see + (int64_t)(q0 + tok[z]) * ta.ld_see;
            auto word = [&](int k) -> uint32_t { return k < 0 ? ~0u : rok[z] && k < ta.ld_see ? words[k] : 0u; };
            const uint64_t two = (uint64_t)word((t >> 5) + 1) << 32 | word(t >> 5);
            const unsigned bits = (unsigned)(two >> (t & 31)) & 0xffu;
            return !rok[z] || have <= 0 ? 0u : have < 8 ? bits & ((1u << have) - 1) : bits;
        };

        v4f o[NQ][NT] = {};
        float m[NQ], l[NQ];  // the reference of the weights, in log2, and their sum
#pragma unroll
        for (int z = 0; z < NQ; z++) m[z] = -INFINITY, l[z] = 0.0f;
        auto scale_sums = [&](int z, float f) {
            l[z] *= f;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) o[z][t][r] *= f;
        };
        int cleaned = 0;
        auto step = [&](Kv4Tile<NB>& t, int k0) {
#pragma clang fp contract(off)
            v4f s[NQ][2] = {};
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
                        for (int z = 0; z < NQ; z++)
#pragma unroll
                            for (int p = PQ - 1; p >= 0; p--) s[z][sub] = mfma16(k, qv[z][p][BS + i], s[z][sub]);
                    }
                });
            float x[NQ][8];  // of keys k0 + 8 g + i
#pragma unroll
            for (int z = 0; z < NQ; z++)
#pragma unroll
                for (int i = 0; i < 8; i++) x[z][i] = s[z][i >> 2][i & 3] * c2;
            const int kl = k0 + 8 * g;
            if (k0 + kTile > base || !t.there) {
#pragma unroll
                for (int z = 0; z < NQ; z++) {
                    const unsigned bits = seen(z, kl);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        if (!t.there) x[z][i] = NAN;
                        if (!(bits >> i & 1u) || kl + i >= k_end) x[z][i] = -INFINITY;
                    }
                }
                // What no row sees is taken out, it may be anything; and so is, of the new tokens' keys,
                // what may not be finite and must not meet the zero weights of rows that do not see it:
                // it is put in as NaN at the end.
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int u = 0; u < NL; u++) {
                        const bool nan = kl + i >= base && t.vbyte(i, u) >= kKv4LargeByte;
                        if (nan || kl + i >= k_end) t.hide(i, u);
                        cleaned |= nan;
                    }
            }
            U4 pb[NQ][PP];
#pragma unroll
            for (int z = 0; z < NQ; z++) {
                float mx = x[z][0];
#pragma unroll
                for (int i = 1; i < 8; i++) mx = fmaxf(mx, x[z][i]);
                mx = rows_max(mx);
                // The reference only has to keep the weights in range: it follows the
                // maximum when a row's has grown by 2^6, so most tiles rescale nothing.
                if (__any(mx > m[z] + 6.0f)) {
                    const float mn = fmaxf(m[z], mx);
                    const float alpha = __builtin_amdgcn_exp2f(m[z] - (mn == -INFINITY ? 0.0f : mn));
                    m[z] = mn;
                    scale_sums(z, alpha);
                }
                // Weights reach 2^6, and no sum over all keys may leave fp32's range: they are 2^-lift as large, in the
                // product alone where they have 24 bits, as their exponent's rounding to 2^-19 would show. (Subtracted behind the
                // reference: a sum of both is rounded by a power of two where scores pass 2^24, and not the same one for every reference.)
                const float mu = m[z] == -INFINITY ? 0.0f : m[z];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    x[z][i] = __builtin_amdgcn_exp2f(PP == 3 ? x[z][i] - mu : x[z][i] - mu - run.lift);
                    l[z] += x[z][i];
                    if (PP == 3) x[z][i] *= run.wscale;
                }
#pragma unroll
                for (int q = 0; q < PP; q++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        pb[z][q].u[j] = pack_upper(x[z][2 * j], x[z][2 * j + 1]);
                        x[z][2 * j] -= upper_part(x[z][2 * j]);
                        x[z][2 * j + 1] -= upper_part(x[z][2 * j + 1]);
                    }
            }
            each_load<NL>([&]<int u>() {
                constexpr int VB = G::vb(u), BS = G::bs(u);
#pragma unroll
                for (int b = 0; b < VB; b++) {
                    U4 lo, hi;
                    t.vfrag(u, b, lo, hi);
                    const int d = 2 * (BS + b);
#pragma unroll
                    for (int z = 0; z < NQ; z++)
#pragma unroll
                        for (int q = PP - 1; q >= 0; q--) {
                            o[z][d] = mfma16(lo, pb[z][q], o[z][d]);
                            o[z][d + 1] = mfma16(hi, pb[z][q], o[z][d + 1]);
                        }
                }
            });
        };
        if constexpr (NB <= 4) {  // two tiles in turn: one is loaded while the other is worked on
            Kv4Tile<NB> t_b;
            for (int k0 = k_first; k0 < k_end;) {
                const int k1 = k0 + W * kTile;
                load(t_b, k1);
                step(t_a, k0);
                if (k1 >= k_end) break;
                k0 = k1 + W * kTile;
                load(t_a, k0);
                step(t_b, k1);
            }
        } else {  // (registers for one)
            for (int k0 = k_first; k0 < k_end; k0 += W * kTile) {
                if (k0 != k_first) load(t_a, k0);
                step(t_a, k0);
            }
        }
        if (__any(cleaned)) {
            const size_t nc = kv4_code_bytes(a.n_kv, HD, a.page_size), ns = kv4_scale_bytes(a.n_kv, HD, a.page_size);
            for (int j = base < 0 ? 0 : base; j < len; j++) {
                const unsigned pn = page_no(run, (unsigned)j / kTile);
                const int page = uniform_page(table, a.ld_table, a.n_pages, pn);
                if (page < 0) continue;  // NaN through its scores
                const uint8_t* vs = a.cache + (size_t)page * (2 * (nc + ns)) + 2 * nc + ns + (size_t)kvh * NB * a.page_size + (j - pn * a.page_size);
#pragma unroll
                for (int z = 0; z < NQ; z++) {
                    const bool sees = seen(z, j) & 1u;
                    each_load<NL>([&]<int u>() {
                        constexpr int VB = G::vb(u), BS = G::bs(u);
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const bool nan = vs[(size_t)(BS + (4 * g + r) * VB / 16) * a.page_size] >= kKv4LargeByte;
#pragma unroll
                            for (int e = 0; e < 2 * VB; e++)
                                if (nan && sees) o[z][2 * BS + e][r] = NAN;
                        }
                    });
                }
            }
        }

        // join the waves, a row tile at a time: rows of LDS hold a row's dims in their own order
#pragma unroll
        for (int z = 0; z < NQ; z++) {
            const float sum_l = rows_sum(l[z]);
            if (g == 0) {
                sml[wave][0][c] = m[z];
                sml[wave][1][c] = sum_l;
            }
            each_load<NL>([&]<int u>() {
                constexpr int VB = G::vb(u), BS = G::bs(u);
#pragma unroll
                for (int e = 0; e < 2 * VB; e++)
#pragma unroll
                    for (int r = 0; r < 4; r++) so[(wave * 16 + c) * MO + 32 * BS + (4 * g + r) * 2 * VB + e] = o[z][2 * BS + e][r];
            });
            __syncthreads();
            for (int i = threadIdx.x; i < 16 * HD; i += W * 64) {
                const int r = i / HD, d = i % HD;
                const int rtok = t0[z] + r / heads, rhh = h0[z] + r % heads;
                if (r >= heads * toks || rtok >= n || rhh >= group) continue;
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
}

// ---- many rows: tiles converted once for all waves of a block ----
//
// Where a sequence has more row tiles than a wave holds, the four waves of a block take rows of their own
// and share the converted tiles: a stage of one or two tiles is loaded and converted by all waves, a
// part each, into LDS, where it lies as the matrix cores take it (16 bytes a lane, no bank conflicts);
// while a stage is worked on the next one is put into the other buffer and the one behind it is loaded.
//
// Values c * 2^e with e in [-23, 8] are exact in fp16, and so a stage of such values meets weights in
// fp16, in two parts as in bf16. (fp16 queries then meet
// keys in fp16 too, in one part instead of two.) Weights are 2^9 times as large, up to 2^15, and where a
// row's are all below 2^-16 of its largest they are raised for that stage, the sums with them, so that
// a weight is off by 2^-22 of itself or by 2^-18 of the stage's largest, whichever is more. The first
// stage with other values, with what may not be finite, without a page or with a row that is further down than
// sums can be raised turns the block to bf16 parts for good. (Scores of a deviation of 4, or a key 20 above all others, raise sums in
// most stages: 2 x 131072 in bf16 579 and 569 us for 488; 80 above, in bf16 parts 731.)
//
// 2 x 131072 keys, 64 new tokens, 32 heads on 8 of 128: 501 us in fp16, 488 in bf16 (563 TFLOP/s of the product's own
// operations); 48 mixed up to 8192, 32 new, bf16: 172. What bounds it are the vector instructions (257 for 32 rows and keys) and the matrix
// instructions (48) together: a SIMD's two waves hardly overlap them, nor does conversion between
// the products of a stage, or the exponentials of its second tile between those of the first, gain anything.

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

__device__ __forceinline__ v4f mfma16h(const U4& a, const U4& b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
// the scale of byte I of four, which the converters read from the exponent bits alone
template <int I>
__device__ __forceinline__ float scale_at(unsigned w) {
    return __uint_as_float(I == 0 ? w << 23 : I == 1 ? w << 15 : I == 2 ? w << 7 : w >> 1);
}
template <int SEL, bool HALF>
__device__ __forceinline__ unsigned pair_of(unsigned codes, float scale) {
    if constexpr (HALF) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, SEL));
    else return bf16_of<SEL>(codes, scale);
}
// four scale bytes with e in [-23, 8]: 104 .. 135 (a byte past 231 disturbs the next one, and is found itself)
__device__ __forceinline__ bool in_window(unsigned bytes) { return ((bytes + 0x18181818u) & 0xe0e0e0e0u) == 0x80808080u; }
__device__ __forceinline__ unsigned pack_half(float a, float b) {
    const v2f x = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(x, v2h));
}

// x less the lower or upper half of two fp16 numbers, exact for what was rounded from it: one instruction, where the compiler
// takes a conversion and a subtraction (48 trees of 32 175 us, now 172; 2 x 131072 in fp16 515, now 501)
template <int UPPER>
__device__ __forceinline__ float less_half(float x, unsigned h) {
    float d;
    if constexpr (UPPER) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "v"(x));
    else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "v"(x));
    return d;
}

// a barrier for what is in LDS: __syncthreads would wait for the loads of later stages too
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <class T, int NB>
struct TreeGeo {
    static constexpr bool KHALF = !__is_same(T, bf16_t);      // keys in fp16 too
    static constexpr int W = 4, HD = 32 * NB;
    static constexpr int NQ = 2;                              // row tiles of a wave
    static constexpr int TILES = 2;                           // of a stage
    static constexpr int KU = 2 * NB * TILES, VU = NB * TILES;  // units of a stage: a step's 16 keys of 32 dims, a tile's values of 32 dims
    static constexpr int KN = (KU + W - 1) / W, VN = (VU + W - 1) / W;
    static constexpr int KBYTES = KU * 1024, STAGE = KBYTES + VU * 2048;
};

template <class T, int NB>
__global__ __launch_bounds__(256, 2) void kv4_tree_shared_kernel(Kv4TreeArgs ta, Kv4Run run) {
    using G = TreeGeo<T, NB>;
    constexpr int W = G::W, NQ = G::NQ, TILES = G::TILES, HD = G::HD, NT = 2 * NB;
    const Kv4Args& a = ta.kv;
    __shared__ __attribute__((aligned(16))) unsigned char mem[2 * G::STAGE];
    __shared__ int slow_at, redo, cleaned;  // the first stage that fp16 does not take; the first that some wave has left; whether values were taken out

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int kvh = __builtin_amdgcn_readfirstlane(blockIdx.x % a.n_kv), rt = __builtin_amdgcn_readfirstlane(blockIdx.x / a.n_kv);
    const int block = blockIdx.y;
    const int group = a.n_q / a.n_kv;
    const int heads = group < 16 ? group : 16;         // heads of a row tile
    const int toks = group < 16 ? 16 / group : 1;      // tokens of a row tile
    const float c2 = fabsf(a.scale) * kLog2e;
    const unsigned flip = a.scale < 0.0f ? 0x80008000u : 0u;  // of the queries' signs
    const size_t nc = kv4_code_bytes(a.n_kv, HD, a.page_size), ns = kv4_scale_bytes(a.n_kv, HD, a.page_size), pb = 2 * (nc + ns);
    const uint8_t* codes = a.cache + (size_t)kvh * a.page_size * (HD / 2);
    const uint8_t* scales = a.cache + 2 * nc + (size_t)kvh * NB * a.page_size;

    // A wave's share of a stage as loaded. Unit u of the keys is the 16 keys of step s and the 32 dims of block b of
    // tile t, u = (t * 2 + s) * NB + b; of the values the 32 keys and the 32 dims of block b, u = t * NB + b. (A wave whose last
    // unit is behind the last one loads unit 0 instead.)
    // (The bytes of scales and of values' codes are loaded as the four that hold them: of a byte that is kept for later
    // the compiler clears the rest at once, and so waits for it.)
    struct Raw {
        unsigned kc[G::KN], kb[G::KN], vc[G::VN][8], vb[G::VN][2];
        unsigned gone;  // bits of the tiles that have no page
    };
    const unsigned sh = 8 * (c & 3);  // of the lane's byte in the four
    unsigned k_at[G::KN], ks_at[G::KN], v_at[G::VN], vs_at[G::VN];  // offsets of the lane's bytes from the tile's first
    int k_tile[G::KN], v_tile[G::VN], k_to[G::KN], v_to[G::VN];     // the unit's tile, and where it goes
#pragma unroll
    for (int i = 0; i < G::KN; i++) {
        const int u = i * W + wave < G::KU ? i * W + wave : 0, b = u % NB, row = 8 * (c >> 2) + (c & 3) + 4 * (u / NB & 1);
        k_tile[i] = u / (2 * NB);
        k_at[i] = row * (HD / 2) + b * 16 + g * 4;
        ks_at[i] = b * a.page_size + (row & ~3);
        k_to[i] = u * 1024;
    }
#pragma unroll
    for (int i = 0; i < G::VN; i++) {
        const int u = i * W + wave < G::VU ? i * W + wave : 0, b = u % NB;
        v_tile[i] = u / NB;
        v_at[i] = 8 * g * (HD / 2) + b * 16 + (c & ~3);
        vs_at[i] = b * a.page_size + 8 * g;
        v_to[i] = G::KBYTES + u * 2048;
    }

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
    const int s0 = uniform_entry(a.start, seq), s1 = uniform_entry(a.start, seq + 1);
    const int q0 = s0 < 0 ? 0 : s0;
    const int n = (s1 < a.total ? s1 : a.total) - q0;
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
    const int base = len - n;  // the first new token, before the first key where more are new than there are
    const int k_begin = t_begin * kTile, k_end = t_end * kTile < len ? t_end * kTile : len;
    const int stages = k_end > k_begin ? (k_end - k_begin + TILES * kTile - 1) / (TILES * kTile) : 0;
    const int open = base < k_end ? base : k_end;  // behind the last key that all rows see
    const int open_stages = (k_end - k_begin) / (TILES * kTile);  // of keys that are all there
    const int subs = (n + toks - 1) / toks * run.head_tiles;  // row tiles of the sequence

    for (int r0 = rt * (NQ * W); r0 < subs; r0 += run.tok_tiles * (NQ * W)) {
        // the pages of a stage's tiles (behind the last tile the first once more, not used)
        struct Pages {
            int at[TILES];
        };
        auto tile_of = [&](int stage, int t) {
            const int k = k_begin + (stage * TILES + t) * kTile;
            return k < k_end ? (unsigned)k / kTile : 0u;
        };
        auto pages_of = [&](int stage) {
            Pages p;
#pragma unroll
            for (int t = 0; t < TILES; t++) {  // (a number behind the table is looked at when it is used: a scalar load is not waited for here)
                const int pn = (int)page_no(run, tile_of(stage, t));
                p.at[t] = uniform_entry(table, pn < a.ld_table ? pn : 0);
            }
            return p;
        };
        // (always as many loads, so that the waits for one stage can count those of the next)
        auto load = [&](int stage, const Pages& p, Raw& x) {
            const uint8_t *tc[TILES], *ts[TILES];
            x.gone = 0;
#pragma unroll
            for (int t = 0; t < TILES; t++) {
                const unsigned tile = tile_of(stage, t), pn = page_no(run, tile), slot = (tile - pn * run.per_page) * kTile;
                const bool there = pn < (unsigned)a.ld_table && (unsigned)p.at[t] < (unsigned)a.n_pages;
                const size_t at = (size_t)__builtin_amdgcn_readfirstlane(there ? p.at[t] : 0) * pb;
                x.gone |= (there ? 0u : 1u) << t;
                tc[t] = codes + at + slot * (HD / 2);
                ts[t] = scales + at + slot;
            }
#pragma unroll
            for (int i = 0; i < G::KN; i++) {
                const int t = k_tile[i];
                x.kc[i] = *reinterpret_cast<const uint32_t*>((t ? tc[1] : tc[0]) + k_at[i]);
                x.kb[i] = *reinterpret_cast<const uint32_t*>((t ? ts[1] : ts[0]) + ks_at[i]);
            }
#pragma unroll
            for (int i = 0; i < G::VN; i++) {
                const int t = v_tile[i];
                const auto w = *reinterpret_cast<const Pack<unsigned, 2>*>((t ? ts[1] : ts[0]) + ns + vs_at[i]);
                x.vb[i][0] = w.v[0];
                x.vb[i][1] = w.v[1];
                const uint8_t* vp = (t ? tc[1] : tc[0]) + nc;
#pragma unroll
                for (int k = 0; k < 8; k++) x.vc[i][k] = *reinterpret_cast<const uint32_t*>(vp + (v_at[i] + k * (HD / 2)));
            }
        };
        // whether a lane holds a value that fp16 does not take exactly; zeros do not count, but what may not be finite does
        auto outside = [&](const Raw& x) -> bool {
            bool ok = true;
#pragma unroll
            for (int i = 0; i < G::KN; i++) ok = ok && (!G::KHALF || in_window(x.kb[i]));
#pragma unroll
            for (int i = 0; i < G::VN; i++) ok = ok && in_window(x.vb[i][0]) && in_window(x.vb[i][1]);
            if (__builtin_expect(!__any(!ok), 1)) return false;
            bool bad = false;
#pragma unroll
            for (int i = 0; i < G::KN; i++) {
                const unsigned byte = x.kb[i] >> sh & 255u;
                if (G::KHALF) bad |= byte >= kKv4LargeByte || (byte - 104u >= 32u && (x.kc[i] & 0x77777777u));
            }
#pragma unroll
            for (int i = 0; i < G::VN; i++)
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const unsigned byte = x.vb[i][k >> 2] >> (8 * (k & 3)) & 255u;
                    bad |= byte >= kKv4LargeByte || (byte - 104u >= 32u && (x.vc[i][k] >> sh & 0x77u));
                }
            return __any(bad);
        };
        // converts a wave's share of a stage into LDS
        auto put = [&]<bool SLOW>(int stage, const Raw& x) {
            unsigned char* buf = mem + (stage & 1) * G::STAGE + lane * 16;
#pragma unroll
            for (int i = 0; i < G::KN; i++) {
                constexpr bool H = G::KHALF && !SLOW;
                const float sc = __uint_as_float(__builtin_amdgcn_alignbit(x.kb[i], x.kb[i], sh + 9));  // the byte at the exponent's bits
                const U4 k{{pair_of<0, H>(x.kc[i], sc), pair_of<1, H>(x.kc[i], sc), pair_of<2, H>(x.kc[i], sc), pair_of<3, H>(x.kc[i], sc)}};
                if (G::KU % W == 0 || i * W + wave < G::KU) *reinterpret_cast<U4*>(buf + k_to[i]) = k;
            }
#pragma unroll
            for (int i = 0; i < G::VN; i++) {
                constexpr bool H = !SLOW;
                unsigned z[8];
                z[0] = pair_of<0, H>(x.vc[i][0] >> sh, scale_at<0>(x.vb[i][0]));
                z[1] = pair_of<0, H>(x.vc[i][1] >> sh, scale_at<1>(x.vb[i][0]));
                z[2] = pair_of<0, H>(x.vc[i][2] >> sh, scale_at<2>(x.vb[i][0]));
                z[3] = pair_of<0, H>(x.vc[i][3] >> sh, scale_at<3>(x.vb[i][0]));
                z[4] = pair_of<0, H>(x.vc[i][4] >> sh, scale_at<0>(x.vb[i][1]));
                z[5] = pair_of<0, H>(x.vc[i][5] >> sh, scale_at<1>(x.vb[i][1]));
                z[6] = pair_of<0, H>(x.vc[i][6] >> sh, scale_at<2>(x.vb[i][1]));
                z[7] = pair_of<0, H>(x.vc[i][7] >> sh, scale_at<3>(x.vb[i][1]));
                U4 lo, hi;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    lo.u[j] = __builtin_amdgcn_perm(z[2 * j + 1], z[2 * j], 0x05040100u);
                    hi.u[j] = __builtin_amdgcn_perm(z[2 * j + 1], z[2 * j], 0x07060302u);
                }
                if (G::VU % W == 0 || i * W + wave < G::VU) {
                    *reinterpret_cast<U4*>(buf + v_to[i]) = lo;
                    *reinterpret_cast<U4*>(buf + v_to[i] + 1024) = hi;
                }
            }
        };
        // What no row sees is taken out, it may be anything; and so is, of the new tokens, what may not be
        // finite and must not meet the zero weights of rows that do not see it: it is put in as NaN at the end.
        auto clean = [&]<bool SLOW>(int stage, Raw& x) {
#pragma unroll
            for (int i = 0; i < G::VN; i++) {
                const int t = v_tile[i], key = k_begin + (stage * TILES + t) * kTile + 8 * g;
                const bool gone = x.gone >> t & 1u;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const unsigned byte = x.vb[i][k >> 2] >> (8 * (k & 3)) & 255u;
                    const bool nan = SLOW && !gone && key + k >= base && key + k < k_end && byte >= kKv4LargeByte;
                    if (nan) cleaned = 1;
                    if (nan || gone || key + k >= k_end) {
                        x.vc[i][k] = 0;
                        x.vb[i][k >> 2] = (x.vb[i][k >> 2] & ~(255u << (8 * (k & 3)))) | 127u << (8 * (k & 3));
                    }
                }
            }
        };

        if (threadIdx.x == 0) {
            slow_at = redo = 0x7fffffff;
            cleaned = 0;
        }
        Raw now;
        load(0, pages_of(0), now);
        Pages pages = pages_of(1);

        int tok[NQ];  // this lane's row of each row tile, -1 for none
        U4 qv[NQ][NB];
#pragma unroll
        for (int z = 0; z < NQ; z++) {
            const int sub = r0 + wave * NQ + z, hh = sub % run.head_tiles * 16 + c % heads, t = sub / run.head_tiles * toks + c / heads;
            const bool ok = c < heads * toks && t < n && hh < group;
            tok[z] = ok ? t : -1;
            // (rows without a query read the sequence's first one and take zeros)
            const T* qrow = static_cast<const T*>(a.Q) + (size_t)(q0 + (ok ? t : 0)) * a.ldq + (kvh * group + (ok ? hh : 0)) * HD + 8 * g;
            unsigned keep = ok ? ~0u : 0u;
            asm volatile("" : "+v"(keep));
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const U4 q = *reinterpret_cast<const U4*>(qrow + 32 * b);
#pragma unroll
                for (int j = 0; j < 4; j++) qv[z][b].u[j] = (q.u[j] ^ flip) & keep;
            }
        }
        // bits of the keys key .. key + 7 that this lane's row of row tile z sees
        auto seen = [&](int z, int key) -> unsigned {
            const int t = key - base, have = n - t;
            const uint32_t* words = ta.see + (int64_t)(q0 + tok[z]) * ta.ld_see;
            auto word = [&](int k) -> uint32_t { return k < 0 ? ~0u : tok[z] >= 0 && k < ta.ld_see ? words[k] : 0u; };
            const uint64_t two = (uint64_t)word((t >> 5) + 1) << 32 | word(t >> 5);
            const unsigned bits = (unsigned)(two >> (t & 31)) & 0xffu;
            return tok[z] < 0 || have <= 0 ? 0u : have < 8 ? bits & ((1u << have) - 1) : bits;
        };

        v4f o[NQ][NT] = {};
        float m[NQ], l[NQ];  // the reference of the weights, in log2, and their sum
#pragma unroll
        for (int z = 0; z < NQ; z++) m[z] = -INFINITY, l[z] = 0.0f;
        // The reference only has to keep the weights in range: it follows when a row's maximum has passed it by `most`, to `lead` below
        // that, so most tiles rescale nothing. It is a whole number, to which others are added without rounding up to 2^24. (Past 2^26,
        // where fp32's steps are above 2 `lead`, it takes the maximum itself.)
        auto follow = [&](const float (&top)[NQ], float lead, float most) {
            bool grown = false;
#pragma unroll
            for (int z = 0; z < NQ; z++) grown |= top[z] - m[z] > most;  // (not where a row has seen nothing)
            if (__builtin_expect(__any(grown), 0)) {
#pragma unroll
                for (int z = 0; z < NQ; z++) {
                    const float mx = rows_max(top[z]), to = floorf(mx - lead);
                    const float mn = fmaxf(m[z], mx - to > most ? mx : to);
                    const float alpha = __builtin_amdgcn_exp2f(m[z] - (mn == -INFINITY ? 0.0f : mn));
                    m[z] = mn;
                    l[z] *= alpha;
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int r = 0; r < 4; r++) o[z][t][r] *= alpha;
                }
            }
        };

        // A wave's tiles of a stage, in fp16. Weights come from the rounded scores that their reference was taken from, and it is
        // subtracted as it is: from unrounded ones, or with the 2^9 added to it first, they would pass fp16's range
        // where scores pass 2^24 (48 trees of 32 took 171 us without this, 176 with it).
        int next = 0x7fffffff;  // the stage from which on this wave leaves all of them to the parts in bf16
        auto fast_step = [&](int stage) {
#pragma clang fp contract(off)
            const unsigned char* buf = mem + (stage & 1) * G::STAGE + lane * 16;
            const int k0 = k_begin + stage * TILES * kTile;
            v4f s[NQ][TILES][2] = {};
#pragma unroll
            for (int ch = 0; ch < TILES; ch++)
#pragma unroll
                for (int sub = 0; sub < 2; sub++)
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const U4 k = *reinterpret_cast<const U4*>(buf + ((ch * 2 + sub) * NB + b) * 1024);
#pragma unroll
                        for (int z = 0; z < NQ; z++) s[z][ch][sub] = G::KHALF ? mfma16h(k, qv[z][b], s[z][ch][sub]) : mfma16(k, qv[z][b], s[z][ch][sub]);
                    }
#pragma unroll
            for (int z = 0; z < NQ; z++)
#pragma unroll
                for (int i = 0; i < 8 * TILES; i++) s[z][i >> 3][i >> 2 & 1][i & 3] *= c2;
            if (k0 + TILES * kTile > open) {
#pragma unroll
                for (int z = 0; z < NQ; z++)
#pragma unroll
                    for (int ch = 0; ch < TILES; ch++) {  // (behind the last tile of a run there may be more keys that the row sees)
                        const unsigned bits = k0 + ch * kTile < k_end ? seen(z, k0 + ch * kTile + 8 * g) : 0u;
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            if (!(bits >> i & 1u)) s[z][ch][i >> 2][i & 3] = -INFINITY;
                    }
            }
            float top[NQ];
#pragma unroll
            for (int z = 0; z < NQ; z++) {
                float mx = s[z][0][0][0];
#pragma unroll
                for (int i = 1; i < 8 * TILES; i++) mx = fmaxf(mx, s[z][i >> 3][i >> 2 & 1][i & 3]);
                top[z] = mx;
            }
            follow(top, 9.0f, 15.0f);
            // Where the weights of a row are all below 2^-16 of its largest, its sums are raised by what is missing for this stage, as
            // far as fp32's range goes (sums are below 2^26 times the number of keys). What lies further down is left to the parts in bf16.
            float mu[NQ], up[NQ];
            bool low = false;
#pragma unroll
            for (int z = 0; z < NQ; z++) {
                mu[z] = m[z] == -INFINITY ? 0.0f : m[z];
                low |= top[z] - m[z] < -7.0f && top[z] > -INFINITY;
            }
            low = __any(low);
            auto raise = [&](int sign) {
#pragma unroll
                for (int z = 0; z < NQ; z++) {
                    const float f = __builtin_ldexpf(1.0f, sign * (int)up[z]);
                    l[z] *= f;
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int r = 0; r < 4; r++) o[z][t][r] *= f;
                }
            };
            if (__builtin_expect(low, 0)) {
                const float up_most = 106.0f - run.lift;  // 100 less log2 of the keys
                bool far = false;
#pragma unroll
                for (int z = 0; z < NQ; z++) {
                    const float mx = rows_max(top[z]), k = mx > -INFINITY ? floorf(m[z] - mx + 9.0f) : 0.0f, base = mu[z];
                    mu[z] -= fminf(fmaxf(k, 0.0f), up_most);
                    up[z] = base - mu[z];
                    far |= k > up_most + 16.0f || mx - mu[z] > 15.0f;  // (the latter where the reference had to be rounded)
                }
                if (__any(far)) {
                    next = stage;
                    if (lane == 0) {
                        atomicMin(&slow_at, stage + 2);  // (which the others find out behind the next barrier)
                        atomicMin(&redo, stage);
                    }
                    return;
                }
                raise(1);
            }
#pragma unroll
            for (int ch = 0; ch < TILES; ch++) {
                U4 pw[NQ][2];
#pragma unroll
                for (int z = 0; z < NQ; z++) {
                    float x[8], sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        x[i] = __builtin_amdgcn_exp2f(s[z][ch][i >> 2][i & 3] - mu[z]);
                        sum += x[i];
                    }
                    l[z] += sum;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        pw[z][0].u[j] = pack_half(x[2 * j], x[2 * j + 1]);
                        pw[z][1].u[j] = pack_half(less_half<0>(x[2 * j], pw[z][0].u[j]), less_half<1>(x[2 * j + 1], pw[z][0].u[j]));
                    }
                }
                const unsigned char* vbuf = buf + G::KBYTES + ch * NB * 2048;
#pragma unroll
                for (int d = 0; d < NT; d++) {
                    const U4 v = *reinterpret_cast<const U4*>(vbuf + d * 1024);
#pragma unroll
                    for (int z = 0; z < NQ; z++)
#pragma unroll
                        for (int q = 1; q >= 0; q--) o[z][d] = mfma16h(v, pw[z][q], o[z][d]);
                }
            }
            if (__builtin_expect(low, 0)) raise(-1);
        };
        // one tile of any values and masks, in bf16: fp16 queries and all weights in two parts
        auto slow_step = [&](const unsigned char* buf, int tile, int k0, bool there) {
#pragma clang fp contract(off)
            v4f s[NQ][2] = {};
#pragma unroll
            for (int sub = 0; sub < 2; sub++)
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const U4 k = *reinterpret_cast<const U4*>(buf + ((tile * 2 + sub) * NB + b) * 1024);
#pragma unroll
                    for (int z = 0; z < NQ; z++) {
                        if constexpr (!G::KHALF) {
                            s[z][sub] = mfma16(k, qv[z][b], s[z][sub]);
                        } else {
                            U4 hi, lo;
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const v2h h = __builtin_bit_cast(v2h, qv[z][b].u[j]);
                                const float x = (float)h[0], y = (float)h[1];
                                hi.u[j] = pack_upper(x, y);
                                lo.u[j] = pack_upper(x - upper_part(x), y - upper_part(y));
                            }
                            s[z][sub] = mfma16(k, lo, s[z][sub]);
                            s[z][sub] = mfma16(k, hi, s[z][sub]);
                        }
                    }
                }
            float top[NQ];
            unsigned bits[NQ];
#pragma unroll
            for (int z = 0; z < NQ; z++) {
                bits[z] = seen(z, k0 + 8 * g);
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float x = there ? s[z][i >> 2][i & 3] * c2 : NAN;
                    s[z][i >> 2][i & 3] = x;
                    if (bits[z] >> i & 1u) mx = fmaxf(mx, x);
                }
                top[z] = mx;
            }
            follow(top, 0.0f, 6.0f);
            U4 pw[NQ][2];
#pragma unroll
            for (int z = 0; z < NQ; z++) {
                const float mu = m[z] == -INFINITY ? 0.0f : m[z];
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    x[i] = bits[z] >> i & 1u ? __builtin_amdgcn_exp2f(s[z][i >> 2][i & 3] - mu - run.lift) : 0.0f;
                    l[z] += x[i];
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    pw[z][0].u[j] = pack_upper(x[2 * j], x[2 * j + 1]);
                    pw[z][1].u[j] = pack_upper(x[2 * j] - upper_part(x[2 * j]), x[2 * j + 1] - upper_part(x[2 * j + 1]));
                }
            }
            const unsigned char* vbuf = buf + G::KBYTES + tile * NB * 2048;
#pragma unroll
            for (int d = 0; d < NT; d++) {
                const U4 v = *reinterpret_cast<const U4*>(vbuf + d * 1024);
#pragma unroll
                for (int z = 0; z < NQ; z++) {
                    o[z][d] = mfma16(v, pw[z][1], o[z][d]);
                    o[z][d] = mfma16(v, pw[z][0], o[z][d]);
                }
            }
        };

        __syncthreads();  // slow_at is set
        // Stage i + 1 is converted behind the barrier that ends the work on stage i - 1, whose buffer it takes, and stage i + 2
        // loaded while stage i is worked on. A stage's scales are looked at before that barrier, so that all waves agree.
        int i = -1;
        for (bool go = true; go; ) {
            const int j = i + 1;
            go = j < stages;
            if (go && j >= open_stages) clean.template operator()<false>(j, now);
            if (go && (now.gone || outside(now)) && lane == 0) atomicMin(&slow_at, j);
            lds_barrier();
            go = go && __builtin_amdgcn_readfirstlane(slow_at) > j;
            if (go) {
                put.template operator()<false>(j, now);
                load(j + 1, pages, now);
                pages = pages_of(j + 2);
            }
            if (i >= 0 && i < next) fast_step(i);
            i = j;
        }
        __syncthreads();
        next = next < i ? next : i;
        i = __builtin_amdgcn_readfirstlane(redo) < i ? __builtin_amdgcn_readfirstlane(redo) : i;
        // what is left, from stage i on, for a wave from `next` on: sums are of weights 2^-lift as large
        const float to_slow = __builtin_amdgcn_exp2f(-run.lift);
        if (i < stages) {
#pragma unroll
            for (int z = 0; z < NQ; z++) {
                l[z] *= to_slow;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) o[z][t][r] *= to_slow;
            }
            load(i, pages_of(i), now);
            for (;;) {
                clean.template operator()<true>(i, now);
                put.template operator()<true>(i, now);
                const unsigned gone = now.gone;
                load(i + 1, pages_of(i + 1), now);
                __syncthreads();
#pragma unroll 1
                for (int ch = 0; ch < TILES; ch++) {
                    const int k0 = k_begin + (i * TILES + ch) * kTile;
                    if (i >= next && k0 < k_end) slow_step(mem + (i & 1) * G::STAGE + lane * 16, ch, k0, !(gone >> ch & 1u));
                }
                if (++i >= stages) break;
            }
        } else {
#pragma unroll
            for (int z = 0; z < NQ; z++) {
                l[z] *= to_slow;
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) o[z][t][r] *= to_slow;
            }
        }
        __syncthreads();
        if (__builtin_amdgcn_readfirstlane(cleaned)) {
            for (int j = base < k_begin ? k_begin : base; j < k_end; j++) {
                const unsigned pn = page_no(run, (unsigned)j / kTile);
                const int page = uniform_page(table, a.ld_table, a.n_pages, pn);
                if (page < 0) continue;  // NaN through its scores
                const uint8_t* vs = scales + (size_t)page * pb + ns + (j - pn * a.page_size);
#pragma unroll
                for (int z = 0; z < NQ; z++) {
                    const bool sees = seen(z, j) & 1u;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const bool nan = sees && vs[(size_t)b * a.page_size] >= kKv4LargeByte;
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (nan) o[z][2 * b][r] = o[z][2 * b + 1][r] = NAN;
                    }
                }
            }
        }

        // a lane holds 8 neighbouring dims of its row in each block
#pragma unroll
        for (int z = 0; z < NQ; z++) l[z] = rows_sum(l[z]);
#pragma unroll
        for (int z = 0; z < NQ; z++) {
            if (tok[z] < 0) continue;
            const int rhead = kvh * group + (r0 + wave * NQ + z) % run.head_tiles * 16 + c % heads;
            if (pieces == 1) {
                const float inv = l[z] == 0.0f ? 0.0f : 1.0f / l[z];
                T* to = static_cast<T*>(a.out) + (size_t)(q0 + tok[z]) * a.ldo + rhead * HD + 8 * g;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    Pack<T, 8> y;
#pragma unroll
                    for (int r = 0; r < 4; r++) y.v[2 * r] = (T)(o[z][2 * b][r] * inv), y.v[2 * r + 1] = (T)(o[z][2 * b + 1][r] * inv);
                    *reinterpret_cast<Pack<T, 8>*>(to + 32 * b) = y;
                }
            } else {
                const size_t rr = ((size_t)slot * run.tok_cap + tok[z]) * a.n_q + rhead;
                float* to = run.o + rr * HD + 8 * g;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    *reinterpret_cast<float4*>(to + 32 * b) = make_float4(o[z][2 * b][0], o[z][2 * b + 1][0], o[z][2 * b][1], o[z][2 * b + 1][1]);
                    *reinterpret_cast<float4*>(to + 32 * b + 4) = make_float4(o[z][2 * b][2], o[z][2 * b + 1][2], o[z][2 * b][3], o[z][2 * b + 1][3]);
                }
                if (g == 0) *reinterpret_cast<float2*>(run.ml + rr * 2) = make_float2(m[z], l[z]);
            }
        }
        __syncthreads();  // (the next rows' or sequence's first stages take the buffers)
    }
    }
}

// row tiles of 16 queries over `rows` tokens of a sequence
int64_t row_tiles(int64_t rows, int n_q, int n_kv) {
    const int group = n_q / n_kv, toks = group <= 16 ? 16 / group : 1;
    return (rows + toks - 1) / toks * ((group + 15) / 16);
}

constexpr int attn_waves(int head_dim) { return head_dim >= 192 ? 2 : 4; }

// Row tiles that blocks have where each sequence has its own: of all that there can be, not of as many in every sequence.
int64_t row_blocks(int64_t most, int total_q, int n_seqs, int n_q, int n_kv, int nq) {
    const int64_t spread = most * n_seqs, sum = row_tiles(total_q, n_q, n_kv) / nq + (int64_t)n_seqs * ((n_q / n_kv + 15) / 16);
    return n_kv * (spread < sum ? spread : sum);
}

// Which kernel takes a call, and the row tiles of one of its blocks. Every row tile that has keys to itself reads and converts
// them again: two in registers (heads up to 128 in 16-bit types) halve that, from five on four waves share
// what is converted. Measured, us, 48 sequences mixed up to 8192 keys, 32 heads on 8, bf16, one in registers | two |
// shared: heads of 128, 4 new tokens (one row tile) 49 | 67 | 150, 8 (two) 86 | 74 | 154, 16 (four) 118 | 116 | 160, 20 (five) 146 | 158 | 163, 24 176 |
// 162 | 165, 32 (eight) 204 | 201 | 172; of 96, 16 137 | 112 | 141, 20 159 | 159 | 143; of 64, 16 83 | 98 | 110, 20 107 | 120 | 113, 32 152 | 139 | 121; of
// 32, 16 84 | 81 | 92, 20 97 | 107 | 94; 2 x 131072, heads of 128, 16 new 167 | 144 | 251, 20 258 | 262 | 252, of 64 125 | 101 | 164, 195 | 184 | 165; fp16 alike. Heads
// above 128 leave a wave no room for two row tiles, and sharing for four gains nothing: of 256, 16 new 215 | - | 230, 32 new
// 385 | - | 418, 64 new 706 | - | 1157. (Two waves sharing for four row tiles of 128: 117 and 164 for 114 and 132.)
constexpr int kSharedTiles = 5, kSharedRows = 8;  // row tiles from which on waves share, and of a block then
int rows_per_block(int total_q, int max_new, int n_q, int n_kv, int head_dim, bool half) {
    if (!half || head_dim > 128) return 1;
    const int64_t tiles = row_tiles(max_new < total_q ? max_new : total_q, n_q, n_kv);
    return tiles >= kSharedTiles ? kSharedRows : tiles == 1 ? 1 : 2;
}

// How a call runs, from sizes the host knows: equal runs of tiles (and a second kernel), or a
// block per sequence and row tiles. In registers as the attention of a causal chunk, by the same measure: a block's steps against the blocks
// that the card is short of. Shared tiles: runs, each of at least two stages, unless blocks of sequences fill the card four times (us, runs |
// sequences, heads of 128: 4 x 1000 keys, 32 new 30 | 54, 16 x 3000, 64 new 127 | 149, 48 mixed up to 8192, 32 new 180 | 407, 100 new 581 | 703, 200
// new 1023 | 1077, 64 x 4000, 64 new 507 | 475, 120 new 999 | 927, 200 x 800, 40 new 419 | 359; of 64 21 | 37, 90 | 97, 128 | 270, 402 | 492, 708 | 711, 341 |
// 309, 674 | 603, 301 | 237); no more runs than are under way at once (2 x 131072, 200 new: 9 runs 1692, 10 2614).
Kv4Run plan(int total_q, int n_seqs, int max_new, int64_t max_len, int n_q, int n_kv, int head_dim, int nq) {
    Kv4Run r{};
    max_new = max_new < total_q ? max_new : total_q;
    r.head_tiles = (n_q / n_kv + 15) / 16;
    const int64_t tiles_of_rows = (row_tiles(max_new, n_q, n_kv) + nq - 1) / nq;
    const int64_t most = ((int64_t)1 << 23) / n_kv;  // (a launch has less than 2^32 threads; a block loops over the rest)
    r.tok_tiles = (int)(tiles_of_rows < most ? tiles_of_rows : most);
    const int64_t blocks = row_blocks(r.tok_tiles, total_q, n_seqs, n_q, n_kv, nq);
    const bool shared = nq == kSharedRows;
    const int64_t card = shared || attn_waves(head_dim) == 4 ? 512 : 1024;
    const int64_t steps = max_len / (kTile * attn_waves(head_dim));
    if (shared ? blocks >= 4 * card || max_len <= 8 * kTile : steps <= 64 && steps * (card - blocks) <= 12 * card) return r;
    const int64_t tiles = (max_len + kTile - 1) / kTile * n_seqs;
    int64_t runs = (card * n_seqs + (shared ? 0 : blocks - 1)) / blocks;
    const int64_t rounds = tiles / (shared ? 4 : 2 * attn_waves(head_dim));
    runs = runs < rounds ? runs : rounds;
    runs = runs < kMaxPieces ? runs : kMaxPieces;
    r.runs = runs <= 1 ? 0 : (int)runs;
    r.tok_cap = max_new;
    r.slots = r.runs + n_seqs;
    if (plan_bytes(r, 0, n_q, head_dim) > (size_t)1 << 28) r.runs = 0;  // pieces of long chunks
    return r;
}

template <class T, int PQ, int PP, int NB, int NQ>
void run_tree_nb(const Kv4TreeArgs& a, const Kv4Run& r, hipStream_t st) {
    constexpr int W = attn_waves(32 * NB);
    kv4_tree_kernel<T, NB, PQ, PP, W, NQ><<<dim3(a.kv.n_kv * r.tok_tiles, r.runs ? r.runs : a.kv.n_seqs), W * 64, 0, st>>>(a, r);
    VLA_LAUNCH_CHECK();
}

template <class T, int PQ, int PP, int NB>
void run_tree_nq(const Kv4TreeArgs& a, const Kv4Run& r, int nq, hipStream_t st) {
    if constexpr (sizeof(T) == 2 && NB <= 4) {
        if (nq == kSharedRows) {
            kv4_tree_shared_kernel<T, NB><<<dim3(a.kv.n_kv * r.tok_tiles, r.runs ? r.runs : a.kv.n_seqs), 256, 0, st>>>(a, r);
            VLA_LAUNCH_CHECK();
            return;
        }
        if (nq == 2) return run_tree_nb<T, PQ, PP, NB, 2>(a, r, st);
    }
    run_tree_nb<T, PQ, PP, NB, 1>(a, r, st);
}

template <class T, int PQ, int PP>
void run_tree(const Kv4TreeArgs& ta, const Kv4Run& r, int nq, hipStream_t st) {
    const Kv4Args& a = ta.kv;
    switch (a.head_dim / 32) {
    case 1: run_tree_nq<T, PQ, PP, 1>(ta, r, nq, st); break;
    case 2: run_tree_nq<T, PQ, PP, 2>(ta, r, nq, st); break;
    case 3: run_tree_nq<T, PQ, PP, 3>(ta, r, nq, st); break;
    case 4: run_tree_nq<T, PQ, PP, 4>(ta, r, nq, st); break;
    case 6: run_tree_nq<T, PQ, PP, 6>(ta, r, nq, st); break;
    default: run_tree_nq<T, PQ, PP, 8>(ta, r, nq, st); break;
    }
    if (!r.runs) return;
    if (r.runs > 8 * a.n_seqs) kv4_join_kernel<T, 256><<<a.total * a.n_q, 256, 0, st>>>(a, r);
    else kv4_join_kernel<T, 64><<<a.total * a.n_q, 64, 0, st>>>(a, r);
    VLA_LAUNCH_CHECK();
}

}  // namespace

size_t kv4_tree_attention_work_bytes(int total_q, int n_seqs, int max_new, int max_len, int n_q, int n_kv, int head_dim) {
    if (total_q <= 0 || n_seqs <= 0 || max_new <= 0 || max_len <= 0 || n_kv <= 0 || n_q <= 0 || n_q % n_kv || head_dim <= 0) return 0;
    // sizes that the call refuses, or that it does not split
    if (!kv4_head_dim_ok(head_dim) || n_kv > 1024 || n_q > 65536 || n_seqs > kMaxSeqs || !joins(total_q, n_q)) return 0;
    size_t most = 0;
    for (bool half : {false, true}) {
        const int nq = rows_per_block(total_q, max_new, n_q, n_kv, head_dim, half);
        const size_t b = plan_bytes(plan(total_q, n_seqs, max_new, max_len, n_q, n_kv, head_dim, nq), total_q, n_q, head_dim);
        most = b > most ? b : most;
    }
    return most;
}

void launch_kv4_tree_attention(const Kv4TreeArgs& ta, hipStream_t st) {
    const Kv4Args& a = ta.kv;
    const std::string w = "kv4_tree_attention";
    check_cache(a, "kv4_tree_attention");
    VLA_REQUIRE(a.n_q > 0 && a.n_q <= 65536 && a.n_q % a.n_kv == 0, w + ": n_q must be a multiple of n_kv up to 65536");
    VLA_REQUIRE(std::isfinite(a.scale), w + ": scale must be finite");
    VLA_REQUIRE(a.max_new >= 0 && a.max_len >= 0, w + ": max_new and max_len must not be negative");
    VLA_REQUIRE(ta.ld_see >= 1 && ta.ld_see <= 1 << 20, w + ": rows of 1 to 2^20 words");
    if (a.n_seqs == 0 || a.total == 0) return;
    VLA_REQUIRE(a.max_new >= 1, w + ": max_new must be at least 1");
    VLA_REQUIRE(a.n_seqs <= kMaxSeqs, w + ": at most 65535 sequences");
    VLA_REQUIRE(a.n_pages > 0 && a.cache && aligned(a.cache, 16), w + ": the cache must hold a page and be 16-byte aligned");
    VLA_REQUIRE(a.table && a.ld_table > 0 && a.lens && a.start, w + ": page table, lens or q_start missing");
    VLA_REQUIRE(a.out && a.Q && ta.see, w + ": null buffer");
    const int sz = dtype_size(a.dtype);
    VLA_REQUIRE(a.ldq >= a.n_q * a.head_dim && a.ldo >= a.n_q * a.head_dim, w + ": row stride shorter than heads * head_dim");
    VLA_REQUIRE(aligned(a.Q, 16) && aligned(a.out, 16) && a.ldq * sz % 16 == 0 && a.ldo * sz % 16 == 0, w + ": rows must be 16-byte aligned");
    VLA_REQUIRE((int64_t)a.total * a.n_q < (int64_t)1 << 31, w + ": too many query rows times heads");
    const int nq = rows_per_block(a.total, a.max_new, a.n_q, a.n_kv, a.head_dim, sz == 2);
    Kv4Run r = plan(a.total, a.n_seqs, a.max_new, a.max_len, a.n_q, a.n_kv, a.head_dim, nq);
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
    // is not known, there are 2^16 blocks or twice as many as can have work; they take several row tiles then.
    const int64_t busy = row_blocks(r.tok_tiles, a.total, a.n_seqs, a.n_q, a.n_kv, nq), grid = 2 * busy > 1 << 16 ? 2 * busy : 1 << 16;
    const int64_t most = grid / ((int64_t)a.n_kv * (r.runs ? r.runs : a.n_seqs));
    if (r.tok_tiles > most) r.tok_tiles = (int)(most < 1 ? 1 : most);
    int log2_n = 0;
    while ((int64_t)1 << log2_n < (int64_t)a.ld_table * a.page_size) log2_n++;
    r.lift = 6.0f + (float)log2_n;
    r.wscale = a.dtype == kF32 ? std::ldexp(1.0f, -6 - log2_n) : 1.0f;
    if (a.dtype == kF32) run_tree<float, 3, 3>(ta, r, nq, st);
    else if (a.dtype == kBf16) run_tree<bf16_t, 1, 2>(ta, r, nq, st);
    else run_tree<f16_t, 2, 2>(ta, r, nq, st);
}

}  // namespace hip
}  // namespace vla
