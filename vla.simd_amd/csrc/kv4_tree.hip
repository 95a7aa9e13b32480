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
        int cleaned = 0;
        auto step = [&](Kv4Tile<NB>& t, int k0) {
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
                    l[z] *= alpha;
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int r = 0; r < 4; r++) o[z][t][r] *= alpha;
                }
                // Weights reach 2^6, and no sum over all keys may leave fp32's range: they are 2^-lift as large, in the
                // product alone where they have 24 bits, as their exponent's rounding to 2^-19 would show.
                const float mu = (m[z] == -INFINITY ? 0.0f : m[z]) + (PP == 3 ? 0.0f : run.lift);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    x[z][i] = __builtin_amdgcn_exp2f(x[z][i] - mu);
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

// How a call runs, from sizes the host knows: equal runs of tiles (and a second kernel), or a
// block per sequence and row tile.
Kv4Run plan(int total_q, int n_seqs, int max_new, int64_t max_len, int n_q, int n_kv, int head_dim, int nq) {
    Kv4Run r{};
    max_new = max_new < total_q ? max_new : total_q;
    r.head_tiles = (n_q / n_kv + 15) / 16;
    const int64_t tiles_of_rows = (row_tiles(max_new, n_q, n_kv) + nq - 1) / nq;
    const int64_t most = ((int64_t)1 << 23) / n_kv;  // (a launch has less than 2^32 threads; a block loops over the rest)
    r.tok_tiles = (int)(tiles_of_rows < most ? tiles_of_rows : most);
    const int64_t blocks = row_blocks(r.tok_tiles, total_q, n_seqs, n_q, n_kv, nq);
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

int rows_per_wave(int max_new, int n_q, int n_kv, int head_dim) { return 1; }

template <class T, int PQ, int PP, int NB, int NQ>
void run_tree_nb(const Kv4TreeArgs& a, const Kv4Run& r, hipStream_t st) {
    constexpr int W = attn_waves(32 * NB);
    kv4_tree_kernel<T, NB, PQ, PP, W, NQ><<<dim3(a.kv.n_kv * r.tok_tiles, r.runs ? r.runs : a.kv.n_seqs), W * 64, 0, st>>>(a, r);
    VLA_LAUNCH_CHECK();
}

template <class T, int PQ, int PP>
void run_tree(const Kv4TreeArgs& ta, const Kv4Run& r, int nq, hipStream_t st) {
    const Kv4Args& a = ta.kv;
    switch (a.head_dim / 32) {
    case 1: run_tree_nb<T, PQ, PP, 1, 1>(ta, r, st); break;
    case 2: run_tree_nb<T, PQ, PP, 2, 1>(ta, r, st); break;
    case 3: run_tree_nb<T, PQ, PP, 3, 1>(ta, r, st); break;
    case 4: run_tree_nb<T, PQ, PP, 4, 1>(ta, r, st); break;
    case 6: run_tree_nb<T, PQ, PP, 6, 1>(ta, r, st); break;
    default: run_tree_nb<T, PQ, PP, 8, 1>(ta, r, st); break;
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
    const int nq = rows_per_wave(max_new, n_q, n_kv, head_dim);
    return plan_bytes(plan(total_q, n_seqs, max_new, max_len, n_q, n_kv, head_dim, nq), total_q, n_q, head_dim);
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
    const int nq = rows_per_wave(a.max_new, a.n_q, a.n_kv, a.head_dim);
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
    while (1 << log2_n < a.ld_table * a.page_size) log2_n++;
    r.lift = 6.0f + (float)log2_n;
    r.wscale = a.dtype == kF32 ? std::ldexp(1.0f, -6 - log2_n) : 1.0f;
    if (a.dtype == kF32) run_tree<float, 3, 3>(ta, r, nq, st);
    else if (a.dtype == kBf16) run_tree<bf16_t, 1, 2>(ta, r, nq, st);
    else run_tree<f16_t, 2, 2>(ta, r, nq, st);
}

}  // namespace hip
}  // namespace vla
