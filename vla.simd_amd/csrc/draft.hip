// draft.hip - what a step with drafted tokens needs around its attention: a
// tree's positions and bits, the choice of an accepted path, and that path's place in the cache.
//
// A sequence's packed rows are the nodes of a tree: row 0 its last certain token, behind it
// the drafted ones, each with a parent of a smaller number.

#include "kv4_device.h"
#include "wave.h"

namespace vla {
namespace hip {
namespace {

// rows of sequence s, clamped to the buffer
struct Nodes {
    int first, n;
};
__device__ __forceinline__ Nodes nodes_of(const int32_t* start, int s, int total) {
    const int s0 = start[s], s1 = start[s + 1];
    const int first = s0 < 0 ? 0 : s0, end = s1 < total ? s1 : total;
    return {first, end > first ? end - first : 0};
}

// ---------------------------------------------------------------- tree ----
// depth and bits of row i: those of its parent, and its own. Latency bounds it.

// Row i of a sequence by a walk up to its root. Numbers fall on the way, so its words are
// written from the last to the first. up(at): the parent of row `at` as given.
template <class F>
__device__ __forceinline__ void walk_up(const DraftTreeArgs& a, const Nodes& nd, int s, int i, F&& up) {
    const int row = nd.first + i;
    uint32_t* see = a.see + (int64_t)row * a.ld_see;
    for (int w = a.ld_see - 1; w > i >> 5; w--) see[w] = 0;
    int depth = 0, w = i >> 5;
    uint32_t bits = 0;
    for (int at = i;;) {
        for (; w > at >> 5; w--) {
            if (w < a.ld_see) see[w] = bits;
            bits = 0;
        }
        bits |= 1u << (at & 31);
        const int p = up(at);
        if (p < 0 || p >= at) break;
        at = p;
        depth++;
    }
    for (; w >= 0; w--) {
        if (w < a.ld_see) see[w] = bits;
        bits = 0;
    }
    a.pos[row] = (int)((unsigned)a.lens[s] - (unsigned)nd.n + (unsigned)depth);
}

// A thread for each row; the parents of a block's rows are in LDS.
__global__ __launch_bounds__(256) void draft_tree_rows_kernel(DraftTreeArgs a) {
    __shared__ int32_t parent[256];
    const int row0 = blockIdx.x * 256, row = row0 + threadIdx.x;
    if (a.parent) {
        parent[threadIdx.x] = row < a.total ? a.parent[row] : -1;
        __syncthreads();
    }
    if (row >= a.total) return;
    const int s = seq_of_row(a.start, a.n_seqs, row);
    if (s >= a.n_seqs) return;
    const Nodes nd = nodes_of(a.start, s, a.total);
    if (row < nd.first || row >= nd.first + nd.n) return;
    walk_up(a, nd, s, row - nd.first, [&](int at) {
        if (!a.parent) return at - 1;
        const int r = nd.first + at;
        return r >= row0 ? parent[r - row0] : a.parent[r];
    });
}

// A wave for each sequence, 64 rows at a time: they take as many steps as the depth among them has bits, each joining a row's
// bits and depth with those of the row that it has got to; what is in front of the 64 stands in memory already.
// (256 trees of 64 rows 2.6 us, by walks 5.4; as many chains 2.8 and 13.7.)
__global__ __launch_bounds__(64) void draft_tree_wave_kernel(DraftTreeArgs a) {
    const int lane = threadIdx.x;
    for (int s = blockIdx.x; s < a.n_seqs; s += gridDim.x) {
        const Nodes nd = nodes_of(a.start, s, a.total);
        const unsigned first_pos = (unsigned)a.lens[s] - (unsigned)nd.n;
        for (int c0 = 0; c0 < nd.n; c0 += 64) {
            const int i = c0 + lane;
            int up = i < nd.n ? a.parent ? a.parent[nd.first + i] : i - 1 : -1;
            up = up >= 0 && up < i ? up : -1;
            uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
            unsigned depth = up >= 0;
            while (__any(up >= c0)) {
                const int from = up >= c0 ? up - c0 : lane;
                const uint32_t l = __shfl(lo, from), h = __shfl(hi, from), d = __shfl(depth, from);
                const int u = __shfl(up, from);
                if (up >= c0) {
                    lo |= l;
                    hi |= h;
                    depth += d;
                    up = u;
                }
            }
            if (i < nd.n) {  // (no lane reads what another one writes here: `up` is in front of the 64)
                uint32_t* see = a.see + (int64_t)(nd.first + i) * a.ld_see;
                const uint32_t* front = up >= 0 ? a.see + (int64_t)(nd.first + up) * a.ld_see : nullptr;
                const int w0 = c0 >> 5;
                for (int w = 0; w < w0 && w < a.ld_see; w++) see[w] = front ? front[w] : 0;
                if (w0 < a.ld_see) see[w0] = lo;
                if (w0 + 1 < a.ld_see) see[w0 + 1] = hi;
                for (int w = w0 + 2; w < a.ld_see; w++) see[w] = 0;
                if (up >= 0) depth += (unsigned)a.pos[nd.first + up] - first_pos;
                a.pos[nd.first + i] = (int)(first_pos + depth);
            }
            __syncthreads();  // (one wave: its stores before the loads of the next 64)
        }
    }
}

// -------------------------------------------------------------- verify ----
// A walk down the tree. At node x with children c in order, p and q the rows of x:
//   with q:    a = 0, S = 1; c is taken if u_c S q(c) < p(c) - a q(c), else
//              a += S, S = sum_v max(p(v) - a q(v), 0)
//   without:   S = 1; c is taken if u_c S < p(c) (0 for a token refused before), else S -= p(c)
// The next token is drawn from what is left at the last node, w = max(p - a q, 0) or p without
// the refused: the first v with sum of w up to v > u_next * sum of w. With r = max(p - a q, 0) / S the
// distribution left after some refusals, max(r - q, 0) is max(p - (a + S) q, 0) / S: one number stands for
// all of them, and the rows are never written.
//
// Sums are of 64 bits, so that their order moves a result only where a random number lies
// within 2^-50 of a border. A block takes a sequence. Children in front of the first refusal
// need two probabilities each; every refusal with q, and the draw, go through rows of the vocabulary. What bounds that
// is one CU: the loads' latency, four chunks at a time, and 64-bit instructions, five a value (bf16 takes as long as fp32: 29 us, 31).
// A chain of four drafted tokens over 49280 values takes 12.8 us, over 131072 17.4; 48 trees of 32 take 31, the time of the tree with most
// refusals, under 3 us each. (More blocks to a sequence would have to wait for each other.)
constexpr int kVerifyNodes = 512;   // probabilities held in LDS
constexpr int kVerifyThreads = 1024;

__device__ __forceinline__ double above_zero(double x) { return fmax(x, 0.0); }  // (0 for NaN)

template <class T>
__global__ __launch_bounds__(kVerifyThreads) void verify_kernel(VerifyArgs a) {
    constexpr int W = kVerifyThreads / 64, VEC = 16 / sizeof(T);
    __shared__ int32_t up[kVerifyNodes], tok[kVerifyNodes], refused[kVerifyNodes];
    __shared__ float us[kVerifyNodes], pc[kVerifyNodes], qc[kVerifyNodes];
    __shared__ double sums[2][W];
    __shared__ int found;
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Nodes nd = nodes_of(a.start, s, a.total);
    const int n = nd.n, V = a.vocab;
    const T* P = static_cast<const T*>(a.p) + (int64_t)nd.first * a.ldp;
    const T* Q = a.q ? static_cast<const T*>(a.q) + (int64_t)nd.first * a.ldq : nullptr;
    const int32_t* parent = a.parent ? a.parent + nd.first : nullptr;
    const int32_t* tokens = a.tokens + nd.first;
    const float* u = a.u + nd.first;
    int32_t* path = a.path + nd.first;
    if (n == 0) {
        if (tid == 0) {
            a.count[s] = 0;
            a.token[s] = -1;
        }
        return;
    }
    auto parent_at = [&](int i) { return parent ? parent[i] : i - 1; };
    auto prob = [&](const T* rows, int64_t ld, int node, int t) {
        return rows && node >= 0 && t >= 0 && t < V ? to_f32(rows[(int64_t)node * ld + t]) : 0.0f;
    };
    for (int i = tid; i < n && i < kVerifyNodes; i += kVerifyThreads) {
        const int x = parent_at(i), t = tokens[i];
        const bool ok = x >= 0 && x < i;
        up[i] = ok ? x : -1;
        tok[i] = t;
        us[i] = u[i];
        pc[i] = prob(P, a.ldp, ok ? x : -1, t);
        qc[i] = prob(Q, a.ldq, ok ? x : -1, t);
    }
    if (tid == 0) found = -1;
    __syncthreads();

    // the share of wave w: whole chunks of 64 * VEC values
    const int chunk = 64 * VEC;
    const int share = ((V + VEC + chunk - 1) / chunk + W - 1) / W * chunk;
    const T* pr = nullptr;
    const T* qr = nullptr;
    int phase = 0;
    bool wide = false;
    auto at_node = [&](int node) {
        pr = P + (int64_t)node * a.ldp;
        qr = Q ? Q + (int64_t)node * a.ldq : nullptr;
        phase = (int)(reinterpret_cast<uintptr_t>(pr) / sizeof(T) % VEC);
        wide = !qr || (int)(reinterpret_cast<uintptr_t>(qr) / sizeof(T) % VEC) == phase;
    };
    auto difference = [&](const Pack<T, VEC>& x, const Pack<T, VEC>& y, bool two, double coef, double (&w)[VEC]) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const double pv = to_f32(x.v[e]);
            w[e] = above_zero(two ? fma(-coef, (double)to_f32(y.v[e]), pv) : pv);
        }
    };
    // the weights of values v .. v + VEC - 1 (v + phase a multiple of VEC), 0 outside the row
    auto weights = [&](int v, double coef, double (&w)[VEC]) {
        const bool two = qr && coef != 0.0;
        Pack<T, VEC> x, y{};
        if (wide && v >= 0 && v + VEC <= V) {
            x = *reinterpret_cast<const Pack<T, VEC>*>(pr + v);
            if (two) y = *reinterpret_cast<const Pack<T, VEC>*>(qr + v);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const bool in = v + e >= 0 && v + e < V;
                x.v[e] = in ? pr[v + e] : (T)0.0f;
                if (two) y.v[e] = in ? qr[v + e] : (T)0.0f;
            }
        }
        difference(x, y, two, coef, w);
    };
    // Tokens refused at the node: in LDS, and past its room at the end of the path, of whose n places
    // those kept and refused never need more.
    int n_refused = 0;
    auto refused_at = [&](int j) { return j < kVerifyNodes ? refused[j] : path[n - 1 - (j - kVerifyNodes)]; };
    // (A lane holds the one of its number among the first 64, so that a chunk without any is seen at once.)
    int held = -1;
    auto drop = [&](int v, double (&w)[VEC]) {
        const int at = v - lane * VEC;
        if (n_refused <= 64 && !__any(held >= at && held < at + chunk)) return;
        for (int i = 0; i < n_refused; i++) {
            const int t = refused_at(i);
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (v + e == t) w[e] = 0.0;
        }
    };
    int turn = 0;
    // the sums of the waves, the same bits in every thread; they stay in sums[turn]
    auto all_of = [&](double sum) {
        sum = wave_sum_f64(sum);
        turn ^= 1;
        if (lane == 0) sums[turn][wave] = sum;
        __syncthreads();
        double all = 0.0;
        for (int i = 0; i < W; i++) all += sums[turn][i];
        return all;
    };
    auto plus = [&](int v, double (&w)[VEC]) {
        double sum = 0.0;
        if (n_refused) drop(v, w);
#pragma unroll
        for (int e = 0; e < VEC; e++) sum += w[e];
        return sum;
    };
    auto sum_of = [&](int v0, double coef) {  // of a lane's values of the chunk at v0, which all lanes go through
        const int v = v0 + lane * VEC;
        double w[VEC];
        weights(v, coef, w);
        return plus(v, w);
    };
    // the same of U chunks in the row, whose loads are all under way before the first is used; `two`: with q
    auto sums_of = [&]<int U, bool TWO>(int v0, double coef, double (&part)[U]) {
        Pack<T, VEC> x[U], y[U];
        const int v = v0 + lane * VEC;
#pragma unroll
        for (int i = 0; i < U; i++) {
            x[i] = *reinterpret_cast<const Pack<T, VEC>*>(pr + v + i * chunk);
            if constexpr (TWO) y[i] = *reinterpret_cast<const Pack<T, VEC>*>(qr + v + i * chunk);
        }
#pragma unroll
        for (int i = 0; i < U; i++) {
            double w[VEC];
            difference(x[i], y[i], TWO, coef, w);
            part[i] = plus(v + i * chunk, w);
        }
    };
    // the sum of what is left
    auto total_of = [&](double coef) {
        constexpr int U = 4;
        const int begin = wave * share - phase, end = begin + share < V ? begin + share : V;
        const bool two = qr && coef != 0.0;
        double sum = 0.0;
        for (int v = begin; v < end;) {
            if (wide && v >= 0 && v + U * chunk <= V && v + (U - 1) * chunk < end) {
                double part[U];
                if (two) sums_of.template operator()<U, true>(v, coef, part);
                else sums_of.template operator()<U, false>(v, coef, part);
#pragma unroll
                for (int i = 0; i < U; i++) sum += part[i];
                v += U * chunk;
            } else {
                sum += sum_of(v, coef);
                v += chunk;
            }
        }
        return all_of(sum);
    };

    int node = 0, kept = 1;
    double coef = 0.0, S = 1.0;
    bool known = false;  // S is the sum of what is left, and sums[turn] its parts
    at_node(0);
    if (tid == 0) path[0] = 0;
    for (int base = 1; base < n; base += 64) {
        const int mine = base + lane;
        unsigned long long todo = ~0ull;
        while (todo) {
            // the next child of the node among these rows
            const int x = mine < n ? (mine < kVerifyNodes ? up[mine] : parent_at(mine)) : -2;
            todo &= __ballot(x == node);
            if (!todo) break;
            const int l = __ffsll(todo) - 1, i = base + l;
            todo = l == 63 ? 0 : ~0ull << (l + 1);
            const int t = i < kVerifyNodes ? tok[i] : tokens[i];
            const double ui = i < kVerifyNodes ? us[i] : u[i];
            double pi = i < kVerifyNodes ? pc[i] : prob(P, a.ldp, node, t);
            const double qi = i < kVerifyNodes ? qc[i] : prob(Q, a.ldq, node, t);
            bool yes;
            if (Q) {
                yes = ui * S * qi < fma(-coef, qi, pi);
            } else {
                for (int j = 0; j < n_refused; j++)
                    if (refused_at(j) == t) pi = 0.0;
                yes = ui * S < pi;
            }
            if (yes) {
                node = i;
                at_node(i);
                if (tid == 0) path[kept] = i;
                kept++;
                coef = 0.0;
                S = 1.0;
                known = false;
                n_refused = 0;
                held = -1;
            } else if (Q) {
                coef += S;
                S = total_of(coef);
                known = true;
                if (!(S > 0.0)) {
                    base = n;
                    break;
                }
            } else {
                S -= pi;
                __syncthreads();
                if (tid == 0) (n_refused < kVerifyNodes ? refused[n_refused] : path[n - 1 - (n_refused - kVerifyNodes)]) = t;
                if (lane == n_refused) held = t;
                n_refused++;
                __syncthreads();
            }
        }
    }

    // the next token
    if (!known) S = total_of(coef);
    if (!(S > 0.0)) {
        n_refused = 0;
        held = -1;
        coef = 0.0;
        S = total_of(0.0);
    }
    const double want = fmax((double)a.u_next[s], 0.0) * S;
    // The part that holds it, or the last with any weight where rounding leaves none; `before`: what lies in front of it.
    auto pick = [&](double& before) {
        int at = -1, last = -1;
        double front = before;
        for (int i = 0; i < W; i++) {
            const double x = sums[turn][i];
            if (at < 0 && x > 0.0) {
                last = i;
                before = front;
                if (front + x > want) at = i;
            }
            front += x;
        }
        return at >= 0 ? at : last;
    };
    // first the wave's share, then, with all waves on that share, a 16th of it, which its wave goes through
    double before = 0.0;
    const int outer = pick(before);
    if (outer >= 0) {
        const int part = (share / chunk + W - 1) / W * chunk;
        const int first = outer * share - phase, stop = first + share < V ? first + share : V;
        const int begin = first + wave * part, end = begin + part < stop ? begin + part : stop;
        double sum = 0.0;
        for (int v = begin; v < end; v += chunk) sum += sum_of(v, coef);
        all_of(sum);
        const int inner = pick(before);
        if (wave == inner) {
            int best = -1, some = -1;  // the first value past `want`, the last with weight
            for (int v0 = begin; v0 < end && best < 0; v0 += chunk) {
                const int v = v0 + lane * VEC;
                double w[VEC], mass = 0.0;
                weights(v, coef, w);
                if (n_refused) drop(v, w);
                int mine = -1;
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    mass += w[e];
                    if (w[e] > 0.0) mine = v + e;
                }
                double incl = mass;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const double o = __shfl_up(incl, d);
                    if (lane >= d) incl += o;
                }
                const unsigned long long has = __ballot(mine >= 0), over = __ballot(mine >= 0 && before + incl > want);
                if (has) some = __builtin_amdgcn_readlane(mine, 63 - __clzll(has));
                if (over) {
                    double at = before + (incl - mass);
                    int choice = -1;
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        at += w[e];
                        if (choice < 0 && at > want && w[e] > 0.0) choice = v + e;
                    }
                    best = __builtin_amdgcn_readlane(choice < 0 ? mine : choice, __ffsll(over) - 1);
                }
                before += __shfl(incl, 63);
            }
            if (lane == 0) found = best >= 0 ? best : some;
        }
    }
    __syncthreads();
    for (int i = kept + tid; i < n; i += kVerifyThreads) path[i] = -1;
    if (tid == 0) {
        a.count[s] = kept;
        a.token[s] = found;
    }
}

// ---------------------------------------------------------------- keep ----
// Token len - n + path[i] of the cache becomes token len - n + i, in place. A block takes one head
// of a sequence; a thread moves the codes and the scale of a block of 32 values. Rows move
// forward (path[i] >= i, ascending), so what a pass over some tokens has read before
// it writes is all that its own writes can reach. Latency bounds it, of the offsets, the path, two
// entries of the table and the codes, one after the other: 8 drafted rows of one sequence, 5 heads of 64, 2.5 us; 64 rows of each of
// 64 sequences, 8 heads of 128, 3.3 us, an empty launch 2.2.
constexpr int kKeepThreads = 128;

// (a vector: an array that lives over the barriers would go to LDS by way of the launch's packet, which is in host memory: 17 us)
typedef uint32_t Codes16 __attribute__((ext_vector_type(4)));

__global__ __launch_bounds__(kKeepThreads) void kv4_keep_kernel(Kv4KeepArgs k) {
    const Kv4Args& a = k.kv;
    const int head = blockIdx.x, s = blockIdx.y, nb = a.head_dim / kKv4Block;
    const Nodes nd = nodes_of(a.start, s, a.total);
    const int len = a.lens[s], n = nd.n;
    int count = k.count[s];
    count = count < 0 ? 0 : count > n ? n : count;
    const int64_t base = (int64_t)len - n;
    if (head == 0 && threadIdx.x == 0 && k.new_lens) k.new_lens[s] = (int)(base + count);
    const size_t nc = kv4_code_bytes(a.n_kv, a.head_dim, a.page_size), ns = kv4_scale_bytes(a.n_kv, a.head_dim, a.page_size);
    const int units = 2 * nb, per = kKeepThreads / units;  // of a token; tokens of a pass
    const int tt = threadIdx.x / units, x = threadIdx.x - tt * units, part = x >= nb, b = x - part * nb;
    const int32_t* table = a.table + (size_t)s * a.ld_table;
    // the addresses of codes and scale of this thread's block at a token
    auto place = [&](int64_t tok, uint8_t*& codes, uint8_t*& scale) {
        if (tok < 0) return false;
        const int64_t no = (uint64_t)tok / (unsigned)a.page_size;
        const int slot = (int)(tok - no * a.page_size), page = kv4_page(table, a.ld_table, a.n_pages, no);
        if (page < 0) return false;
        uint8_t* pg = a.cache + (size_t)page * (2 * (nc + ns));
        codes = pg + part * nc + ((size_t)head * a.page_size + slot) * (a.head_dim / 2) + b * (kKv4Block / 2);
        scale = pg + 2 * nc + part * ns + ((size_t)head * nb + b) * a.page_size + slot;
        return true;
    };
    for (int i0 = 0; i0 < count; i0 += per) {
        const int i = i0 + tt;
        const bool on = tt < per && i < count;
        const int from = on ? k.path[nd.first + i] : 0;
        uint8_t *codes = nullptr, *scale = nullptr, *codes_to = nullptr, *scale_to = nullptr;
        const bool to = on && place(base + i, codes_to, scale_to);  // (looked up while the path is on its way)
        const bool moves = to && from != i;
        Codes16 c = {0, 0, 0, 0};
        int byte = kKv4NanByte;  // a token without a page reads as NaN
        if (moves && place(base + from, codes, scale)) {
            c = *reinterpret_cast<const Codes16*>(codes);
            byte = *scale;
        }
        __syncthreads();
        if (moves) {
            *reinterpret_cast<Codes16*>(codes_to) = c;
            *scale_to = (uint8_t)byte;
        }
        __syncthreads();
    }
}

}  // namespace

void launch_draft_tree(const DraftTreeArgs& a, hipStream_t st) {
    VLA_REQUIRE(a.n_seqs >= 0 && a.total >= 0 && a.n_seqs <= 1 << 28 && a.total <= 1 << 28, "draft_tree: need 0 to 2^28 sequences and rows");
    VLA_REQUIRE(a.ld_see >= 1 && a.ld_see <= 1 << 20, "draft_tree: rows of 1 to 2^20 words");
    if (a.n_seqs == 0 || a.total == 0) return;
    VLA_REQUIRE(a.pos && a.see && a.lens && a.start, "draft_tree: null buffer");
    VLA_REQUIRE(a.pos != a.parent, "draft_tree: pos must not be parent, which other rows still read");
    // A wave for each sequence where they are short on average, or up to 512 rows with words for no more: a long one among short
    // ones keeps one wave busy with its words (48 sequences, one a chain of 8192: 3295 us, by threads 1548). Otherwise, by the depth, a thread for each
    // row. Wave | threads, us, 64 sequences:
    // chains of 65 rows 3.9 | 15, 256 7.9 | 50, 512 21 | 101, 1024 67 | 203, 4096 925 | 1095; parents among the 8 before of 256 7.4 | 15,
    // 512 21 | 29, 1024 66 | 57, 4096 939 | 349; among all before of 256 6.7 | 6.1, 512 19 | 9.7, 1024 67 | 17. One sequence: the same less a tenth.
    if (a.total <= (int64_t)64 * a.n_seqs || (a.ld_see <= 16 && a.total <= (int64_t)512 * a.n_seqs))
        draft_tree_wave_kernel<<<a.n_seqs < 1 << 20 ? a.n_seqs : 1 << 20, 64, 0, st>>>(a);
    else draft_tree_rows_kernel<<<(a.total + 255) / 256, 256, 0, st>>>(a);
    VLA_LAUNCH_CHECK();
}

void launch_verify_drafts(const VerifyArgs& a, hipStream_t st) {
    VLA_REQUIRE(dtype_ok(a.dtype), "verify_drafts: dtype must be VLA_F32, VLA_BF16 or VLA_F16");
    VLA_REQUIRE(a.n_seqs >= 0 && a.total >= 0 && a.total <= 1 << 28, "verify_drafts: need n_seqs >= 0 and 0 to 2^28 rows");
    VLA_REQUIRE(a.n_seqs <= kMaxSeqs, "verify_drafts: at most 65535 sequences");
    VLA_REQUIRE(a.vocab >= 1 && a.vocab <= 1 << 30, "verify_drafts: a vocabulary of 1 to 2^30 tokens");
    if (a.n_seqs == 0) return;
    VLA_REQUIRE(a.count && a.token && a.start && a.u_next, "verify_drafts: null buffer");
    VLA_REQUIRE(a.total == 0 || (a.path && a.p && a.tokens && a.u), "verify_drafts: null buffer");
    VLA_REQUIRE(a.total == 0 || (a.ldp >= a.vocab && (!a.q || a.ldq >= a.vocab)), "verify_drafts: row stride shorter than the vocabulary");
    const int sz = dtype_size(a.dtype);
    VLA_REQUIRE(aligned(a.p, sz) && aligned(a.q, sz), "verify_drafts: probabilities must be aligned to their type");
    if (a.dtype == kF32) verify_kernel<float><<<a.n_seqs, kVerifyThreads, 0, st>>>(a);
    else if (a.dtype == kBf16) verify_kernel<bf16_t><<<a.n_seqs, kVerifyThreads, 0, st>>>(a);
    else verify_kernel<f16_t><<<a.n_seqs, kVerifyThreads, 0, st>>>(a);
    VLA_LAUNCH_CHECK();
}

void launch_kv4_keep(const Kv4KeepArgs& a, hipStream_t st) {
    const Kv4Args& c = a.kv;
    check_cache(c, "kv4_keep");
    VLA_REQUIRE(c.n_seqs <= kMaxSeqs, "kv4_keep: at most 65535 sequences");
    if (c.n_seqs == 0) return;
    VLA_REQUIRE(c.n_pages > 0 && c.cache && aligned(c.cache, 16), "kv4_keep: the cache must hold a page and be 16-byte aligned");
    VLA_REQUIRE(c.table && c.ld_table > 0, "kv4_keep: page table missing");
    VLA_REQUIRE(c.lens && c.start && a.count && (a.path || c.total == 0), "kv4_keep: null buffer");
    VLA_REQUIRE(!a.new_lens || (a.new_lens != c.lens && a.new_lens != a.count), "kv4_keep: new_lens must not be lens or count, which other blocks still read");
    kv4_keep_kernel<<<dim3(c.n_kv, c.n_seqs), kKeepThreads, 0, st>>>(a);
    VLA_LAUNCH_CHECK();
}

}  // namespace hip
}  // namespace vla
