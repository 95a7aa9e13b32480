// rope_append.hip - norms and rotation of packed rows on their way into the 4-bit
// cache, in one pass.
//
// Per token t and head of queries and keys: y = x / sqrt(mean(x^2) + eps) * w (left out where
// w is null), then with angle = pos[t] * freqs[i], for the pairs i < rot / 2 at
// (i, i + rot / 2), or (2 i, 2 i + 1) where they are interleaved, the values (a, b) become
//   magnitude * (a cos(angle) - b sin(angle)), magnitude * (a sin(angle) + b cos(angle))
// and those from rot on stay. Queries go to q_out, keys to k_out where it is given and, as
// values do, into the cache (kv4.h).
//
// Codes lie next to borders, where the last bit of a value moves it by a whole step, so keys
// are normed and turned in 64 bits and quantized from there: a code then is the nearest of
// the exact value but where that lies within 2^-40 or so of a border. A result is rounded once.
//
// Few rows are bound by latency (from the offsets to the table, the sines, a store: 4 us), many by HBM: 16 prompts of 20500 tokens
// (484 MB with the fp16 rows of the keys) 104 us, 4.6 TB/s where a copy has 5.1, with pairs as halves 118; 1536 rows with norms
// 13.8 us, 2.4 TB/s; 5005 rows of fp32 38 us.
// A block takes a few tokens and fills a table of their sines and cosines in LDS, the same for all heads. A group of lanes stays
// with one token, a lane with 16 bytes of a row at the same place of every head, so that it keeps its sines and cosines in registers. The other
// value of a pair is another lane's of the group where pairs are halves.

#include "kv4_device.h"
#include "wave.h"

#include <cmath>

namespace vla {
namespace hip {
namespace {

constexpr int kMaxTokens = 16;   // of a block
constexpr int kTableEntries = 1024;  // sines and cosines of a block: half of the values that turn for each token (16 tokens of 128 fill it)
constexpr int kCus = 256;

// d for a later rounding to fewer bits than an fp32 has: cut off, the last bit set where anything
// was lost. Past fp32's range it is infinite.
__device__ __forceinline__ float to_odd(double d) {
    const uint64_t u = (uint64_t)__double_as_longlong(d);
    const uint32_t lo = (uint32_t)u, rest = lo & 0x1fffffffu;
    const uint32_t cut = (lo & 0xe0000000u) | (rest ? 0x20000000u : 0u);
    return (float)__longlong_as_double((long long)((u & 0xffffffff00000000ull) | cut));
}

template <class T>
__device__ __forceinline__ T round_once(double d) {
    if constexpr (sizeof(T) == 4) return (float)d;
    else return (T)to_odd(d);
}

// 16 bytes of a row
struct alignas(16) Words {
    unsigned w[4];
};

template <class T>
__device__ __forceinline__ float value_of(const Words& x, int e) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(x.w[e]);
    else return to_f32(__builtin_bit_cast(T, (unsigned short)(x.w[e >> 1] >> (16 * (e & 1)))));
}

// 1 / sqrt(x) to the last bits of a double: the hardware's number and two steps of Newton's. (Their factor is about 1; where
// x is infinite it is NaN, and the maximum leaves the 0 as it is. A choice of results would take registers that the fourth wave needs.)
__device__ __forceinline__ double rsqrt_wide(double x) {
    double y = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 2; i++) y = y * fmax(fma(-0.5 * x * y, y, 1.5), 0.5);
    return y;
}

// Sums over the lp lanes of a group, a power of two, in all of them: by lane permutations of the vector ALU.
template <class F>
__device__ __forceinline__ F group_sum(F x, int lp) {
    auto step = [&]<int CTRL>() {
        if constexpr (sizeof(F) == 8) x += dpp_f64<CTRL, 0xf>(0.0, x);
        else x += dpp_f32<CTRL, 0xf>(0.0f, x);
    };
    if (lp > 1) step.template operator()<0xb1>();   // quad_perm [1,0,3,2]
    if (lp > 2) step.template operator()<0x4e>();   // quad_perm [2,3,0,1]
    if (lp > 4) step.template operator()<0x141>();  // row_half_mirror
    if (lp > 8) step.template operator()<0x140>();  // row_mirror
    if (lp > 16) x += __shfl_xor(x, 16);
    if (lp > 32) x += __shfl_xor(x, 32);
    return x;
}

template <class T, bool INTER>
__global__ __launch_bounds__(256) void rope_append_kernel(RopeAppendArgs a, int lp) {
    constexpr int EPL = RowGeo<T>::EPL;
    __shared__ double2 cs[kTableEntries];
    __shared__ int32_t starts[kStartsInLds];
    __shared__ Where place[kMaxTokens];
    __shared__ __attribute__((aligned(16))) float norm[2][256];  // the norms' weights
    const Kv4Args& c = a.kv;
    const int tb = a.tokens_per_block, t0 = blockIdx.x * tb;
    const int nt = c.total - t0 < tb ? c.total - t0 : tb;
    const int half = a.rot >> 1, hd = c.head_dim;
    const int group = threadIdx.x / lp, ln = threadIdx.x & (lp - 1);
    const int tt = group % tb, i0 = ln * EPL;
    const bool in = i0 < hd && tt < nt;
    const size_t t = t0 + (tt < nt ? tt : 0);
    const int step = gridDim.y * (256 / lp / tb);
    int h = blockIdx.y * (256 / lp / tb) + group / tb;
    // a row's 16 bytes of query, key or value head h
    auto row = [&](int h) -> Words {
        const T* src = h < a.n_q ? static_cast<const T*>(a.q) + t * a.ldq + h * hd
                     : h < a.n_q + c.n_kv ? static_cast<const T*>(c.K) + t * c.ldk + (h - a.n_q) * hd
                                          : static_cast<const T*>(c.V) + t * c.ldv + (h - a.n_q - c.n_kv) * hd;
        return *reinterpret_cast<const Words*>(src + (i0 < hd ? i0 : 0));
    };
    const int n_all = a.n_q + c.n_kv + (c.cache ? c.n_kv : 0);
    // A head's load is under way while the one before it is worked on, the first one while the table is filled. All lanes load
    // in every turn (those without a row another one's, which is not used), so that a wait is for one load and not for a branch's.
    Words x = row(h < n_all ? h : n_all - 1);
    if (a.wq && threadIdx.x < hd) norm[0][threadIdx.x] = a.wq[threadIdx.x];
    if (a.wk && threadIdx.x < hd) norm[1][threadIdx.x] = a.wk[threadIdx.x];

    auto fill = [&](int threads) {
        for (int idx = threadIdx.x; idx < nt * half; idx += threads) {
            const int k = idx / half, i = idx - k * half;
            int p;
            if (a.pos) {
                p = a.pos[t0 + k];
            } else {  // its number in its sequence
                const int s = place[k].seq;
                p = s < 0 ? 0 : c.lens[s] - (c.start[s + 1] - c.start[s]) + (t0 + k - c.start[s]);
            }
            double sn, co;
            sincos((double)p * a.freqs[i], &sn, &co);
            cs[idx] = make_double2(co * a.magnitude, sn * a.magnitude);
        }
    };
    if (a.pos) {  // the last wave finds the tokens' places meanwhile
        if (threadIdx.x < 192) {
            fill(192);
        } else {
            const int i = threadIdx.x - 192;
            const int32_t* start = c.start;
            if (c.n_seqs < kStartsInLds) {
                for (int s = i; s <= c.n_seqs; s += 64) starts[s] = c.start[s];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                start = starts;
            }
            if (i < nt) place[i] = locate(c, start, t0 + i, false);
        }
        __syncthreads();
    } else {
        locate_rows(c, t0, nt, false, starts, place);
        fill(256);
        __syncthreads();
    }
    const Where where = place[tt < nt ? tt : 0];
    const bool on = in && where.seq >= 0;  // (rows behind the last sequence are left as they are)
    // This lane's sines and cosines, by fours; the sine's sign is that of the other value's share. (Behind the part that turns they are not used.)
    bool turns[EPL / 4];
#pragma unroll
    for (int j = 0; j < EPL / 4; j++) turns[j] = on && i0 + 4 * j < a.rot;
    auto angles = [&]<class F>(F (&co)[EPL], F (&si)[EPL]) {
#pragma unroll
        for (int j = 0; j < EPL / 4; j++) {
            const int v = i0 + 4 * j;
            const bool second = !INTER && v >= half;
            const double2* z = cs + (turns[j] ? tt * half + (INTER ? v >> 1 : second ? v - half : v) : 0);
            double2 at[INTER ? 2 : 4];
#pragma unroll
            for (int e = 0; e < (INTER ? 2 : 4); e++) at[e] = z[e];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double sn = at[INTER ? e >> 1 : e].y;
                co[4 * j + e] = (F)at[INTER ? e >> 1 : e].x;
                si[4 * j + e] = (F)((INTER ? e & 1 : second) ? sn : -sn);
            }
        }
    };
    // Where the other values of the lane's pairs are: of halves, four neighbours belong to four neighbours of one lane, in the same
    // half of it or (odd) the other. Behind the part that turns they are not used.
    const int d = half >> 2;  // fours between them
    const unsigned odd = EPL == 8 && (d & 1) ? ~0u : 0u;
    int from[EPL / 4], other[EPL / 4];  // the lane, and the first of the other values, for the weights
#pragma unroll
    for (int j = 0; j < EPL / 4; j++) {
        const int g = ln * (EPL / 4) + j, o = g < d ? g + d : g < 2 * d ? g - d : g;
        from[j] = (threadIdx.x & 63 & ~(lp - 1)) + o / (EPL / 4);
        other[j] = 4 * o;
    }
    auto others = [&](const Words& x) {
        Words z;
        if constexpr (INTER) {
#pragma unroll
            for (int i = 0; i < 4; i++) z.w[i] = EPL == 8 ? __builtin_amdgcn_alignbit(x.w[i], x.w[i], 16) : x.w[i ^ 1];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (EPL == 4) z.w[i] = __shfl(x.w[i], from[0]);
                else z.w[i] = __shfl((x.w[i ^ 2] & odd) | (x.w[i] & ~odd), from[i >> 1]);
            }
        }
        return z;
    };
    // the norm's weights of the lane's values and of the others
    auto weights = [&](const float (&w)[256], float (&mine)[EPL], float (&theirs)[EPL]) {
#pragma unroll
        for (int j = 0; j < EPL / 4; j++) {
            const int at = i0 < hd ? i0 + 4 * j : 0, there = INTER ? at : i0 < hd ? other[j] : 0;
#pragma unroll
            for (int e = 0; e < 4; e++) mine[4 * j + e] = w[at + e], theirs[4 * j + e] = w[there + (INTER ? e ^ 1 : e)];
        }
    };

    const unsigned mine = i0 < hd ? ~0u : 0u;
    auto take = [&] {
        Words now = x;
        x = row(h + step < n_all ? h + step : n_all - 1);
#pragma unroll
        for (int i = 0; i < 4; i++) now.w[i] &= mine;
        return now;
    };
    if (h < a.n_q) {  // queries, in 32 bits
        float cf[EPL], sf[EPL], wy[EPL], wz[EPL];
        if (a.wq) weights(norm[0], wy, wz);
        angles(cf, sf);
        T* dst = static_cast<T*>(a.q_out) + t * a.ldqo + i0;
        const float inv_hd = 1.0f / (float)hd;
        for (; h < a.n_q; h += step) {
            const Words x = take(), xo = others(x);
            float y[EPL], z[EPL];
#pragma unroll
            for (int e = 0; e < EPL; e++) y[e] = value_of<T>(x, e), z[e] = value_of<T>(xo, e);
            if (a.wq) {
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < EPL; e++) sum += y[e] * y[e];
                const float mean = group_sum(sum, lp) * inv_hd + a.eps;
                if (mean > 1e-30f && mean < 1e30f) {
                    const float r = rsqrtf(mean);
#pragma unroll
                    for (int e = 0; e < EPL; e++) y[e] = y[e] * r * wy[e], z[e] = z[e] * r * wz[e];
                } else {  // the squares leave fp32's range, or are about to
                    double wide = 0.0;
#pragma unroll
                    for (int e = 0; e < EPL; e++) wide += (double)y[e] * y[e];
                    const double r = 1.0 / sqrt(group_sum(wide, lp) / hd + a.eps);
#pragma unroll
                    for (int e = 0; e < EPL; e++) y[e] = (float)(y[e] * r) * wy[e], z[e] = (float)(z[e] * r) * wz[e];
                }
            }
            Pack<T, EPL> out;
#pragma unroll
            for (int e = 0; e < EPL; e++) out.v[e] = (T)(turns[e >> 2] ? fmaf(cf[e], y[e], sf[e] * z[e]) : y[e]);
            if (on) *reinterpret_cast<Pack<T, EPL>*>(dst + h * hd) = out;
        }
    }
    if (h < a.n_q + c.n_kv) {  // keys, in 64 bits
        float wy[EPL], wz[EPL];
        double co[EPL], si[EPL];
        const double inv_hd = 1.0 / hd;
        if (a.wk) weights(norm[1], wy, wz);
        angles(co, si);
        for (; h < a.n_q + c.n_kv; h += step) {
            const Words x = take(), xo = others(x);
            double y[EPL], z[EPL];
#pragma unroll
            for (int e = 0; e < EPL; e++) y[e] = value_of<T>(x, e), z[e] = value_of<T>(xo, e);
            if (a.wk) {
                double sum = 0.0;
#pragma unroll
                for (int e = 0; e < EPL; e++) sum = fma(y[e], y[e], sum);
                const double r = rsqrt_wide(fma(group_sum(sum, lp), inv_hd, (double)a.eps));
#pragma unroll
                for (int e = 0; e < EPL; e++) y[e] = y[e] * r * wy[e], z[e] = z[e] * r * wz[e];
            }
            float f[EPL];
            Pack<T, EPL> out;
#pragma unroll
            for (int e = 0; e < EPL; e++) {
                const double v = turns[e >> 2] ? fma(co[e], y[e], si[e] * z[e]) : y[e];
                f[e] = to_odd(v);
                out.v[e] = round_once<T>(v);
            }
            if (a.k_out && on) *reinterpret_cast<Pack<T, EPL>*>(static_cast<T*>(a.k_out) + t * a.ldko + (h - a.n_q) * hd + i0) = out;
            const Kv4Lane q = quantize_lane(f);
            if (on && where.page >= 0) store_lane<EPL>(c, where, 0, h - a.n_q, ln, q);
        }
    }
    for (; h < n_all; h += step) {
        const Words x = take();
        float f[EPL];
#pragma unroll
        for (int e = 0; e < EPL; e++) f[e] = value_of<T>(x, e);
        const Kv4Lane q = quantize_lane(f);
        if (on && where.page >= 0) store_lane<EPL>(c, where, 1, h - a.n_q - c.n_kv, ln, q);
    }
}

template <class T>
void run_rope_append(RopeAppendArgs a, hipStream_t st) {
    const Kv4Args& c = a.kv;
    const int lanes = c.head_dim / RowGeo<T>::EPL;
    int lp = 1;
    while (lp < lanes) lp <<= 1;
    const int groups = 256 / lp;
    const int n_all = a.n_q + c.n_kv + (c.cache ? c.n_kv : 0);
    // As many tokens to a block as bring the blocks down to those that run at once, three to a CU, and where that is not to be had eight
    // turns of a group, over which its table is worth it. One token | 2 | 4 | 8 | 16, 32 heads of queries and 8 of keys of 128, us:
    // 256 rows with norms 6.6 | 8.4 | 11.4 | 18.2 | 32, 1536 16.4 | 14.0 | 16.0 | 20.4 | 34, 4800 42 | 35 | 30 | 28 | 41; 20500 without 140 | 110 |
    // 104 | 110 | 134, of heads of 64 with norms 89 | 63 | 52 | 47 | 51, of 12 and 2 heads 77 | 48 | 35 | 31 | 33.
    int tb = 1;
    while (tb < kMaxTokens && tb * 2 <= groups && tb * a.rot <= kTableEntries && c.total > (int64_t)tb * 3 * kCus &&
           (n_all * tb < 8 * groups || c.total <= (int64_t)tb * 6 * kCus || c.total > (int64_t)tb << 23)) tb <<= 1;  // (a launch has less than 2^32 threads)
    a.tokens_per_block = tb;
    // and more blocks to a token while the card has CUs without any (one such row 3.9 us, 64 4.7)
    const int rounds = (n_all * tb + groups - 1) / groups;
    const int spare = kCus / c.total;
    const unsigned blocks = (unsigned)(((int64_t)c.total + tb - 1) / tb);
    const dim3 grid(blocks, rounds < spare ? rounds : spare > 1 ? spare : 1);
    if (a.interleaved) rope_append_kernel<T, true><<<grid, 256, 0, st>>>(a, lp);
    else rope_append_kernel<T, false><<<grid, 256, 0, st>>>(a, lp);
    VLA_LAUNCH_CHECK();
}

void check_strided(const void* p, int64_t ld, int heads, const Kv4Args& c, const char* what) {
    const std::string w = std::string("rope_kv4_append: ") + what;
    const int sz = dtype_size(c.dtype);
    VLA_REQUIRE(p, w + " missing");
    VLA_REQUIRE(ld >= (int64_t)heads * c.head_dim, w + ": row stride shorter than heads * head_dim");
    VLA_REQUIRE(aligned(p, 16) && ld * sz % 16 == 0, w + ": rows must be 16-byte aligned");
}

}  // namespace

void launch_rope_kv4_append(RopeAppendArgs a, hipStream_t st) {
    const Kv4Args& c = a.kv;
    check_cache(c, "rope_kv4_append");
    VLA_REQUIRE(c.total < (1 << 26) - 3, "rope_kv4_append: fewer than 2^26 - 3 rows");  // (4 or more to a block then)
    VLA_REQUIRE(a.n_q >= 0 && a.n_q <= 65536, "rope_kv4_append: 0 to 65536 query heads");
    VLA_REQUIRE(a.rot >= 0 && a.rot <= c.head_dim && a.rot % 8 == 0, "rope_kv4_append: rot_dim must be a multiple of 8 up to head_dim");
    VLA_REQUIRE(std::isfinite(a.magnitude), "rope_kv4_append: magnitude must be finite");
    VLA_REQUIRE(a.eps >= 0.0f && std::isfinite(a.eps), "rope_kv4_append: eps must not be negative");
    if (c.n_seqs == 0 || c.total == 0) return;
    VLA_REQUIRE(c.lens && c.start, "rope_kv4_append: lens or start missing");
    VLA_REQUIRE(a.freqs || a.rot == 0, "rope_kv4_append: frequencies missing");
    check_strided(c.K, c.ldk, c.n_kv, c, "keys");
    if (a.n_q) {
        check_strided(a.q, a.ldq, a.n_q, c, "queries");
        check_strided(a.q_out, a.ldqo, a.n_q, c, "q_out");
        VLA_REQUIRE(a.q_out != a.q || a.ldqo == a.ldq || c.total == 1, "rope_kv4_append: q_out over q needs the same stride");
    }
    if (a.k_out) {
        check_strided(a.k_out, a.ldko, c.n_kv, c, "k_out");
        VLA_REQUIRE(a.k_out != c.K || a.ldko == c.ldk || c.total == 1, "rope_kv4_append: k_out over the keys needs the same stride");
    }
    if (c.cache) {
        VLA_REQUIRE(c.n_pages > 0 && aligned(c.cache, 16), "rope_kv4_append: the cache must hold a page and be 16-byte aligned");
        VLA_REQUIRE(c.table && c.ld_table > 0, "rope_kv4_append: page table missing");
        check_strided(c.V, c.ldv, c.n_kv, c, "values");
    }
    if (c.dtype == kF32) run_rope_append<float>(a, st);
    else if (c.dtype == kBf16) run_rope_append<bf16_t>(a, st);
    else run_rope_append<f16_t>(a, st);
}

}  // namespace hip
}  // namespace vla
