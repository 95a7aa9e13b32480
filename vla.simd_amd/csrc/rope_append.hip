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
// HBM bounds it. A block takes a few tokens and fills a table of their sines and cosines in
// LDS, the same for all heads. A group of lanes stays with one token, a lane with 16 bytes of a row
// at the same place of every head, so that it keeps its sines and cosines in registers. The other
// value of a pair is another lane's of the group where pairs are halves.

#include "kv4_device.h"

#include <cmath>

namespace vla {
namespace hip {
namespace {

constexpr int kMaxTokens = 16;   // of a block
constexpr int kTableEntries = 1024;

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

template <class T, bool INTER>
__global__ __launch_bounds__(256) void rope_append_kernel(RopeAppendArgs a, int lp) {
    constexpr int EPL = RowGeo<T>::EPL;
    __shared__ double2 cs[kTableEntries];
    __shared__ int32_t starts[kStartsInLds];
    __shared__ Where place[kMaxTokens];
    const Kv4Args& c = a.kv;
    const int tb = a.tokens_per_block, t0 = blockIdx.x * tb;
    const int nt = c.total - t0 < tb ? c.total - t0 : tb;
    const int half = a.rot >> 1, hd = c.head_dim;
    locate_rows(c, t0, nt, false, starts, place);

    for (int idx = threadIdx.x; idx < nt * half; idx += 256) {
        const int tt = idx / half, i = idx - tt * half;
        int p;
        if (a.pos) {
            p = a.pos[t0 + tt];
        } else {  // its number in its sequence
            const int s = place[tt].seq;
            p = s < 0 ? 0 : c.lens[s] - (c.start[s + 1] - c.start[s]) + (t0 + tt - c.start[s]);
        }
        double sn, co;
        sincos((double)p * a.freqs[i], &sn, &co);
        cs[idx] = make_double2(co * a.magnitude, sn * a.magnitude);
    }
    __syncthreads();

    const int group = threadIdx.x / lp, ln = threadIdx.x & (lp - 1);
    const int tt = group % tb, step = 256 / lp / tb;
    const int i0 = ln * EPL;
    const bool on = i0 < hd && tt < nt && place[tt].seq >= 0;  // (rows behind the last sequence are left as they are)
    const Where w = place[tt < nt ? tt : 0];
    // this lane's sines and cosines: 1 and 0 behind the part that turns; the sign is that of b's share
    double co[EPL], si[EPL];
#pragma unroll
    for (int e = 0; e < EPL; e++) {
        const int v = i0 + e;
        co[e] = 1.0;
        si[e] = 0.0;
        if (on && v < a.rot) {
            const int pair = INTER ? v >> 1 : v < half ? v : v - half;
            const bool second = INTER ? v & 1 : v >= half;
            const double2 z = cs[tt * half + pair];
            co[e] = z.x;
            si[e] = second ? z.y : -z.y;
        }
    }
    const size_t t = t0 + tt;
    const int nh = a.n_q + c.n_kv + (c.cache ? c.n_kv : 0);
    for (int h = blockIdx.y * step + group / tb; h < nh; h += gridDim.y * step) {
        const int kind = h < a.n_q ? 0 : h < a.n_q + c.n_kv ? 1 : 2;  // query, key, value
        const int head = kind == 0 ? h : kind == 1 ? h - a.n_q : h - a.n_q - c.n_kv;
        const T* src = kind == 0 ? static_cast<const T*>(a.q) + t * a.ldq
                     : kind == 1 ? static_cast<const T*>(c.K) + t * c.ldk : static_cast<const T*>(c.V) + t * c.ldv;
        Pack<T, EPL> x{};
        if (on) x = *reinterpret_cast<const Pack<T, EPL>*>(src + head * hd + i0);
        float f[EPL];
        if (kind == 2) {
#pragma unroll
            for (int e = 0; e < EPL; e++) f[e] = to_f32(x.v[e]);
        } else {
            double y[EPL], z[EPL];  // the lane's values, and the others of their pairs
#pragma unroll
            for (int e = 0; e < EPL; e++) y[e] = to_f32(x.v[e]);
            const float* wt = kind ? a.wk : a.wq;
            if (wt) {
                double sum = 0.0;
#pragma unroll
                for (int e = 0; e < EPL; e++) sum = fma(y[e], y[e], sum);
                for (int m = 1; m < lp; m <<= 1) sum += __shfl_xor(sum, m);
                const double r = 1.0 / sqrt(sum / hd + a.eps);
#pragma unroll
                for (int e = 0; e < EPL; e++) y[e] = on ? y[e] * r * wt[i0 + e] : 0.0;
            }
            if constexpr (INTER) {
#pragma unroll
                for (int e = 0; e < EPL; e++) z[e] = y[e ^ 1];
            } else {
                // four values at a time, whose others are four neighbours too
#pragma unroll
                for (int j = 0; j < EPL / 4; j++) {
                    const int g = ln * (EPL / 4) + j, d = half >> 2;
                    const int o = g < d ? g + d : g < 2 * d ? g - d : g;
                    const int from = (threadIdx.x & 63 & ~(lp - 1)) + o / (EPL / 4);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if constexpr (EPL == 4) {
                            z[e] = __shfl(y[e], from);
                        } else {
                            const double lo = __shfl(y[e], from), hi = __shfl(y[4 + e], from);
                            z[4 * j + e] = o & 1 ? hi : lo;
                        }
                    }
                }
            }
            Pack<T, EPL> out;
#pragma unroll
            for (int e = 0; e < EPL; e++) {
                const double v = i0 + e < a.rot ? fma(co[e], y[e], si[e] * z[e]) : y[e];
                f[e] = to_odd(v);
                out.v[e] = round_once<T>(v);
            }
            T* dst = kind == 0 ? static_cast<T*>(a.q_out) + t * a.ldqo : a.k_out ? static_cast<T*>(a.k_out) + t * a.ldko : nullptr;
            if (dst && on) *reinterpret_cast<Pack<T, EPL>*>(dst + head * hd + i0) = out;
            if (kind == 0) continue;
        }
        if (!c.cache) continue;
        const Kv4Lane z = quantize_lane(f);
        if (on && w.page >= 0) store_lane<EPL>(c, w, kind - 1, head, ln, z);
    }
}

template <class T>
void run_rope_append(RopeAppendArgs a, hipStream_t st) {
    const Kv4Args& c = a.kv;
    const int lanes = c.head_dim / RowGeo<T>::EPL;
    int lp = 1;
    while (lp < lanes) lp <<= 1;
    const int groups = 256 / lp;
    int tb = c.total < 4096 ? 1 : 16;
    while (tb > groups || tb * (a.rot / 2) > kTableEntries) tb >>= 1;
    a.tokens_per_block = tb;
    const dim3 grid((unsigned)(((int64_t)c.total + tb - 1) / tb), 1);
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
    VLA_REQUIRE(c.total < 1 << 26, "rope_kv4_append: fewer than 2^26 rows");  // a launch has less than 2^32 threads
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
    }
    if (a.k_out) check_strided(a.k_out, a.ldko, c.n_kv, c, "k_out");
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
