// rope_heads.hip - norms of queries and keys per head and their rotation by
// positions of one or several axes, in one pass.
//
// Per token t and head: y = x / sqrt(mean(x^2) + eps) * w (left out where w is
// null), then for every pair i < head_dim / 2 of axis a (its section):
//   angle = pos[a][t] * base^(-2 i / head_dim)
//   out[i]        = y[i] cos(angle) - y[i + half] sin(angle)
//   out[i + half] = y[i] sin(angle) + y[i + half] cos(angle)
//
// HBM bounds it: every value is read and written once, some ten operations
// each (32768 tokens of 40 heads of 128 in 125 us, 5.4 TB/s, where a large copy reaches 4.75; one
// token of 20 heads of 64 in 3.9). The angle needs 64 bits (a position of 10^6 leaves 4 bits of an fp32
// fraction), the rest 32: the product in double is brought to a fraction of a
// turn, [-1/2, 1/2], whose fp32 sine and cosine, turned on by what the fraction's own rounding
// left out, carry fp32 errors of their size whatever the position. That costs a few hundred cycles per (token, pair) and is the same for
// every head, so a block first fills a table of its tokens' sines and cosines
// in LDS and then streams all their heads past it.
//
// Lanes: a lane owns VEC pairs (16-byte loads of both halves where the type and
// head_dim allow), so the rotation needs no other lane and in-place calls are
// safe; `lp` lanes, a power of two, share a head and its sum of squares.

#include "serving.h"

#include <cmath>

namespace vla {
namespace hip {
namespace {

constexpr int kMaxHalf = 128;
constexpr int kMaxTokens = 4;  // of a block

template <class T, int VEC>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeHeadsArgs a, int lp) {
    __shared__ float2 cs[kMaxTokens * kMaxHalf];
    const int half = a.head_dim >> 1;
    const int t0 = blockIdx.x * a.tokens_per_block;
    const int nt = a.seq - t0 < a.tokens_per_block ? a.seq - t0 : a.tokens_per_block;

    int last = -1;
    double turns = 0.0;  // of a position, for pair `last`
    const int32_t* pos = nullptr;
    for (int idx = threadIdx.x; idx < nt * half; idx += 256) {
        const int tt = idx / half, i = idx - tt * half;
        if (i != last) {  // a thread keeps its pair where half divides 256
            last = i;
            turns = exp2((double)(-2 * i) / a.head_dim * a.log2_base) * 0.15915494309189533577;
            int axis = 0;
#pragma unroll
            for (int x = 0; x < kMaxAxes - 1; x++) axis += x < a.n_axes - 1 && i >= a.ends[x];
            pos = a.pos + axis * a.ld_pos + t0;
        }
        double r = (double)pos[tt] * turns;
        r -= rint(r);
        const float f = (float)r, rest = 6.28318530717958648f * (float)(r - f);  // rest: at most 2^-23
        float s, c;
        sincospif(2.0f * f, &s, &c);
        cs[idx] = make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
    }
    __syncthreads();

    const int nh = a.n_q + a.n_kv;
    const int j = threadIdx.x & (lp - 1), groups = 256 / lp;
    const int i0 = j * VEC;
    const bool on = i0 < half;
    for (int item = threadIdx.x / lp; item < nt * nh; item += groups) {
        const int tt = item / nh, h = item - tt * nh;
        const bool key = h >= a.n_q;
        const size_t t = t0 + tt;
        const T* x = key ? static_cast<const T*>(a.k) + t * a.ldk + (h - a.n_q) * a.head_dim
                         : static_cast<const T*>(a.q) + t * a.ldq + h * a.head_dim;
        T* y = key ? static_cast<T*>(a.k_out) + t * a.ldko + (h - a.n_q) * a.head_dim
                   : static_cast<T*>(a.q_out) + t * a.ldqo + h * a.head_dim;
        const float* w = key ? a.wk : a.wq;
        float lo[VEC] = {}, hi[VEC] = {};
        if (on) {
            const auto l = *reinterpret_cast<const Pack<T, VEC>*>(x + i0);
            const auto u = *reinterpret_cast<const Pack<T, VEC>*>(x + half + i0);
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                lo[v] = to_f32(l.v[v]);
                hi[v] = to_f32(u.v[v]);
            }
        }
        if (w) {
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < VEC; v++) sum += lo[v] * lo[v] + hi[v] * hi[v];
            for (int m = 1; m < lp; m <<= 1) sum += __shfl_xor(sum, m);
            const float mean = sum / (float)a.head_dim + a.eps;
            if (mean > 1e-30f && mean < 1e30f) {
                const float r = 1.0f / sqrtf(mean);
#pragma unroll
                for (int v = 0; v < VEC; v++) lo[v] *= r, hi[v] *= r;
            } else {  // the squares leave fp32's range, or are about to (all in double: 142 us for 127)
                double wide = 0.0;
#pragma unroll
                for (int v = 0; v < VEC; v++) wide += (double)lo[v] * lo[v] + (double)hi[v] * hi[v];
                for (int m = 1; m < lp; m <<= 1) wide += __shfl_xor(wide, m);
                const double r = 1.0 / sqrt(wide / a.head_dim + a.eps);
#pragma unroll
                for (int v = 0; v < VEC; v++) lo[v] = (float)(lo[v] * r), hi[v] = (float)(hi[v] * r);
            }
            if (on) {
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    lo[v] *= w[i0 + v];
                    hi[v] *= w[half + i0 + v];
                }
            }
        }
        if (on) {
            Pack<T, VEC> l, u;
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                const float2 z = cs[tt * half + i0 + v];
                l.v[v] = (T)(lo[v] * z.x - hi[v] * z.y);
                u.v[v] = (T)(lo[v] * z.y + hi[v] * z.x);
            }
            *reinterpret_cast<Pack<T, VEC>*>(y + i0) = l;
            *reinterpret_cast<Pack<T, VEC>*>(y + half + i0) = u;
        }
    }
}

template <class T, int VEC>
void run_rope(const RopeHeadsArgs& a, hipStream_t st) {
    int lp = 1;
    while (lp * VEC < a.head_dim / 2) lp <<= 1;
    qk_norm_rope_kernel<T, VEC><<<(unsigned)(((int64_t)a.seq + a.tokens_per_block - 1) / a.tokens_per_block), 256, 0, st>>>(a, lp);
    VLA_LAUNCH_CHECK();
}

}  // namespace

void launch_qk_norm_rope(RopeHeadsArgs a, hipStream_t st) {
    VLA_REQUIRE(dtype_ok(a.dtype), "qk_norm_rope: dtype must be VLA_F32, VLA_BF16 or VLA_F16");
    VLA_REQUIRE(a.seq < 1 << 26, "qk_norm_rope: seq must be below 2^26");  // a launch has less than 2^32 threads
    VLA_REQUIRE(a.seq >= 0 && a.n_q >= 0 && a.n_kv >= 0 && a.n_q + a.n_kv > 0 && a.n_q <= 4096 && a.n_kv <= 4096,
                "qk_norm_rope: need seq >= 0 and heads");
    VLA_REQUIRE(a.head_dim >= 8 && a.head_dim <= 2 * kMaxHalf && a.head_dim % 8 == 0,
                "qk_norm_rope: head_dim must be a multiple of 8 in [8, 256]");
    VLA_REQUIRE(a.n_axes >= 1 && a.n_axes <= kMaxAxes, "qk_norm_rope: 1 to 8 axes");
    VLA_REQUIRE(a.ends[a.n_axes - 1] == a.head_dim / 2, "qk_norm_rope: the sections must add up to head_dim / 2");
    VLA_REQUIRE(std::isfinite(a.log2_base), "qk_norm_rope: base must be positive");
    VLA_REQUIRE(a.eps >= 0.0f && std::isfinite(a.eps), "qk_norm_rope: eps must not be negative");
    if (a.seq == 0) return;
    const int sz = dtype_size(a.dtype);
    VLA_REQUIRE(a.pos && a.ld_pos >= a.seq, "qk_norm_rope: positions missing, or their rows shorter than seq");
    if (a.n_q) {
        VLA_REQUIRE(a.q && a.q_out, "qk_norm_rope: null queries");
        VLA_REQUIRE(a.ldq >= a.n_q * a.head_dim && a.ldqo >= a.n_q * a.head_dim,
                    "qk_norm_rope: row stride shorter than heads * head_dim");
        VLA_REQUIRE(aligned(a.q, 16) && aligned(a.q_out, 16) && a.ldq * sz % 16 == 0 && a.ldqo * sz % 16 == 0,
                    "qk_norm_rope: rows must be 16-byte aligned");
    }
    if (a.n_kv) {
        VLA_REQUIRE(a.k && a.k_out, "qk_norm_rope: null keys");
        VLA_REQUIRE(a.ldk >= a.n_kv * a.head_dim && a.ldko >= a.n_kv * a.head_dim,
                    "qk_norm_rope: row stride shorter than heads * head_dim");
        VLA_REQUIRE(aligned(a.k, 16) && aligned(a.k_out, 16) && a.ldk * sz % 16 == 0 && a.ldko * sz % 16 == 0,
                    "qk_norm_rope: rows must be 16-byte aligned");
    }
    // Tokens of a block: several share the first half's latency, but blocks for every CU come
    // first. By the tokens alone, as measured, us, 1 | 2 | 4 tokens (24 heads of 128, bf16): 100 tokens 4.4 | 5.5 | 6.5, 2371
    // 9.0 | 9.2 | 10.2, 4000 13.2 | 12.5 | 12.7, 8000 20.8 | 19.9 | 19.3, 16000 35.2 | 34.0 | 33.5 (5.9 TB/s);
    // 32768 of 40 heads 129 | 126 | 127 (5.3 TB/s).
    a.tokens_per_block = a.seq < 4000 ? 1 : a.seq < 8000 ? 2 : 4;
    const bool wide = a.head_dim % 16 == 0;  // 8 pairs of a 16-bit type: 16 bytes of each half
    if (a.dtype == kF32) run_rope<float, 4>(a, st);
    else if (a.dtype == kBf16) wide ? run_rope<bf16_t, 8>(a, st) : run_rope<bf16_t, 4>(a, st);
    else wide ? run_rope<f16_t, 8>(a, st) : run_rope<f16_t, 4>(a, st);
}

}  // namespace hip
}  // namespace vla
