// kv4_attn.h - what the attention kernels over the 4-bit cache share: a lane's bytes of a tile of
// 32 keys and the operands made of them, equal runs of tiles over all sequences, and
// the kernel that joins the pieces of sequences cut by runs.
#pragma once

#include "kv4_device.h"
#include "wave.h"

namespace vla {
namespace hip {
namespace {

template <int NB>
struct Kv4Geo {
    static constexpr int NL = NB == 3 || NB > 4 ? 2 : 1;  // loads of a row, each of vb blocks from block bs on
    static constexpr int vb(int u) { return u == 0 ? (NB >= 4 ? 4 : NB >= 2 ? 2 : 1) : NB - vb(0); }
    static constexpr int bs(int u) { return u * vb(0); }
    static constexpr int NT = 2 * NB;                     // 16-dim tiles of O
};
// f<u>() for the loads of a row
template <int NL, class F>
__device__ __forceinline__ void each_load(F&& f) {
    f.template operator()<0>();
    if constexpr (NL == 2) f.template operator()<1>();
}

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

// An entry of an array that nothing writes while the kernel runs, at an index that is the same in
// all lanes: a scalar load, although the kernel stores elsewhere. (As a vector load, a page
// number waits behind the tile loads issued before it: 54 us became 64 over 64 x 4096 tokens.)
__device__ __forceinline__ int32_t uniform_entry(const int32_t* p, int64_t i) {
    return reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p))[i];
}
// kv4_page of such a row
__device__ __forceinline__ int uniform_page(const int32_t* row, int ld_table, int n_pages, unsigned page_no) {
    if (page_no >= (unsigned)ld_table) return -1;
    const int32_t p = uniform_entry(row, page_no);
    return p >= 0 && p < n_pages ? p : -1;
}

struct Kv4Run {
    int runs;          // blocks of a head: equal runs of tiles; 0: one block per sequence
    int tok_tiles;     // row tiles over the new tokens; with head_tiles in gridDim.y / n_kv
    int head_tiles;
    int tok_cap;       // tokens of a sequence that a piece has room for
    int slots;         // pieces in the workspace
    unsigned per_page; // tiles of a page, and 2^32 / per_page rounded up
    unsigned magic;
    float lift;        // the weights' scale in log2, negated
    float wscale;      // of the weights in the product with V against those in their sum: 2^-lift with 24 bits, else 1
    int4* info;        // workspace: [total queries] first piece, pieces, token in its sequence
    float* ml;         // [slots][tok_cap * n_q][2]
    float* o;          // [slots][tok_cap * n_q][head_dim]
};

// tile / per_page; exact while tile * per_page < 2^32
__device__ __forceinline__ unsigned page_no(const Kv4Run& r, unsigned tile) {
    return r.per_page == 1 ? tile : __umulhi(tile, r.magic);
}

// The loaded bytes of a tile of 32 keys, as a lane holds them. Rows of the first product's
// operand are keys in this order: row c of step s is key 8 (c / 4) + 4 s + c % 4, so that the
// scores a lane holds, rows 4 g + r of both steps, are of 8 neighbouring keys 8 g + 4 s + r.
template <int NB>
struct Kv4Tile {
    using G = Kv4Geo<NB>;
    unsigned kd[2][NB], kb[2][G::NL], vd[8][G::NL], vw[2][G::NL];
    bool there;  // the table names a page

    __device__ __forceinline__ void load(const Kv4Args& a, const Kv4Run& run, const int32_t* table, int kvh, int c, int g,
                                         unsigned tile) {
        constexpr int HD = 32 * NB;
        const size_t nc = kv4_code_bytes(a.n_kv, HD, a.page_size), ns = kv4_scale_bytes(a.n_kv, HD, a.page_size);
        const unsigned pn = page_no(run, tile), slot = (tile - pn * run.per_page) * kTile;
        const int page = uniform_page(table, a.ld_table, a.n_pages, pn);
        there = page >= 0;
        const uint8_t* pg = a.cache + (size_t)__builtin_amdgcn_readfirstlane(there ? page : 0) * (2 * (nc + ns));  // not there: read, and not used
        const uint8_t* kc = pg + ((size_t)kvh * a.page_size + slot) * (HD / 2);
        const uint8_t* vc = kc + nc;
        const uint8_t* ks = pg + 2 * nc + (size_t)kvh * NB * a.page_size + slot;
        const uint8_t* vs = ks + ns;
        const unsigned krow = 8 * (c >> 2) + (c & 3);
        each_load<G::NL>([&]<int u>() {
            constexpr int VB = G::vb(u), BS = G::bs(u);
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const auto z = *reinterpret_cast<const Pack<unsigned, VB>*>(kc + ((krow + 4 * s) * (HD / 2) + BS * 16 + g * 4 * VB));
#pragma unroll
                for (int i = 0; i < VB; i++) kd[s][BS + i] = z.v[i];
                kb[s][u] = ks[(unsigned)(BS + g * VB / 4) * a.page_size + krow + 4 * s];
            }
        });
        each_load<G::NL>([&]<int u>() {
            constexpr int VB = G::vb(u), BS = G::bs(u);
            const auto w = *reinterpret_cast<const Pack<unsigned, 2>*>(vs + ((unsigned)(BS + c * VB / 16) * a.page_size + 8 * g));
            vw[0][u] = w.v[0];
            vw[1][u] = w.v[1];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const uint8_t* p = vc + ((unsigned)(8 * g + k) * (HD / 2) + BS * 16 + c * VB);
                vd[k][u] = VB == 4 ? *reinterpret_cast<const uint32_t*>(p) : VB == 2 ? *reinterpret_cast<const uint16_t*>(p) : *p;
            }
        });
    }

    __device__ __forceinline__ unsigned vbyte(int k, int u) const { return vw[k >> 2][u] >> (8 * (k & 3)) & 255u; }

    // V's operands of the pair of 16-dim tiles (u, b): the even and the odd value of a byte
    __device__ __forceinline__ void vfrag(int u, int b, U4& lo, U4& hi) const {
        unsigned z[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float sc = scale_of(vbyte(k, u));
            const unsigned w = vd[k][u];
            z[k] = b == 0 ? bf16_of<0>(w, sc) : b == 1 ? bf16_of<1>(w, sc) : b == 2 ? bf16_of<2>(w, sc) : bf16_of<3>(w, sc);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            lo.u[j] = __builtin_amdgcn_perm(z[2 * j + 1], z[2 * j], 0x05040100u);
            hi.u[j] = __builtin_amdgcn_perm(z[2 * j + 1], z[2 * j], 0x07060302u);
        }
    }

    // takes V's value k out (2^-127 of nothing: zeros)
    __device__ __forceinline__ void hide(int k, int u) {
        vd[k][u] = 0;
        vw[k >> 2][u] &= ~(255u << (8 * (k & 3)));
    }
};

// Tiles of a sequence: at least one, whose block writes the zeros of an empty one. Of a length
// beyond the table the first tile behind it is among them and makes NaN of the rows that see it.
__device__ __forceinline__ int seq_tiles(const Kv4Args& a, int cached, int& len) {
    len = cached < 0 ? 0 : cached;
    const int all = a.ld_table * (a.page_size / kTile) + 1;
    const int tiles = len / kTile + (len % kTile != 0);
    return tiles > all ? all : tiles > 0 ? tiles : 1;
}

// Where the run of tiles [run * per, (run + 1) * per) begins: sequence `seq`, whose first tile
// is number `first` of all. False for a run behind the last tile. Every wave does the same sums.
__device__ __forceinline__ bool find_run(const Kv4Args& a, int runs, int run, int& per, int& seq, int& first, int& cached) {
    const int lane = threadIdx.x & 63;
    int incl = 0, tiles = 0, lens = 0;
    auto load = [&](int base) {
        int len;
        lens = base + lane < a.n_seqs ? a.lens[base + lane] : 0;
        incl = tiles = base + lane < a.n_seqs ? seq_tiles(a, lens, len) : 0;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d);
            if (lane >= d) incl += o;
        }
        return __builtin_amdgcn_readlane(incl, 63);
    };
    int total = load(0);
    if (a.n_seqs > 64)
        for (int base = 64; base < a.n_seqs; base += 64) total += load(base);
    per = (total + runs - 1) / runs;
    int want = run * per, base = 0;
    if (want >= total) return false;
    first = 0;
    if (a.n_seqs > 64) {
        for (;; base += 64) {
            const int sum = load(base);
            if (want < sum) break;
            want -= sum;
            first += sum;
        }
    }
    const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(incl > want)) - 1);
    seq = base + l;
    cached = __builtin_amdgcn_readlane(lens, l);
    first += __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(tiles, l);
    return true;
}

// Joins the pieces, one block per row (query token and head). Every thread first takes some
// pieces' maxima and sums, so that their loads are under way together; then hd / 4 lanes
// carry a piece's values, as many pieces at once as the block has room for.
constexpr int kMaxPieces = 256;

template <class T, int N>
__global__ __launch_bounds__(N) void kv4_join_kernel(Kv4Args a, Kv4Run run) {
    __shared__ float factor[kMaxPieces], red[N / 64][2];
    __shared__ __attribute__((aligned(16))) float4 part[N];
    const int row = blockIdx.x, tok = row / a.n_q, head = row - tok * a.n_q;
    const int tid = threadIdx.x, wave = tid >> 6;
    if (tok < (a.start ? a.start[0] : 0) || tok >= (a.start ? a.start[a.n_seqs] : a.n_seqs)) return;
    const int4 in = run.info[tok];
    // (offsets out of order can leave a token without a sequence and its entry unwritten)
    if (in.y <= 1 || in.y > kMaxPieces || in.x < 0 || in.x > run.slots - in.y || in.z < 0 || in.z >= run.tok_cap) return;
    const int pieces = in.y;
    const size_t stride = (size_t)run.tok_cap * a.n_q;
    const float* pml = run.ml + (in.x * stride + (size_t)in.z * a.n_q + head) * 2;
    const float* po = run.o + (in.x * stride + (size_t)in.z * a.n_q + head) * a.head_dim;
    const int lanes = a.head_dim / 4, groups = N / lanes;
    const int gr = tid / lanes, ln = tid - gr * lanes;
    // (values of two pieces are under way with the maxima; a lane without a piece loads the last one's)
    auto value = [&](int s) { return *reinterpret_cast<const float4*>(po + (s < pieces ? s : pieces - 1) * stride * a.head_dim + ln * 4); };
    const float4 first = value(gr), second = value(gr + groups);
    float2 z[kMaxPieces / N];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMaxPieces / N; i++) {
        z[i] = make_float2(-INFINITY, 0.0f);
        if (tid + i * N < pieces) z[i] = *reinterpret_cast<const float2*>(pml + (tid + i * N) * stride * 2);
        m = fmaxf(m, z[i].x);
    }
    const float wm = wave_max_f32(m);
    if ((tid & 63) == 0) red[wave][0] = wm;
    __syncthreads();
    float top = red[0][0];
#pragma unroll
    for (int w = 1; w < N / 64; w++) top = fmaxf(top, red[w][0]);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxPieces / N; i++) {
        const float f = __builtin_amdgcn_exp2f(z[i].x - (top == -INFINITY ? 0.0f : top));
        factor[tid + i * N] = f;
        sum += f * z[i].y;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    if ((tid & 63) == 0) red[wave][1] = sum;
    __syncthreads();
    sum = red[0][1];
#pragma unroll
    for (int w = 1; w < N / 64; w++) sum += red[w][1];

    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (gr < groups) {
        auto add = [&](int s, const float4& v) {
            const float w = factor[s];
            acc.x += w * v.x;
            acc.y += w * v.y;
            acc.z += w * v.z;
            acc.w += w * v.w;
        };
        if (gr < pieces) add(gr, first);
        if (gr + groups < pieces) add(gr + groups, second);
#pragma unroll 4
        for (int s = gr + 2 * groups; s < pieces; s += groups) add(s, value(s));
    }
    part[tid] = acc;
    __syncthreads();
    if (gr) return;
    for (int g = 1; g < groups; g++) {
        const float4 v = part[g * lanes + ln];
        acc.x += v.x;
        acc.y += v.y;
        acc.z += v.z;
        acc.w += v.w;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / (sum * run.wscale);
    Pack<T, 4> o;
    o.v[0] = (T)(acc.x * inv);
    o.v[1] = (T)(acc.y * inv);
    o.v[2] = (T)(acc.z * inv);
    o.v[3] = (T)(acc.w * inv);
    *reinterpret_cast<Pack<T, 4>*>(static_cast<T*>(a.out) + (size_t)tok * a.ldo + head * a.head_dim + ln * 4) = o;
}

// the workspace's parts, each 16-byte aligned
inline size_t info_bytes(int total_q) { return ((size_t)total_q * sizeof(int4) + 255) / 256 * 256; }
inline size_t ml_bytes(const Kv4Run& r, int n_q) { return ((size_t)r.slots * r.tok_cap * n_q * 2 * sizeof(float) + 255) / 256 * 256; }
inline size_t plan_bytes(const Kv4Run& r, int total_q, int n_q, int head_dim) {
    return r.runs ? info_bytes(total_q) + ml_bytes(r, n_q) + (size_t)r.slots * r.tok_cap * n_q * head_dim * sizeof(float) : 0;
}

// rows times heads that the second kernel has blocks of 256 threads for
inline bool joins(int total_q, int n_q) { return (int64_t)total_q * n_q < (int64_t)1 << 24; }

}  // namespace
}  // namespace hip
}  // namespace vla
