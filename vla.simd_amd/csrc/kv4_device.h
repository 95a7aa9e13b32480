// kv4_device.h - what the kernels of the 4-bit cache share: where a packed row lives
// in the cache, and how a lane's share of a row becomes codes and a scale byte.
#pragma once

#include "kv4.h"
#include "serving.h"

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

// The places of the block's rows row0 .. row0 + n - 1, a thread for each: the chain of the
// search (in LDS where the starts fit) and the reads of length and table is walked once.
__device__ __forceinline__ void locate_rows(const Kv4Args& a, int row0, int n, bool gather, int32_t* starts, Where* out) {
    const int32_t* start = a.start;
    if (a.n_seqs < kStartsInLds) {
        for (int i = threadIdx.x; i <= a.n_seqs; i += blockDim.x) starts[i] = a.start[i];
        __syncthreads();
        start = starts;
    }
    for (int i = threadIdx.x; i < n; i += blockDim.x) out[i] = row0 + i < a.total ? locate(a, start, row0 + i, gather) : Where{-1, -1, 0};
    __syncthreads();
}

template <class T>
struct RowGeo {
    static constexpr int EPL = 16 / sizeof(T);      // values of a lane
    static constexpr int LPB = kKv4Block / EPL;     // lanes of a block
};


// A lane's share of a block of 32 values: its codes, and the block's scale byte.
struct Kv4Lane {
    unsigned codes;
    int byte;
};

// The codes of a lane's EPL values, whose 32 / EPL neighbouring lanes hold the rest of the block.
template <int EPL>
__device__ __forceinline__ Kv4Lane quantize_lane(const float (&f)[EPL]) {
    unsigned top = 0;  // bits of the largest magnitude: NaN above infinity above all numbers
#pragma unroll
    for (int e = 0; e < EPL; e++) {
        const unsigned u = __float_as_uint(f[e]) & 0x7fffffffu;
        top = u > top ? u : top;
    }
#pragma unroll
    for (int m = 1; m < kKv4Block / EPL; m <<= 1) {
        const unsigned u = __shfl_xor(top, m);
        top = u > top ? u : top;
    }
    // 1.f * 2^(E - 127) <= 1.75 * 2^(e + 2), so e + 127 = E - 2, one more where 1.f > 1.75
    int byte = (int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x600000u);
    byte = byte < kKv4MinByte ? kKv4MinByte : byte;
    const float sc = scale_of(byte);
    unsigned codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, f[0], f[1], sc, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[2], f[3], sc, 1);
    if constexpr (EPL == 8) {
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[4], f[5], sc, 2);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[6], f[7], sc, 3);
    }
    if (top >= 0x7f800000u) {
        codes = 0;
        byte = kKv4NanByte;
    }
    return {codes, byte};
}

// Lane ln of a row stores its share, the first lane of a block the scale byte.
template <int EPL>
__device__ __forceinline__ void store_lane(const Kv4Args& a, const Where& w, int part, int head, int ln, const Kv4Lane& z) {
    const size_t nc = kv4_code_bytes(a.n_kv, a.head_dim, a.page_size), ns = kv4_scale_bytes(a.n_kv, a.head_dim, a.page_size);
    uint8_t* pg = a.cache + (size_t)w.page * (2 * (nc + ns));
    uint8_t* cd = pg + part * nc + ((size_t)head * a.page_size + w.slot) * (a.head_dim / 2) + ln * (EPL / 2);
    if (EPL == 8) *reinterpret_cast<uint32_t*>(cd) = z.codes;
    else *reinterpret_cast<uint16_t*>(cd) = (uint16_t)z.codes;
    constexpr int LPB = kKv4Block / EPL;
    if (ln % LPB == 0)
        pg[2 * nc + part * ns + ((size_t)head * (a.head_dim / kKv4Block) + ln / LPB) * a.page_size + w.slot] = (uint8_t)z.byte;
}

constexpr int kTile = 32;         // keys that the attention takes at once; pages hold whole tiles
constexpr int kMaxSeqs = 65535;  // blocks of a launch in y

inline void check_cache(const Kv4Args& a, const char* who) {
    const std::string w(who);
    VLA_REQUIRE(dtype_ok(a.dtype), w + ": dtype must be VLA_F32, VLA_BF16 or VLA_F16");
    VLA_REQUIRE(a.n_seqs >= 0 && a.total >= 0 && a.n_kv > 0 && a.n_kv <= 1024, w + ": need n_seqs, rows >= 0 and 1 to 1024 kv heads");
    VLA_REQUIRE(a.n_seqs <= 1 << 28 && a.total <= 1 << 28, w + ": at most 2^28 sequences and rows");
    VLA_REQUIRE(kv4_head_dim_ok(a.head_dim), w + ": head_dim must be 32, 64, 96, 128, 192 or 256");
    VLA_REQUIRE(a.page_size > 0 && a.page_size % kTile == 0 && a.page_size <= kKv4MaxPage,
                w + ": page_size must be a multiple of 32 in [32, 2048]");
    VLA_REQUIRE(a.n_pages >= 0 && a.ld_table >= 0 && (int64_t)a.ld_table * a.page_size <= (int64_t)1 << 30,
                w + ": a sequence has at most 2^30 tokens");
}

}  // namespace
}  // namespace hip
}  // namespace vla
