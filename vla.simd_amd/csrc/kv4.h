// kv4.h - the paged cache of 4-bit keys and values, for host and device code.
//
// A page holds page_size tokens (a multiple of 32) of every kv head:
//   K codes  [n_kv][page_size][head_dim / 2] bytes, value 2i of a row in the low half of byte i
//   V codes  the same
//   K scales [n_kv][head_dim / 32][page_size] bytes
//   V scales the same
// 32 neighbouring values of a head (a block) share a scale byte e + 127, that
// is 2^e, with the smallest e >= -100 for which the block's largest magnitude
// is at most 7 * 2^e; a code is a sign bit over three bits that choose from
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 (one bit of mantissa, two of exponent: what the
// matrix cores and converters of gfx950 call fp4), the nearest of them, ties to
// the even code. With amax <= 7 * 2^e no value is off by more than half a step,
// as 6 takes everything from 5 to 7. A block with an infinity or a NaN has
// scale byte 255 and reads as NaN throughout. Scaling by 2^e is exact, so
// quantization and reading are exact functions of the values, whatever runs them.
//
// Scales lie block-major over the page's tokens because the attention reads,
// per lane, the scales of neighbouring tokens for one block.
#pragma once

#include <cstddef>
#include <cstdint>

#ifndef __HIPCC__
#define VLA_HD inline
#else
#include <hip/hip_runtime.h>
#define VLA_HD __host__ __device__ __forceinline__
#endif

namespace vla {
namespace hip {

constexpr int kKv4Block = 32;
constexpr int kKv4MinByte = 27;    // e = -100
constexpr int kKv4NanByte = 255;
constexpr int kKv4LargeByte = 253; // from here on the largest codes pass fp32's range
constexpr int kKv4MaxPage = 2048;  // tokens of a page

inline bool kv4_head_dim_ok(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 192 || hd == 256; }

VLA_HD size_t kv4_code_bytes(int n_kv, int head_dim, int page_size) {
    return (size_t)n_kv * page_size * (head_dim / 2);
}
VLA_HD size_t kv4_scale_bytes(int n_kv, int head_dim, int page_size) {
    return (size_t)n_kv * page_size * (head_dim / kKv4Block);
}
VLA_HD size_t kv4_page_bytes(int n_kv, int head_dim, int page_size) {
    return 2 * (kv4_code_bytes(n_kv, head_dim, page_size) + kv4_scale_bytes(n_kv, head_dim, page_size));
}

// The page that a table row names as its page_no-th, or -1 where the row does not
// reach that far or names no page of the cache.
VLA_HD int kv4_page(const int32_t* row, int ld_table, int n_pages, int64_t page_no) {
    if (page_no < 0 || page_no >= ld_table) return -1;
    const int32_t p = row[page_no];
    return p >= 0 && p < n_pages ? p : -1;
}

}  // namespace hip
}  // namespace vla
