// The 8-bit paged KV cache: e4m3 codes and one power-of-two scale for each
// block of tokens and KV head.
//
// Layout: codes [num_pages, Hkv, page_size, 128] (keys and values apart),
// scales [num_pages, Hkv, page_size / block] as biased exponents (e8m0: scale
// = 2^(byte - 127)).  An entry stands for code * scale, which a bf16 holds
// exactly.  A (page, head) is one contiguous run of page_size * 128 bytes:
// reading split by split and head by head, token-major rows (128-byte pieces
// Hkv * 128 apart, the bf16 cache's order) reach 5.26 TB/s over 262,144 tokens
// of 8 heads and 4.5 over 32,768, head-major pages 5.98 and 5.0.
#pragma once

#include "d3d_common.hpp"

namespace d3d {
namespace fp8 {

constexpr int D = 128;      // head dimension
constexpr int kMinExp = -117;  // every code times its scale is a normal float
constexpr int kMaxExp = 119;   // and 448 * 2^119 a finite bf16
constexpr int kMinBlock = 16, kMaxBlock = 256;

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// The least exponent e in [kMinExp, kMaxExp] with amax <= 448 * 2^e: 448 is
// 1.75 * 2^8, so e is amax's exponent - 8, plus one past a mantissa of 1.75.
__device__ __forceinline__ int need_exp(float amax) {
    const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
    return min(max(e, kMinExp), kMaxExp);
}

// Four values as e4m3 codes (nearest, ties to even; not finite -> NaN).
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

}  // namespace fp8
}  // namespace d3d

// Page and block sizes that the cache's entry points take.
static inline int fp8_block_shift(int page_size, int block) {
    if (block < d3d::fp8::kMinBlock || block > d3d::fp8::kMaxBlock || (block & (block - 1)) || page_size < block ||
        page_size % block)
        return -1;
    int sh = 0;
    while ((1 << sh) < block) ++sh;
    return sh;
}
