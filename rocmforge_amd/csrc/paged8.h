// paged8.h -- 8-bit pages: e4m3 codes and the exponents of their blocks.
//
// Exponents are powers of two from 2^-15 to 2^7, so that all that a code can stand for is one of
// fp16's values: gfx950 converts two codes times a power of two in one instruction, and
// nothing is rounded.  An exponent that grows shifts its block's codes, exactly but for those
// that become subnormal.
#pragma once
#include "paged_common.h"
#include "qk_common.h"

namespace rf {

constexpr int kBlock8 = 16;                      // positions of a block, or a page's where it has fewer
constexpr int kScaleLo = 112, kScaleHi = 134;    // exponents -15 and 7, + 127

inline bool cache8_ok(const rf_paged_cache8& c) {
    if (!c.k || !c.v || !c.k_scale || !c.v_scale || c.num_kv_heads <= 0 || c.num_kv_heads > 65535 ||
        !page_size_ok(c.page_size) || c.num_pages <= 0 || (int64_t)c.num_pages * c.page_size > INT_MAX)
        return false;
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return false;
    if (((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15u) != 0) return false;
    return c.page_stride > 0 && c.row_stride > 0 && c.head_stride > 0 && c.row_stride <= (1 << 27) &&
           ((c.page_stride | c.row_stride | c.head_stride) & 15) == 0;
}

typedef _Float16 h2 __attribute__((ext_vector_type(2)));

// log2 of a block's positions
__device__ __forceinline__ int block_shift(const rf_paged_cache8& c) { return __ffs(min(c.page_size, kBlock8)) - 1; }
// Where the exponent of a page's row is, of KV head 0.
__device__ __forceinline__ int64_t scale_at(const rf_paged_cache8& c, int page, int row, int bsh) {
    return (((int64_t)page * c.page_size + row) >> bsh) * c.num_kv_heads;
}
__device__ __forceinline__ int scale_byte(int v) { return min(max(v, kScaleLo), kScaleHi); }
__device__ __forceinline__ float pow2_of(int byte) { return __uint_as_float((uint32_t)byte << 23); }

// The smallest exponent (+ 127) with amax <= 448 2^e, within the range: 448 is 1.75 2^8.
__device__ __forceinline__ int scale_for(float amax) {
    const uint32_t b = __float_as_uint(amax);
    return scale_byte((int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0));
}

// Two codes (the low or the high half of w) times a power of two, exact.
template <bool HIGH>
__device__ __forceinline__ h2 two_of(uint32_t w, float scale) {
    return __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HIGH));
}

// x - x: 0, or NaN for infinities and NaN.
__device__ __forceinline__ float nan_unless_finite(float x) { return x - x; }

// The nearest codes of four values times a power of two: at most 448, NaN for what is not finite.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[4], float by) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = __builtin_amdgcn_fmed3f(x[i] * by, -448.0f, 448.0f) + nan_unless_finite(x[i]);
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
}

// Four codes under a grown exponent: by = 2^(old - new) <= 1.
__device__ __forceinline__ uint32_t recoded(uint32_t w, float by) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * by, a[1] * by, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(b[0] * by, b[1] * by, lo, true);
}

}  // namespace rf
