// Rows held in 8 bits: a row x (a position's key or value head, a token, a row of a matrix) is kept as codes
//     c_i = rint(x_i * (127 / top)),   top = max |x_i|,
// and the scale top / 127 in float32: c_i * scale is x_i to within half a step, top / 254.  For bfloat16 rows the codes are
// the exact quotient's: 254 x_i and an odd multiple of top are at least one part in 2^16 apart, and the two roundings of the product
// come to one in 2^23, or they are equal because 127 / top is a power of two and nothing rounds, or because x_i is just half of the top
// (63.5 steps: either neighbour is as near).  A row whose top is below 2^-100 is a row of zeros (127 / top would pass the range of
// float32); one that holds an infinity or a NaN has the scale NaN and codes of zero, so that whatever is computed from it is NaN,
// as it would be from the row itself.
#pragma once

#include "common.cuh"

namespace nnis {

struct RowScale {
    float inverse, scale;
};

// The magnitude as its bits: as whole numbers they compare like the magnitudes, and a NaN is above every number.
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ RowScale row_scale(uint32_t top_bits) {
    const float top = __uint_as_float(top_bits);
    if (top_bits >= 0x7f800000u) return {0.f, __uint_as_float(0x7fc00000u)};
    if (top < 0x1p-100f) return {0.f, 0.f};
    return {__fdiv_rn(127.f, top), __fdiv_rn(top, 127.f)};
}

// (a NaN's or an infinity's product with 0 is NaN, whose code is 0)
__device__ __forceinline__ int row_code(float x, float inverse) { return __float2int_rn(__fmul_rn(x, inverse)); }

// Four codes as a word: a product of at most 127 plus 1.5 * 2^23 is rounded to a whole number, ties to even, whose low byte is the
// code (a conversion to a whole number runs at a quarter of an addition's rate).  `good` 0: a row that is no number.
__device__ __forceinline__ uint32_t code_word(float a, float b, float c, float d, float inverse, uint32_t good) {
    constexpr float kWhole = 12582912.f;
    const uint32_t x = __float_as_uint(__fadd_rn(__fmul_rn(a, inverse), kWhole)), y = __float_as_uint(__fadd_rn(__fmul_rn(b, inverse), kWhole));
    const uint32_t z = __float_as_uint(__fadd_rn(__fmul_rn(c, inverse), kWhole)), w = __float_as_uint(__fadd_rn(__fmul_rn(d, inverse), kWhole));
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410) & good;
}
__device__ __forceinline__ uint32_t good_row(float scale) { return scale == scale ? 0xffffffffu : 0u; }

__device__ __forceinline__ uint32_t pack_codes(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}

// The largest of a group of G lanes (a power of two); every lane of the warp calls it.
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ float code_value(uint32_t word, int i) { return (float)(int8_t)(word >> (8 * i)); }

}  // namespace nnis
