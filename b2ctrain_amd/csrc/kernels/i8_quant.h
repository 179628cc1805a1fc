// Rounding to 8 bits by rows, as the 8-bit operators do it.
#pragma once
#include "dense.h"

namespace b2c {
namespace dev {

// A row's divisor: scale = top / 127, from its largest magnitude as bits, in which an infinity or NaN orders last.
struct RowScale {
  float scale, inverse;
  bool plain;  // the quotient may be formed from the inverse: neither under- nor overflows
  __device__ __forceinline__ explicit RowScale(uint32_t top) {
    const bool fine = top < 0x7f800000u;
    scale = fine ? __builtin_bit_cast(float, top) / 127.f : __builtin_nanf("");
    plain = scale > 1e-30f;
    inverse = plain ? 1.f / scale : 0.f;
  }
  // x / scale rounded to nearest even twice, to single precision and to an integer, as two's complement in the low
  // byte. With the correctly rounded inverse y, q = x y and the remainder r = x - q scale (exact in one fused
  // operation), q + r y is the correctly rounded quotient (Markstein 1990): three operations in place of a division's ten.
  // Adding 1.5 2^23 then leaves the integer in the low bits (the bits above the lowest byte are not cleared). The scale of a row of
  // subnormals may be rounded down so far that a quotient passes 127 (160 units in the last place have a scale of one): it is held there.
  __device__ __forceinline__ uint32_t operator()(float x) const {
    float q = 0.f;
    if (plain) {
      q = x * inverse;
      q = fmaf(fmaf(-q, scale, x), inverse, q);
    } else if (scale > 0.f) {
      q = fminf(fmaxf(x / scale, -127.f), 127.f);
    }
    return __builtin_bit_cast(uint32_t, q + 12582912.f);
  }
  // The same for values that were computed in single precision themselves: one rounding of x inverse, which may fall to the
  // other side where x / scale lies within 2^-17 of the middle of two integers. Of a plain row, or one of zeros.
  __device__ __forceinline__ uint32_t near(float x) const { return __builtin_bit_cast(uint32_t, fmaf(x, inverse, 12582912.f)); }
};
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
// The lowest bytes of four words.
__device__ __forceinline__ uint32_t bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}

}  // namespace dev
}  // namespace b2c
