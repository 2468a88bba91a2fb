// The two scales of a block of e4m3 products.
//
// A block's sum p is to be multiplied by a row's scale a and a tile's b, any
// fp32 numbers.  One multiplication by fl(a b) is within a rounding of that
// while the product is a normal number.  Where it overflows, p a b may be finite
// (and is zero for p = 0, not NaN); where it is subnormal, it has lost bits that p
// (up to 2^24.7) brings back into the normal range.  Then p is multiplied by the
// larger scale first: if a b overflows, both are above 1 and no step exceeds the
// result; if it is subnormal, the larger is below 2^23 and p times it does not
// overflow, nor underflow unless the result does.
#pragma once

#include <cstdint>

namespace col {

__device__ __forceinline__ bool normal_f32(float v) {
  return (__float_as_uint(v) << 1) - (0x00800000u << 1) < ((0x7f800000u - 0x00800000u) << 1);
}

__device__ __forceinline__ bool finite_nonzero(float v) {
  return (__float_as_uint(v) << 1) - 1u < (0x7f800000u << 1) - 1u;
}

// p a b = (p first) rest
struct BlockScales {
  float first;
  float rest;
};

__device__ __forceinline__ BlockScales block_scales(float a, float b) {
  const float product = a * b;
  // a zero, an infinity or a NaN among the scales is in the product too
  if (normal_f32(product) || !finite_nonzero(a) || !finite_nonzero(b)) return {1.0f, product};
  return fabsf(a) > fabsf(b) ? BlockScales{a, b} : BlockScales{b, a};
}

}  // namespace col
