// Numbers for the matrix instruction in float16 with a power of two beside them: x = f 2^e.  float16 has three bits more than
// bfloat16 and the same rate, but not its range, so a set of numbers (a query; the keys, or the values, of 32 tokens) that does
// not fit has an exponent other than 0.
#pragma once
#include "common.h"

// The exponent of numbers up to `most` in magnitude.  None between 2^-8 and 2^15: there float16 holds all of them within 2^-12 of
// themselves, or within 2^-25, which is 2^-17 of the largest, where they are smaller than 2^-14.  Not below `least`.
__device__ __forceinline__ int half_exponent(float most, int least = -60) {
  const int e = (int)(__float_as_uint(most) >> 23) - 127;  // 128 for an infinity
  return most == 0.f || (e >= -8 && e <= 14) ? 0 : min(max(e - 6, least), 121);
}
// The lowest exponent of values: sums of up to 2^67, with weights of 2^7 times their own, can be brought to any.
#define VALUES_LEAST -53
__device__ __forceinline__ float power_of_two(int e) { return e < -126 ? 0.f : __uint_as_float((uint32_t)(min(e, 127) + 127) << 23); }
// Two floats rounded (nearest, ties to even) to a pair of float16.
__device__ __forceinline__ uint32_t pack2_f16(float lo, float hi) {
  typedef float two_floats __attribute__((ext_vector_type(2)));
  typedef _Float16 two_halves __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((two_floats){lo, hi}, two_halves));
}
