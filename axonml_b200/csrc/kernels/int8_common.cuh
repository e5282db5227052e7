// Shared by the int8 serving kernels: exact rounding of a value to the int8 grid of a group
// (a row of activations, a page of the cache).
//
//   q = rint(127 t / a),  a = the group's largest magnitude,  value = q a / 127
//
// Products of two bf16 values are exact in fp32, and so is that times 127 (8 + 8 + 7 bits), so the
// correctly rounded quotient decides every rounding as the real number would, ties included: the
// result does not depend on the order in which anything was summed.
#pragma once
#include "common.cuh"

namespace ax {

// Largest magnitudes are kept as the bits of |x|: integer order is the order of non-negative
// floats, and NaN lies above infinity, so a NaN in a group reaches the group's magnitude.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

constexpr uint32_t kTinyBits = 0x00800000u;   // smallest normal number: below it a group counts as zero

// The division only runs for values next to a border between two steps: t * inv is off by at most
// two roundings of a number <= 127, i.e. by 1.6e-5, so a fraction at least 1e-4 from one half
// already shows the side.  One value in 5000 takes the division; a NaN (inv infinite) takes it too.
__device__ __forceinline__ int int8_step(float t, float amax, float inv) {
  const float f = t * inv;
  float n = rintf(f);
  if (!(fabsf(fabsf(f - n) - 0.5f) >= 1e-4f)) n = rintf(__fdiv_rn(__fmul_rn(t, 127.f), amax));
  return __float2int_rn(n);
}

__device__ __forceinline__ uint32_t pack_int8x4(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | ((uint32_t)(b & 255) << 8) | ((uint32_t)(c & 255) << 16) | ((uint32_t)d << 24);
}

}  // namespace ax
