// Shared by the int8 serving kernels: exact rounding of a value to the int8 grid of a group
// (a row of activations, a page of the cache).
//
//   q = rint(127 t / a),  a = the group's largest magnitude,  value = q a / 127
//
// The quotient is formed from 127 / a in two floats, so that it is the real one rounded once to fp32: a quotient
// that lies on a border between two steps (a value of exactly half the largest is 63.5 steps, and bf16 values
// are that often) is that border exactly and goes to the even step.  Products of two bf16 values are exact in
// fp32, so no rounding depends on the order in which anything was summed.
#pragma once
#include "common.cuh"

namespace ax {

// Programmatic dependent launch: a kernel launched with launch_chained may start while the one before it on
// the stream still runs, and sets itself up (barriers, TMEM, descriptors) until chain_wait returns, which is when that
// kernel has ended and its writes are visible.  Every thread that touches memory calls chain_wait first, in
// every block, so that a grid never ends before the one it follows.  chain_ready lets the next grid start.
__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void chain_ready() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Largest magnitudes travel as the bits of |x|: integer order is the order of non-negative floats, and
// NaN lies above infinity, so a NaN in a group reaches the group's magnitude.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// max(a, |x|) that keeps a NaN; one instruction per value inside a thread.
__device__ __forceinline__ float amax_nan(float a, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(x)));
  return r;
}

// What a group's largest magnitude means for its values: t -> t (n / a), n = 127 for values, the old
// magnitude for steps that move to a larger one.
struct Int8Grid {
  float hi, lo;        // n / a as a sum of two floats; 0 for a group whose steps are all 0
};
// 2^-118: below it a group counts as zero.  From there on a / 127 is a normal number, and a value that is not (the files are
// compiled with those flushed to zero) is less than half a step.
constexpr uint32_t kTinyBits = 9u << 23;
__device__ __forceinline__ Int8Grid two_float_quotient(float n, float a) {
  Int8Grid g;
  g.hi = __fdiv_rn(n, a);
  // (the small part of 127 / a is below the normal numbers from a = 2^108 on: kept, to 2^-150, which times a value below 2^128
  // is far less than the quotient's last bit)
  asm("div.full.f32 %0, %1, %2;" : "=f"(g.lo) : "f"(__fmaf_rn(-g.hi, a, n)), "f"(a));
  return g;
}
__device__ __forceinline__ Int8Grid int8_grid(uint32_t top) {
  if (top < kTinyBits || top >= 0x7f800000u) return Int8Grid{0.f, 0.f};
  return two_float_quotient(127.f, __uint_as_float(top));
}
// From magnitude `old_bits` to a larger one, both times 2^64 where the quotient's remainder would be below the normal numbers.
__device__ __forceinline__ Int8Grid int8_ratio(uint32_t old_bits, uint32_t top) {
  if (top < kTinyBits || top >= 0x7f800000u) return Int8Grid{0.f, 0.f};
  const float f = top < (87u << 23) ? 18446744073709551616.f : 1.f;      // 2^-40
  return two_float_quotient(__uint_as_float(old_bits) * f, __uint_as_float(top) * f);
}

// Adding 1.5 * 2^23 rounds a number below 2^22 to the nearest whole one (ties to even) and leaves that number,
// in two's complement, in the low bits of the sum: no conversion instruction, which the SM has at a
// sixteenth of the rate of additions.
__device__ __forceinline__ uint32_t int8_bits(float t, const Int8Grid& g) {
  float low, q;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(low) : "f"(t), "f"(g.lo));
  asm("fma.rn.f32 %0, %1, %2, %3;" : "=f"(q) : "f"(t), "f"(g.hi), "f"(low));
  return __float_as_uint(__fadd_rn(q, 12582912.f));
}

__device__ __forceinline__ uint32_t pack_low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Steps of eight values as packed bytes.  (A value that is not finite makes its group's grid zero and its own
// byte something; the group's magnitude says that none of them mean anything.)
__device__ __forceinline__ uint2 int8_steps(const float (&t)[8], const Int8Grid& g) {
  uint32_t b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) b[j] = int8_bits(t[j], g);
  return make_uint2(pack_low_bytes(b[0], b[1], b[2], b[3]), pack_low_bytes(b[4], b[5], b[6], b[7]));
}

// Eight consecutive values, as they lie in memory and as numbers.
template <typename T>
struct Raw8;
template <>
struct Raw8<__nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), c = unpack_bf16x2(u.z), d = unpack_bf16x2(u.w);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  }
  // rounds to bf16; v becomes what was kept
  __device__ __forceinline__ void set(float (&v)[8]) {
    u.x = pack_bf16x2(v[0], v[1]); u.y = pack_bf16x2(v[2], v[3]); u.z = pack_bf16x2(v[4], v[5]); u.w = pack_bf16x2(v[6], v[7]);
    get(v);
  }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = u; }
};
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ void set(float (&v)[8]) {
    a = make_float4(v[0], v[1], v[2], v[3]);
    b = make_float4(v[4], v[5], v[6], v[7]);
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<float4*>(p) = a;
    *reinterpret_cast<float4*>(p + 4) = b;
  }
};

}  // namespace ax

namespace axh {
// Launch with the attribute above, and in clusters of `cluster` blocks along x where that is more than one.
template <typename... P, typename... A>
int launch_chained(void (*kern)(P...), dim3 grid, dim3 block, int smem, int cluster, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kern, args...);
}
}  // namespace axh
