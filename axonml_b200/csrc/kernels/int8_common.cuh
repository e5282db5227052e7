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

// What a group's largest magnitude means for its values.
struct Int8Grid {
  float amax, inv;     // inv = 127 / amax
  bool live;           // false: the magnitude is zero, below the normal numbers, or not finite; all steps are 0
  bool exact;          // the inverse overflows: divide for every value
};
__device__ __forceinline__ Int8Grid int8_grid(uint32_t top) {
  Int8Grid g;
  g.live = top >= 0x00800000u && top < 0x7f800000u;
  g.amax = __uint_as_float(top);
  g.inv = g.live ? __fdiv_rn(127.f, g.amax) : 0.f;
  g.exact = !(g.inv < 3.0e38f);
  return g;
}

// Adding 1.5 * 2^23 rounds a number below 2^22 to the nearest whole one (ties to even) and leaves that number,
// in two's complement, in the low bits of the sum: no conversion instruction, which the SM has at a
// sixteenth of the rate of additions.
constexpr float kRound = 12582912.f;

// t * inv is off by at most two roundings of a number <= 127, i.e. by 1.6e-5: a value further than 3e-5 from
// the border between two steps is on its side already.  Only the others (one in 16000) take the division.
constexpr float kBorder = 0.5f - 3.0e-5f;

__device__ __forceinline__ uint32_t int8_exact_bits(float t, float amax) {
  return __float_as_uint(__fadd_rn(__fdiv_rn(__fmul_rn(t, 127.f), amax), kRound));
}

__device__ __forceinline__ uint32_t pack_low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Steps of N values (N a multiple of 4) as packed bytes.
template <int N>
__device__ __forceinline__ void int8_steps(const float (&t)[N], const Int8Grid& g, uint32_t (&packed)[N / 4]) {
  uint32_t b[N];
  float worst = g.exact ? 1.f : 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float f = t[j] * g.inv;
    const float r = __fadd_rn(f, kRound);
    worst = fmaxf(worst, fabsf(f - __fadd_rn(r, -kRound)));
    b[j] = __float_as_uint(r);
  }
  if (worst > kBorder) {
#pragma unroll
    for (int j = 0; j < N; ++j) b[j] = int8_exact_bits(t[j], g.amax);
  }
#pragma unroll
  for (int j = 0; j < N; j += 4) packed[j / 4] = g.live ? pack_low_bytes(b[j], b[j + 1], b[j + 2], b[j + 3]) : 0u;
}

// One value.
__device__ __forceinline__ int8_t int8_step(float t, const Int8Grid& g) {
  const float f = t * g.inv;
  float r = __fadd_rn(f, kRound);
  if (fabsf(f - __fadd_rn(r, -kRound)) > kBorder || g.exact) r = __uint_as_float(int8_exact_bits(t, g.amax));
  return g.live ? (int8_t)(__float_as_uint(r) & 255u) : (int8_t)0;
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
