// Producers of int8 rows with one scale a row (the activations of an int8 matrix product):
//
//   RMS norm   h = x + r (rounded to the stream's type), t = h w,  y = t / sqrt(mean h^2 + eps)
//   SwiGLU     y = silu(g) u
//   plain      y = x
//   a = max |y| over the row,  q = rint(127 y / a),  scale = a / 127
//
// The norm's 1 / sqrt(...) is one number for the row, so it cancels in q: q = rint(127 t / max |t|),
// and only the scale carries it.  One block per row; the row is read once and stays in registers
// between the reduction (sum of squares and largest magnitude together) and the rounding; rows too
// wide for that are read twice, the second time from L2.  The kernels are bound by the bytes of
// x, r, h and q.
#include "int8_common.cuh"

namespace {
using namespace ax;

enum Mode : int { kPlain = 0, kNorm = 1, kSwiglu = 2 };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float v, float* p) { *p = v; }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }

// Eight consecutive values.
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), c = unpack_bf16x2(u.z), d = unpack_bf16x2(u.w);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  uint4 u;
  u.x = pack_bf16x2(v[0], v[1]); u.y = pack_bf16x2(v[2], v[3]); u.z = pack_bf16x2(v[4], v[5]); u.w = pack_bf16x2(v[6], v[7]);
  *reinterpret_cast<uint4*>(p) = u;
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ float round_to(float v, const float*) { return v; }
__device__ __forceinline__ float round_to(float v, const __nv_bfloat16*) { return __bfloat162float(__float2bfloat16_rn(v)); }

struct RowArgs {
  const void* x;      // [rows, D], or [rows, 2 D] gate | up
  const void* res;    // [rows, D] or null
  const void* w;      // [D]
  void* h;            // [rows, D], the updated stream (with res)
  int8_t* q;          // [rows, D], row stride a multiple of 16
  float* scale;       // [rows]
  long xs, rs, hs, qs;
  int D;
  float eps;
};

// One value of element c of the row, the product t (norm), the gated value (SwiGLU) or x itself.
// `sq` gets the square that the norm sums.
template <int MODE, typename T, typename WT>
__device__ __forceinline__ float one_value(const RowArgs& a, const T* x, const T* r, T* h, int c, bool write_h, float& sq) {
  float v = to_f(x[c]);
  if (MODE == kSwiglu) return siluf_(v) * to_f(x[a.D + c]);
  if (MODE == kPlain) return v;
  if (r != nullptr) {
    v = round_to(v + to_f(r[c]), h);
    if (write_h) from_f(v, h + c);
  }
  sq = v * v;
  return __fmul_rn(v, to_f(((const WT*)a.w)[c]));
}
template <int MODE, typename T, typename WT>
__device__ __forceinline__ void eight_values(const RowArgs& a, const T* x, const T* r, T* h, int c, bool write_h, float (&t)[8], float& sq) {
  load8(x + c, t);
  if (MODE == kSwiglu) {
    float u[8];
    load8(x + a.D + c, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = siluf_(t[j]) * u[j];
  } else if (MODE == kNorm) {
    if (r != nullptr) {
      float rv[8];
      load8(r + c, rv);
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = round_to(t[j] + rv[j], h);
      if (write_h) store8(h + c, t);
    }
    float wv[8];
    load8((const WT*)a.w + c, wv);
#pragma unroll
    for (int j = 0; j < 8; ++j) { sq += t[j] * t[j]; t[j] = __fmul_rn(t[j], wv[j]); }
  }
}

// Sum and largest bits over the block; every thread gets both.
__device__ __forceinline__ void block_stats(float& sum, uint32_t& top) {
  __shared__ float s_sum[32];
  __shared__ uint32_t s_top[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  sum = warp_sum(sum);
  top = __reduce_max_sync(0xffffffffu, top);
  if (warps == 1) return;
  if (lane == 0) { s_sum[warp] = sum; s_top[warp] = top; }
  __syncthreads();
  sum = warp_sum(lane < warps ? s_sum[lane] : 0.f);
  top = __reduce_max_sync(0xffffffffu, lane < warps ? s_top[lane] : 0u);
}

// KEEP: VPT groups of eight values stay in registers (D <= VPT * 8 * threads).  Otherwise the row
// is walked twice.  VEC: rows and D allow 16-byte accesses; otherwise a thread's values lie
// blockDim apart, so that a warp's accesses are still contiguous.
template <int MODE, typename T, typename WT, int VPT, bool KEEP, bool VEC>
__global__ void __launch_bounds__(1024) int8_rows_kernel(const RowArgs a) {
  const long row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.xs;
  const T* r = (MODE == kNorm && a.res != nullptr) ? (const T*)a.res + row * a.rs : nullptr;
  T* h = (MODE == kNorm && a.res != nullptr) ? (T*)a.h + row * a.hs : nullptr;
  int8_t* q = a.q + row * a.qs;
  const int tid = threadIdx.x, n = blockDim.x;
  float t[KEEP ? VPT : 1][8];
  float sum = 0.f;
  uint32_t top = 0;
  if (VEC) {
    const int steps = KEEP ? VPT : (a.D + 8 * n - 1) / (8 * n);
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int c = (i * n + tid) * 8;
      if (c < a.D) {
        float (&v)[8] = t[KEEP ? i : 0];
        eight_values<MODE, T, WT>(a, x, r, h, c, true, v, sum);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[j]));
      }
    }
  } else {
    const int steps = KEEP ? VPT * 8 : (a.D + n - 1) / n;
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int c = i * n + tid;
      if (c < a.D) {
        float sq = 0.f;
        float& v = t[KEEP ? i / 8 : 0][KEEP ? i % 8 : 0];
        v = one_value<MODE, T, WT>(a, x, r, h, c, true, sq);
        sum += sq;
        top = max(top, abs_bits(v));
      }
    }
  }
  block_stats(sum, top);
  if (top < kTinyBits) top = 0;
  const float amax = __uint_as_float(top);
  const float inv = top ? __fdiv_rn(127.f, amax) : 0.f;
  if (tid == 0) {
    const float rstd = MODE == kNorm ? __frsqrt_rn(__fdiv_rn(sum, (float)a.D) + a.eps) : 1.f;
    a.scale[row] = __fdiv_rn(__fmul_rn(amax, rstd), 127.f);
  }
  if (VEC) {
    const int steps = KEEP ? VPT : (a.D + 8 * n - 1) / (8 * n);
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int c = (i * n + tid) * 8;
      if (c < a.D) {
        float (&v)[8] = t[KEEP ? i : 0];
        // the second walk reads the inputs again, not h: with r, x + r rounds to the same h
        if (!KEEP) eight_values<MODE, T, WT>(a, x, r, h, c, false, v, sum);
        int s[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = top ? int8_step(v[j], amax, inv) : 0;
        *reinterpret_cast<uint2*>(q + c) = make_uint2(pack_int8x4(s[0], s[1], s[2], s[3]), pack_int8x4(s[4], s[5], s[6], s[7]));
      }
    }
  } else {
    const int steps = KEEP ? VPT * 8 : (a.D + n - 1) / n;
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int c = i * n + tid;
      if (c < a.D) {
        float& v = t[KEEP ? i / 8 : 0][KEEP ? i % 8 : 0];
        float sq;
        if (!KEEP) v = one_value<MODE, T, WT>(a, x, r, h, c, false, sq);
        q[c] = (int8_t)(top ? int8_step(v, amax, inv) : 0);
      }
    }
  }
}

// Threads and groups per thread: the fewest groups that 1024 threads cover for few rows (latency:
// all loads of the row are in flight at once), two or more groups a thread for many rows (fewer
// warps wait at the reduction).
template <int MODE, typename T, typename WT, bool VEC>
int launch(const RowArgs& a, int rows, cudaStream_t stream) {
  const int groups = (a.D + 7) / 8;
  int vpt = 1;
  if (rows > 2 * axh::sm_count() && groups > 64) vpt = groups > 1024 ? 4 : 2;
  while (vpt < 4 && (long)vpt * 1024 < groups) vpt *= 2;
  int threads = ((groups + vpt - 1) / vpt + 31) / 32 * 32;
  if (threads > 1024) {
    int8_rows_kernel<MODE, T, WT, 1, false, VEC><<<rows, 1024, 0, stream>>>(a);
  } else if (vpt == 1) {
    int8_rows_kernel<MODE, T, WT, 1, true, VEC><<<rows, threads, 0, stream>>>(a);
  } else if (vpt == 2) {
    int8_rows_kernel<MODE, T, WT, 2, true, VEC><<<rows, threads, 0, stream>>>(a);
  } else {
    int8_rows_kernel<MODE, T, WT, 4, true, VEC><<<rows, threads, 0, stream>>>(a);
  }
  return (int)cudaGetLastError();
}

template <int MODE, typename T, typename WT>
int launch_vec(const RowArgs& a, int rows, cudaStream_t stream) {
  constexpr int kPer16 = 16 / (int)sizeof(T);
  const bool vec = a.D % 8 == 0 && a.xs % kPer16 == 0 && a.rs % kPer16 == 0 && a.hs % kPer16 == 0 && a.qs % 8 == 0 &&
                   (((uintptr_t)a.x | (uintptr_t)a.res | (uintptr_t)a.h | (uintptr_t)a.w) & 15) == 0 && ((uintptr_t)a.q & 7) == 0;
  return vec ? launch<MODE, T, WT, true>(a, rows, stream) : launch<MODE, T, WT, false>(a, rows, stream);
}

}  // namespace

// mode 0 plain, 1 RMS norm, 2 SwiGLU (x is [rows, 2 D]).  dt / wdt: 1 bf16, 0 fp32 (the weight may be fp32
// beside bf16 rows).  res / h may be null (norm without a residual).  Strides in elements.
AX_API int ax_int8_rows(int mode, int dt, int wdt, const void* x, long xs, const void* res, long rs, const void* w, float eps,
                        void* h, long hs, int8_t* q, long qs, float* scale, int rows, int D, cudaStream_t stream) {
  if (rows <= 0 || D <= 0) return 0;
  if (mode < 0 || mode > 2 || (mode == kNorm && w == nullptr) || ((res == nullptr) != (h == nullptr))) return -1;
  RowArgs a{x, res, w, h, q, scale, xs, rs, hs, qs, D, eps};
  using bf = __nv_bfloat16;
  if (mode == kNorm) {
    if (dt == 1 && wdt == 1) return launch_vec<kNorm, bf, bf>(a, rows, stream);
    if (dt == 1 && wdt == 0) return launch_vec<kNorm, bf, float>(a, rows, stream);
    if (dt == 0 && wdt == 0) return launch_vec<kNorm, float, float>(a, rows, stream);
    return -2;
  }
  if (mode == kSwiglu) return dt == 1 ? launch_vec<kSwiglu, bf, bf>(a, rows, stream) : launch_vec<kSwiglu, float, float>(a, rows, stream);
  return dt == 1 ? launch_vec<kPlain, bf, bf>(a, rows, stream) : launch_vec<kPlain, float, float>(a, rows, stream);
}
