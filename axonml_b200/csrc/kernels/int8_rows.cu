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
// blockDim apart, so that a warp's accesses are still contiguous.  All loads of a walk come before its
// stores of h: the compiler may not move a load across a store that could alias it.
template <int MODE, typename T, typename WT, int VPT, bool KEEP, bool VEC>
__global__ void __launch_bounds__(VPT == 4 ? 512 : 1024) int8_rows_kernel(const RowArgs a) {
  const long row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.xs;
  const bool res = MODE == kNorm && a.res != nullptr;
  const T* r = res ? (const T*)a.res + row * a.rs : nullptr;
  T* h = res ? (T*)a.h + row * a.hs : nullptr;
  const WT* w = (const WT*)a.w;
  int8_t* q = a.q + row * a.qs;
  const int tid = threadIdx.x, n = blockDim.x;
  constexpr int W = VEC ? 8 : 1;                 // values of an access
  constexpr int S = VEC ? VPT : VPT * 8;         // accesses of a thread (KEEP)
  float t[VPT][8];
  float sum = 0.f, most = 0.f;
  chain_ready();
  chain_wait();

  // values of accesses [i0, i0 + S) of this thread into t; `out` says whether h is written
  auto walk = [&](int i0, bool out) {
    if constexpr (VEC) {
      Raw8<T> xv[VPT], second[MODE == kPlain ? 1 : VPT];
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = ((i0 + i) * n + tid) * 8;
        if (c < a.D) {
          xv[i].load(x + c);
          if (MODE == kSwiglu) second[i].load(x + a.D + c);
          if (MODE == kNorm && res) second[i].load(r + c);
        }
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = ((i0 + i) * n + tid) * 8;
        if (c < a.D) {
          xv[i].get(t[i]);
          if (MODE == kSwiglu) {
            float u[8];
            second[i].get(u);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[i][j] = siluf_(t[i][j]) * u[j];
          }
          if (MODE == kNorm) {
            Raw8<WT> wr;
            wr.load(w + c);
            if (res) {
              float u[8];
              second[i].get(u);
#pragma unroll
              for (int j = 0; j < 8; ++j) t[i][j] += u[j];
              xv[i].set(t[i]);
              if (out) xv[i].store(h + c);
            }
            float wv[8];
            wr.get(wv);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              sum += t[i][j] * t[i][j];
              t[i][j] = __fmul_rn(t[i][j], wv[j]);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) t[i][j] = 0.f;
        }
      }
    } else {
      float second[MODE == kPlain ? 1 : VPT * 8], wv[MODE == kNorm ? VPT * 8 : 1];
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const int c = (i0 + i) * n + tid;
        const bool in = c < a.D;
        t[i / 8][i % 8] = in ? to_f(x[c]) : 0.f;
        if (MODE == kSwiglu) second[i] = in ? to_f(x[a.D + c]) : 0.f;
        if (MODE == kNorm) {
          second[i] = in && res ? to_f(r[c]) : 0.f;
          wv[i] = in ? to_f(w[c]) : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const int c = (i0 + i) * n + tid;
        float& v = t[i / 8][i % 8];
        if (MODE == kSwiglu) v = siluf_(v) * second[i];
        if (MODE == kNorm) {
          if (res) {
            v = round_to(v + second[i], h);
            if (out && c < a.D) from_f(v, h + c);
          }
          sum += v * v;
          v = __fmul_rn(v, wv[i]);
        }
      }
    }
  };
  const int rounds = KEEP ? 1 : (a.D + W * S * n - 1) / (W * S * n);
#pragma unroll 1
  for (int k = 0; k < rounds; ++k) {
    walk(k * S, true);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) most = amax_nan(most, t[i][j]);
  }
  uint32_t top = abs_bits(most);
  block_stats(sum, top);
  const Int8Grid grid = int8_grid(top);
  if (tid == 0) {
    const float rstd = MODE == kNorm ? __frsqrt_rn(__fdiv_rn(sum, (float)a.D) + a.eps) : 1.f;
    const float amax = top < 0x00800000u ? 0.f : grid.amax;
    a.scale[row] = __fdiv_rn(__fmul_rn(amax, rstd), 127.f);
  }
#pragma unroll 1
  for (int k = 0; k < rounds; ++k) {
    // the second walk reads x and r again, not h: they round to the same sum
    if (!KEEP) walk(k * S, false);
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = ((k * S + i) * n + tid) * 8;
        uint32_t b[2];
        int8_steps<8>(t[i], grid, b);
        if (c < a.D) *reinterpret_cast<uint2*>(q + c) = make_uint2(b[0], b[1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        uint32_t b[2];
        int8_steps<8>(t[i], grid, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = (k * S + i * 8 + j) * n + tid;
          if (c < a.D) q[c] = (int8_t)(b[j / 4] >> (8 * (j % 4)));
        }
      }
    }
  }
}

// Threads and groups per thread: one group each for few rows (latency: all loads of the row are in flight
// at once), four for many rows (a warp's share of the reduction and of the row's divisions is paid once per
// 1024 values: 508 instructions a warp at two groups, of which 150 do not depend on them); rows up to 16384
// wide stay in registers.
template <int MODE, typename T, typename WT, bool VEC>
int launch(const RowArgs& a, int rows, cudaStream_t stream) {
  const int groups = (a.D + 7) / 8;
  int vpt = groups > 1024 ? 2 : 1;   // (the scalar path stops at two: its values are 8 x as many accesses)
  if (rows > 2 * axh::sm_count() && groups > 64) vpt = VEC && groups >= 256 ? 4 : 2;
  const int threads = ((groups + vpt - 1) / vpt + 31) / 32 * 32;
  if (threads > (vpt == 4 ? 512 : 1024)) return axh::launch_chained(int8_rows_kernel<MODE, T, WT, 1, false, VEC>, dim3(rows), dim3(1024), 0, 1, stream, a);
  if (vpt == 1) return axh::launch_chained(int8_rows_kernel<MODE, T, WT, 1, true, VEC>, dim3(rows), dim3(threads), 0, 1, stream, a);
  if (vpt == 2) return axh::launch_chained(int8_rows_kernel<MODE, T, WT, 2, true, VEC>, dim3(rows), dim3(threads), 0, 1, stream, a);
  if constexpr (VEC) return axh::launch_chained(int8_rows_kernel<MODE, T, WT, 4, true, VEC>, dim3(rows), dim3(threads), 0, 1, stream, a);
  return -1;
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
