// Producers of int8 rows with one scale a row (the activations of an int8 matrix product):
//
//   RMS norm   h = x + r (rounded to the stream's type), t = h w,  y = t / sqrt(mean h^2 + eps)
//   SwiGLU     y = silu(g) u
//   plain      y = x
//   a = max |y| over the row,  q = rint(127 y / a),  scale = a / 127
//
// The norm's 1 / sqrt(...) is one number for the row, so it cancels in q: q = rint(127 t / max |t|),
// and only the scale carries it.  A block takes a row at a time; the row is read once and stays in registers
// between the reduction (sum of squares and largest magnitude together) and the rounding, and the block's
// next row is requested before that reduction, so that its loads travel while this row is rounded.  Rows too
// wide for registers are read twice, the second time from L2.  The kernels are bound by the bytes of x, r, h
// and q, in so far as a row's 15 to 24 instructions a value leave room: norm of 8192 x 4096 bf16 with a
// residual 37.4 us (6.3 TB/s), SwiGLU of 4096 x 11008 45.4 us (5.0 TB/s: two special-function results and some 20
// instructions a value), 1021 x 5125 fp32 rows off the 16-byte grid 11 us.
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

// x + r as the stream's type rounds it.  The files are compiled with subnormal results flushed to zero; the stream keeps its own.
__device__ __forceinline__ float add_stream(float x, float r) {
  float h;
  asm("add.rn.f32 %0, %1, %2;" : "=f"(h) : "f"(x), "f"(r));
  return h;
}

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
  float least;        // sums of squares below this may lack some that vanished: 2^-100 D without an eps that hides it, else 0
};

// Sum (where SUM) and largest bits over the block; every thread gets both.  `turn` alternates between two sets of
// shared words, so that one barrier a row is enough.
template <bool SUM>
__device__ __forceinline__ void block_stats(float& sum, uint32_t& top, int turn) {
  __shared__ float s_sum[2][32];
  __shared__ uint32_t s_top[2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (SUM) sum = warp_sum(sum);
  top = __reduce_max_sync(0xffffffffu, top);
  if (warps == 1) return;
  if (lane == 0) { s_sum[turn][warp] = sum; s_top[turn][warp] = top; }
  __syncthreads();
  if (SUM) sum = warp_sum(lane < warps ? s_sum[turn][lane] : 0.f);
  top = __reduce_max_sync(0xffffffffu, lane < warps ? s_top[turn][lane] : 0u);
}

template <int MODE>
__device__ __forceinline__ void write_scale(const RowArgs& a, long row, float sum, uint32_t top) {
  const float rstd = MODE == kNorm ? __frsqrt_rn(__fdiv_rn(sum, (float)a.D) + a.eps) : 1.f;
  a.scale[row] = __fdiv_rn(__fmul_rn(top < kTinyBits ? 0.f : __uint_as_float(top), rstd), 127.f);
}

// A norm whose sums left fp32's range: squares that overflow (values above about 1e19), t = h w that does, or squares that
// vanish beside an eps that is nothing either.  (A row with a value that is not finite comes here too, and keeps its scale that is not.)
__device__ __forceinline__ bool norm_out_of_range(const RowArgs& a, float sum, uint32_t top) {
  return !(sum >= a.least && sum <= 3.402823466e38f) || top >= 0x7f800000u;
}
// Such a row again, when the block has nothing else left: its values scaled by the power of two that brings the largest |h| near
// one and cancels, y = t f / sqrt(mean (h f)^2 + eps f^2).  Three walks; h has been stored.
template <bool RES, typename T, typename WT>
__device__ __forceinline__ void norm_scaled_row(const RowArgs& a, long row) {
  const int tid = threadIdx.x, n = blockDim.x;
  const T* x = (const T*)a.x + row * a.xs;
  const T* r = RES ? (const T*)a.res + row * a.rs : x;
  const WT* w = (const WT*)a.w;
  auto value = [&](int c) {
    const float v = to_f(x[c]);
    return RES ? round_to(add_stream(v, to_f(r[c])), (const T*)nullptr) : v;
  };
  float most = 0.f, sum = 0.f;
#pragma unroll 1
  for (int c = tid; c < a.D; c += n) most = amax_nan(most, value(c));
  __syncthreads();                                             // what the first pass wrote lies before what follows
  uint32_t top = abs_bits(most);
  block_stats<false>(sum, top, 0);
  if (top >= 0x7f800000u) {                                    // a value that is not finite: so is the scale
    if (tid == 0) a.scale[row] = __uint_as_float(0x7fffffffu);
    return;
  }
  const int up = min(max(127 - (int)(top >> 23), -126), 100);
  const float f = __uint_as_float((uint32_t)(127 + up) << 23);
  sum = most = 0.f;
#pragma unroll 1
  for (int c = tid; c < a.D; c += n) {
    const float v = value(c) * f;
    sum += v * v;
    most = amax_nan(most, __fmul_rn(v, to_f(w[c])));
  }
  top = abs_bits(most);
  block_stats<true>(sum, top, 0);
  const Int8Grid grid = int8_grid(top);
  RowArgs b = a;
  b.eps = a.eps * f * f;
  if (tid == 0) write_scale<kNorm>(b, row, sum, top);
#pragma unroll 1
  for (int c = tid; c < a.D; c += n) a.q[row * a.qs + c] = (int8_t)int8_bits(__fmul_rn(value(c) * f, to_f(w[c])), grid);
}

// Inlined behind the loop over rows it costs that loop 6 % without a residual (8192 x 4096 bf16: 22.4 us, 21.3 as a call), and as a call
// 3 % with one (fp32: 83.7 inlined, 86.2).
template <typename T, typename WT>
__device__ __noinline__ void norm_scaled_row_call(const RowArgs a, long row) { norm_scaled_row<false, T, WT>(a, row); }

// Rows and D allow 16-byte accesses, and VPT groups of eight values a thread cover a row.
template <int MODE, bool RES, typename T, typename WT, int VPT>
__global__ void __launch_bounds__(VPT == 4 ? 512 : 1024, VPT == 4 && MODE == kSwiglu ? 2 : 1) int8_rows_kernel(const RowArgs a, int rows) {
  const WT* w = (const WT*)a.w;
  const int tid = threadIdx.x, n = blockDim.x;
  constexpr bool kTwo = MODE == kSwiglu || RES;
  // SwiGLU's two inputs a value leave no registers for another row: with it requested ahead only one block
  // fits an SM at 11008 columns (70 us for 4096 rows against 50 with a block a row)
  constexpr bool kAhead = MODE != kSwiglu;
  Raw8<T> first[VPT], second[kTwo ? VPT : 1];
  Raw8<WT> wv[MODE == kNorm ? VPT : 1];
  auto request = [&](long row) {
    const T* x = (const T*)a.x + row * a.xs;
    const T* r = RES ? (const T*)a.res + row * a.rs : x + a.D;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * n + tid) * 8;
      if (c < a.D) {
        first[i].load(x + c);
        if (kTwo) second[i].load(r + c);
      }
    }
  };
  chain_ready();
  chain_wait();
  bool again = false;
  long row = blockIdx.x;
  if (kAhead) request(row);
  if (MODE == kNorm) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if ((i * n + tid) * 8 < a.D) wv[i].load(w + (i * n + tid) * 8);
  }
#pragma unroll 1
  for (int turn = 0; row < rows; row += gridDim.x, turn ^= 1) {
    float t[VPT][8];
    float sum = 0.f, most = 0.f;
    if (!kAhead) request(row);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * n + tid) * 8;
      if (c < a.D) {
        first[i].get(t[i]);
        float u[8];
        if (kTwo) second[i].get(u);
        if (MODE == kSwiglu) {
#pragma unroll
          for (int j = 0; j < 8; ++j) t[i][j] = siluf_(t[i][j]) * u[j];
        }
        if (MODE == kNorm) {
          if (RES) {
#pragma unroll
            for (int j = 0; j < 8; ++j) t[i][j] = add_stream(t[i][j], u[j]);
            first[i].set(t[i]);                              // the stream's own rounding
            first[i].store((T*)a.h + row * a.hs + c);
          }
          float v[8];
          wv[i].get(v);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            sum += t[i][j] * t[i][j];
            t[i][j] = __fmul_rn(t[i][j], v[j]);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) t[i][j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) most = amax_nan(most, t[i][j]);
    }
    if (kAhead && row + gridDim.x < rows) request(row + gridDim.x);
    uint32_t top = abs_bits(most);
    block_stats<MODE == kNorm>(sum, top, turn);
    const Int8Grid grid = int8_grid(top);
    const bool out = MODE == kNorm && norm_out_of_range(a, sum, top);
    again |= out;                                            // (uniform)
    if (tid == 0) {
      if (out) a.scale[row] = __uint_as_float(0x7fffffffu);  // found below: no other row's scale is a NaN
      else write_scale<MODE>(a, row, sum, top);
    }
    int8_t* q = a.q + row * a.qs;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * n + tid) * 8;
      const uint2 b = int8_steps(t[i], grid);
      if (c < a.D) *reinterpret_cast<uint2*>(q + c) = b;
    }
  }
  if constexpr (MODE == kNorm) {
    if (again) {
      __syncthreads();
#pragma unroll 1
      for (row = blockIdx.x; row < rows; row += gridDim.x) {
        const bool marked = abs_bits(a.scale[row]) > 0x7f800000u;
        __syncthreads();                                     // all have read the mark, and the row before is done
        if (!marked) continue;
        if constexpr (RES) norm_scaled_row<true, T, WT>(a, row);
        else norm_scaled_row_call<T, WT>(a, row);
      }
    }
  }
}

// SwiGLU of many wide rows: the gated values wait in shared memory (D floats), not in registers, so that enough
// warps are there to load other rows meanwhile.
template <typename T>
__global__ void __launch_bounds__(512) swiglu_int8_rows_kernel(const RowArgs a) {
  extern __shared__ float4 held[];                           // [2][groups]: values 0-3 and 4-7 of every group of eight
  const long row = blockIdx.x;
  const int tid = threadIdx.x, groups = a.D / 8;
  const T* x = (const T*)a.x + row * a.xs;
  chain_ready();
  chain_wait();
  float most = 0.f, none = 0.f;
#pragma unroll 3
  for (int i = tid; i < groups; i += 512) {
    Raw8<T> g, u;
    g.load(x + 8 * i);
    u.load(x + a.D + 8 * i);
    float v[8], w[8];
    g.get(v);
    u.get(w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = siluf_(v[j]) * w[j];
      most = amax_nan(most, v[j]);
    }
    held[i] = make_float4(v[0], v[1], v[2], v[3]);
    held[groups + i] = make_float4(v[4], v[5], v[6], v[7]);
  }
  uint32_t top = abs_bits(most);
  block_stats<false>(none, top, 0);
  const Int8Grid grid = int8_grid(top);
  if (tid == 0) write_scale<kSwiglu>(a, row, 0.f, top);
  int8_t* q = a.q + row * a.qs;
#pragma unroll 3
  for (int i = tid; i < groups; i += 512) {
    const float4 p = held[i], r = held[groups + i];
    const float v[8] = {p.x, p.y, p.z, p.w, r.x, r.y, r.z, r.w};
    *reinterpret_cast<uint2*>(q + 8 * i) = int8_steps(v, grid);
  }
}

// Any alignment: a thread's values lie blockDim apart, so that a warp's accesses are contiguous.  KEEP: G
// groups of eight of them stay in registers; otherwise the row is walked twice.
template <int MODE, bool RES, typename T, typename WT, int G, bool KEEP>
__global__ void __launch_bounds__(KEEP ? 512 : 1024) int8_rows_any_kernel(const RowArgs a) {
  const long row = blockIdx.x;
  const int tid = threadIdx.x, n = blockDim.x;
  const T* x = (const T*)a.x + row * a.xs + tid;
  const T* r = (RES ? (const T*)a.res + row * a.rs : (const T*)a.x + row * a.xs + a.D) + tid;
  const WT* w = (const WT*)a.w + tid;
  constexpr bool kTwo = MODE == kSwiglu || RES;
  float t[G][8];
  float sum = 0.f, most = 0.f;
  chain_ready();
  chain_wait();
  // eight accesses of this thread, n apart, from column c0 + tid on
  auto walk = [&](float (&v)[8], int c0, bool out) {
    float u[8], wv[8];
    const int left = a.D - c0 - tid;                         // columns from this thread's first one on
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = j * n < left;
      v[j] = in ? to_f(x[c0 + j * n]) : 0.f;
      if (kTwo) u[j] = in ? to_f(r[c0 + j * n]) : 0.f;
      if (MODE == kNorm) wv[j] = in ? to_f(w[c0 + j * n]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (MODE == kSwiglu) v[j] = siluf_(v[j]) * u[j];
      if (MODE == kNorm) {
        if (RES) {
          v[j] = round_to(add_stream(v[j], u[j]), (const T*)nullptr);
          if (out && j * n < left) from_f(v[j], (T*)a.h + row * a.hs + c0 + tid + j * n);
        }
        sum += v[j] * v[j];
        v[j] = __fmul_rn(v[j], wv[j]);
      }
    }
  };
  const int groups = KEEP ? G : (a.D + 8 * n - 1) / (8 * n);
#pragma unroll
  for (int k = 0; k < groups; ++k) {
    float (&v)[8] = t[KEEP ? k : 0];
    walk(v, 8 * n * k, true);
#pragma unroll
    for (int j = 0; j < 8; ++j) most = amax_nan(most, v[j]);
  }
  uint32_t top = abs_bits(most);
  block_stats<MODE == kNorm>(sum, top, 0);
  const Int8Grid grid = int8_grid(top);
  const bool again = MODE == kNorm && norm_out_of_range(a, sum, top);
  if (tid == 0) write_scale<MODE>(a, row, sum, top);
  int8_t* q = a.q + row * a.qs + tid;
#pragma unroll
  for (int k = 0; k < groups; ++k) {
    float (&v)[8] = t[KEEP ? k : 0];
    if (!KEEP) walk(v, 8 * n * k, false);                    // x and r again, not h: they round to the same sum
    const uint2 b = int8_steps(v, grid);
    const int left = a.D - 8 * n * k - tid;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * n < left) q[8 * n * k + j * n] = (int8_t)((j < 4 ? b.x : b.y) >> (8 * (j % 4)));
  }
  if constexpr (MODE == kNorm) {
    if (again) norm_scaled_row<RES, T, WT>(a, row);
  }
}

// Blocks of Kern that the device holds at once.
template <auto Kern>
int resident(int threads) {
  static int known[64][33] = {{0}};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return axh::sm_count();
  int& k = known[dev][threads / 32];
  if (k == 0) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kern, threads, 0) != cudaSuccess || n < 1) n = 1;
    k = n * axh::sm_count();
  }
  return k;
}
template <auto Kern>
int launch_rows(const RowArgs& a, int rows, int threads, bool ahead, cudaStream_t stream) {
  const int most = ahead ? resident<Kern>(threads) : rows;   // a kernel that does not request ahead takes a block a row
  return axh::launch_chained(Kern, dim3(rows < most ? rows : most), dim3(threads), 0, 1, stream, a, rows);
}

// Threads and groups per thread: one group each for few rows (latency: all loads of the row are in flight
// at once), four for many rows (a warp's share of the reduction and of the row's divisions is paid once per
// 1024 values: 508 instructions a warp at two groups, of which 150 do not depend on them); rows up to 16384
// wide stay in registers.
template <int MODE, bool RES, typename T, typename WT>
int launch_vec(const RowArgs& a, int rows, cudaStream_t stream) {
  const int groups = (a.D + 7) / 8;
  int vpt = groups > 1024 ? 2 : 1;
  if (rows > 2 * axh::sm_count() && groups > 64) vpt = groups >= 256 ? 4 : 2;
  const int threads = ((groups + vpt - 1) / vpt + 31) / 32 * 32;
  if constexpr (MODE == kSwiglu) {
    // Values in shared memory where registers would leave one or two blocks an SM.  Registers / shared memory, us:
    // 4096 rows of bf16, 8192 wide 31.3 / 36.9, 9728 40.4 / 41.9, 11008 51.5 / 45.2, 14336 60.2 / 57.6; fp32, 4096 wide
    // 35.8 / 25.3, 8192 67.1 / 45.8.
    if (vpt == 4 && a.D >= (sizeof(T) == 2 ? 10240 : 4096)) {
      static bool configured[64] = {false};
      int dev = 0;
      cudaGetDevice(&dev);
      if (dev < 0 || dev >= 64 || !configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(swiglu_int8_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 16384 * 4);
        if (e != cudaSuccess) return (int)e;
        if (dev >= 0 && dev < 64) configured[dev] = true;
      }
      return axh::launch_chained(swiglu_int8_rows_kernel<T>, dim3(rows), dim3(512), a.D * 4, 1, stream, a);
    }
  }
  if (vpt == 1) return launch_rows<int8_rows_kernel<MODE, RES, T, WT, 1>>(a, rows, threads, MODE != kSwiglu, stream);
  if (vpt == 2) return launch_rows<int8_rows_kernel<MODE, RES, T, WT, 2>>(a, rows, threads, MODE != kSwiglu, stream);
  return launch_rows<int8_rows_kernel<MODE, RES, T, WT, 4>>(a, rows, threads, MODE != kSwiglu, stream);
}

template <int MODE, bool RES, typename T, typename WT>
int launch(const RowArgs& a, int rows, cudaStream_t stream) {
  constexpr int kPer16 = 16 / (int)sizeof(T);
  const bool vec = a.D % 8 == 0 && a.D <= 16384 && a.xs % kPer16 == 0 && a.rs % kPer16 == 0 && a.hs % kPer16 == 0 && a.qs % 8 == 0 &&
                   (((uintptr_t)a.x | (uintptr_t)a.res | (uintptr_t)a.h | (uintptr_t)a.w) & 15) == 0 && ((uintptr_t)a.q & 7) == 0;
  if (vec) return launch_vec<MODE, RES, T, WT>(a, rows, stream);
  // one group of eight a thread up to 4096 columns, two up to 8192
  const int threads = ((a.D + 7) / 8 + 31) / 32 * 32;
  if (threads <= 512) return axh::launch_chained(int8_rows_any_kernel<MODE, RES, T, WT, 1, true>, dim3(rows), dim3(threads), 0, 1, stream, a);
  if (threads <= 1024) {
    const int half = ((a.D + 15) / 16 + 31) / 32 * 32;
    return axh::launch_chained(int8_rows_any_kernel<MODE, RES, T, WT, 2, true>, dim3(rows), dim3(half), 0, 1, stream, a);
  }
  return axh::launch_chained(int8_rows_any_kernel<MODE, RES, T, WT, 1, false>, dim3(rows), dim3(1024), 0, 1, stream, a);
}

template <typename T, typename WT>
int launch_norm(const RowArgs& a, int rows, cudaStream_t stream) {
  return a.res != nullptr ? launch<kNorm, true, T, WT>(a, rows, stream) : launch<kNorm, false, T, WT>(a, rows, stream);
}

}  // namespace

// mode 0 plain, 1 RMS norm, 2 SwiGLU (x is [rows, 2 D]).  dt / wdt: 1 bf16, 0 fp32 (the weight may be fp32
// beside bf16 rows).  res / h may be null (norm without a residual).  Strides in elements.
AX_API int ax_int8_rows(int mode, int dt, int wdt, const void* x, long xs, const void* res, long rs, const void* w, float eps,
                        void* h, long hs, int8_t* q, long qs, float* scale, int rows, int D, cudaStream_t stream) {
  if (rows <= 0 || D <= 0) return 0;
  if (mode < 0 || mode > 2 || (mode == kNorm && w == nullptr) || ((res == nullptr) != (h == nullptr))) return -1;
  constexpr float kLeast = 7.888609052e-31f;                   // 2^-100: a square that vanishes (below 2^-126) is 2^-26 of that
  RowArgs a{x, res, w, h, q, scale, xs, rs, hs, qs, D, eps, eps < kLeast ? kLeast * (float)D : 0.f};
  using bf = __nv_bfloat16;
  if (mode == kNorm) {
    if (dt == 1 && wdt == 1) return launch_norm<bf, bf>(a, rows, stream);
    if (dt == 1 && wdt == 0) return launch_norm<bf, float>(a, rows, stream);
    if (dt == 0 && wdt == 0) return launch_norm<float, float>(a, rows, stream);
    return -2;
  }
  if (mode == kSwiglu) return dt == 1 ? launch<kSwiglu, false, bf, bf>(a, rows, stream) : launch<kSwiglu, false, float, float>(a, rows, stream);
  return dt == 1 ? launch<kPlain, false, bf, bf>(a, rows, stream) : launch<kPlain, false, float, float>(a, rows, stream);
}
