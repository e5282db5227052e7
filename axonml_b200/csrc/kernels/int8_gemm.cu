// Matrix product of int8 rows with an int8 weight, a scale for each row and each output channel:
//
//   y[m, n] = sx[m] sw[n] sum_k q[m, k] w[n, k]  (+ b[n])
//
// The sum runs on the tensor cores as tcgen05.mma kind::i8 (int8 x int8 -> int32 in TMEM), so it is
// exact: |sum| <= 2^14 K fits 31 bits up to K = 131071, and splitting K over blocks changes nothing.
// The two scales, the bias and the one rounding to the output's type are the epilogue.
//
// Two kernels.
//  * few rows (int8_stream_kernel): bound by the weight's bytes.  The weight takes the MMA's 128-row
//    side and the tokens its narrow side (N = 16 .. 128), so that one MMA per 32 bytes of K serves
//    all tokens; K is split over a cluster of up to 8 blocks so that even a narrow matrix keeps every
//    SM loading, and the blocks add their int32 accumulators through distributed shared memory.
//  * many rows (int8_pair_kernel): bound by the tensor cores.  CTA pairs (cta_group::2) on 256 x 256
//    or 256 x 128 tiles, persistent, the accumulator double-buffered in TMEM so that a tile's epilogue
//    runs beside the next tile's products.
#include "int8_common.cuh"

namespace {
using namespace ax;

constexpr int kRowsA = 128;    // rows of the MMA's M side per CTA
constexpr int kBytesK = 128;   // bytes (= int8 values) of K per stage: one 128-byte swizzle row
constexpr int kMmaK = 32;      // K of one kind::i8 MMA

// Instruction descriptor of kind::i8: int32 accumulator, signed operands, both K-major.
__host__ __device__ constexpr uint32_t idesc_s8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_s8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_s8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ int4 ld_cluster4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_out(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_out4(float* p, float a, float b, float c, float d) { *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d); }
__device__ __forceinline__ void store_out4(__nv_bfloat16* p, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
}

struct GemmArgs {
  int M, N, K;
  const float* sx;     // [M]
  const float* sw;     // [N]
  const float* bias;   // [N] or null
  void* out;           // [M, N], row stride ldo
  long ldo;
  int tma_out;         // rows of `out` start on 16-byte boundaries: tiles leave by TMA, channels four at a time
  int group;           // row blocks that sweep the columns together (many rows)
  int* status;
};

// ------------------------------------------------------------------------------ few rows
// Grid (S * ceil(N / 128), ceil(M / BN)), clusters of S along x: rank r of a cluster takes its share of
// the k blocks of one tile of 128 channels and BN tokens.  Warp 0 loads, warp 1 multiplies, all four read
// TMEM.  (256 channels a block, which halve how often the tokens are read, were 0 to 10 % slower at every size tried.)
template <int BN>
struct StreamCfg {
  static constexpr int kStageA = kRowsA * kBytesK, kStageB = BN * kBytesK, kStage = kStageA + kStageB;
  // half of an SM's shared memory: two blocks share it, and where the tiles do not fill the device evenly
  // the bandwidth still does (128 x 28672 x 4096: 27.9 us, 40.6 with one block an SM)
  static constexpr int kStages = 102 * 1024 / kStage;
  static constexpr int kTmem = BN < 32 ? 32 : BN;
  static constexpr int kSmem = 1024 + kStages * kStage + 256;
  static_assert(BN * kRowsA * 4 <= kStages * kStage, "the exchange buffer lies over the stages");
};

template <int BN, typename OutT>
__global__ void __launch_bounds__(128)
int8_stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const GemmArgs p, int S) {
  using C = StreamCfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(smem + C::kStages * C::kStage);
  uint64_t* empty = full + C::kStages;
  uint64_t* done = empty + C::kStages;
  uint32_t* tmem_slot = (uint32_t*)(done + 1);
  volatile int* dead = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int n0 = ((int)blockIdx.x / S) * kRowsA, m0 = (int)blockIdx.y * BN;
  const int num_kb = (p.K + kBytesK - 1) / kBytesK;
  const int kb0 = (int)((long)num_kb * rank / S), kb1 = (int)((long)num_kb * (rank + 1) / S);

  if (threadIdx.x == 0) {
    *dead = 0;
    for (int i = 0; i < C::kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    mbar_init(done, 1);
    mbar_fence_init();
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_x);
  }
  if (warp == 1) { tmem_alloc<C::kTmem>(tmem_slot); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  chain_ready();
  chain_wait();

  if (warp == 0) {
    if (lane == 0) {
      for (int kb = kb0; kb < kb1; ++kb) {
        const int it = kb - kb0, s = it % C::kStages;
        if (!mbar_wait(&empty[s], (uint32_t)(((it / C::kStages) & 1) ^ 1), dead, p.status, 1100)) break;
        uint8_t* dst = smem + s * C::kStage;
        mbar_expect_tx(&full[s], C::kStage);
        tma_load_2d(dst, &map_w, &full[s], kb * kBytesK, n0);
        tma_load_2d(dst + C::kStageA, &map_x, &full[s], kb * kBytesK, m0);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_s8(kRowsA, BN);
      const uint32_t s0 = smem_u32(smem);
      const uint64_t da0 = umma_desc_sw128(s0, 16, 1024), db0 = umma_desc_sw128(s0 + C::kStageA, 16, 1024);
      uint32_t accum = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int it = kb - kb0, s = it % C::kStages;
        if (!mbar_wait(&full[s], (uint32_t)((it / C::kStages) & 1), dead, p.status, 1101)) break;
        tc_fence_after();
        const uint64_t off = (uint64_t)((uint32_t)(s * C::kStage) >> 4);
#pragma unroll
        for (int k = 0; k < kBytesK / kMmaK; ++k) {
          umma_s8(tmem, da0 + off + (uint64_t)(k * kMmaK >> 4), db0 + off + (uint64_t)(k * kMmaK >> 4), idesc, accum);
          accum = 1;
        }
        umma_commit(&empty[s]);
      }
      umma_commit(done);
    }
  }
  __syncwarp();
  bool ok = mbar_wait(done, 0, dead, p.status, 1102);
  ok = __all_sync(0xffffffffu, ok);
  tc_fence_after();

  // epilogue: thread = output channel n0 + row, column j of the accumulator = token m0 + j
  const int row = warp * 32 + lane, n = n0 + row;
  const uint32_t t_row = tmem + ((uint32_t)(warp * 32) << 16);
  const int cols = min(BN, p.M - m0);
  if (S == 1) {
    const float sw = n < p.N ? p.sw[n] : 0.f;
    const float bias = (p.bias != nullptr && n < p.N) ? p.bias[n] : 0.f;
    OutT* out = (OutT*)p.out + (long)m0 * p.ldo + n;
    if (ok) {
#pragma unroll 1
      for (int c = 0; c < cols; c += 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(t_row + c, v);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c + j < cols && n < p.N)
            store_out(out + (long)(c + j) * p.ldo, __int2float_rn((int)v[j]) * __ldg(p.sx + m0 + c + j) * sw + bias);
      }
    }
  } else {
    // every block leaves its partial sums in its own shared memory, [column][row]; then a warp of block r
    // adds whole columns r, r + S, ... of all of them, four channels a lane (integers: any order gives the
    // same sum)
    int* red = (int*)smem;
    if (ok) {
#pragma unroll 1
      for (int c = 0; c < cols; c += 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(t_row + c, v);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) red[(c + j) * kRowsA + row] = (int)v[j];
      }
    }
    __syncwarp();
    cluster_sync_all();
    if (ok) {
      const int n4 = n0 + 4 * lane;
      uint32_t peer[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) peer[s] = s < S ? mapa_shared(smem_u32(red + 4 * lane), s) : 0;
      float sw[4], bias[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sw[j] = n4 + j < p.N ? p.sw[n4 + j] : 0.f;
        bias[j] = (p.bias != nullptr && n4 + j < p.N) ? p.bias[n4 + j] : 0.f;
      }
#pragma unroll 4
      for (int c = rank + S * warp; c < cols; c += 4 * S) {
        int4 sum = make_int4(0, 0, 0, 0);
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          if (s < S) {
            const int4 v = ld_cluster4(peer[s] + (uint32_t)(c * kRowsA * 4));
            sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
          }
        }
        const float sx = __ldg(p.sx + m0 + c);
        const float y0 = __int2float_rn(sum.x) * sx * sw[0] + bias[0], y1 = __int2float_rn(sum.y) * sx * sw[1] + bias[1];
        const float y2 = __int2float_rn(sum.z) * sx * sw[2] + bias[2], y3 = __int2float_rn(sum.w) * sx * sw[3] + bias[3];
        OutT* o = (OutT*)p.out + (long)(m0 + c) * p.ldo + n4;
        if (p.tma_out && n4 + 3 < p.N) {      // rows on 16-byte boundaries: four channels are one store
          store_out4(o, y0, y1, y2, y3);
        } else {
          if (n4 < p.N) store_out(o, y0);
          if (n4 + 1 < p.N) store_out(o + 1, y1);
          if (n4 + 2 < p.N) store_out(o + 2, y2);
          if (n4 + 3 < p.N) store_out(o + 3, y3);
        }
      }
    }
    __syncwarp();
    cluster_sync_all();   // nobody leaves while another block still reads its sums
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc<C::kTmem>(tmem);
}

// ----------------------------------------------------------------------------- many rows
constexpr int kThreads = 192;                  // warp 0 loads, warp 1 multiplies, warps 2..5 epilogue
constexpr int kEpiWarps = 4;
constexpr int kStageBuf = 32 * 128;            // 32 rows x 128 bytes of output

template <int BN>
struct PairCfg {
  static constexpr int kStageA = kRowsA * kBytesK, kStageB = (BN / 2) * kBytesK, kStage = kStageA + kStageB;
  static constexpr int kStages = BN == 256 ? 6 : 8;
  static constexpr int kTmem = 512;            // all of it: the pair addresses both SMs' accumulators by one column
  static constexpr int kSmem = 1024 + kStages * kStage + kEpiWarps * 2 * kStageBuf + 256;
};

// Tile t of `num_m` x `num_n`: groups of row blocks sweep the columns, so that pairs at work together share tiles in
// L2.  `group` is at most num_m, so a group's tiles are at most all tiles, which the launch keeps below 2^31.
__host__ __device__ __forceinline__ void pair_tile(int t, int num_m, int num_n, int group, int& mb, int& nb) {
  const int per = group * num_n, g = t / per, first = g * group, size = group < num_m - first ? group : num_m - first, r = t - g * per;
  mb = first + r % size;
  nb = r / size;
}
// Row blocks that sweep together: as many as fill a quarter of L2 with 256 K bytes each, so that they stay there while the
// weight passes once for all of them.  Back to back under the power cap, 8192 x 28672 x 4096 takes 770 / 740 /
// 718 / 707 us with 4 / 8 / 16 / 32 together (33 MB), 8192 x 4096 x 14336 365 / 361 / 368 / 394 us (118 MB).
int pair_group(int M, int K) {
  const long num_m = ((long)M + 2 * kRowsA - 1) / (2 * kRowsA), fit = (34L << 20) / (256L * K), group = fit < 4 ? 4 : (fit < 1024 ? fit : 1024);
  return (int)(group < num_m ? group : num_m);
}

template <int BN, typename OutT>
__global__ void __launch_bounds__(kThreads, 1)
int8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                 const __grid_constant__ CUtensorMap map_out, const GemmArgs p) {
  using C = PairCfg<BN>;
  constexpr int HB = BN / 2, PM = 2 * kRowsA;
  constexpr int CC = 128 / (int)sizeof(OutT);   // output columns of one 128-byte staging row
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* epi = smem + C::kStages * C::kStage;
  uint64_t* full = (uint64_t*)(epi + kEpiWarps * 2 * kStageBuf);
  uint64_t* empty = full + C::kStages;
  uint64_t* tfull = empty + C::kStages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = (uint32_t*)(tempty + 2);
  volatile int* dead = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  const int pair_id = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int num_m = (p.M + PM - 1) / PM, num_n = (p.N + BN - 1) / BN;
  const int num_tiles = num_m * num_n, num_kb = (p.K + kBytesK - 1) / kBytesK;

  if (threadIdx.x == 0) {
    *dead = 0;
    for (int i = 0; i < C::kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&tfull[i], 1); mbar_init(&tempty[i], 2 * kEpiWarps); }
    mbar_fence_init();
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_out);
  }
  if (warp == 1) { tmem_alloc_pair<C::kTmem>(tmem_slot); tmem_relinquish_pair(); }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  chain_ready();
  chain_wait();

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      for (int t = pair_id; t < num_tiles; t += num_pairs) {
        int mb, nb;
        pair_tile(t, num_m, num_n, p.group, mb, nb);
        const int m0 = mb * PM + (int)crank * kRowsA, n0 = nb * BN + (int)crank * HB;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[s], ph ^ 1, dead, p.status, 1110)) break;
          uint8_t* dst = smem + s * C::kStage;
          if (crank == 0) mbar_expect_tx(&full[s], 2 * C::kStage);
          const uint32_t fb = mapa_shared(smem_u32(&full[s]), 0);
          tma_load_2d_pair(dst, &map_x, fb, kb * kBytesK, m0);
          tma_load_2d_pair(dst + C::kStageA, &map_w, fb, kb * kBytesK, n0);
          if (++s == C::kStages) { s = 0; ph ^= 1; }
        }
        if (*dead) break;
      }
      // every arrival that the leader's commits still owe this CTA lands before it leaves
      for (int i = 0; i < C::kStages && !*dead; ++i) {
        if (!mbar_wait(&empty[s], ph ^ 1, dead, p.status, 1111)) break;
        if (++s == C::kStages) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && crank == 0) {
      constexpr uint32_t idesc = idesc_s8(PM, BN);
      const uint32_t s0 = smem_u32(smem);
      const uint64_t da0 = umma_desc_sw128(s0, 16, 1024), db0 = umma_desc_sw128(s0 + C::kStageA, 16, 1024);
      int s = 0, it = 0;
      uint32_t ph = 0;
      for (int t = pair_id; t < num_tiles; t += num_pairs, ++it) {
        const int acc = it & 1;
        if (!mbar_wait(&tempty[acc], (uint32_t)(((it >> 1) & 1) ^ 1), dead, p.status, 1112)) break;
        tc_fence_after();
        uint32_t accum = 0;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full[s], ph, dead, p.status, 1113)) break;
          tc_fence_after();
          const uint64_t off = (uint64_t)((uint32_t)(s * C::kStage) >> 4);
#pragma unroll
          for (int k = 0; k < kBytesK / kMmaK; ++k) {
            umma_s8_pair(tmem + acc * BN, da0 + off + (uint64_t)(k * kMmaK >> 4), db0 + off + (uint64_t)(k * kMmaK >> 4), idesc, accum);
            accum = 1;
          }
          umma_commit_pair(&empty[s]);
          if (++s == C::kStages) { s = 0; ph ^= 1; }
        }
        umma_commit_pair(&tfull[acc]);
        if (*dead) break;
      }
    }
  } else {
    const int q = warp & 3, ew = warp - 2;
    uint8_t* stg = epi + ew * 2 * kStageBuf;
    const uint32_t tempty0 = mapa_shared(smem_u32(&tempty[0]), 0);
    int buf = 0, it = 0;
    for (int t = pair_id; t < num_tiles; t += num_pairs, ++it) {
      int mb, nb;
      pair_tile(t, num_m, num_n, p.group, mb, nb);
      const int m_warp = mb * PM + (int)crank * kRowsA + q * 32, n0 = nb * BN;
      const int acc = it & 1;
      const int m = m_warp + lane;
      const float sx = m < p.M ? p.sx[m] : 0.f;
      bool ok = mbar_wait(&tfull[acc], (uint32_t)((it >> 1) & 1), dead, p.status, 1114);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_row = tmem + ((uint32_t)(q * 32) << 16) + acc * BN;
#pragma unroll 1
      for (int ch = 0; ch < BN / CC; ++ch) {
        uint32_t r[CC];
#pragma unroll
        for (int j = 0; j < CC; j += 32) tmem_ld_32x32b_x32(t_row + ch * CC + j, *reinterpret_cast<uint32_t(*)[32]>(&r[j]));
        tc_wait_ld();
        if (ch == BN / CC - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(tempty0 + acc * 8);
        }
        const int c0 = n0 + ch * CC;
        if (c0 >= p.N || m_warp >= p.M) continue;     // (warp-uniform)
        if (c0 + CC <= p.N && (((uintptr_t)p.sw | (uintptr_t)p.bias) & 15) == 0) {
          const float4* w4 = reinterpret_cast<const float4*>(p.sw + c0);
          const float4* b4 = p.bias != nullptr ? reinterpret_cast<const float4*>(p.bias + c0) : nullptr;
#pragma unroll
          for (int j = 0; j < CC; j += 4) {
            const float4 w = __ldg(w4 + j / 4);
            const float4 b = b4 != nullptr ? __ldg(b4 + j / 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            r[j] = __float_as_uint(__int2float_rn((int)r[j]) * sx * w.x + b.x);
            r[j + 1] = __float_as_uint(__int2float_rn((int)r[j + 1]) * sx * w.y + b.y);
            r[j + 2] = __float_as_uint(__int2float_rn((int)r[j + 2]) * sx * w.z + b.z);
            r[j + 3] = __float_as_uint(__int2float_rn((int)r[j + 3]) * sx * w.w + b.w);
          }
        } else {
#pragma unroll
          for (int j = 0; j < CC; ++j) {
            const int n = c0 + j;
            const float w = n < p.N ? __ldg(p.sw + n) : 0.f;
            const float b = (p.bias != nullptr && n < p.N) ? __ldg(p.bias + n) : 0.f;
            r[j] = __float_as_uint(__int2float_rn((int)r[j]) * sx * w + b);
          }
        }
        // 16-byte pieces of the staging row, swizzled by the row so that the warp's stores spread over the banks
        uint8_t* dst = stg + buf * kStageBuf;
        if (p.tma_out) {
          if (lane == 0) tma_store_wait_read<1>();
          __syncwarp();
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint4 o;
          if (sizeof(OutT) == 2) {
            o.x = pack_bf16x2(__uint_as_float(r[c * 8 % CC]), __uint_as_float(r[(c * 8 + 1) % CC]));
            o.y = pack_bf16x2(__uint_as_float(r[(c * 8 + 2) % CC]), __uint_as_float(r[(c * 8 + 3) % CC]));
            o.z = pack_bf16x2(__uint_as_float(r[(c * 8 + 4) % CC]), __uint_as_float(r[(c * 8 + 5) % CC]));
            o.w = pack_bf16x2(__uint_as_float(r[(c * 8 + 6) % CC]), __uint_as_float(r[(c * 8 + 7) % CC]));
          } else {
            o = make_uint4(r[c * 4], r[c * 4 + 1], r[c * 4 + 2], r[c * 4 + 3]);
          }
          *reinterpret_cast<uint4*>(dst + lane * 128 + ((c ^ (lane & 7)) << 4)) = o;
        }
        if (p.tma_out) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_out, dst, c0, m_warp);
            tma_store_commit();
          }
          buf ^= 1;
        } else {
          // rows that start anywhere: one row at a time, neighbouring lanes on neighbouring columns
          __syncwarp();
          const int rows = min(32, p.M - m_warp);
          for (int i = 0; i < rows; ++i) {
            OutT* o = (OutT*)p.out + (long)(m_warp + i) * p.ldo + c0;
#pragma unroll
            for (int j = lane; j < CC; j += 32) {
              const int byte = j * (int)sizeof(OutT);
              if (c0 + j < p.N) o[j] = *reinterpret_cast<const OutT*>(dst + i * 128 + (((byte >> 4) ^ (i & 7)) << 4) + (byte & 15));
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0 && p.tma_out) tma_store_wait<0>();
  }
  // neither CTA leaves while the other can still read its shared memory or signal its barriers
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair<C::kTmem>(tmem);
}

// -------------------------------------------------------------------------------- host side
int make_map(CUtensorMap* m, CUtensorMapDataType dt, const void* ptr, uint64_t inner, uint64_t outer, uint64_t ld_bytes, uint32_t box_inner,
             uint32_t box_outer) {
  uint64_t dims[2] = {inner, outer}, strides[1] = {ld_bytes};
  uint32_t box[2] = {box_inner, box_outer};
  return axh::encode_tensor_map(m, dt, 2, ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int device_slot() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev >= 0 && dev < 64 ? dev : -1;
}

template <int BN, typename OutT>
int launch_stream(const void* q, long ldq, const void* w, long ldw, const GemmArgs& p, int S, cudaStream_t stream) {
  using C = StreamCfg<BN>;
  auto kern = int8_stream_kernel<BN, OutT>;
  static bool configured[64] = {false};
  const int dev = device_slot();
  if (dev < 0 || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0) configured[dev] = true;
  }
  CUtensorMap mw, mx;
  int rc = make_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, p.K, p.N, ldw, kBytesK, kRowsA);
  if (rc) return 1000 + rc;
  rc = make_map(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, q, p.K, p.M, ldq, kBytesK, BN);
  if (rc) return 2000 + rc;
  const dim3 grid(S * ((p.N + kRowsA - 1) / kRowsA), (p.M + BN - 1) / BN);
  return axh::launch_chained(kern, grid, dim3(128), C::kSmem, S, stream, mw, mx, p, S);
}

template <int BN, typename OutT>
int launch_pair(const void* q, long ldq, const void* w, long ldw, const GemmArgs& p, cudaStream_t stream, bool query) {
  using C = PairCfg<BN>;
  auto kern = int8_pair_kernel<BN, OutT>;
  static int max_pairs[64] = {0};
  const int dev = device_slot();
  if (dev < 0) return -3;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (max_pairs[dev] == 0) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return (int)e;
    cfg.gridDim = dim3(2 * axh::sm_count(), 1, 1);
    int n = 0;
    e = cudaOccupancyMaxActiveClusters(&n, (const void*)kern, &cfg);
    if (e != cudaSuccess) return (int)e;
    if (n < 1) return -3;
    max_pairs[dev] = n;
  }
  if (query) return max_pairs[dev];
  CUtensorMap mx, mw, mo;
  int rc = make_map(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, q, p.K, p.M, ldq, kBytesK, kRowsA);
  if (rc) return 1000 + rc;
  rc = make_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, p.K, p.N, ldw, kBytesK, BN / 2);
  if (rc) return 2000 + rc;
  mo = mx;
  if (p.tma_out) {
    rc = make_map(&mo, sizeof(OutT) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, p.out, p.N, p.M,
                  p.ldo * sizeof(OutT), 128 / sizeof(OutT), 32);
    if (rc) return 3000 + rc;
  }
  const long tiles = (long)((p.M + 2 * kRowsA - 1) / (2 * kRowsA)) * ((p.N + BN - 1) / BN);
  if (tiles > 0x7f000000L) return -4;                          // (an output of 2^46 values)
  const int pairs = tiles < max_pairs[dev] ? (int)tiles : max_pairs[dev];
  return axh::launch_chained(kern, dim3(2 * pairs), dim3(kThreads), C::kSmem, 2, stream, mx, mw, mo, p);
}

// Which kernel, token tile and split of K: the lowest estimated time in microseconds.  The constants are fits to
// timings of all forms at 1 to 1024 rows, 1000 to 28672 channels and K of 1024 to 14336 (a chain of
// products, inputs larger than L2); they name what each form waits for:
//   stream  4 to start and end; then the slowest of its k blocks in turn (0.27 each, and 4 more for every
//           wave once there are two), shared-memory fills at 16 TB/s over all blocks, the weight at 6.3 TB/s; 0.03 a column to
//           store, or 1 + 0.015 a column to hand over and 0.04 a column to add and store when K is split.
//           Measured 1 x 6144 x 4096: 12.7 / 9.3 / 8.3 / 13.6 us with K split 1 / 2 / 4 / 8 ways;
//           128 x 4096 x 4096: 14.4 / 11.7 / 9.6 us with 64 tokens and 1 / 2 / 4 ways, 15.0 as pairs.
//   pair    0.3 a k block and wave.  512 x 28672 x 4096: 51 us as 256 x 256 tiles, 74 as 256 x 128, 90 streamed;
//           512 x 4096 x 4096: 16.5 / 15.4 / 18.1.
struct Choice { int bn, split; bool pair; };
Choice choose(int M, int N, int K, int pairs) {
  const double kb = (K + kBytesK - 1) / kBytesK, slots = 2.0 * axh::sm_count();
  Choice best{256, 1, true};
  double least = 1e30;
  auto waves = [](double tiles, double room) { return (double)(long)((tiles + room - 1) / room); };
  if (pairs > 0) {
    const double mb = (M + 255) / 256;
    const double t256 = 6.0 + waves(mb * ((N + 255) / 256), pairs) * (0.3 * kb + 1.6);
    const double t128 = 5.0 + waves(mb * ((N + 127) / 128), pairs) * (0.3 * kb + 0.4);
    least = t256 < t128 ? t256 : t128;
    if (t128 < t256) best.bn = 128;
  }
  for (int bn = 16; bn <= 128; bn *= 2) {
    if (bn > 16 && M <= bn / 2) break;
    if ((M - 1) / bn >= 65535) continue;                       // (the grid's second dimension)
    const double tiles = (double)((N + kRowsA - 1) / kRowsA) * ((M + bn - 1) / bn);
    for (int S = 1; S <= 8 && S <= (int)kb; S *= 2) {
      const double w = waves(tiles * S, slots), each = (kb + S - 1) / S;
      const double end = S == 1 ? 0.03 * bn : 1.0 + 0.015 * bn + 0.04 * bn / S;
      double body = w > 1 ? w * (0.3 * each + 4.0 + end) : 0.27 * each;
      const double fill = tiles * kb * kBytesK * (kRowsA + bn) / 16.0e6, weight = (double)N * K / 6.3e6;
      if (fill > body) body = fill;
      if (weight > body) body = weight;
      const double t = 4.0 + body + end;
      if (t < least) { least = t; best = Choice{bn, S, false}; }
    }
  }
  return best;
}

template <typename OutT>
int dispatch(const void* q, long ldq, const void* w, long ldw, const GemmArgs& p, cudaStream_t stream) {
  const int pairs = launch_pair<256, OutT>(q, ldq, w, ldw, p, stream, true);
  const Choice c = choose(p.M, p.N, p.K, pairs);
  if (c.pair) {
    if (pairs < 1) return pairs ? pairs : -3;
    return c.bn == 256 ? launch_pair<256, OutT>(q, ldq, w, ldw, p, stream, false) : launch_pair<128, OutT>(q, ldq, w, ldw, p, stream, false);
  }
  switch (c.bn) {
    case 16: return launch_stream<16, OutT>(q, ldq, w, ldw, p, c.split, stream);
    case 32: return launch_stream<32, OutT>(q, ldq, w, ldw, p, c.split, stream);
    case 64: return launch_stream<64, OutT>(q, ldq, w, ldw, p, c.split, stream);
    default: return launch_stream<128, OutT>(q, ldq, w, ldw, p, c.split, stream);
  }
}

}  // namespace

// out[M, N] (bf16 with out_bf16, else fp32; row stride ldo elements) from q[M, K] and w[N, K] int8, whose
// row strides ldq / ldw are multiples of 16 bytes and whose base addresses lie on 16-byte boundaries.
// K <= 131071.  Returns a cudaError_t value, -1 / -2 for unsupported arguments.
AX_API int ax_int8_gemm(const void* q, long ldq, const float* sx, const void* w, long ldw, const float* sw, const float* bias, void* out,
                        long ldo, int out_bf16, int M, int N, int K, int* status, cudaStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K > 131071) return -1;
  if ((ldq % 16) || (ldw % 16) || (((uintptr_t)q | (uintptr_t)w) & 15)) return -2;
  GemmArgs p{M, N, K, sx, sw, bias, out, ldo, 0, pair_group(M, K), status};
  const int size = out_bf16 ? 2 : 4;
  p.tma_out = (ldo * size) % 16 == 0 && ((uintptr_t)out & 15) == 0;
  return out_bf16 ? dispatch<__nv_bfloat16>(q, ldq, w, ldw, p, stream) : dispatch<float>(q, ldq, w, ldw, p, stream);
}

// Where the many-row kernel puts its tile `t` of `bn` channels for a product of M x N x K: out = {row block, column block}.
// Returns the number of tiles.  (Host arithmetic alone: what the kernel walks, for its tests.)
AX_API long ax_int8_gemm_tile(int M, int N, int K, int bn, int t, int* out) {
  if (M <= 0 || N <= 0 || K <= 0 || bn <= 0) return 0;
  const int num_m = (M + 2 * kRowsA - 1) / (2 * kRowsA), num_n = (N + bn - 1) / bn;
  const long tiles = (long)num_m * num_n;
  if (t >= 0 && t < tiles && tiles <= 0x7f000000L) pair_tile(t, num_m, num_n, pair_group(M, K), out[0], out[1]);
  return tiles;
}
