// Paged K/V cache in 8 bits: pages of P tokens, one magnitude a for each (page, KV head) of K and of V;
// a stored byte q stands for q a / 127.
//
//   k_cache [pages, Hkv, P, D]            k_amax [pages, Hkv]
//   v_cache [pages, Hkv, P / 16, D, 16]   v_amax [pages, Hkv]
//
// K keeps a token's dims side by side, V keeps sixteen tokens of one dim side by side: both are the order
// in which the two matrix products contract (over dims, over tokens), so a lane's bytes become MMA
// operands without a transposition, and sixteen tokens of a head are one contiguous 16 D byte piece of
// either, which one bulk copy fetches.
//
// Writing: a page's magnitude grows to the largest it holds; what it held is scaled to the new one
// (rint(q a_old / a_new)), new rows are rint(127 x / a).  A page written from its first slot starts anew.
//
// Attention of one query token per sequence: softmax(q K^T scale) V over the first ctx tokens.
#include "int8_common.cuh"

namespace {
using namespace ax;

// ------------------------------------------------------------------------------------ write
struct WriteArgs {
  const void *k, *v;          // [T, Hkv, D]
  int8_t *kc, *vc;
  float *ka, *va;
  const int* table;           // [B, max_pages]
  const int* starts;          // [B] position of the first new token
  const int* cu;              // [B + 1] first token of each row in k / v, or null: T / B tokens each
  long k_ts, k_hs, v_ts, v_hs;
  int T, B, Hkv, D, P, max_pages, num_pages;
  int per_row, each;          // blocks and tokens of a row without cu
  int shift;                  // log2(P), or -1 where P is no power of two
  int magic;                  // i * magic / 65536 is i / (D / 8) for a thread's index i (i (D / 8) < 65536)
  int* status;
};

struct Piece { int page, first, count, src; };   // slots [first, first + count) of a page, from token src

// x / P.  A block waits for a chain of these and of loads before its first value arrives.
template <typename I>
__device__ __forceinline__ int page_of(const WriteArgs& a, I x) { return (int)(a.shift >= 0 ? x >> a.shift : x / a.P); }

// Pages touched by row b: 0 for an empty row or one that does not fit.
__device__ __forceinline__ int row_pieces(const WriteArgs& a, int b, int& start, int& src, int& len) {
  start = a.starts[b];
  if (a.cu != nullptr) {
    src = a.cu[b];
    len = a.cu[b + 1] - src;
  } else {
    len = a.each;
    src = b * len;
  }
  if (len <= 0) return 0;
  if (start < 0 || src < 0 || (long)src + len > a.T || (long)start + len > min((long)a.max_pages * a.P, 0x7fffffffL)) {
    set_status(a.status, kBadArgument, 1200);
    return 0;
  }
  return page_of(a, start + len - 1) - page_of(a, start) + 1;
}

// The piece that block `slot` of the grid works on.  n tokens touch at most (n + 2 P - 2) / P pages, so row b's slots begin
// at (cu[b] + b (2 P - 2)) / P: a warp looks for the row 128 at a time, and slots past a row's pages have nothing to do.
// (A token of each of 2048 sequences, 8 heads: 79 us; 568 when a warp counted the pages of the rows before.)
__device__ __forceinline__ bool find_piece(const WriteArgs& a, int slot, Piece& out) {
  int b = 0, start = 0, src = 0, len = 0, j, pages;
  if (a.cu == nullptr) {
    b = a.per_row == 1 ? slot : slot / a.per_row;
    j = slot - b * a.per_row;
    pages = row_pieces(a, b, start, src, len);
  } else {
    const int lane = threadIdx.x & 31;
    auto at = [&](int r) { return (long)min(max(a.cu[r], 0), a.T) + (long)r * (2 * a.P - 2); };
    const long below = ((long)slot + 1) * a.P;
    if (a.B <= 32) {                                         // a lane a row
      long x = below;
      pages = 0;
      if (lane < a.B) {
        x = at(lane);
        pages = row_pieces(a, lane, start, src, len);
      }
      b = max(__popc(__ballot_sync(0xffffffffu, x < below)) - 1, 0);
      j = slot - __shfl_sync(0xffffffffu, page_of(a, x), b);
      pages = __shfl_sync(0xffffffffu, pages, b);
      start = __shfl_sync(0xffffffffu, start, b);
      src = __shfl_sync(0xffffffffu, src, b);
      len = __shfl_sync(0xffffffffu, len, b);
    } else {
      for (int n = a.B;;) {                                    // the row is one of n from b on
        const int step = (n + 127) / 128;
        int count = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = (k * 32 + lane) * step;
          count += __popc(__ballot_sync(0xffffffffu, i < n && at(b + i) < below));
        }
        const int skip = max(count - 1, 0) * step;
        b += skip;
        if (step == 1) break;
        n = min(step, n - skip);
      }
      j = slot - page_of(a, at(b));
      pages = row_pieces(a, b, start, src, len);
    }
  }
  if (j < 0 || j >= pages) return false;
  const int idx = page_of(a, start) + j, page0 = idx * a.P;        // which page of the row
  const int lo = max(start, page0), n = min(start + len - page0, a.P) + page0 - lo;
  out.page = a.table[(long)b * a.max_pages + idx];
  out.first = lo - page0;
  out.count = n;
  out.src = src + lo - start;
  if (out.page < 0 || out.page >= a.num_pages) { set_status(a.status, kBadArgument, 1201); return false; }
  return true;
}

// rint(q a_old / a_new) of four bytes
__device__ __forceinline__ uint32_t rescale4(uint32_t w, const Int8Grid& g) {
  uint32_t b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = int8_bits((float)(int8_t)((w >> (8 * j)) & 255u), g);
  return pack_low_bytes(b[0], b[1], b[2], b[3]);
}

// 0xff in byte j of word w where lo <= 4 w + j < hi
__device__ __forceinline__ uint32_t byte_mask(int w, int lo, int hi) {
  const int a = min(max(lo - 4 * w, 0), 4), b = min(max(hi - 4 * w, 0), 4);
  const uint32_t below_b = b == 4 ? 0xffffffffu : (1u << (8 * b)) - 1u, below_a = a == 4 ? 0xffffffffu : (1u << (8 * a)) - 1u;
  return below_b & ~below_a;
}

// Grid (pieces, Hkv): a block takes a page piece of a head; kHalf of its threads take K, as many V.  A thread holds
// four times eight dims, so that 16 tokens of 128 dims on 64 threads are read once and stay in registers between
// the magnitude and the rounding; larger pieces are read a second time, from L1.
// K: a thread rounds eight dims of a token.  V: four lanes take eight dims of sixteen slots, four slots each,
// and exchange words so that each lane stores two dims' sixteen slots whole.
template <typename T, int kHalf>
__global__ void __launch_bounds__(2 * kHalf, 512 / kHalf) kv_write_int8_kernel(const WriteArgs a) {
  __shared__ uint32_t s_top[2 * kHalf / 32];
  chain_ready();
  chain_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __shared__ Piece s_piece;                                  // (found by one warp: the issue slots are what the kernel lacks)
  if (warp == 0) {
    Piece found;
    if (!find_piece(a, (int)blockIdx.x, found)) found.count = 0;
    if (lane == 0) s_piece = found;
  }
  __syncthreads();
  const Piece pc = s_piece;
  if (pc.count == 0) return;
  const bool is_v = threadIdx.x >= kHalf;
  const int tid = threadIdx.x & (kHalf - 1), i4 = tid & 3;
  const long ts = is_v ? a.v_ts : a.k_ts, hs = is_v ? a.v_hs : a.k_hs;
  const T* rows = (const T*)(is_v ? a.v : a.k) + (long)pc.src * ts;
  const int per_row = a.D / 8, end = pc.first + pc.count;

  // K: threads side by side along a token's dims, 64 / per_row tokens at once, four of those a round.
  // V: a unit is 16 slots x 8 dims on four lanes, 16 units a round.
  const int g0 = pc.first / 16, g1 = (end + 15) / 16, units = (g1 - g0) * per_row;
  const int across = kHalf / per_row, row0 = (tid * a.magic) >> 16, tokens = 4 * across;
  const int rounds = is_v ? (units + kHalf / 4 - 1) / (kHalf / 4) : (pc.count + tokens - 1) / tokens;
  Raw8<T> raw[4];
  int t0, step, col = (tid - row0 * per_row) * 8, slot0 = 0;  // this thread's tokens of the round: t0, t0 + step, ...
  bool in = row0 < across;                                   // K: the thread has tokens; V: its unit exists
  auto token = [&](int k) { return t0 + k * step; };
  auto live = [&](int k) { return in && (unsigned)token(k) < (unsigned)pc.count; };
  auto request = [&](const T* x, int round) {
    if (is_v) {
      const int u = round * (kHalf / 4) + tid / 4, g = u / per_row;
      in = u < units;
      col = (u - g * per_row) * 8;
      slot0 = (g0 + g) * 16;                                 // the unit's first slot
      t0 = slot0 + 4 * i4 - pc.first;
      step = 1;
    } else {
      t0 = round * tokens + row0;
      step = across;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (live(k)) raw[k].load(x + token(k) * ts + col);
  };
  const int h = blockIdx.y;
  const T* x = rows + (long)h * hs;
  const long group = (long)pc.page * a.Hkv + h;
  float* amax_p = (is_v ? a.va : a.ka) + group;
  int8_t* dst = (is_v ? a.vc : a.kc) + group * a.P * a.D;
  const float before = pc.first > 0 ? *amax_p : 0.f;
  float most = 0.f;
#pragma unroll 1
  for (int round = 0; round < rounds; ++round) {
    request(x, round);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (live(k)) {
        float v[8];
        raw[k].get(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) most = amax_nan(most, v[j]);
      }
    }
  }
  uint32_t top = __reduce_max_sync(0xffffffffu, abs_bits(most));
  if (lane == 0) s_top[warp] = top;
  __syncthreads();                                         // also: every thread has read the old magnitude
  const int w0 = is_v ? kHalf / 32 : 0;
#pragma unroll
  for (int i = 0; i < kHalf / 32; ++i) top = max(top, s_top[w0 + i]);
  const uint32_t old_bits = abs_bits(before) < kTinyBits ? 0u : abs_bits(before);
  top = max(top, old_bits);
  if (top < kTinyBits) top = 0;
  const Int8Grid grid = int8_grid(top);
  const bool again = top > old_bits && pc.first > 0;       // the page's magnitude grows
  const Int8Grid shrink = int8_ratio(old_bits, again ? top : 0u);
  if (tid == 0) *amax_p = __uint_as_float(top);

  if (again) {                                               // what the page held: whole tokens of K, whole 16-slot groups of V
    uint4* held = reinterpret_cast<uint4*>(dst);
    const int words = (is_v ? g0 * 16 : pc.first) * a.D / 16;
#pragma unroll 1
    for (int i = tid; i < words; i += kHalf) {
      const uint4 w = held[i];
      held[i] = make_uint4(rescale4(w.x, shrink), rescale4(w.y, shrink), rescale4(w.z, shrink), rescale4(w.w, shrink));
    }
  }
#pragma unroll 1
  for (int round = 0; round < rounds; ++round) {
    if (rounds > 1) request(x, round);
    uint32_t steps[4][2];                                    // [token][dims 0-3 | 4-7]
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      steps[k][0] = steps[k][1] = 0u;
      if (live(k)) {
        float v[8];
        raw[k].get(v);
        const uint2 b = int8_steps(v, grid);
        steps[k][0] = b.x;
        steps[k][1] = b.y;
        if (!is_v) *reinterpret_cast<uint2*>(dst + (pc.first + token(k)) * a.D + col) = b;
      }
    }
    if (!is_v) continue;
    __syncwarp();
    // bytes [slot][dim] -> words word[dim] of this lane's four slots
    uint32_t word[8];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t lo01 = __byte_perm(steps[0][half], steps[1][half], 0x5140), hi01 = __byte_perm(steps[0][half], steps[1][half], 0x7362);
      const uint32_t lo23 = __byte_perm(steps[2][half], steps[3][half], 0x5140), hi23 = __byte_perm(steps[2][half], steps[3][half], 0x7362);
      word[4 * half] = __byte_perm(lo01, lo23, 0x5410);
      word[4 * half + 1] = __byte_perm(lo01, lo23, 0x7632);
      word[4 * half + 2] = __byte_perm(hi01, hi23, 0x5410);
      word[4 * half + 3] = __byte_perm(hi01, hi23, 0x7632);
    }
    // four lanes hold four slots each of dims col .. col + 7; lane i4 collects dims col + i4 and col + 4 + i4 in two
    // exchanges (with the neighbour at distance 1, then 2)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t* m = word + 4 * half;
      const bool odd = i4 & 1, up = i4 & 2;
      const uint32_t s1 = __shfl_xor_sync(0xffffffffu, odd ? m[0] : m[1], 1), s2 = __shfl_xor_sync(0xffffffffu, odd ? m[2] : m[3], 1);
      // dims {i4 & 1, 2 + (i4 & 1)}, slots of the pair's even and odd lane
      const uint32_t d0e = odd ? s1 : m[0], d0o = odd ? m[1] : s1;
      const uint32_t d2e = odd ? s2 : m[2], d2o = odd ? m[3] : s2;
      // lanes 0, 1 keep dims 0, 1; lanes 2, 3 keep dims 2, 3
      const uint32_t r0 = __shfl_xor_sync(0xffffffffu, up ? d0e : d2e, 2), r1 = __shfl_xor_sync(0xffffffffu, up ? d0o : d2o, 2);
      uint32_t out[4] = {up ? r0 : d0e, up ? r1 : d0o, up ? d2e : r0, up ? d2o : r1};
      if (in) {
        const int s0 = slot0;
        uint4* p = reinterpret_cast<uint4*>(dst + (long)s0 * a.D + (col + 4 * half + i4) * 16);
        if (s0 < pc.first || s0 + 16 > end) {                // slots that are neither old nor new keep their byte
          const uint4 o = *p;
          const uint32_t was[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t fresh = byte_mask(k, pc.first - s0, end - s0), held = again ? byte_mask(k, 0, pc.first - s0) : 0u;
            const uint32_t scaled = held ? rescale4(was[k], shrink) : 0u;
            out[k] = (out[k] & fresh) | (scaled & held) | (was[k] & ~(fresh | held));
          }
        }
        *p = make_uint4(out[0], out[1], out[2], out[3]);
      }
    }
  }
}

// -------------------------------------------------------------------------------- attention
// Every warp is a worker of its own: it takes an equal, contiguous share of all 16-token tiles of the
// batch, counted over sequences, KV heads and tokens in that order, whatever the context lengths are.
// Its tiles arrive in a ring of stages in shared memory, K and V of a tile by one bulk copy each, several
// tiles ahead; page numbers and magnitudes of 32 tiles are fetched by the 32 lanes at once, a batch ahead.
//
// Products (mma.m16n8k16, fp16 operands, fp32 sums), the cache on the 16-row side so that no row is idle
// with up to eight query heads on the other:
//   S^T[16 tokens x heads] = K Q^T,      O^T[16 dims x heads] += V^T P^T for each 16 dims
// int8 becomes fp16 exactly (byte | 0x6400 is 1024 + byte).  Q is scaled by a power of two to lie near one,
// where fp16 holds every bf16 significand.  P carries the page's V magnitude relative to the largest one met so
// far, so that O stays in the accumulators; a page below 1/8 of that is summed apart and added in fp32.
// Weights are counted in 2^-7 of the running maximum's, which only moves when a score exceeds it by 2^8 (a vote of the warp
// finds out), so that the usual tile needs no exchange and no rescaling: P lies in 0 .. 2^15 and fills fp16's range from
// above.  Rounding it costs 2^-11 of a weight (below bf16's own rounding of the result) down to 2^-21 of the
// largest one, and below that 2^-32 of the largest: a long flat tail behind one strong token is still summed, where
// weights counted from one would vanish at 2^-25.
//
// A worker writes a head's result itself when all its tokens were in the worker's share, and otherwise a
// partial (O, maximum, sum) that a second kernel merges.  Where contexts are short or heads few, the second
// launch and its wait cost more than even shares gain: then a cluster of blocks takes a head (ONE), its warps equal
// parts of the context, and they add up through shared memory.
constexpr int kWarps = 4;
constexpr int kTile = 16;

struct AttnArgs {
  const __nv_bfloat16* q;      // [B, Hq, D]
  const int8_t *kc, *vc;
  const float *ka, *va;
  const int *table, *ctx;
  __nv_bfloat16* out;          // [B, Hq, D]
  float* part;                 // [workers][2][HG][D]
  float* ml;                   // [workers][2][HG][2]
  int B, Hq, Hkv, G, nblk, P, max_pages, num_pages, min_chunk, workers;
  int* seen;                   // [B + 1] tiles of the sequences before, for the merge
  int cluster;                 // ONE: blocks that share a head
  float scale_log2;            // scale * log2(e) / 127
  int* status;
};

__device__ __forceinline__ int tiles_of(const AttnArgs& a, int b) {
  int n = a.ctx[b];
  const long cap = (long)a.max_pages * a.P;
  if (n < 0 || n > cap) {
    set_status(a.status, kBadArgument, 1210);
    n = n < 0 ? 0 : (int)cap;                                    // (below n, so it fits)
  }
  return n / kTile + (n % kTile != 0);
}
__device__ __forceinline__ int chunk_of(const AttnArgs& a, int total) {
  const int even = (total + a.workers - 1) / a.workers;
  return even > a.min_chunk ? even : a.min_chunk;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"((uint64_t)src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four int8 to two fp16 pairs: the byte with its sign bit flipped is value + 128; over 0x64 it is 1024 + that.
__device__ __forceinline__ void int8x4_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  w ^= 0x80808080u;
  const uint32_t l = __byte_perm(w, 0x64646464u, 0x4140), h = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 off = __half2half2(__ushort_as_half((unsigned short)0x6480));   // 1152
  const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&l), off), b = __hsub2(*reinterpret_cast<const __half2*>(&h), off);
  lo = *reinterpret_cast<const uint32_t*>(&a);
  hi = *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Transposes an 8 x 8 matrix of 16-bit values spread over the warp (lane 4 r + c holds columns 2 c, 2 c + 1 of row r).
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <int D>
struct AttnCfg {
  static constexpr int kStage = 2 * kTile * D;                   // K and V of a tile
  static constexpr int kStages = D == 64 ? 6 : 3;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kBlocks = D == 256 ? 2 : 4;               // blocks per SM that registers and shared memory allow
};
constexpr float kUnit = 7.f;                                     // log2 of the weight of a score at the running maximum
constexpr float kMost = 15.f;                                    // log2 of the largest weight
constexpr float kNone = -3.402823466e38f;                        // reference before the first score (-FLT_MAX: not above a finite one)
constexpr float kFaint = 1.f / 8.f;

// NB: blocks of eight query heads.
template <int D, int NB, bool ONE>
__global__ void __launch_bounds__(kWarps * 32, NB == 1 ? AttnCfg<D>::kBlocks : 2) decode_int8_kernel(const AttnArgs a) {
  using C = AttnCfg<D>;
  constexpr int HG = 8 * NB;
  constexpr int NJ = D / 64;                                     // 64-dim groups: a lane's 16-byte pieces of a K row
  constexpr int MT = D / 16;                                     // 16-dim tiles of O^T
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* bars = (uint64_t*)(smem + C::kRing);
  volatile int* dead = (volatile int*)(bars + kWarps * C::kStages);
  int* prefix = (int*)(bars + kWarps * C::kStages) + 2;          // [B + 1] tiles of the sequences before (not ONE)
  float* part_ml = reinterpret_cast<float*>(prefix);             // ONE: [warps][HG] maximum, sum
  float* block_ml = part_ml + kWarps * HG * 2;                   // ONE: [HG] maximum, sum
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    *dead = 0;
    for (int i = 0; i < kWarps * C::kStages; ++i) mbar_init(&bars[i], 1);
    mbar_fence_init();
  }
  chain_ready();                                                 // the merge may be set up
  chain_wait();
  const int VH = a.Hkv * a.nblk;
  uint8_t* ring = smem + warp * C::kStages * C::kStage;
  uint64_t* full = bars + warp * C::kStages;
  int w = 0, f0 = 0, f1 = 0, n;                                  // worker, its share of the flat tiles
  int b = 0, vh = 0, tb = 0, tile = 0;                           // sequence, KV head (block of query heads), its tiles, the next one
  if constexpr (ONE) {
    const int seg = (int)blockIdx.x / a.cluster, part = (a.cluster > 1 ? (int)cluster_ctarank() : 0) * kWarps + warp;
    b = seg / VH;
    vh = seg - b * VH;
    tb = tiles_of(a, b);
    const int share = (tb + a.cluster * kWarps - 1) / (a.cluster * kWarps);
    tile = part * share;
    n = max(0, min(share, tb - tile));
    __syncthreads();                                             // the barriers are set up
  } else {
    if (warp == 0) {
      int sum = 0;
      for (int b0 = 0; b0 < a.B; b0 += 32) {
        int m = b0 + lane < a.B ? tiles_of(a, b0 + lane) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int t = __shfl_up_sync(0xffffffffu, m, o);
          if (lane >= o) m += t;
        }
        if (b0 + lane < a.B) prefix[b0 + lane + 1] = sum + m;
        sum += __shfl_sync(0xffffffffu, m, 31);
      }
      if (lane == 0) prefix[0] = 0;
    }
    __syncthreads();
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i <= a.B; i += kWarps * 32) a.seen[i] = prefix[i];
    const int total = prefix[a.B] * VH, chunk = chunk_of(a, total);
    w = warp * (int)gridDim.x + (int)blockIdx.x;                 // neighbouring workers on different SMs
    const long first = (long)w * chunk;
    if (first >= total) return;
    f0 = (int)first;
    f1 = min(total, f0 + chunk);
    n = f1 - f0;
  }

  // sequence whose tiles (times VH) contain flat tile f
  auto find_seq = [&](int f) {
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid + 1] * VH > f) hi = mid; else lo = mid + 1;
    }
    return lo;
  };
  // what lane l knows about tile (t0 + l): where its bytes lie (in tiles; -1: no such page), and its magnitudes
  auto load_ids = [&](int t0, int& at, int& group) {
    at = -1;
    group = -1;
    if (t0 + lane < n) {
      int sb = b, sv = vh, tok = (tile + t0 + lane) * kTile;
      if (!ONE) {
        const int f = f0 + t0 + lane;
        sb = find_seq(f);
        const int st = prefix[sb + 1] - prefix[sb], r = f - prefix[sb] * VH;
        sv = r / st;
        tok = (r - sv * st) * kTile;
      }
      const int page = a.table[(long)sb * a.max_pages + tok / a.P];
      if (page < 0 || page >= a.num_pages) {
        set_status(a.status, kBadArgument, 1211);
      } else {
        group = page * a.Hkv + sv / a.nblk;
        at = group * (a.P / kTile) + (tok % a.P) / kTile;
      }
    }
  };
  auto load_amax = [&](int group, float& ka, float& va) {
    ka = group >= 0 ? a.ka[group] : -1.f;                        // negative: the tile is masked
    va = group >= 0 ? a.va[group] : 0.f;
  };
  int at_c, at_n = -1, grp = -1;
  float ka_c, va_c, ka_n = -1.f, va_n = 0.f;
  load_ids(0, at_c, grp);
  load_amax(grp, ka_c, va_c);
  auto issue = [&](int s, int at) {                              // a tile into stage s
    if (lane == 0) {
      if (at < 0) {
        mbar_arrive(&full[s]);                                   // nothing is fetched
      } else {
        uint8_t* dst = ring + s * C::kStage;
        const long off = (long)at * (kTile * D);
        mbar_expect_tx(&full[s], C::kStage);
        bulk_load(dst, a.kc + off, kTile * D, &full[s]);
        bulk_load(dst + kTile * D, a.vc + off, kTile * D, &full[s]);
      }
    }
  };
#pragma unroll 1
  for (int t = 0; t < C::kStages && t < n; ++t) issue(t, __shfl_sync(0xffffffffu, at_c, t));

  const int g = lane >> 2, i4 = lane & 3;
  if (!ONE) {
    b = find_seq(f0);
    tb = prefix[b + 1] - prefix[b];
    vh = (f0 - prefix[b] * VH) / tb;
    tile = f0 - prefix[b] * VH - vh * tb;
  }
  int ctx = 0, s = 0;
  uint32_t ph = 0;
  uint32_t qb[NB][NJ * 4][2];                                    // Q^T: head g of each block, four dims a step
  // of heads 2 i4 and 2 i4 + 1: scale, reference (log2 of the running maximum's weight less kUnit), this lane's share of the sum
  float qs[NB][2], m[NB][2], l[NB][2], o[NB][MT][4];
  float vref = 0.f, vinv = 1.f;                                  // V magnitude (/ 127) that O is counted in, and 1 / it
#pragma unroll 1
  for (int t = 0; t < n;) {
    // ---- a head: all or part of its tokens
    ctx = (int)min((long)a.ctx[b], (long)a.max_pages * a.P);
    const int h0 = (vh / a.nblk) * a.G, first = (vh % a.nblk) * HG;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int head = first + 8 * nb + g;
      const bool live = head < a.G;
      const __nv_bfloat16* qp = a.q + ((long)b * a.Hq + h0 + head) * D;
      Raw8<__nv_bfloat16> raw[NJ][2];
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          raw[j][e].u = make_uint4(0u, 0u, 0u, 0u);
          if (live) raw[j][e].load(qp + (i4 + 4 * j) * 16 + 8 * e);
        }
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v[8];
          raw[j][e].get(v);
#pragma unroll
          for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(v[k]));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the power of two at or below the head's largest value (clamped: its inverse is a normal number too);
      // a negative scale goes into Q, so that the factor of the scores is never negative
      const uint32_t e2 = min(max(__float_as_uint(top) >> 23, 2u), 252u);
      const float scale = __uint_as_float(e2 << 23) * fabsf(a.scale_log2);
      const float down = copysignf(__uint_as_float((254u - e2) << 23), a.scale_log2);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v[8];
          raw[j][e].get(v);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            qb[nb][j * 4 + 2 * e + k][0] = pack_half2(v[4 * k] * down, v[4 * k + 1] * down);
            qb[nb][j * 4 + 2 * e + k][1] = pack_half2(v[4 * k + 2] * down, v[4 * k + 3] * down);
          }
        }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        qs[nb][c] = __shfl_sync(0xffffffffu, scale, (2 * i4 + c) * 4);
        m[nb][c] = kNone;
        l[nb][c] = 0.f;
      }
#pragma unroll
      for (int x = 0; x < MT; ++x) o[nb][x][0] = o[nb][x][1] = o[nb][x][2] = o[nb][x][3] = 0.f;
    }
    vref = 0.f;
    vinv = 1.f;
    const int run = min(tb - tile, n - t);
#pragma unroll 1
    for (int e = 0; e < run; ++e, ++t) {
      const int bi = t & 31;
      if (bi == 0) {
        if (t > 0) { at_c = at_n; ka_c = ka_n; va_c = va_n; }
        if (t + 32 < n) load_ids(t + 32, at_n, grp);
      }
      if (bi == 8 && t - 8 + 32 < n) load_amax(grp, ka_n, va_n);
      bool ok = mbar_wait(&full[s], ph, dead, a.status, 1212);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {                                                 // (recorded) no more tiles
        t = n;
        break;
      }
      const uint8_t* kt = ring + s * C::kStage;
      const uint8_t* vt = kt + kTile * D;
      const float ka = __shfl_sync(0xffffffffu, ka_c, bi), va = __shfl_sync(0xffffffffu, va_c, bi) * (1.f / 127.f);
      const int left = ka < 0.f ? 0 : ctx - (tile + e) * kTile;          // tokens of the tile that count (a NaN magnitude counts)

      // ---- S^T: row r of the MMA is token 4 (r / 2 % 4) + r % 2 + 2 (r / 8), so that after the transposition below a lane
      // has the weights of tokens 4 i4 .. 4 i4 + 3, whose V bytes are one word
      float sc[NB][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) sc[nb][0] = sc[nb][1] = sc[nb][2] = sc[nb][3] = 0.f;
      const int tok = 4 * (g >> 1) + (g & 1);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const uint4 k0 = *reinterpret_cast<const uint4*>(kt + tok * D + (i4 + 4 * j) * 16);
        const uint4 k1 = *reinterpret_cast<const uint4*>(kt + (tok + 2) * D + (i4 + 4 * j) * 16);
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t f[4];
          int8x4_to_half(w0[k], f[0], f[2]);
          int8x4_to_half(w1[k], f[1], f[3]);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma_f16(sc[nb], f, qb[nb][j * 4 + k][0], qb[nb][j * 4 + k][1]);
        }
      }
      // ---- weights.  Column c of sc is head 2 i4 + c % 2.
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 4; ++c) sc[nb][c] *= ka * qs[nb][c & 1];
      if (left < kTile) {                                        // (uniform) tokens behind the context
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (tok + (c & 2) >= left) sc[nb][c] = -INFINITY;
      }
      bool move = va > vref;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c) move |= fmaxf(sc[nb][c], sc[nb][2 + c]) > m[nb][c] + kMost;
      if (__any_sync(0xffffffffu, move)) {
        const float vnew = fmaxf(vref, va), down = vnew > 0.f ? __fdiv_rn(vref, vnew) : 1.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = fmaxf(sc[nb][c], sc[nb][2 + c]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float mn = mx > m[nb][c] + kMost ? mx - kUnit : m[nb][c];
            const float alpha = exp2f(m[nb][c] - mn);
            m[nb][c] = mn;
            l[nb][c] *= alpha;
            const float all = alpha * down;
#pragma unroll
            for (int x = 0; x < MT; ++x) {
              o[nb][x][c] *= all;
              o[nb][x][2 + c] *= all;
            }
          }
        vref = vnew;
        vinv = vnew > 0.f ? __fdiv_rn(1.f, vnew) : 1.f;
      }
      const float ratio = va * vinv;
      const bool faint = ratio < kFaint;                           // (uniform; a NaN magnitude is not)
      const float pr = faint ? 1.f : ratio;
      uint32_t pb[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float pv[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) pv[c] = exp2f(sc[nb][c] - m[nb][c & 1]);
        l[nb][0] += pv[0] + pv[2];
        l[nb][1] += pv[1] + pv[3];
        pb[nb][0] = transpose8x8(pack_half2(pv[0] * pr, pv[1] * pr));
        pb[nb][1] = transpose8x8(pack_half2(pv[2] * pr, pv[3] * pr));
      }
      // ---- O^T: dims g and g + 8 of each tile, tokens 4 i4 .. 4 i4 + 3
      const uint32_t* vw = reinterpret_cast<const uint32_t*>(vt) + g * 4 + i4;
      if (!faint) {
#pragma unroll
        for (int x = 0; x < MT; ++x) {
          uint32_t f[4];
          int8x4_to_half(vw[x * 64], f[0], f[2]);
          int8x4_to_half(vw[x * 64 + 32], f[1], f[3]);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) mma_f16(o[nb][x], f, pb[nb][0], pb[nb][1]);
        }
      } else {
#pragma unroll
        for (int x = 0; x < MT; ++x) {
          uint32_t f[4];
          int8x4_to_half(vw[x * 64], f[0], f[2]);
          int8x4_to_half(vw[x * 64 + 32], f[1], f[3]);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            mma_f16(c, f, pb[nb][0], pb[nb][1]);
#pragma unroll
            for (int k = 0; k < 4; ++k) o[nb][x][k] += c[k] * ratio;
          }
        }
      }
      __syncwarp();                                                // the stage has been read by all lanes
      {
        const int ahead = bi + C::kStages;
        const int at = __shfl_sync(0xffffffffu, ahead < 32 ? at_c : at_n, ahead & 31);
        if (t + C::kStages < n) issue(s, at);
      }
      if (++s == C::kStages) { s = 0; ph ^= 1; }
    }
    if constexpr (ONE) {
      // this warp's part, [head][dim], over its own ring: the tiles in it have been read
      float* po = reinterpret_cast<float*>(ring);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int row = 8 * nb + 2 * i4 + c;
          l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], 4);
          l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], 8);
          l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], 16);
#pragma unroll
          for (int x = 0; x < MT; ++x) {
            po[row * D + x * 16 + g] = o[nb][x][c] * vref;
            po[row * D + x * 16 + 8 + g] = o[nb][x][2 + c] * vref;
          }
          if (g == 0) {
            part_ml[(warp * HG + row) * 2] = m[nb][c];
            part_ml[(warp * HG + row) * 2 + 1] = l[nb][c];
          }
        }
      break;                                                     // a worker has one head
    }
    // ---- end of this head's tokens, or of this worker's share
    const int seg = prefix[b] * VH + vh * tb;                  // flat tile the head begins with
    const bool whole = seg >= f0 && seg + tb <= f1;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      __syncwarp();
      float up[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], 4);
        l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], 8);
        l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], 16);
        up[c] = whole ? (l[nb][c] != 0.f ? __fdividef(vref, l[nb][c]) : 0.f) : vref;
      }
      if (whole) {
        // pairs of heads of a dim -> pairs of dims of a head
        const int head = first + 8 * nb + g;
        __nv_bfloat16* op = a.out + ((long)b * a.Hq + h0 + head) * D + 2 * i4;
#pragma unroll
        for (int x = 0; x < MT; ++x) {
          const uint32_t lo = transpose8x8(pack_bf16x2(o[nb][x][0] * up[0], o[nb][x][1] * up[1]));
          const uint32_t hi = transpose8x8(pack_bf16x2(o[nb][x][2] * up[0], o[nb][x][3] * up[1]));
          if (head < a.G) {
            *reinterpret_cast<uint32_t*>(op + x * 16) = lo;
            *reinterpret_cast<uint32_t*>(op + x * 16 + 8) = hi;
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int row = 8 * nb + 2 * i4 + c;
          if (first + row < a.G) {
            const long slot = ((long)w * 2 + (seg < f0 ? 0 : 1)) * HG + row;
            float* pp = a.part + slot * D + g;
#pragma unroll
            for (int x = 0; x < MT; ++x) {
              pp[x * 16] = o[nb][x][c] * up[c];
              pp[x * 16 + 8] = o[nb][x][2 + c] * up[c];
            }
            if (g == 0) { a.ml[slot * 2] = m[nb][c]; a.ml[slot * 2 + 1] = l[nb][c]; }
          }
        }
      }
    }
    // ---- the next KV head or non-empty sequence
    tile = 0;
    if (++vh == VH) {
      vh = 0;
      do { ++b; } while (b < a.B && prefix[b + 1] == prefix[b]);
      if (b < a.B) tb = prefix[b + 1] - prefix[b];
    }
  }
  if constexpr (ONE) {
    if (n == 0) {                                                // no part of the context
      for (int i = lane; i < HG * D; i += 32) reinterpret_cast<float*>(ring)[i] = 0.f;
      for (int i = lane; i < HG; i += 32) {
        part_ml[(warp * HG + i) * 2] = kNone;
        part_ml[(warp * HG + i) * 2 + 1] = 0.f;
      }
    }
    __syncthreads();
    const int first = (vh % a.nblk) * HG, heads = min(HG, a.G - first), items = heads * (D / 4);
    __nv_bfloat16* op = a.out + ((long)b * a.Hq + (vh / a.nblk) * a.G + first) * D;
    float* sum0 = reinterpret_cast<float*>(smem);                // the block's sum takes the place of warp 0's
    constexpr int kNext = C::kStages * C::kStage / 4;            // floats from one warp's part to the next
    auto put = [&](int i, const float4& v, float L) {
      const float inv = L != 0.f ? __fdividef(1.f, L) : 0.f;
      *reinterpret_cast<uint2*>(op + i * 4) = make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
    };
    for (int i = threadIdx.x; i < items; i += kWarps * 32) {
      const int h = i / (D / 4);
      float M = kNone, L = 0.f;
#pragma unroll
      for (int x = 0; x < kWarps; ++x) M = fmaxf(M, part_ml[(x * HG + h) * 2]);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int x = 0; x < kWarps; ++x) {
        const float f = exp2f(part_ml[(x * HG + h) * 2] - M);
        const float4 p = *reinterpret_cast<const float4*>(sum0 + x * kNext + i * 4);
        L += part_ml[(x * HG + h) * 2 + 1] * f;
        v.x += p.x * f; v.y += p.y * f; v.z += p.z * f; v.w += p.w * f;
      }
      if (a.cluster == 1) {
        put(i, v, L);
      } else {
        *reinterpret_cast<float4*>(sum0 + i * 4) = v;            // (read by this thread only)
        if (i % (D / 4) == 0) { block_ml[2 * h] = M; block_ml[2 * h + 1] = L; }
      }
    }
    if (a.cluster > 1) {
      __syncwarp();
      cluster_sync_all();
      for (int i = (int)cluster_ctarank() * kWarps * 32 + threadIdx.x; i < items; i += a.cluster * kWarps * 32) {
        const int h = i / (D / 4);
        float M = kNone, L = 0.f, ms[8], ls[8];
        float4 p[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          ms[x] = kNone;
          ls[x] = 0.f;
          p[x] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (x < a.cluster) {
            const uint32_t ml = mapa_shared(smem_u32(block_ml + 2 * h), x);
            ms[x] = ld_cluster_f32(ml);
            ls[x] = ld_cluster_f32(ml + 4);
            p[x] = ld_cluster_f32x4(mapa_shared(smem_u32(sum0 + i * 4), x));
          }
          M = fmaxf(M, ms[x]);
        }
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float f = exp2f(ms[x] - M);
          L += ls[x] * f;
          v.x += p[x].x * f; v.y += p[x].y * f; v.z += p[x].z * f; v.w += p[x].w * f;
        }
        put(i, v, L);
      }
      __syncwarp();
      cluster_sync_all();                                        // nobody leaves while another block still reads its sums
    }
  }
}

// Adds up the partials of the heads whose tokens went to several workers, and writes zeros for an empty
// context.  Grid (B Hq, D / SL): a block has SL dims of a head, a group of lanes holds them (four or eight a
// lane), and the block's groups take the partials in turn; the largest maximum is found first, so that the
// loads of the sums do not wait for one another.  SL = D for many heads (few blocks and few partials each),
// 32 for few heads whose tokens went to many workers: 1 sequence of 60000 tokens and one KV head takes 20 us
// that way, 48 with whole heads a block; 300 sequences of up to 200 tokens 42 us with whole heads, 60 in slices.
// HP: heads of a block, a warp each (1: the whole block works on one).  Most heads of a large batch lie in one worker's share and
// need nothing: 8000 sequences of 500 tokens, 32 query heads, take 1646 us with eight heads a block, 1696 with one.
template <int D, int HG, int SL, int HP>
__global__ void __launch_bounds__(SL == 32 ? 1024 : 256) merge_int8_kernel(const AttnArgs a) {
  constexpr int LG = SL / 4 < 32 ? SL / 4 : 32;                  // lanes of a group
  constexpr int NV = SL / 4 / LG;                                // float4s of a lane
  constexpr int GW = 32 / LG;                                    // groups of a warp
  __shared__ float s_top[32], s_sum[32];
  __shared__ float4 s_acc[SL == 32 ? 32 : 8][SL / 4];            // [warps]
  const int lane = threadIdx.x & 31, warp = HP > 1 ? 0 : threadIdx.x >> 5, warps = HP > 1 ? 1 : blockDim.x >> 5;
  const int tid = warp * 32 + lane, threads = warps * 32;
  const int item = blockIdx.x * HP + (HP > 1 ? threadIdx.x >> 5 : 0), b = item / a.Hq, hq = item - b * a.Hq;
  const int h = hq / a.G, hg = hq % a.G, vh = h * a.nblk + hg / HG, row = hg % HG;
  const int VH = a.Hkv * a.nblk;
  chain_wait();
  if (HP > 1 && b >= a.B) return;
  const int before = a.seen[b], tb = a.seen[b + 1] - before, total = a.seen[a.B];
  __nv_bfloat16* op = a.out + ((long)b * a.Hq + hq) * D + blockIdx.y * SL;
  if (tb == 0) {
    for (int d = tid; d < SL; d += threads) op[d] = __float2bfloat16(0.f);
    return;
  }
  const int chunk = chunk_of(a, total * VH), seg = before * VH + vh * tb;
  const int w0 = seg / chunk, w1 = (seg + tb - 1) / chunk, pieces = w1 - w0 + 1;
  if (pieces == 1) return;                                       // one worker had it all and wrote it
  auto slot_of = [&](int i) { return ((long)(w0 + i) * 2 + (i == 0 ? 1 : 0)) * HG + row; };
  float M = -INFINITY;
  for (int i = tid; i < pieces; i += threads) M = fmaxf(M, a.ml[slot_of(i) * 2]);
  M = warp_max(M);
  if (warps > 1) {
    if (lane == 0) s_top[warp] = M;
    __syncthreads();
    M = warp_max(lane < warps ? s_top[lane] : -INFINITY);
  }
  const int sub = lane % LG, group = warp * GW + lane / LG, groups = warps * GW;
  float4 acc[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  float L = 0.f;
#pragma unroll 4
  for (int i = group; i < pieces; i += groups) {
    const long slot = slot_of(i);
    const float2 ml = *reinterpret_cast<const float2*>(a.ml + slot * 2);
    const float4* pp = reinterpret_cast<const float4*>(a.part + slot * D + blockIdx.y * SL) + sub;
    const float f = exp2f(ml.x - M);
    L += ml.y * f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const float4 v = pp[k * LG];
      acc[k].x += v.x * f; acc[k].y += v.y * f; acc[k].z += v.z * f; acc[k].w += v.w * f;
    }
  }
  auto add_groups = [&](float4& v) {
#pragma unroll
    for (int o = LG; o < 32; o *= 2) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
      v.z += __shfl_xor_sync(0xffffffffu, v.z, o);
      v.w += __shfl_xor_sync(0xffffffffu, v.w, o);
    }
  };
#pragma unroll
  for (int o = LG; o < 32; o *= 2) L += __shfl_xor_sync(0xffffffffu, L, o);
#pragma unroll
  for (int k = 0; k < NV; ++k) add_groups(acc[k]);
  if (warps > 1) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (lane < LG) s_acc[warp][k * LG + sub] = acc[k];
    if (lane == 0) s_sum[warp] = L;
    __syncthreads();
    if (warp != 0) return;
    L = warp_sum(lane < warps ? s_sum[lane] : 0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int x = lane / LG; x < warps; x += GW) {
        const float4 v = s_acc[x][k * LG + sub];
        acc[k].x += v.x; acc[k].y += v.y; acc[k].z += v.z; acc[k].w += v.w;
      }
      add_groups(acc[k]);
    }
  }
  const float inv = L != 0.f ? __fdividef(1.f, L) : 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (lane < LG)
      *reinterpret_cast<uint2*>(op + (k * LG + sub) * 4) =
          make_uint2(pack_bf16x2(acc[k].x * inv, acc[k].y * inv), pack_bf16x2(acc[k].z * inv, acc[k].w * inv));
}

// Sequences of a launch: their running counts lie in shared memory, where four blocks an SM leave 4 KB each (2048 of 2048
// tokens, 8 KV heads: 1826 us in one launch with three blocks an SM, 1429 in two).
constexpr int kMaxSeqs = 1024;
template <int D, int HG, bool ONE>
int launch_decode(const AttnArgs& a, int blocks, int smem, cudaStream_t stream) {
  auto kern = decode_int8_kernel<D, HG / 8, ONE>;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {                // the most that any call takes: host threads in a race set the same
    const int most = ONE ? smem : smem + (kMaxSeqs - a.B) * 4;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  return axh::launch_chained(kern, dim3(blocks), dim3(kWarps * 32), smem, ONE ? a.cluster : 1, stream, a);
}

template <int D, int HG>
int launch_attn(const AttnArgs& a, int blocks, cudaStream_t stream) {
  using C = AttnCfg<D>;
  const int fixed = C::kRing + kWarps * C::kStages * 8 + 8;
  if (a.cluster > 0) return launch_decode<D, HG, true>(a, blocks, fixed + (kWarps + 1) * HG * 8, stream);
  int rc = launch_decode<D, HG, false>(a, blocks, fixed + (a.B + 1) * 4, stream);
  if (rc) return rc;
  // partials of a head, at the most if heads are alike
  const long heads = (long)a.B * a.Hkv * a.nblk, per = a.workers / heads + 2;
  int warps = 1;
  if ((long)a.B * a.Hq >= 4 * axh::sm_count()) {
    while (warps < 8 && warps * 2 < per) warps *= 2;
    if (warps == 1) return axh::launch_chained(merge_int8_kernel<D, HG, D, 8>, dim3((a.B * a.Hq + 7) / 8), dim3(256), 0, 1, stream, a);
    return axh::launch_chained(merge_int8_kernel<D, HG, D, 1>, dim3(a.B * a.Hq), dim3(32 * warps), 0, 1, stream, a);
  }
  while (warps < 32 && warps * 4 < per) warps *= 2;
  return axh::launch_chained(merge_int8_kernel<D, HG, 32, 1>, dim3(a.B * a.Hq, D / 32), dim3(32 * warps), 0, 1, stream, a);
}

}  // namespace

// New K/V rows [T, Hkv, D] (dt 1 bf16, 0 fp32; inner stride 1, token and head strides in elements, rows on 16-byte
// boundaries) of B sequences into their pages.  Row b brings tokens cu[b] .. cu[b + 1] (cu null: T / B each) at positions
// starts[b], starts[b] + 1, ...  Tokens behind cu[B] are not read.  A row that does not fit its table, or a page number outside
// the cache, is recorded in `status` and skipped.
AX_API int ax_kv_write_int8(int dt, const void* k, long k_ts, long k_hs, const void* v, long v_ts, long v_hs, int8_t* kc, int8_t* vc,
                            float* ka, float* va, const int* table, const int* starts, const int* cu, int T, int B, int Hkv, int D, int P,
                            int max_pages, int num_pages, int* status, cudaStream_t stream) {
  if (T <= 0 || B <= 0 || Hkv <= 0) return 0;
  if (D % 16 || D > 512 || P % 16 || P <= 0 || (long)P * D > (1L << 30) || Hkv > 65535 || (cu == nullptr && T % B)) return -1;
  const int vec = dt == 1 ? 8 : 4;
  if ((k_ts % vec) || (k_hs % vec) || (v_ts % vec) || (v_hs % vec) || (((uintptr_t)k | (uintptr_t)v | (uintptr_t)kc | (uintptr_t)vc) & 15)) return -2;
  // a row of n tokens touches at most (n + 2 P - 2) / P pages; a single token one
  const int per_row = T == B ? 1 : (int)((T / B + 2L * P - 2) / P);
  const long pieces = cu == nullptr ? (long)B * per_row : (T + B * (2L * P - 2)) / P + 1;
  if (pieces > 0x7fffffffL) return -3;
  WriteArgs a{k, v, kc, vc, ka, va, table, starts, cu, k_ts, k_hs, v_ts, v_hs, T, B, Hkv, D, P, max_pages, num_pages, per_row, T / B, (P & (P - 1)) == 0 ? __builtin_ctz((unsigned)P) : -1, (65536 + D / 8 - 1) / (D / 8), status};
  const dim3 grid((unsigned)pieces, Hkv);
  // Larger blocks shorten the latency of a big page where few blocks leave room (200 tokens, pages of 64 x 128: 6.2 us
  // against 8.4); full devices prefer the small ones (8192 tokens, pages of 16 x 128: 18.5 against 32.1).
  const bool big = (long)P * D >= 4096 && pieces * Hkv < 8L * axh::sm_count();
  auto go = [&](auto kern, int half) { return axh::launch_chained(kern, grid, dim3(2 * half), 0, 1, stream, a); };
  if (dt == 1) return big ? go(kv_write_int8_kernel<__nv_bfloat16, 128>, 128) : go(kv_write_int8_kernel<__nv_bfloat16, 64>, 64);
  return big ? go(kv_write_int8_kernel<float, 128>, 128) : go(kv_write_int8_kernel<float, 64>, 64);
}

// How the attention kernel is launched for a cache of this capacity.  The contexts lie on the device, so the table's width
// stands for them: in a table much wider than they are, a few sequences get shares that are too large (1 sequence of 777 tokens, 8 KV
// heads: 6.1 us in a table of 1024 tokens, 12.6 in 8192, 18.2 in 32768, 26.7 in 131072; 8 of 777 10.4 in all; 64 of 777 23.8 and 31.1).
struct AttnShape { int HG, nblk, min_chunk, blocks, cluster; };
static AttnShape attn_shape(int B, int Hq, int Hkv, int D, int max_pages, int P) {
  AttnShape r;
  const int G = Hq / Hkv;
  r.HG = G <= 8 ? 8 : 16;
  r.nblk = (G + r.HG - 1) / r.HG;
  const long per_head = (long)max_pages * P / kTile, heads = (long)B * Hkv * r.nblk, tiles = heads * per_head;
  const long most = (long)axh::sm_count() * (r.HG == 16 || D == 256 ? 2 : 4);
  // The fewest tiles a worker takes: every tile in turn costs it about 0.45 us, every worker a partial that the
  // merge has to read, so a share grows with the root of the context (1 sequence of 4096 tokens, 8 KV
  // heads: 13.8 us with shares of one tile, 12.1 with four; 100 tokens: 7.3 and 10.9).
  long chunk = 1;
  while ((chunk + 1) * (chunk + 1) * 16 < per_head) ++chunk;
  r.min_chunk = (int)(chunk < 64 ? chunk : 64);
  const long even = (tiles + most * kWarps - 1) / (most * kWarps);
  if (even > chunk) chunk = even;
  // A cluster a head, as many blocks as fit the device at once and have tiles to read, when its warps then take at
  // most eight tiles more than even shares would.  Cluster / even shares and merge, us (32 heads, 8 KV heads): 1 sequence of
  // 777 tokens 6.2 / 8.8, 4096 11.9 / 13.1, 8192 17.8 / 15.3, 30000 50 / 24; 8 of 777 10.4 / 15.5; 64 of 777 23.8 / 31.9,
  // of up to 2048 with lengths spread over 0.3 to 1 44.7 / 44.8.
  r.cluster = 0;
  // More heads than blocks at once: a block a head by estimated time (us, fits to full tables).  Even shares cost 9 and, a
  // tile of a worker, 2.2 up to 14 of them, 1.55 beyond; a block a head 2.6 and, in turn, 2 and 1.6 a tile of its warps; the last
  // turn is half full on average.  Block a head / even shares: 128 x 500 tokens, 8 KV heads 32.0 / 39.5; 300 x 200 37.8 / 45.7;
  // 64 x 777, 32 KV heads 72.9 / 82.1; 24 x 8192, 32 KV heads 232 / 203; 64 x 16, 32 KV heads 14.9 / 11.2.
  if (heads > most) {
    const double turns = (double)heads / most, whole = (double)((heads + most - 1) / most);
    const double part = per_head > kWarps ? (double)per_head / kWarps : 1.0;
    const double block = 2.6 + 0.5 * (turns + whole) * (1.6 * part + 2.0);
    const double shares = 9.0 + 2.2 * (chunk < 14 ? chunk : 14) + 1.55 * (chunk > 14 ? chunk - 14 : 0);
    if (block < shares) {
      r.cluster = 1;
      r.blocks = (int)heads;
      return r;
    }
  }
  if (heads <= most) {
    int c = 8;
    while (c > 1 && (heads * c > most || (c / 2) * kWarps >= per_head)) c /= 2;
    if ((per_head + c * kWarps - 1) / (c * kWarps) <= chunk + 8) {
      r.cluster = c;
      r.blocks = (int)(heads * c);
      return r;
    }
  }
  // Blocks whose warps all have a share; where that leaves SMs without a block, fewer warps a block.
  long n = (tiles + chunk * kWarps - 1) / (chunk * kWarps);
  if (n < axh::sm_count()) {
    n = (tiles + chunk - 1) / chunk;
    if (n > axh::sm_count()) n = axh::sm_count();
  }
  r.blocks = (int)(n < 1 ? 1 : (n < most ? n : most));
  return r;
}

// Floats of workspace that ax_decode_int8 needs (0: none).
AX_API long ax_decode_int8_workspace(int B, int Hq, int Hkv, int D, int max_pages, int P) {
  if (Hkv <= 0 || Hq % Hkv || P <= 0) return 0;
  const AttnShape r = attn_shape(B, Hq, Hkv, D, max_pages, P);
  return r.cluster ? 0 : (long)r.blocks * kWarps * 2 * r.HG * (D + 2) + B + 1;
}

// out[B, Hq, D] = attention of q[B, Hq, D] (bf16, contiguous) over the first ctx[b] tokens of each sequence.
// D in {64, 128, 256}; P a multiple of 16.  A context longer than the table and a page number outside the cache are
// recorded in `status`; such tokens do not count.
AX_API int ax_decode_int8(const void* q, const int8_t* kc, const int8_t* vc, const float* ka, const float* va, const int* table,
                          const int* ctx, void* out, int B, int Hq, int Hkv, int D, int P, int max_pages, int num_pages, float scale,
                          float* workspace, int* status, cudaStream_t stream) {
  if (B <= 0) return 0;
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv || P <= 0 || P % 16 || B > kMaxSeqs || (long)B * Hq > 0x7fffffffL) return -1;
  if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)out | (uintptr_t)workspace) & 15) return -2;
  const AttnShape r = attn_shape(B, Hq, Hkv, D, max_pages, P);
  const int HG = r.HG, blocks = r.blocks, workers = blocks * kWarps;
  // flat tiles and the end of a share are ints
  if ((long)B * Hkv * r.nblk * ((long)max_pages * P / kTile) > 0x7f000000L || (long)num_pages * Hkv * (P / kTile) > 0x7fffffffL) return -3;
  AttnArgs a{(const __nv_bfloat16*)q, kc, vc, ka, va, table, ctx, (__nv_bfloat16*)out, workspace, workspace + (long)workers * 2 * HG * D,
             B, Hq, Hkv, Hq / Hkv, r.nblk, P, max_pages, num_pages, r.min_chunk, workers, (int*)(workspace + (long)workers * 2 * HG * (D + 2)), r.cluster, scale * 1.4426950408889634f / 127.f, status};
#define AX_ATTN(DD)                                                      \
  return HG == 8 ? launch_attn<DD, 8>(a, blocks, stream) : launch_attn<DD, 16>(a, blocks, stream)
  switch (D) {
    case 64: AX_ATTN(64);
    case 128: AX_ATTN(128);
    case 256: AX_ATTN(256);
    default: return -4;
  }
#undef AX_ATTN
}
