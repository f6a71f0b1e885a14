// Products of a few rows with a weight held in 4 bits: y[m, n] = sum_k x[m, k] w[n, k] (+ bias[n]), w ~ scale c + low by groups of 32, 64 or 128 along K (int4.cuh).
//
// A weight is tiles of 16 output rows x 128 channels: weight words [row][t][j] of 128 channels, then the group words [row][group].  Eight tiles of 128 rows lie one behind
// the other, then those of the next 128 channels (a copy of the eight is one of 9 KB: eight copies of 1 KB each streamed 2.8 TB/s where one streamed 4.4), then the next rows'.
// Rows beyond N and channels beyond K hold codes, scales and lowest values of 0.
//
// Few rows (up to 16): a block of eight warps has 32 output rows, its warps walk along K in blocks of 128 channels, one in eight each, and add their sums up at the end; where that
// leaves SMs idle, the blocks of a cluster share K.  Codes become exact 16-bit numbers (a mask that leaves a code in the low bits of 128 or 1024, and a subtraction) and are the
// left operand, 16 output rows at a time; rows of x, read from L2 and L1 as the operands' lanes want them, are the right one, eight at a time.  Scale and lowest value stay out: a
// group's product is scaled in fp32 when its channels are through, and the lowest value times the sum of x over the group (one more product, with ones) is added.
// More rows: a block has 128 output rows and all rows of x (in pieces of 128), and the products run on tcgen05.  Eight warps turn a block of 128 channels of codes into a swizzled
// operand tile in shared memory, rows of x come by TMA, one warp issues the products of a group of channels into an accumulator of its own in tensor memory, and eight warps
// scale it into sums in registers (and add the lowest values times the sums of x, which they take from the operand tile) while the next group is multiplied.
#include "attn_common.cuh"
#include "int4.cuh"

#include <algorithm>
#include <atomic>

namespace {

constexpr int kFewWarps = 8, kFewThreads = kFewWarps * 32, kFewRows = 32;
constexpr int kMaxSplits = 8;      // blocks of a portable cluster

template <int G> struct WTile {
  static constexpr int kGroups = 128 / G, kWords = 16 * 16 + 16 * kGroups;
};

// where tile i of block kb begins
template <int G> RB_DEVICE int64_t tile_at(int i, int kb, int kblocks) { return (((int64_t)(i >> 3) * kblocks + kb) * 8 + (i & 7)) * WTile<G>::kWords; }

template <typename T, int G>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ w, uint32_t* __restrict__ q, int N, int K, int64_t ld) {
  const int r = threadIdx.x / 16, sub = threadIdx.x % 16, n = blockIdx.x * 16 + r, kblocks = RB_CEIL_DIV(K, 128);
  rb::pdl_trigger();
  rb::pdl_wait();
  for (int kb = blockIdx.y; kb < kblocks; kb += gridDim.y) {
    const int k = kb * 128 + sub * 8;
    const bool mine = n < N && k < K;
    uint4 a = make_uint4(0, 0, 0, 0);
    if (mine) a = *reinterpret_cast<const uint4*>(w + n * ld + k);
    float lo, hi;
    q4::extremes<T, G / 8>(a, lo, hi);
    const q4::Coded c = q4::code8<T, q4::kWeight>(a, lo, hi);
    uint32_t* at = q + tile_at<G>(blockIdx.x, kb, kblocks);
    at[r * 16 + q4::word_place<4>(sub)] = mine ? c.word : 0u;
    if (sub % (G / 8) == 0) at[256 + r * WTile<G>::kGroups + sub / (G / 8)] = mine ? c.group : 0u;
  }
}

// The same from codes, a byte each, and 16-bit steps and lowest values.
template <int G> __global__ void __launch_bounds__(256) pack_kernel(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scale, const uint16_t* __restrict__ low,
                                                                    uint32_t* __restrict__ q, int N, int K) {
  const int r = threadIdx.x / 16, sub = threadIdx.x % 16, n = blockIdx.x * 16 + r, kblocks = RB_CEIL_DIV(K, 128);
  rb::pdl_trigger();
  rb::pdl_wait();
  for (int kb = blockIdx.y; kb < kblocks; kb += gridDim.y) {
    const int k = kb * 128 + sub * 8;
    const bool mine = n < N && k < K;
    uint2 c = make_uint2(0, 0);
    if (mine) c = *reinterpret_cast<const uint2*>(codes + (int64_t)n * K + k);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (c.x >> (8 * i) & 15u) << q4::bit_of<q4::kWeight>(i) | (c.y >> (8 * i) & 15u) << q4::bit_of<q4::kWeight>(4 + i);
    uint32_t* at = q + tile_at<G>(blockIdx.x, kb, kblocks);
    at[r * 16 + q4::word_place<4>(sub)] = w;
    if (sub % (G / 8) == 0) {
      const int64_t g = (int64_t)n * (K / G) + k / G;
      at[256 + r * WTile<G>::kGroups + sub / (G / 8)] = mine ? (uint32_t)scale[g] << 16 | low[g] : 0u;
    }
  }
}

template <typename T> RB_DEVICE void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same onto zeros
template <typename T> RB_DEVICE void mma16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
template <typename T> constexpr uint32_t kOnes = std::is_same<T, __half>::value ? 0x3c003c00u : 0x3f803f80u;

// The codes of a word as pairs of neighbouring channels of type T, exact.  `magic`, 1024 or 128 in both halves, comes as a number that the compiler does not know: mask and
// magic as two immediates are two instructions where an immediate and a register are one.
template <typename T> constexpr uint32_t kMagic = std::is_same<T, __half>::value ? 0x64006400u : 0x43004300u;
template <typename T> RB_DEVICE void expand(uint32_t w, uint32_t (&h)[4], uint32_t magic) {
  if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = (i < 2 ? w : w >> 8) & (i & 1 ? 0x00f000f0u : 0x000f000fu) | magic;       // 1024 + c, or 1024 + 16 c
      const __half2 x = *reinterpret_cast<const __half2*>(&u);
      const __half2 y = i & 1 ? __hfma2(x, __float2half2_rn(0.0625f), __float2half2_rn(-64.f)) : __hadd2(x, __float2half2_rn(-1024.f));
      h[i] = *reinterpret_cast<const uint32_t*>(&y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = w >> (4 * i) & 0x000f000fu | magic;                                       // 128 + c
      const __nv_bfloat162 y = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&u), __float2bfloat162_rn(-128.f));
      h[i] = *reinterpret_cast<const uint32_t*>(&y);
    }
  }
}

struct LinearParams {
  const void *x, *bias;
  const uint32_t* q;
  void* y;
  int M, N, K, kblocks, splits;
  int64_t ldx, ldy;
  int* status;              // rb_attn_status()
  uint32_t magic;           // kMagic<T>
};

// One block of 128 channels of 16 rows: a lane's words of rows g and g + 8, and their groups', from a tile in shared memory.
template <int G> struct Block {
  uint32_t w[2][4], g[2][128 / G];
  RB_DEVICE void load(uint32_t tile, int lane) {
    const int r = lane >> 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 v = ld_shared_v4(tile + h * 512 + lane * 16);
      w[h][0] = v.x; w[h][1] = v.y; w[h][2] = v.z; w[h][3] = v.w;
#pragma unroll
      for (int i = 0; i < 128 / G; ++i)
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(g[h][i]) : "r"(tile + 1024 + ((r + 8 * h) * (128 / G) + i) * 4) : "memory");
    }
  }
};
// A warp's ring of blocks on their way, 2176 to 2560 bytes each (registers hold one ahead, and 35 KB an SM were on their way: 2.1 TB/s at any number of rows)
constexpr int kFewRing = 4;
template <int G> constexpr int kFewBytes = kFewRows / 16 * WTile<G>::kWords * 4;
template <int G> constexpr size_t kFewSmem = kFewWarps * kFewRing * kFewBytes<G>;

// NT: sets of eight rows of x
template <typename T, int G, int NT>
__global__ void __launch_bounds__(kFewThreads, 2) few_rows_kernel(const LinearParams p) {
  constexpr int MT = kFewRows / 16, NG = 128 / G;
  extern __shared__ __align__(128) unsigned char few_ring[];
  __shared__ __align__(16) float sums[2][kFewWarps][NT * 8][kFewRows + 1];    // (of a tile of rows and of the next: a warp may be that far ahead)
  __shared__ float part[NT * 8][kFewRows];
  __shared__ __align__(8) uint64_t bar[kFewWarps][kFewRing];
  __shared__ uint32_t dead_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  volatile uint32_t* dead = &dead_flag;
  if (threadIdx.x == 0) *dead = 0;
  if (lane < kFewRing) ptx::mbar_init(ptx::smem_u32(&bar[warp][lane]), 1);
  ptx::fence_barrier_init();
  __syncthreads();
  rb::pdl_trigger();
  // the warp's blocks of a set of 32 output rows, then those of the next set of this block of threads: one sequence, whose copies run ahead of the sums at a set's end
  const int step = kFewWarps * p.splits, first = blockIdx.y * kFewWarps + warp, sets = RB_CEIL_DIV(p.N, kFewRows);
  const uint32_t ring = ptx::smem_u32(few_ring) + warp * (kFewRing * kFewBytes<G>);
  int ask_set = first < p.kblocks ? blockIdx.x : sets, ask_kb = first;
  const uint32_t* ask = p.q + tile_at<G>(ask_set * MT, first, p.kblocks);
  auto fetch = [&](int slot) {
    if (ask_set >= sets) return;
    if (ptx::elect_one()) {
      const uint32_t full = ptx::smem_u32(&bar[warp][slot]);
      ptx::mbar_arrive_expect_tx(full, kFewBytes<G>);
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(ring + slot * kFewBytes<G>),
                   "l"(ask), "r"(kFewBytes<G>), "r"(full) : "memory");
    }
    ask_kb += step;
    ask += step * (8 * WTile<G>::kWords);
    if (ask_kb >= p.kblocks) {
      ask_kb = first;
      ask_set += gridDim.x;
      ask = p.q + tile_at<G>(ask_set * MT, first, p.kblocks);
    }
  };
  rb::pdl_wait();
#pragma unroll
  for (int i = 0; i < kFewRing; ++i) fetch(i);
  // rows beyond M repeat the last one and are not stored; channels beyond K read the row's first ones: they meet codes, scales and lowest values of 0
  const T* x[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) x[n] = reinterpret_cast<const T*>(p.x) + min(n * 8 + g, p.M - 1) * p.ldx + 8 * t;
  const int cols = min(p.M, NT * 8);
  int slot = 0, half = 0;
  uint32_t round = 0;
#pragma unroll 1
  for (int set = blockIdx.x; set < sets; set += gridDim.x, half ^= 1) {
    float acc[MT][NT][4] = {};
#pragma unroll 1
  for (int kb = first; kb < p.kblocks; kb += step) {
    uint4 xv[NT][4];
    if (kb * 128 + 128 <= p.K) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4* from = reinterpret_cast<const uint4*>(x[n] + kb * 128);
#pragma unroll
        for (int j = 0; j < 4; ++j) xv[n][j] = __ldg(from + 4 * j);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) xv[n][j] = __ldg(reinterpret_cast<const uint4*>(x[n] + (kb * 128 + 32 * j < p.K ? kb * 128 + 32 * j : 0)));   // (K is a multiple of 32)
    }
    bounded_wait(ptx::smem_u32(&bar[warp][slot]), round, dead);
    Block<G> cur[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) cur[i].load(ring + slot * kFewBytes<G> + i * (WTile<G>::kWords * 4), lane);
    __syncwarp();
    fetch(slot);
    if (++slot == kFewRing) { slot = 0; round ^= 1; }
#pragma unroll
    for (int q = 0; q < NG; ++q) {                  // a group
      float c[MT][NT][4], one[NT][4];
#pragma unroll
      for (int j = q * 4 / NG; j < (q + 1) * 4 / NG; ++j) {
        uint32_t e0[MT][4], e1[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          expand<T>(cur[i].w[0][j], e0[i], p.magic);
          expand<T>(cur[i].w[1][j], e1[i], p.magic);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint32_t b0 = s ? xv[n][j].z : xv[n][j].x, b1 = s ? xv[n][j].w : xv[n][j].y;
            if (j == q * 4 / NG && s == 0) {
              mma16_first<T>(one[n], kOnes<T>, kOnes<T>, kOnes<T>, kOnes<T>, b0, b1);
#pragma unroll
              for (int i = 0; i < MT; ++i) mma16_first<T>(c[i][n], e0[i][0], e1[i][0], e0[i][1], e1[i][1], b0, b1);
              continue;
            }
            mma16<T>(one[n], kOnes<T>, kOnes<T>, kOnes<T>, kOnes<T>, b0, b1);
#pragma unroll
            for (int i = 0; i < MT; ++i) mma16<T>(c[i][n], e0[i][2 * s], e1[i][2 * s], e0[i][2 * s + 1], e1[i][2 * s + 1], b0, b1);
          }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float scale = q4::scale_of<T>(cur[i].g[h][q]), low = q4::low_of<T>(cur[i].g[h][q]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) acc[i][n][2 * h + e] = fmaf(scale, c[i][n][2 * h + e], fmaf(low, one[n][e], acc[i][n][2 * h + e]));
        }
    }
  }
  // ---- the warps' sums, then the cluster's: columns (rows of x) 2t, 2t + 1, output rows g and g + 8
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[half][warp][n * 8 + 2 * t + (e & 1)][i * 16 + g + 8 * (e >> 1)] = acc[i][n][e];
  __syncthreads();
  auto finish = [&](int m, int r, float v) {
    const int n = set * kFewRows + r;
    if (n < p.N) reinterpret_cast<T*>(p.y)[m * p.ldy + n] = rb::from_f<T>(v + (p.bias ? rb::to_f(reinterpret_cast<const T*>(p.bias)[n]) : 0.f));
  };
  for (int i = threadIdx.x; i < cols * kFewRows; i += kFewThreads) {
    const int m = i / kFewRows, r = i % kFewRows;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) v += sums[half][w][m][r];
    if (p.splits == 1) finish(m, r, v); else part[m][r] = v;
  }
  if (p.splits == 1) continue;
  ptx::cluster_sync();                              // (a cluster has one set)
  for (int i = blockIdx.y * kFewThreads + threadIdx.x; i < cols * kFewRows; i += p.splits * kFewThreads) {
    const int m = i / kFewRows, r = i % kFewRows;
    float v = 0.f;
    for (int c = 0; c < p.splits; ++c) {
      uint32_t a;
      float f;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(ptx::smem_u32(&part[m][r])), "r"(c));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(a) : "memory");
      v += f;
    }
    finish(m, r, v);
  }
  }
  rb::report_given_up(dead, p.status);
  if (p.splits > 1) ptx::cluster_sync();  // nobody leaves while its sums are being read
}

template <typename T, int G, int NT> int few_rows(LinearParams p, cudaStream_t s) {
  static std::atomic<uint64_t> opted_in{0};           // the attribute is the kernel's on one device: a bit per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -3;
  if (dev >= 64 || !(opted_in.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(few_rows_kernel<T, G, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFewSmem<G>) != cudaSuccess) return -3;
    if (dev < 64) opted_in.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  }
  const int sets = RB_CEIL_DIV(p.N, kFewRows), blocks = std::min(sets, 2 * rb::kNumSMs);
  p.splits = 1;
  while (p.splits < kMaxSplits && sets * p.splits * 2 <= 2 * rb::kNumSMs && p.kblocks >= kFewWarps * p.splits * 2) p.splits *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks, p.splits);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = kFewSmem<G>;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (p.splits > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = attr[n].val.clusterDim.z = 1;
    attr[n++].val.clusterDim.y = p.splits;
  }
  if (rb::pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, few_rows_kernel<T, G, NT>, p) == cudaSuccess ? 0 : -3;
}

// ---------------------------------------------------------------------------------------------- many rows

constexpr int kManyRows = 128, kTeams = 2, kScale = 8;                               // output rows; teams of warps that expand (each has every second block), warps that scale
template <int NP> constexpr int kTeam = NP == 128 ? 2 : 4;                           // warps of a team (128 rows: scaling takes longer, and needs the registers)
template <int NP> constexpr int kManyThreads = (kTeams * kTeam<NP> + kScale + 2) * 32;
constexpr int kCodeBytes = kManyRows * 256;                                          // 128 rows x 128 channels of 16 bits: two halves of 64 channels
constexpr int kBufs = 4;                                                             // accumulators
template <int NP> constexpr int kManyStages = NP == 32 ? 4 : NP == 64 ? 3 : 2;       // operand tiles
template <int NP> constexpr int kRaw = NP == 32 ? 5 : 6;                             // blocks of packed codes, 9 or 10 KB each
template <int G> constexpr int kRawBytes = 8 * WTile<G>::kWords * 4;
template <int G, int NP> constexpr size_t kManySmem = 1024 + kManyStages<NP> * (kCodeBytes + NP * 256) + kRaw<NP> * kRawBytes<G>;

RB_DEVICE void tc_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
}
// (x0, x1) <- (x0, x1) + (m, m) * (a0, a1), one instruction
RB_DEVICE void fma2(float2& x, float m, float a0, float a1) {
  asm("{\n\t.reg .b64 x, m, a;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 m, {%2, %2};\n\tmov.b64 a, {%3, %4};\n\tfma.rn.f32x2 x, m, a, x;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(x.x), "+f"(x.y) : "f"(m), "f"(a0), "f"(a1));
}
template <typename T> RB_DEVICE float2 pair_of(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// NP: rows of x, padded (rows beyond M read as zeros)
template <typename T, int G, int NP>
__global__ void __launch_bounds__(kManyThreads<NP>, 1) many_rows_kernel(const __grid_constant__ CUtensorMap xmap, const LinearParams p) {
  constexpr int NG = 128 / G, ND = kBufs, kCols = NP / 2, kX = NP * 256, kStages = kManyStages<NP>, kR = kRaw<NP>, kSums = 3;
  constexpr int kExpand = kTeams * kTeam<NP>, kLoadWarp = kExpand + kScale, kMmaWarp = kLoadWarp + 1;
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], d_full[ND], d_empty[ND], raw_full[kR], raw_empty[kR];
  __shared__ __align__(16) float xsum[kSums][NG][NP];
  __shared__ uint32_t groups[kStages][kManyRows * NG];
  __shared__ uint32_t tmem_ptr, dead_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile uint32_t* dead = &dead_flag;
  const uint32_t base = (ptx::smem_u32(raw) + 1023u) & ~1023u, codes = base, xs = base + kStages * kCodeBytes, packed = xs + kStages * kX;
  auto bar = [](uint64_t* b, int i) { return ptx::smem_u32(&b[i]); };
  // ring slot n % size, in its (n / size)-th round: what fills it waits for the other parity
  auto wait_full = [&](uint64_t* b, int n, int size) { bounded_wait(ptx::smem_u32(&b[n % size]), n / size & 1, dead); };
  auto wait_empty = [&](uint64_t* b, int n, int size) { bounded_wait(ptx::smem_u32(&b[n % size]), (n / size & 1) ^ 1, dead); };
  if (threadIdx.x == 0) {
    *dead = 0;
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(bar(full, i), kTeam<NP> + 1);       // the codes' warps and the copy of x
      ptx::mbar_init(bar(empty, i), 1 + kScale);
    }
    for (int i = 0; i < ND; ++i) {
      ptx::mbar_init(bar(d_full, i), 1);
      ptx::mbar_init(bar(d_empty, i), kScale);
    }
    for (int i = 0; i < kR; ++i) {
      ptx::mbar_init(bar(raw_full, i), 1);
      ptx::mbar_init(bar(raw_empty, i), kTeam<NP>);
    }
    ptx::fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(ptx::smem_u32(&tmem_ptr), ND * NP);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_ptr);
  rb::pdl_trigger();
  rb::pdl_wait();
  // this block's part of the channels
  const int per = RB_CEIL_DIV(p.kblocks, p.splits), k0 = min(p.kblocks, (int)blockIdx.y * per), blocks = min(p.kblocks, k0 + per) - k0;
  float2 acc[kCols / 2];
#pragma unroll
  for (int i = 0; i < kCols / 2; ++i) acc[i] = make_float2(0.f, 0.f);

  if (warp < kExpand) {
    // ---- codes to operands: a team of warps has every second block (its waits, fences and stores pass beside the other's arithmetic), a warp two or four tiles of it, a lane the words
    // of rows g and g + 8 of their four steps; odd rows store them in another order, so that the eight lanes of a store meet all banks
    constexpr int kMine = 8 / (kTeam<NP>);
    const int g = lane >> 2, t = lane & 3, odd = g & 1, w0 = warp / kTeams * kMine;
    for (int n = warp % kTeams; n < blocks; n += kTeams) {
      wait_full(raw_full, n, kR);
      const uint32_t from = packed + n % kR * kRawBytes<G> + w0 * (WTile<G>::kWords * 4) + lane * 16;
      wait_empty(empty, n, kStages);
      const uint32_t to = codes + n % kStages * kCodeBytes + (w0 * 16 + g) * 128;
#pragma unroll
      for (int u = 0; u < kMine; ++u) {
#pragma unroll
        for (int i = lane; i < 16 * NG; i += 32) {
          uint32_t word;
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(word) : "r"(from - lane * 16 + u * (WTile<G>::kWords * 4) + 1024 + i * 4) : "memory");
          groups[n % kStages][(w0 + u) * 16 * NG + i] = word;
        }
        uint4 v[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) v[h] = ld_shared_v4(from + u * (WTile<G>::kWords * 4) + h * 512);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w[4] = {v[h].x, v[h].y, v[h].z, v[h].w};
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            uint32_t e[4];
            expand<T>(odd ? w[jj ^ 1] : w[jj], e, p.magic);
            const int j = jj ^ odd;                 // channels 32 j + 8 t ..: piece 4 (j & 1) + t of half j >> 1
            st_shared_v4(to + u * (16 * 128) + h * (8 * 128) + (j >> 1) * (kManyRows * 128) + ((((j & 1) * 4 + t) ^ g) << 4), e[0], e[1], e[2], e[3]);
          }
        }
      }
      ptx::fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(bar(full, n % kStages));
        ptx::mbar_arrive(bar(raw_empty, n % kR));
      }
    }
  } else if (warp < kLoadWarp) {
    // ---- sums: a warp has 32 output rows, a quarter of the lanes of tensor memory, and half of the rows of x
    const int quarter = warp % 4, half = (warp - kExpand) / 4, tid = (warp - kExpand) * 32 + lane;
    constexpr int kEach = kScale * 32 / NP, kPieces = 16 / kEach;                // threads a row of x, 16-byte pieces a thread of its 128 channels
    constexpr int kSpan = kPieces * 8, kOwn = kSpan > G ? kSpan / G : 1, kShare = kSpan < G ? G / kSpan : 1;   // channels of a thread, groups that it sums alone, threads of a group
    const int col = tid / kEach, sub = tid % kEach, row = quarter * 32 + lane;
    // the sums of x over the groups of block n, one block ahead of the products' use: a thread's pieces lie in one group, or are whole groups
    auto sums_of = [&](int n, uint32_t (&word)[NG]) {
      if (n >= blocks) return;
      wait_full(full, n, kStages);
      float2 s[kOwn];
#pragma unroll
      for (int i = 0; i < kOwn; ++i) s[i] = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int piece = sub * kPieces + i;
        const uint4 v = ld_shared_v4(xs + n % kStages * kX + (piece >> 3) * (NP * 128) + col * 128 + (((piece & 7) ^ (col & 7)) << 4));
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 a = pair_of<T>(u[e]);
          add_pair(s[i * kOwn / kPieces].x, s[i * kOwn / kPieces].y, a.x, a.y);
        }
      }
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        float total = s[i].x + s[i].y;
#pragma unroll
        for (int o = 1; o < kShare; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (sub % kShare == 0) xsum[n % kSums][sub / kShare * kOwn + i][col] = total;
      }
#pragma unroll
      for (int q = 0; q < NG; ++q) word[q] = groups[n % kStages][row * NG + q];
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(empty, n % kStages));
    };
    uint32_t next[NG];
    sums_of(0, next);
    for (int n = 0; n < blocks; ++n) {
      uint32_t word[NG];
#pragma unroll
      for (int q = 0; q < NG; ++q) word[q] = next[q];
      sums_of(n + 1, next);
      asm volatile("bar.sync 1, %0;" ::"n"(kScale * 32) : "memory");             // (sums of block n are there, and those of n - 2 are done with: three sets)
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        const int d_at = n * NG + q;
        wait_full(d_full, d_at, ND);
        ptx::tc_fence_after();
        const float scale = q4::scale_of<T>(word[q]), low = q4::low_of<T>(word[q]);
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + d_at % ND * NP + half * kCols;
        constexpr int kAtOnce = kCols < 32 ? kCols : 32;     // (a wait is for all loads, and takes as long for 32 columns as for 16)
#pragma unroll
        for (int c = 0; c < kCols; c += kAtOnce) {
          uint32_t d[kAtOnce];
          if constexpr (kAtOnce == 32) ptx::tc_ld_32x32(from + c, d); else tc_ld16(from + c, d);
          ptx::tc_wait_ld();
#pragma unroll
          for (int i = 0; i < kAtOnce; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(&xsum[n % kSums][q][half * kCols + c + i]);
            float2 &u = acc[(c + i) / 2], &v = acc[(c + i) / 2 + 1];
            fma2(u, low, x.x, x.y);
            fma2(v, low, x.z, x.w);
            fma2(u, scale, __uint_as_float(d[i]), __uint_as_float(d[i + 1]));
            fma2(v, scale, __uint_as_float(d[i + 2]), __uint_as_float(d[i + 3]));
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(bar(d_empty, d_at % ND));
      }
    }
  } else if (warp == kLoadWarp) {
    // ---- copies: codes run ahead of x by what their rings differ in depth
    constexpr int kLead = kR - kStages;
    const uint32_t* from = p.q + tile_at<G>(blockIdx.x * 8, k0, p.kblocks);
    for (int n = 0; n < blocks + kLead; ++n) {
      if (n < blocks) {
        wait_empty(raw_empty, n, kR);
        if (ptx::elect_one()) {
          ptx::mbar_arrive_expect_tx(bar(raw_full, n % kR), kRawBytes<G>);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(packed + n % kR * kRawBytes<G> + i * (kRawBytes<G> / 2)),
                         "l"(from + (int64_t)n * (8 * WTile<G>::kWords) + i * (4 * WTile<G>::kWords)), "r"(kRawBytes<G> / 2), "r"(bar(raw_full, n % kR)) : "memory");
        }
      }
      const int m = n - kLead;
      if (m >= 0) {
        wait_empty(empty, m, kStages);
        if (ptx::elect_one()) {
          ptx::mbar_arrive_expect_tx(bar(full, m % kStages), kX);
          ptx::tma_load_2d(xs + m % kStages * kX, &xmap, bar(full, m % kStages), (k0 + m) * 128, 0);
          ptx::tma_load_2d(xs + m % kStages * kX + NP * 128, &xmap, bar(full, m % kStages), (k0 + m) * 128 + 64, 0);
        }
      }
    }
  } else {
    constexpr uint32_t idesc = ptx::make_idesc_f16(std::is_same<T, __half>::value ? 0 : 1, 128, NP, 0, 0);
    const uint32_t el = ptx::elect_one() ? 1u : 0u;
    for (int n = 0; n < blocks; ++n) {
      wait_full(full, n, kStages);
      const uint32_t a = ptx::desc_lo(codes + n % kStages * kCodeBytes, 16), b = ptx::desc_lo(xs + n % kStages * kX, 16);
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        const int d_at = n * NG + q;
        wait_empty(d_empty, d_at, ND);
        ptx::tc_fence_after();
#pragma unroll
        for (int k = 0; k < 8 / NG; ++k) {          // 16 channels, 32 bytes of a swizzled row
          const int at = q * (8 / NG) + k;
          ptx::tc_mma_f16_if(el, tmem + d_at % ND * NP, a + (at >> 2) * (kManyRows * 128 >> 4) + (at & 3) * 2, b + (at >> 2) * (NP * 128 >> 4) + (at & 3) * 2, idesc, k != 0);
        }
        ptx::tc_commit_if(el, bar(d_full, d_at % ND));
      }
      ptx::tc_commit_if(el, bar(empty, n % kStages));
      __syncwarp();
    }
  }
  // ---- all products have been read: the ring's place holds the sums where a cluster shares the channels
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == kMmaWarp) ptx::tmem_dealloc(tmem, ND * NP);
  const bool sums = warp >= kExpand && warp < kLoadWarp;
  const int r = warp % 4 * 32 + lane, half = (warp - kExpand) / 4, n = blockIdx.x * kManyRows + r;
  T* y = reinterpret_cast<T*>(p.y);
  const float bias = p.bias && n < p.N ? rb::to_f(reinterpret_cast<const T*>(p.bias)[n]) : 0.f;
  if (p.splits == 1) {
    if (sums && n < p.N) {
#pragma unroll
      for (int i = 0; i < kCols; ++i)
        if (half * kCols + i < p.M) y[(half * kCols + i) * p.ldy + n] = rb::from_f<T>((i & 1 ? acc[i / 2].y : acc[i / 2].x) + bias);
    }
  } else {
    float* part = reinterpret_cast<float*>(raw + (base - ptx::smem_u32(raw)));    // [NP][128]
    if (sums) {
#pragma unroll
      for (int i = 0; i < kCols; ++i) part[(half * kCols + i) * kManyRows + r] = i & 1 ? acc[i / 2].y : acc[i / 2].x;
    }
    ptx::cluster_sync();
    // rows of x are dealt out to the cluster's blocks and their warps
    for (int i = threadIdx.x / kManyRows; i * p.splits + blockIdx.y < p.M; i += kManyThreads<NP> / kManyRows) {
      const int m = i * p.splits + blockIdx.y, c128 = threadIdx.x % kManyRows, out = blockIdx.x * kManyRows + c128;
      if (threadIdx.x >= kManyThreads<NP> / kManyRows * kManyRows) break;
      float v = p.bias && out < p.N ? rb::to_f(reinterpret_cast<const T*>(p.bias)[out]) : 0.f;
      for (int c = 0; c < p.splits; ++c) {
        uint32_t a;
        float f;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(base + (m * kManyRows + c128) * 4), "r"(c));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(a) : "memory");
        v += f;
      }
      if (out < p.N) y[m * p.ldy + out] = rb::from_f<T>(v);
    }
  }
  rb::report_given_up(dead, p.status);
  if (p.splits > 1) ptx::cluster_sync();              // nobody leaves while its sums are being read
}

template <typename T, int G, int NP> int many_rows(LinearParams p, cudaStream_t s) {
  static std::atomic<uint64_t> opted_in{0};           // the attribute is the kernel's on one device: a bit per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -3;
  if (dev >= 64 || !(opted_in.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(many_rows_kernel<T, G, NP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kManySmem<G, NP>) != cudaSuccess) return -3;
    if (dev < 64) opted_in.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  }
  CUtensorMap xmap;
  if (!make_tmap(&xmap, p.x, std::is_same<T, __nv_bfloat16>::value, p.M, p.K, p.ldx, 64, NP)) return -4;
  // Blocks of a cluster: the number whose rounds over the SMs, each a fixed part (about eight blocks' time) and its blocks of channels, take the least
  const int tiles = RB_CEIL_DIV(p.N, kManyRows);
  int64_t best = INT64_MAX;
  for (int c = 1; c <= kMaxSplits && c <= p.kblocks; ++c) {
    const int64_t cost = (int64_t)RB_CEIL_DIV(tiles * (int64_t)c, rb::kNumSMs) * (RB_CEIL_DIV(p.kblocks, c) + 8);
    if (cost < best) { best = cost; p.splits = c; }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles, p.splits);
  cfg.blockDim = dim3(kManyThreads<NP>);
  cfg.dynamicSmemBytes = kManySmem<G, NP>;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (p.splits > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = attr[n].val.clusterDim.z = 1;
    attr[n++].val.clusterDim.y = p.splits;
  }
  if (rb::pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, many_rows_kernel<T, G, NP>, xmap, p) == cudaSuccess ? 0 : -3;
}

template <typename T, int G> int run(const void* x, const void* q, const void* bias, void* y, int M, int N, int K, int64_t ldx, int64_t ldy, cudaStream_t s) {
  int* status = rb_attn_status();
  if (status == nullptr) return -5;
  for (int m0 = 0; m0 < M;) {
    const int rows = std::min(M - m0, 128);
    const LinearParams p{(const T*)x + m0 * ldx, bias, (const uint32_t*)q, (T*)y + m0 * ldy, rows, N, K, RB_CEIL_DIV(K, 128), 1, ldx, ldy, status, kMagic<T>};
    const int rc = rows <= 8 ? few_rows<T, G, 1>(p, s) : rows <= 16 ? few_rows<T, G, 2>(p, s) : rows <= 32 ? many_rows<T, G, 32>(p, s)
                                          : rows <= 64 ? many_rows<T, G, 64>(p, s) : many_rows<T, G, 128>(p, s);
    if (rc != 0) return rc;
    m0 += rows;
  }
  return 0;
}
template <typename T, int G> int quantize(const void* w, void* q, int N, int K, int64_t ld, cudaStream_t s) {
  return rb::launch_pdl(quantize_kernel<T, G>, dim3(RB_CEIL_DIV(N, 128) * 8, min(RB_CEIL_DIV(K, 128), 65535)), dim3(256), 0, s, (const T*)w, (uint32_t*)q, N, K, ld) ==
                 cudaSuccess ? 0 : -3;
}
template <int G> int pack(const void* codes, const void* scale, const void* low, void* q, int N, int K, cudaStream_t s) {
  return rb::launch_pdl(pack_kernel<G>, dim3(RB_CEIL_DIV(N, 128) * 8, min(RB_CEIL_DIV(K, 128), 65535)), dim3(256), 0, s, (const uint8_t*)codes, (const uint16_t*)scale,
                        (const uint16_t*)low, (uint32_t*)q, N, K) == cudaSuccess ? 0 : -3;
}

}  // namespace

// dt: 1 bf16, 2 fp16.  Rows of w and x on 16 bytes; K a multiple of the group.
extern "C" int rb_int4_quantize(const void* w, void* q, int N, int K, int64_t ld, int group, int dt, cudaStream_t s) {
  if (N == 0 || K == 0) return 0;
#define RB_G(T) (group == 32 ? quantize<T, 32>(w, q, N, K, ld, s) : group == 64 ? quantize<T, 64>(w, q, N, K, ld, s) : group == 128 ? quantize<T, 128>(w, q, N, K, ld, s) : -1)
  return dt == 1 ? RB_G(__nv_bfloat16) : dt == 2 ? RB_G(__half) : -2;
#undef RB_G
}

// codes [N, K] and steps and lowest values [N, K / group], contiguous; codes on 8 bytes
extern "C" int rb_int4_pack(const void* codes, const void* scale, const void* low, void* q, int N, int K, int group, cudaStream_t s) {
  if (N == 0 || K == 0) return 0;
  return group == 32 ? pack<32>(codes, scale, low, q, N, K, s) : group == 64 ? pack<64>(codes, scale, low, q, N, K, s) : group == 128 ? pack<128>(codes, scale, low, q, N, K, s) : -1;
}

extern "C" int rb_int4_linear(const void* x, const void* q, const void* bias, void* y, int M, int N, int K, int64_t ldx, int64_t ldy, int group, int dt, cudaStream_t s) {
  if (M == 0 || N == 0) return 0;
#define RB_G(T) \
  (group == 32 ? run<T, 32>(x, q, bias, y, M, N, K, ldx, ldy, s) : group == 64 ? run<T, 64>(x, q, bias, y, M, N, K, ldx, ldy, s) \
                                                                  : group == 128 ? run<T, 128>(x, q, bias, y, M, N, K, ldx, ldy, s) : -1)
  return dt == 1 ? RB_G(__nv_bfloat16) : dt == 2 ? RB_G(__half) : -2;
#undef RB_G
}
