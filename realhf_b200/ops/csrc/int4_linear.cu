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
//   Bound: the weight's bytes.  1 x 4096 x 4096 takes 4.7 us (floor 1.4; 16-bit weights 9.8): launch, first bytes and the last sum.  7 x 1024 x 50257 in groups of 32 takes 13.7
//   (floor 5.0; 27), 16 x 4096 x 22016 24.6 (floor 7.4; 30) and in groups of 32 29.1: copies of 2 KB alone stream 3.3 .. 3.6 TB/s, and products, arithmetic and loads of x fill a third to a
//   half of their pipes each, one after the other in a warp; two of the six products of 16 channels of 16 rows are the sums of x, which each set of 32 output rows forms anew.  Sets dealt
//   out in halves, so that no block has more than others, changed nothing: an SM's two blocks even it out.
// More rows: a block has 128 output rows and all rows of x (in pieces of 128), and the products run on tcgen05.  Teams of four warps turn a block of 128 channels of codes into an
// operand in tensor memory: scale (c - 8) as two numbers of the type, exact, so that one accumulator takes all channels (c - 8 and not c: sums of codes that are all positive would leave
// the accumulator's last places to cancel).  Rows of x come by TMA, one warp issues the products, four warps sum x over the groups (products with ones), and eight add up what is left,
// (lowest value + 8 scale) times those sums, eight output rows and some columns a thread.
//   Bound: none alone.  128 x 11008 x 4096 in groups of 64 takes 36 us (floor 7.2; the 16-bit product 21.3), 64 rows 22.7 (19.3), 32 rows 20.3 (18.4): chains of waits (operands,
//   products, sums, lowest values) of about the same length a block of channels; with half of the products left out 128 rows took 35, with a quarter of the codes expanded 35.  An
//   accumulator a group, scaled out of tensor memory, took 45 (58 in groups of 32, now 39): a group's 64 KB leave tensor memory and its sums of x shared memory at 128 bytes a clock each.
//   The two parts in shared memory took 45 .. 53: 275 KB a block through it.  Sums of x by the lowest values' warps took 25.3 with 64 rows and 22.1 with 32.
// So a weight in 4 bits takes less time than one in 16 up to 16 rows and more beyond (17 rows of 4096 -> 11008 23.8 us against 17.9, of 11008 -> 4096 18.7 against 18.0); it saves memory
// where no 16-bit weight is kept beside it.
//
// Codes and rows are summed over a group before the step goes in: 15 x 128 numbers of a row have to stay inside fp32, so bf16's up to 1e35 do.  A row that holds an infinity or a NaN gives
// numbers that are not finite, which ones is not said (sums that cancel, channels of padding that read the row's first ones against codes of 0).
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
// A warp's ring of blocks on their way, 2176 to 2560 bytes each (registers hold one ahead, and 35 KB an SM were on their way: 2.1 TB/s at any number of rows): four, or three where four would
// leave an SM one block of threads (16 rows in groups of 32)
template <int G> constexpr int kFewBytes = kFewRows / 16 * WTile<G>::kWords * 4;
template <int NT> constexpr size_t kFewSums = 2 * kFewWarps * NT * 8 * (kFewRows + 1) * 4 + NT * 8 * kFewRows * 4;     // a tile of rows' sums and the next one's; a block's
template <int G, int NT, int kRing> constexpr bool kTwoFit = 2 * (kFewWarps * kRing * (kFewBytes<G> + 8) + kFewSums<NT> + 1024 + 64) <= 228 * 1024;
template <int G, int NT> constexpr int kFewRing = kTwoFit<G, NT, 4> ? 4 : 3;
template <int G, int NT> constexpr size_t kFewSmem = kFewWarps * kFewRing<G, NT> * kFewBytes<G>;

// NT: sets of eight rows of x
template <typename T, int G, int NT>
__global__ void __launch_bounds__(kFewThreads, 2) few_rows_kernel(const LinearParams p) {
  constexpr int MT = kFewRows / 16, NG = 128 / G, kRing = kFewRing<G, NT>;
  static_assert(kTwoFit<G, NT, kRing>, "the grid and the splits count on two blocks an SM");
  extern __shared__ __align__(128) unsigned char few_ring[];
  __shared__ __align__(16) float sums[2][kFewWarps][NT * 8][kFewRows + 1];    // (of a tile of rows and of the next: a warp may be that far ahead)
  __shared__ float part[NT * 8][kFewRows];
  __shared__ __align__(8) uint64_t bar[kFewWarps][kRing];
  __shared__ uint32_t dead_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  volatile uint32_t* dead = &dead_flag;
  if (threadIdx.x == 0) *dead = 0;
  if (lane < kRing) ptx::mbar_init(ptx::smem_u32(&bar[warp][lane]), 1);
  ptx::fence_barrier_init();
  __syncthreads();
  rb::pdl_trigger();
  // the warp's blocks of a set of 32 output rows, then those of the next set of this block of threads: one sequence, whose copies run ahead of the sums at a set's end
  const int step = kFewWarps * p.splits, first = blockIdx.y * kFewWarps + warp, sets = RB_CEIL_DIV(p.N, kFewRows);
  const uint32_t ring = ptx::smem_u32(few_ring) + warp * (kRing * kFewBytes<G>);
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
  for (int i = 0; i < kRing; ++i) fetch(i);
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
    if (++slot == kRing) { slot = 0; round ^= 1; }
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
    if (cudaFuncSetAttribute(few_rows_kernel<T, G, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFewSmem<G, NT>) != cudaSuccess) return -3;
    if (dev < 64) opted_in.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  }
  const int sets = RB_CEIL_DIV(p.N, kFewRows), blocks = std::min(sets, 2 * rb::kNumSMs);
  p.splits = 1;
  while (p.splits < kMaxSplits && sets * p.splits * 2 <= 2 * rb::kNumSMs && p.kblocks >= kFewWarps * p.splits * 2) p.splits *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks, p.splits);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = kFewSmem<G, NT>;
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

constexpr int kManyRows = 128, kTeam = 4, kLows = 8;                                 // output rows; warps of a team that expands, a quarter of the rows each; of the lowest values
template <int NP> constexpr int kTeams = NP == 128 ? 1 : 3;                          // teams: every third block each (32 rows 19.5 us, with two 20.5), or one, whose registers the lowest
                                                                                     // values' sums of 128 rows need (39 us for groups of 32, with two 51)
constexpr int kSumWarps = 4;                                                         // warps of the sums of x
template <int NP> constexpr int kManyThreads = (kTeams<NP> * kTeam + kLows + kSumWarps + 2) * 32;
constexpr int kWStages = 3, kWCols = 128;                                            // operand tiles in tensor memory; 64 columns of the larger parts, 64 of the smaller ones
template <int NP> constexpr int kXStages = NP == 128 ? 4 : 6;                        // blocks of x in shared memory
constexpr int kRaw = 6;                                                              // blocks of packed codes, 9 or 10 KB each
template <int G> constexpr int kRawBytes = 8 * WTile<G>::kWords * 4;
template <int G, int NP> constexpr size_t kManySmem = 1024 + kXStages<NP> * NP * 256 + kRaw * kRawBytes<G>;

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

// The numbers c - 8 of a word, as pairs of neighbouring channels of type T
template <typename T> RB_DEVICE void expand_centred(uint32_t w, uint32_t (&h)[4], uint32_t magic) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value) {
      const uint32_t u = (i < 2 ? w : w >> 8) & (i & 1 ? 0x00f000f0u : 0x000f000fu) | magic;       // 1024 + c, or 1024 + 16 c
      const __half2 x = *reinterpret_cast<const __half2*>(&u);
      const __half2 y = i & 1 ? __hfma2(x, __float2half2_rn(0.0625f), __float2half2_rn(-72.f)) : __hadd2(x, __float2half2_rn(-1032.f));
      h[i] = *reinterpret_cast<const uint32_t*>(&y);
    } else {
      const uint32_t u = w >> (4 * i) & 0x000f000fu | magic;                                       // 128 + c
      const __nv_bfloat162 y = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&u), __float2bfloat162_rn(-136.f));
      h[i] = *reinterpret_cast<const uint32_t*>(&y);
    }
  }
}
// scale * e as two numbers of T whose sum it is: a product, and what its rounding left (scale has 8 or 11 bits and e = c - 8 three, or is a power of two, so that fits).  Steps beyond
// an eighth of T's largest number could overflow: there the larger part is half of it, and the smaller one is off by half a step of T at most.
template <typename T> struct Step {
  uint32_t all, first;
  RB_DEVICE explicit Step(uint32_t group) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    all = __byte_perm(group, 0, 0x3232);
    first = (all & 0x7fffu) > (kHalf ? 0x6fffu : 0x7dffu) ? all - (kHalf ? 0x04000400u : 0x00800080u) : all;
  }
  RB_DEVICE void parts(uint32_t e, uint32_t& hi, uint32_t& lo) const {
    if constexpr (std::is_same<T, __half>::value) {
      const __half2 x = *reinterpret_cast<const __half2*>(&e), h = __hmul2_rn(*reinterpret_cast<const __half2*>(&first), x);
      const __half2 l = __hfma2(*reinterpret_cast<const __half2*>(&all), x, __hneg2(h));
      hi = *reinterpret_cast<const uint32_t*>(&h), lo = *reinterpret_cast<const uint32_t*>(&l);
    } else {
      const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&e), h = __hmul2_rn(*reinterpret_cast<const __nv_bfloat162*>(&first), x);
      const __nv_bfloat162 l = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&all), x, __hneg2(h));
      hi = *reinterpret_cast<const uint32_t*>(&h), lo = *reinterpret_cast<const uint32_t*>(&l);
    }
  }
};
template <int N> RB_DEVICE void words_of(uint32_t at, uint32_t (&w)[N]) {
  if constexpr (N == 4) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
  else if constexpr (N == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
  else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(at) : "memory");
}

// NP: rows of x, padded (rows beyond M read as zeros)
template <typename T, int G, int NP>
__global__ void __launch_bounds__(kManyThreads<NP>, 1) many_rows_kernel(const __grid_constant__ CUtensorMap xmap, const LinearParams p) {
  constexpr int NG = 128 / G, kX = NP * 256, kXS = kXStages<NP>, kR = kRaw, kSums = 4, kTms = kTeams<NP>;
  constexpr int kExpand = kTms * kTeam, kSumWarp = kExpand + kLows, kLoadWarp = kSumWarp + kSumWarps, kMmaWarp = kLoadWarp + 1;
  constexpr int kRows = 8, kCols = NP / 16;            // a thread's sums of the lowest values: rows, columns
  // A parity tells a round from the one before it, not from the one two before.  A warp that takes every k-th block knows that the block k before has come (its sums are used, or its
  // product done), so a ring that it waits on has at least k places, or as many as there are teams that take turns.
  static_assert(kXS >= kSumWarps && kR >= kSumWarps && kSums >= kSumWarps, "a warp of the sums of x could take the round before last for its own");
  static_assert(kWStages >= kTms && kR >= kTms, "a team could take the round before last for its own");
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t w_full[kWStages], w_empty[kWStages], x_full[kXS], x_empty[kXS], raw_full[kR], raw_empty[kR], s_full[kSums], s_empty[kSums], done;
  __shared__ __align__(16) float xsum[kSums][NG][NP], lows[kSums][NG][kManyRows];
  __shared__ uint32_t tmem_ptr, dead_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile uint32_t* dead = &dead_flag;
  const uint32_t base = (ptx::smem_u32(raw) + 1023u) & ~1023u, xs = base, packed = xs + kXS * kX;
  auto bar = [](uint64_t* b, int i) { return ptx::smem_u32(&b[i]); };
  // ring slot n % size, in its (n / size)-th round: what fills it waits for the other parity
  auto wait_full = [&](uint64_t* b, int n, int size) { bounded_wait(ptx::smem_u32(&b[n % size]), n / size & 1, dead); };
  auto wait_empty = [&](uint64_t* b, int n, int size) { bounded_wait(ptx::smem_u32(&b[n % size]), (n / size & 1) ^ 1, dead); };
  if (threadIdx.x == 0) {
    *dead = 0;
    for (int i = 0; i < kWStages; ++i) {
      ptx::mbar_init(bar(w_full, i), kTeam);
      ptx::mbar_init(bar(w_empty, i), 1);
    }
    for (int i = 0; i < kXS; ++i) {
      ptx::mbar_init(bar(x_full, i), 1);
      ptx::mbar_init(bar(x_empty, i), 2);              // the products, and the sums
    }
    for (int i = 0; i < kR; ++i) {
      ptx::mbar_init(bar(raw_full, i), 1);
      ptx::mbar_init(bar(raw_empty, i), kTeam + 1);
    }
    for (int i = 0; i < kSums; ++i) {
      ptx::mbar_init(bar(s_full, i), 1);
      ptx::mbar_init(bar(s_empty, i), kLows);
    }
    ptx::mbar_init(bar(&done, 0), 1);
    ptx::fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(ptx::smem_u32(&tmem_ptr), 512);    // sums in columns 0 .. NP - 1, operand tiles from 128 on
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
  float* part = reinterpret_cast<float*>(raw + (base - ptx::smem_u32(raw)));    // [NP][128]: the block's sums, in the place of x once all products are done

  if (warp < kExpand) {
    // ---- codes to operands in tensor memory: a lane has a row, whose 16 words it reads in an order that depends on the lane (eight lanes meet all banks) and puts right again
    const int quarter = warp % 4, team = warp / kTeam, row = quarter * 32 + lane, turn = lane >> 1 & 3;
    const uint32_t into = tmem + ((uint32_t)(quarter * 32) << 16) + 128;
    for (int n = team; n < blocks; n += kTms) {
      wait_full(raw_full, n, kR);
      const uint32_t tile = packed + n % kR * kRawBytes<G> + (row >> 4) * (WTile<G>::kWords * 4);
      uint32_t w[4][4], group[NG];                     // [t][j]
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 v = ld_shared_v4(tile + (row & 15) * 64 + ((i + turn) & 3) * 16);
        w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
      }
      words_of(tile + 1024 + (row & 15) * (NG * 4), group);
#pragma unroll
      for (int j = 0; j < 4; ++j) {                    // w[i] holds piece i + turn: turned on by two and by one
        const uint32_t a0 = turn & 2 ? w[2][j] : w[0][j], a1 = turn & 2 ? w[3][j] : w[1][j], a2 = turn & 2 ? w[0][j] : w[2][j], a3 = turn & 2 ? w[1][j] : w[3][j];
        w[0][j] = turn & 1 ? a3 : a0, w[1][j] = turn & 1 ? a0 : a1, w[2][j] = turn & 1 ? a1 : a2, w[3][j] = turn & 1 ? a2 : a3;
      }
      wait_empty(w_empty, n, kWStages);
      ptx::tc_fence_after();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Step<T> step(group[j * NG / 4]);
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          uint32_t e[4];
          expand_centred<T>(w[t][j], e, p.magic);
#pragma unroll
          for (int i = 0; i < 4; ++i) step.parts(e[i], hi[4 * t + i], lo[4 * t + i]);
        }
        ptx::tc_st_32x16(into + n % kWStages * kWCols + j * 16, hi);
        ptx::tc_st_32x16(into + n % kWStages * kWCols + 64 + j * 16, lo);
      }
      ptx::tc_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(bar(w_full, n % kWStages));
        ptx::mbar_arrive(bar(raw_empty, n % kR));
      }
    }
  } else if (warp < kSumWarp) {
    // ---- lowest values times sums of x, added up in registers: a thread has eight rows and some columns, so that what it reads serves several products
    const int tid = (warp - kExpand) * 32 + lane;
    const int row0 = tid % 16 * kRows, col0 = tid / 16 * kCols;
    float2 acc[kRows][kCols / 2];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int c = 0; c < kCols / 2; ++c) acc[r][c] = make_float2(0.f, 0.f);
#pragma unroll 1
    for (int n = 0; n < blocks; ++n) {
      wait_full(s_full, n, kSums);
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        float2 x[kCols / 2];
#pragma unroll
        for (int c = 0; c < kCols / 2; ++c) x[c] = *reinterpret_cast<const float2*>(&xsum[n % kSums][q][col0 + 2 * c]);
#pragma unroll
        for (int r = 0; r < kRows; r += 4) {
          const float4 v = *reinterpret_cast<const float4*>(&lows[n % kSums][q][row0 + r]);
          const float low[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < kCols / 2; ++c) fma2(acc[r + i][c], low[i], x[c].x, x[c].y);
        }
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar(s_empty, n % kSums));
    }
    if (blocks > 0) bounded_wait(bar(&done, 0), 0, dead);
    ptx::tc_fence_after();
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int r = 0; r < kRows; r += 4) {
        auto of = [&](int i) { return c & 1 ? acc[r + i][c / 2].y : acc[r + i][c / 2].x; };
        *reinterpret_cast<float4*>(&part[(col0 + c) * kManyRows + row0 + r]) = make_float4(of(0), of(1), of(2), of(3));
      }
    asm volatile("bar.sync 1, %0;" ::"n"(kLows * 32) : "memory");
    // ---- and the products: a warp has 32 rows, a quarter of the lanes of tensor memory, and half of the columns
    if (blocks > 0) {
      const int quarter = warp % 4, half = (warp - kExpand) / 4;
#pragma unroll 1
      for (int c = half * (NP / 2); c < (half + 1) * (NP / 2); c += 16) {
        uint32_t d[16];
        tc_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + c, d);
        ptx::tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(c + i) * kManyRows + quarter * 32 + lane] += __uint_as_float(d[i]);
      }
      ptx::tc_fence_before();
    }
  } else if (warp < kLoadWarp) {
    // ---- a block's sums of x over its groups, products with ones 16 rows at a time, and its lowest values: every fourth block a warp
    for (int n = warp - kSumWarp; n < blocks; n += kSumWarps) {
      wait_empty(s_empty, n, kSums);
      wait_full(x_full, n, kXS);
#pragma unroll 4
      for (int rows = 0; rows < NP; rows += 16) {
        const int r = rows + (lane & 15);
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          float c[4] = {};
#pragma unroll
          for (int k = q * (8 / NG); k < (q + 1) * (8 / NG); ++k) {
            const int piece = 2 * k + (lane >> 4);
            uint32_t a[4];
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                         : "r"(xs + n % kXS * kX + (piece >> 3) * (NP * 128) + r * 128 + (((piece & 7) ^ (r & 7)) << 4)) : "memory");
            mma16<T>(c, a[0], a[1], a[2], a[3], kOnes<T>, kOnes<T>);
          }
          if ((lane & 3) == 0) {
            xsum[n % kSums][q][rows + (lane >> 2)] = c[0];
            xsum[n % kSums][q][rows + (lane >> 2) + 8] = c[2];
          }
        }
      }
      wait_full(raw_full, n, kR);
#pragma unroll
      for (int row = lane; row < kManyRows; row += 32) {        // (the products are of c - 8)
        uint32_t word[NG];
        words_of(packed + n % kR * kRawBytes<G> + (row >> 4) * (WTile<G>::kWords * 4) + 1024 + (row & 15) * (NG * 4), word);
#pragma unroll
        for (int q = 0; q < NG; ++q) lows[n % kSums][q][row] = fmaf(8.f, q4::scale_of<T>(word[q]), q4::low_of<T>(word[q]));
      }
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(bar(s_full, n % kSums));
        ptx::mbar_arrive(bar(x_empty, n % kXS));
        ptx::mbar_arrive(bar(raw_empty, n % kR));
      }
    }
  } else if (warp == kLoadWarp) {
    // ---- copies
    const uint32_t* from = p.q + tile_at<G>(blockIdx.x * 8, k0, p.kblocks);
    constexpr int kLead = kR > kXS ? kR - kXS : 0;       // codes run ahead of x by what their rings differ in depth
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
        wait_empty(x_empty, m, kXS);
        if (ptx::elect_one()) {
          ptx::mbar_arrive_expect_tx(bar(x_full, m % kXS), kX);
          ptx::tma_load_2d(xs + m % kXS * kX, &xmap, bar(x_full, m % kXS), (k0 + m) * 128, 0);
          ptx::tma_load_2d(xs + m % kXS * kX + NP * 128, &xmap, bar(x_full, m % kXS), (k0 + m) * 128 + 64, 0);
        }
      }
    }
  } else {
    constexpr uint32_t idesc = ptx::make_idesc_f16(std::is_same<T, __half>::value ? 0 : 1, 128, NP, 0, 0);
    const uint32_t el = ptx::elect_one() ? 1u : 0u;
    for (int n = 0; n < blocks; ++n) {
      wait_full(w_full, n, kWStages);
      wait_full(x_full, n, kXS);
      ptx::tc_fence_after();
      const uint32_t a = tmem + 128 + n % kWStages * kWCols, b = ptx::desc_lo(xs + n % kXS * kX, 16);
#pragma unroll
      for (int k = 0; k < 8; ++k)                     // 16 channels: eight columns of a part, 32 bytes of a swizzled row of x
#pragma unroll
        for (int half = 0; half < 2; ++half)
          ptx::tc_mma_f16_ts_if(el, tmem, a + half * 64 + k * 8, b + (k >> 2) * (NP * 128 >> 4) + (k & 3) * 2, idesc, n + k + half != 0);
      ptx::tc_commit_if(el, bar(w_empty, n % kWStages));
      ptx::tc_commit_if(el, bar(x_empty, n % kXS));
      __syncwarp();
    }
    if (blocks > 0) ptx::tc_commit_if(el, bar(&done, 0));
    __syncwarp();
  }
  // ---- the block's sums lie in shared memory; a cluster's are added up, rows of x dealt out to its blocks and their warps
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == kMmaWarp) ptx::tmem_dealloc(tmem, 512);
  if (p.splits > 1) ptx::cluster_sync();
  T* y = reinterpret_cast<T*>(p.y);
  constexpr int kPasses = kManyThreads<NP> / kManyRows;
  const int r = threadIdx.x % kManyRows, n = blockIdx.x * kManyRows + r;
  if (threadIdx.x < kPasses * kManyRows && n < p.N) {
    const float bias = p.bias ? rb::to_f(reinterpret_cast<const T*>(p.bias)[n]) : 0.f;
    for (int m = threadIdx.x / kManyRows * p.splits + blockIdx.y; m < p.M; m += kPasses * p.splits) {
      float v = bias;
      if (p.splits == 1) {
        v += part[m * kManyRows + r];
      } else {
        for (int c = 0; c < p.splits; ++c) {
          uint32_t at;
          float f;
          asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(base + (m * kManyRows + r) * 4), "r"(c));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(at) : "memory");
          v += f;
        }
      }
      y[m * p.ldy + n] = rb::from_f<T>(v);
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
  // (4096 x 11008 in groups of 128: 16 rows 15 us with few rows' kernel, 20 with the other; 32 rows take two passes of the former, one of 19 of the latter)
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
