// Products of a few rows with a weight held in 4 bits: y[m, n] = sum_k x[m, k] w[n, k] (+ bias[n]), w ~ scale c + low by groups of 32, 64 or 128 along K (int4.cuh).
//
// A weight is tiles of 16 output rows x 128 channels, the tiles of 16 rows one behind the other along K: weight words [row][t][j] of 128 channels,
// then the group words [row][group].  Rows beyond N and channels beyond K hold codes, scales and lowest values of 0.
//
// Few rows (up to 16): a block of eight warps has 32 output rows, its warps walk along K in blocks of 128 channels, one in eight each, and add their sums up at the end; where that
// leaves SMs idle, the blocks of a cluster share K.  Codes become exact 16-bit numbers (a mask that leaves a code in the low bits of 128 or 1024, and a subtraction) and are the
// left operand, 16 output rows at a time; rows of x, read from L2 and L1 as the operands' lanes want them, are the right one, eight at a time.  Scale and lowest value stay out: a
// group's product is scaled in fp32 when its channels are through, and the lowest value times the sum of x over the group (one more product, with ones) is added.
#include "gemm_common.cuh"
#include "int4.cuh"

#include <algorithm>

namespace {

constexpr int kFewWarps = 8, kFewThreads = kFewWarps * 32, kFewRows = 32;
constexpr int kMaxSplits = 8;      // blocks of a portable cluster

template <int G> struct WTile {
  static constexpr int kGroups = 128 / G, kWords = 16 * 16 + 16 * kGroups;
};

template <typename T, int G>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ w, uint32_t* __restrict__ q, int N, int K, int64_t ld) {
  const int r = threadIdx.x / 16, sub = threadIdx.x % 16, n = blockIdx.x * 16 + r, kblocks = RB_CEIL_DIV(K, 128);
  rb::pdl_trigger();
  rb::pdl_wait();
  for (int kb = blockIdx.y; kb < kblocks; kb += gridDim.y) {
    const int k = kb * 128 + sub * 8;
    const bool mine = n < N && k < K;
    rb::Pack<T, 8> a{};
    if (mine) a = *reinterpret_cast<const rb::Pack<T, 8>*>(w + n * ld + k);
    float x[8], lo, hi;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = rb::to_f(a.v[i]);
    q4::extremes<G / 8>(x, lo, hi);
    const uint32_t g = mine ? q4::group_word<T>(lo, hi) : 0u;
    uint32_t* at = q + ((int64_t)blockIdx.x * kblocks + kb) * WTile<G>::kWords;
    at[r * 16 + q4::word_place<4>(sub)] = mine ? q4::pack8<q4::kWeight>(x, q4::scale_of<T>(g), lo) : 0u;
    if (sub % (G / 8) == 0) at[256 + r * WTile<G>::kGroups + sub / (G / 8)] = g;
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
template <typename T> constexpr uint32_t kOnes = std::is_same<T, __half>::value ? 0x3c003c00u : 0x3f803f80u;

// The codes of a word as pairs of neighbouring channels of type T, exact.
template <typename T> RB_DEVICE void expand(uint32_t w, uint32_t (&h)[4]) {
  if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = (i < 2 ? w : w >> 8) & (i & 1 ? 0x00f000f0u : 0x000f000fu) | 0x64006400u;       // 1024 + c, or 1024 + 16 c
      const __half2 x = *reinterpret_cast<const __half2*>(&u);
      const __half2 y = i & 1 ? __hfma2(x, __float2half2_rn(0.0625f), __float2half2_rn(-64.f)) : __hadd2(x, __float2half2_rn(-1024.f));
      h[i] = *reinterpret_cast<const uint32_t*>(&y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = w >> (4 * i) & 0x000f000fu | 0x43004300u;                                       // 128 + c
      const __nv_bfloat162 y = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&u), __float2bfloat162_rn(-128.f));
      h[i] = *reinterpret_cast<const uint32_t*>(&y);
    }
  }
}

struct LinearParams {
  const void *x, *bias;
  const uint32_t* q;
  void* y;
  int M, N, K, kblocks, tiles, splits;
  int64_t ldx, ldy;
};

RB_DEVICE uint4 load_stream(const uint32_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// One block of 128 channels of 16 rows: a lane's words of rows g and g + 8, and their groups'.
template <int G> struct Block {
  uint32_t w[2][4], g[2][128 / G];
  RB_DEVICE void load(const uint32_t* tile, int lane) {
    const int r = lane >> 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 v = load_stream(tile + h * 128 + lane * 4);
      w[h][0] = v.x; w[h][1] = v.y; w[h][2] = v.z; w[h][3] = v.w;
#pragma unroll
      for (int i = 0; i < 128 / G; ++i) g[h][i] = __ldg(tile + 256 + (r + 8 * h) * (128 / G) + i);
    }
  }
};

// NT: sets of eight rows of x
template <typename T, int G, int NT>
__global__ void __launch_bounds__(kFewThreads) few_rows_kernel(const LinearParams p) {
  constexpr int MT = kFewRows / 16, NG = 128 / G;
  __shared__ __align__(16) float sums[kFewWarps][NT * 8][kFewRows + 1];
  __shared__ float part[NT * 8][kFewRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  rb::pdl_trigger();
  const int tile0 = blockIdx.x * MT, step = kFewWarps * p.splits, first = blockIdx.y * kFewWarps + warp;
  const uint32_t* tile[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) tile[i] = p.q + (int64_t)min(tile0 + i, p.tiles - 1) * p.kblocks * WTile<G>::kWords;
  rb::pdl_wait();
  Block<G> next[MT];
  if (first < p.kblocks)
#pragma unroll
    for (int i = 0; i < MT; ++i) next[i].load(tile[i] + (int64_t)first * WTile<G>::kWords, lane);
  float acc[MT][NT][4] = {};
  const T* x = reinterpret_cast<const T*>(p.x);
  for (int kb = first; kb < p.kblocks; kb += step) {
    Block<G> cur[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) cur[i] = next[i];
    uint4 xv[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = n * 8 + g, k = kb * 128 + 32 * j + 8 * t;
        xv[n][j] = m < p.M && k < p.K ? *reinterpret_cast<const uint4*>(x + m * p.ldx + k) : make_uint4(0, 0, 0, 0);
      }
    if (kb + step < p.kblocks)
#pragma unroll
      for (int i = 0; i < MT; ++i) next[i].load(tile[i] + (int64_t)(kb + step) * WTile<G>::kWords, lane);
#pragma unroll
    for (int q = 0; q < NG; ++q) {                  // a group
      float c[MT][NT][4] = {}, one[NT][4] = {};
#pragma unroll
      for (int j = q * 4 / NG; j < (q + 1) * 4 / NG; ++j) {
        uint32_t e0[MT][4], e1[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          expand<T>(cur[i].w[0][j], e0[i]);
          expand<T>(cur[i].w[1][j], e1[i]);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint32_t b0 = s ? xv[n][j].z : xv[n][j].x, b1 = s ? xv[n][j].w : xv[n][j].y;
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
      for (int e = 0; e < 4; ++e) sums[warp][n * 8 + 2 * t + (e & 1)][i * 16 + g + 8 * (e >> 1)] = acc[i][n][e];
  __syncthreads();
  const int cols = min(p.M, NT * 8);
  auto finish = [&](int m, int r, float v) {
    const int n = blockIdx.x * kFewRows + r;
    if (n < p.N) reinterpret_cast<T*>(p.y)[m * p.ldy + n] = rb::from_f<T>(v + (p.bias ? rb::to_f(reinterpret_cast<const T*>(p.bias)[n]) : 0.f));
  };
  for (int i = threadIdx.x; i < cols * kFewRows; i += kFewThreads) {
    const int m = i / kFewRows, r = i % kFewRows;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) v += sums[w][m][r];
    if (p.splits == 1) finish(m, r, v); else part[m][r] = v;
  }
  if (p.splits == 1) return;
  ptx::cluster_sync();
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
  ptx::cluster_sync();  // nobody leaves while its sums are being read
}

template <typename T, int G, int NT> int few_rows(LinearParams p, cudaStream_t s) {
  const int blocks = RB_CEIL_DIV(p.N, kFewRows);
  p.splits = 1;
  while (p.splits < kMaxSplits && blocks * p.splits * 2 <= 2 * rb::kNumSMs && p.kblocks >= kFewWarps * p.splits * 2) p.splits *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks, p.splits);
  cfg.blockDim = dim3(kFewThreads);
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

template <typename T, int G> int run(const void* x, const void* q, const void* bias, void* y, int M, int N, int K, int64_t ldx, int64_t ldy, cudaStream_t s) {
  for (int m0 = 0; m0 < M; m0 += 16) {
    const LinearParams p{(const T*)x + m0 * ldx, bias, (const uint32_t*)q, (T*)y + m0 * ldy, std::min(M - m0, 16), N, K, RB_CEIL_DIV(K, 128), RB_CEIL_DIV(N, 16), 1, ldx, ldy};
    const int rc = p.M <= 8 ? few_rows<T, G, 1>(p, s) : few_rows<T, G, 2>(p, s);
    if (rc != 0) return rc;
  }
  return 0;
}
template <typename T, int G> int quantize(const void* w, void* q, int N, int K, int64_t ld, cudaStream_t s) {
  return rb::launch_pdl(quantize_kernel<T, G>, dim3(RB_CEIL_DIV(N, 16), min(RB_CEIL_DIV(K, 128), 65535)), dim3(256), 0, s, (const T*)w, (uint32_t*)q, N, K, ld) ==
                 cudaSuccess ? 0 : -3;
}

}  // namespace

// dt: 1 bf16, 2 fp16.  Rows of w and x on 16 bytes; K a multiple of the group.
extern "C" int rb_int4_quantize(const void* w, void* q, int N, int K, int64_t ld, int group, int dt, cudaStream_t s) {
  if (N == 0 || K == 0) return 0;
#define RB_G(T) (group == 32 ? quantize<T, 32>(w, q, N, K, ld, s) : group == 64 ? quantize<T, 64>(w, q, N, K, ld, s) : group == 128 ? quantize<T, 128>(w, q, N, K, ld, s) : -1)
  return dt == 1 ? RB_G(__nv_bfloat16) : dt == 2 ? RB_G(__half) : -2;
#undef RB_G
}

extern "C" int rb_int4_linear(const void* x, const void* q, const void* bias, void* y, int M, int N, int K, int64_t ldx, int64_t ldy, int group, int dt, cudaStream_t s) {
  if (M == 0 || N == 0) return 0;
#define RB_G(T) \
  (group == 32 ? run<T, 32>(x, q, bias, y, M, N, K, ldx, ldy, s) : group == 64 ? run<T, 64>(x, q, bias, y, M, N, K, ldx, ldy, s) \
                                                                  : group == 128 ? run<T, 128>(x, q, bias, y, M, N, K, ldx, ldy, s) : -1)
  return dt == 1 ? RB_G(__nv_bfloat16) : dt == 2 ? RB_G(__half) : -2;
#undef RB_G
}
