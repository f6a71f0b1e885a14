// Language-model head with token statistics in its epilogue: logits X = h W^T (h [T, H], W [V, H], 16 bits, fp32 accumulators) never leave the chip.
//
// Forward: a CTA pair forms a 256 x 256 tile of X (tcgen05.mma.cta_group::2, operands by TMA, two accumulators in tensor memory); while the next tile is multiplied, eight
// warps a CTA read theirs, a lane a row of 128 columns, and leave three numbers: maximum, sum and weighted sum (vocab_rows.cuh).  A second kernel merges a row's V / 128
// triples.  Logits are what fp32 accumulators hold; stored in bf16 they would move a log-probability by up to 2^-8 of the logit.
// Backward: d logits, in 16 bits (rounded once) as operand of the products for d h and d W, from the row's log-sum-exp and entropy, either
//   from the product formed again, in its epilogue (2 T V H more operations, no memory), or
//   from the weights e^{x - m} that the forward pass kept, m the maximum of the lane's 128 columns, as fp16 times 2^15: 11 bits for weights down to 2^-29, so that what is kept is
//   rounded by an eighth of what d logits in bf16 are (T V more numbers of 16 bits between the passes).
// `rounded`: each accumulator is rounded to the operands' type first, in both passes, so that log-probabilities are those of stored logits (a ratio of two has to be of one kind).
// In fp16 d logits are stored times a power of two that a bound of all of them gives (vocab_rows.cuh, grad_scale), and both products are taken back from it in fp32, in their epilogues
// where their sum is whole: with row gradients of 1 / T nearly all of them lie below fp16's smallest number.
// d h with few tiles: the sum over the vocabulary in parts, fp32 tiles that a second kernel adds up in order (16 rows of 4096 x 32000: 167 us undivided).
// An epilogue takes 32768 exponentials a CTA, 2048 cycles at least, beside 8 H cycles of products.
// 8192 x 4096 x 32000 bf16, us: forward 1320 .. 1350 (the plain product 1320 .. 1400), 1390 .. 1405 with kept weights, d logits 181 .. 206 from them, 1370 .. 1385 from the product.  fp16: d weight 1570 (the general
// product 1563), d hidden 1514 (1520); the bound of d logits 5 us for 2048 rows.
#include "attn_common.cuh"
#include "cta_pair.cuh"
#include "vocab_rows.cuh"

#include <type_traits>

namespace {

constexpr int HN = 256;                                     // logits of a tile
constexpr int kHeadStages = 6;
constexpr int kHeadA = BM * BK * 2, kHeadB = HN / 2 * BK * 2, kHeadStage = kHeadA + kHeadB;
constexpr int kEpiWarps = 8, kHeadThreads = 64 + 32 * kEpiWarps;
constexpr int kHeadOut = kHeadStages * kHeadStage, kHeadBars = kHeadOut + kEpiWarps * 4096, kHeadSmem = kHeadBars + 1024 + 256;
constexpr int kHeadBand = 8;                                // row tiles walked together, so that the tiles in flight share operands in L2

struct HeadParams {
  int M, N, K;
  float inv_temp;
  const int64_t* labels;
  const uint8_t* mask;
  int64_t mask_stride;
  // forward: [2 tiles_n, M] each, and the label's logit [M]
  float *part_m, *part_s, *part_w, *target;
  // backward
  const float *lse, *entropy, *g_logp, *g_entropy;
  const uint32_t* peak; // fp16: d logits leave times grad_scale of it; null: as they are
  void* out;
  int64_t ld_out;
  int splits;           // d hidden: parts of the sum over the vocabulary, out fp32 [splits, M, N]
  int direct, add;      // gradients of hidden states and weight straight into `out`, over grad_scale: 1 of the operands' type, 2 fp32; add: to what it holds
  int* status;
};

RB_DEVICE void head_tile(int tile, int tiles_m, int tiles_n, int& mt, int& nt) {
  const int per = kHeadBand * tiles_n, band = tile / per, within = tile - band * per, m0 = band * kHeadBand, size = min(kHeadBand, tiles_m - m0);
  mt = m0 + within % size;
  nt = within / size;
}

// two logits as type T holds them
template <typename T> RB_DEVICE void round_pair(float& a, float& b) {
  if constexpr (std::is_same_v<T, __half>) {
    const float2 f = __half22float2(__floats2half2_rn(a, b));
    a = f.x;
    b = f.y;
  } else {
    const float2 f = __bfloat1622float2(__floats2bfloat162_rn(a, b));
    a = f.x;
    b = f.y;
  }
}

// bit i: column col + i of the row is masked out (or beyond the vocabulary)
RB_DEVICE uint32_t gone32(const uint8_t* m, int64_t bytes, int col, int N) {
  uint32_t b = 0;
  if (m) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((col >> 3) + i < bytes) b |= (uint32_t)m[(col >> 3) + i] << (8 * i);
  }
  const int n = N - col;
  return n >= 32 ? b : n <= 0 ? ~0u : b | ~0u << n;
}

// 64 columns of a warp's 32 rows, a lane a row, to 16-bit memory; rows, cols: how many there are from the first on
template <typename T> RB_DEVICE void store_cols(uint32_t stage, const float (&x)[64], T* dst, int64_t ld, int rows, int cols) {
  if (cols >= 64 && rows >= 32) {
    uint32_t r[64];
#pragma unroll
    for (int i = 0; i < 64; ++i) r[i] = __float_as_uint(x[i]);
    store_rows64<T>(stage, r, dst, ld);
  } else {
#pragma unroll
    for (int part = 0; part < 64; part += 32) {
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = x[part + i];
      if (part < cols) store_rows32<T>(stage, v, dst + part, ld, rows, min(32, cols - part), true, false);
    }
  }
}
// (kernels that have no 64 columns)
template <typename T> RB_DEVICE void store_cols(uint32_t, const float (&)[32], T*, int64_t, int, int) {}

enum HeadMode { kStats, kStatsKeep, kLogitGrad, kHiddenGrad, kWeightGrad };
constexpr float kKeepScale = 32768.f;

// kRound: logits are rounded to the operands' type, as a product that stores them leaves them (a variant of its own: asked at run time, it cost every narrow head 3 %)
template <typename T, int kFmt, HeadMode kMode, bool kRound = false>
__global__ void __launch_bounds__(kHeadThreads, 1) head_stats_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                                                                 const HeadParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint32_t dead;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *smem_a = smem, *smem_b = smem + kHeadStages * kHeadA;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kHeadBars);
  uint64_t *full_bar = bars, *empty_bar = bars + kHeadStages, *tmem_full = bars + 2 * kHeadStages, *tmem_empty = tmem_full + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr bool kBwd = kMode == kLogitGrad, kAMN = kMode == kWeightGrad, kSplit = kMode == kHiddenGrad || kAMN;
  constexpr bool kKeep = kMode == kStatsKeep;
  constexpr int kCols = kBwd || kKeep || kAMN ? 64 : 32;    // columns an epilogue warp holds at once
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int tiles_m = RB_CEIL_DIV(p.M, 2 * BM), tiles_n = RB_CEIL_DIV(p.N, HN), all_kb = RB_CEIL_DIV(p.K, BK);
  const int num_tiles = tiles_m * tiles_n * (kSplit ? p.splits : 1);
  // a work item: a tile, and with splits the part [kb0, kb1) of the sum
  auto item = [&](int i, int& mt, int& nt, int& part, int& kb0, int& kb1) {
    part = kSplit ? i / (tiles_m * tiles_n) : 0;
    head_tile(kSplit ? i - part * (tiles_m * tiles_n) : i, tiles_m, tiles_n, mt, nt);
    kb0 = kSplit ? (int)((int64_t)all_kb * part / p.splits) : 0;
    kb1 = kSplit ? (int)((int64_t)all_kb * (part + 1) / p.splits) : all_kb;
  };

  if (threadIdx.x == 0) dead = 0;
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tensormap(&tma_a);
    ptx::prefetch_tensormap(&tma_b);
    for (int i = 0; i < kHeadStages; ++i) {
      ptx::mbar_init(ptx::smem_u32(&full_bar[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&empty_bar[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(ptx::smem_u32(&tmem_full[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&tmem_empty[i]), 2 * kEpiWarps);
    }
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_cg2(ptx::smem_u32(tmem_ptr), 2 * HN);
    tmem_relinquish_cg2();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync();  // the peer's barriers exist
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr;

  if (warp == 0) {
    // both CTAs load their 128 rows of h and their half of the tile's rows of W; every copy completes on the leader's barrier
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int tile = pair; tile < num_tiles; tile += num_pairs) {
        int mt, nt, part, kb0, kb1;
        item(tile, mt, nt, part, kb0, kb1);
        const int m0 = mt * 2 * BM + (int)rank * BM, n0 = nt * HN + (int)rank * (HN / 2);
        for (int kb = kb0; kb < kb1; ++kb) {
          bounded_wait(ptx::smem_u32(&empty_bar[stage]), phase ^ 1, &dead);
          const uint32_t fb_local = ptx::smem_u32(&full_bar[stage]);
          if (leader) ptx::mbar_arrive_expect_tx(fb_local, 2 * kHeadStage);
          const uint32_t fb = mapa_u32(fb_local, 0);
          const uint32_t sa = ptx::smem_u32(smem_a + stage * kHeadA);
          if constexpr (kAMN) {            // d logits as [T, V]: the sum runs over its rows
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) tma_load_2d_cg2(sa + j * (BK * 128), &tma_a, fb, m0 + 64 * j, kb * BK);
          } else {
            tma_load_2d_cg2(sa, &tma_a, fb, kb * BK, m0);
          }
          const uint32_t sb = ptx::smem_u32(smem_b + stage * kHeadB);
          if constexpr (kSplit) {          // W as [V, H], h as [T, H]: the sum runs over its rows
#pragma unroll
            for (int j = 0; j < HN / 2 / 64; ++j) tma_load_2d_cg2(sb + j * (BK * 128), &tma_b, fb, n0 + 64 * j, kb * BK);
          } else {
            tma_load_2d_cg2(sb, &tma_b, fb, kb * BK, n0);
          }
          if (++stage == kHeadStages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (leader) {      // the warp runs converged, one elected lane issues
      constexpr uint32_t idesc = ptx::make_idesc_f16(kFmt, 2 * BM, HN, kAMN ? 1 : 0, kSplit ? 1 : 0);
      constexpr uint32_t kAStep = (kAMN ? 2048 : 32) >> 4, kBStep = (kSplit ? 2048 : 32) >> 4;          // 16 elements of the sum further, in descriptor units
      const uint32_t tm = (uint32_t)ptx::uniform((int)tmem_base);
      int stage = 0, as = 0;
      uint32_t phase = 0, aphase = 0;
      for (int tile = pair; tile < num_tiles; tile += num_pairs) {
        bounded_wait(ptx::smem_u32(&tmem_empty[as]), aphase ^ 1, &dead);
        __syncwarp();
        ptx::tc_fence_after();
        const uint32_t d_tmem = tm + as * HN;
        int mt, nt, part, kb0, kb1;
        item(tile, mt, nt, part, kb0, kb1);
        const int n_kb = ptx::uniform(kb1 - kb0);
        for (int kb = 0; kb < n_kb; ++kb) {
          bounded_wait(ptx::smem_u32(&full_bar[stage]), phase, &dead);
          __syncwarp();
          ptx::tc_fence_after();
          const uint64_t da = ptx::make_smem_desc_sw128(ptx::smem_u32(smem_a + stage * kHeadA), kAMN ? BK * 128 : 16, 1024);
          const uint64_t db = ptx::make_smem_desc_sw128(ptx::smem_u32(smem_b + stage * kHeadB), kSplit ? BK * 128 : 16, 1024);
          if (ptx::elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) tc_mma_f16_cg2(d_tmem, da + k * kAStep, db + k * kBStep, idesc, (kb | k) != 0 ? 1u : 0u);
            tc_commit_cg2(ptx::smem_u32(&empty_bar[stage]), 0b11);
          }
          __syncwarp();
          if (++stage == kHeadStages) { stage = 0; phase ^= 1; }
        }
        if (ptx::elect_one()) tc_commit_cg2(ptx::smem_u32(&tmem_full[as]), 0b11);
        __syncwarp();
        if (++as == 2) { as = 0; aphase ^= 1; }
      }
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) >> 2;        // 32 rows, 128 columns
    const uint32_t stage_out = ptx::smem_u32(smem + kHeadOut + (warp - 2) * 4096);
    const float k = p.inv_temp * rb::kLog2e;
    int as = 0;
    uint32_t aphase = 0;
    for (int tile = pair; tile < num_tiles; tile += num_pairs) {
      int mt, nt, part, kb0, kb1;
      item(tile, mt, nt, part, kb0, kb1);
      const int n0 = nt * HN, row0 = mt * 2 * BM + (int)rank * BM + quad * 32, row = row0 + lane;
      const bool on = row < p.M;
      const int64_t given = !kSplit && on ? p.labels[row] : -1;
      const uint8_t* mr = p.mask && on ? p.mask + row * p.mask_stride : nullptr;
      const int label = given >= n0 && given < min(p.N, n0 + HN) ? (int)(given - n0) : -1;       // within this tile
      float lse = 0.f, H = 0.f, gl = 0.f, ge = 0.f;
      if (kBwd && on) {
        lse = p.lse[row];
        H = p.entropy[row];
        if (p.g_logp && given >= 0) gl = p.g_logp[row] * p.inv_temp;
        if (p.g_entropy) ge = p.g_entropy[row] * p.inv_temp;
        if (gl != 0.f && given >= p.N) gl = NAN;
        if constexpr (std::is_same_v<T, __half>) {
          const float up = p.peak ? rb::grad_scale(*p.peak) : 1.f;
          gl *= up;
          ge *= up;
        }
      }
      const bool zero = (gl == 0.f && ge == 0.f) || lse == -INFINITY;
      const float a = -(gl + ge * H);
      bounded_wait(ptx::smem_u32(&tmem_full[as]), aphase, &dead);
      __syncwarp();
      ptx::tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + as * HN;
      float m = -INFINITY, s = 0.f, w = 0.f;
      if constexpr (kKeep) {           // the maximum of the lane's columns first
#pragma unroll 1
        for (int c = half * (HN / 2); c < (half + 1) * (HN / 2); c += 32) {
          uint32_t r[32];
          __syncwarp();
          ptx::tc_ld_32x32(taddr + c, r);
          const uint32_t gone = p.mask || n0 + c + 32 > p.N ? gone32(mr, p.mask_stride, n0 + c, p.N) : 0u;
          __syncwarp();
          ptx::tc_wait_ld();
          if (gone) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if ((gone >> i) & 1) r[i] = 0xff800000u;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) m = rb::max_nan(m, __uint_as_float(r[i]));
        }
        if (kRound) {
          float same = m;
          round_pair<T>(m, same);
        }
      }
#pragma unroll 1
      for (int c = half * (HN / 2); c < (half + 1) * (HN / 2); c += kCols) {
        uint32_t r[kCols];
        __syncwarp();
        ptx::tc_ld_32x32(taddr + c, r);
        if (kCols == 64) ptx::tc_ld_32x32(taddr + c + 32, r + kCols - 32);
        const int col = n0 + c;
        uint32_t gone = 0, gone_hi = 0;
        if (!kSplit && (p.mask || col + kCols > p.N)) {
          gone = gone32(mr, p.mask_stride, col, p.N);
          if (kCols == 64) gone_hi = gone32(mr, p.mask_stride, col + 32, p.N);
        }
        __syncwarp();
        ptx::tc_wait_ld();
        if (row0 >= p.M || col >= p.N) continue;
        float x[kCols];
#pragma unroll
        for (int i = 0; i < kCols; ++i) x[i] = __uint_as_float(r[i]);
        if (kRound) {
#pragma unroll
          for (int i = 0; i < kCols; i += 2) round_pair<T>(x[i], x[i + 1]);
        }
        const int at = label - c;
        if constexpr (kSplit) {
          if (p.direct) {
            const float down = p.peak ? rb::grad_unscale(*p.peak) : 1.f;
#pragma unroll
            for (int i = 0; i < kCols; ++i) x[i] *= down;
            const int64_t to = (int64_t)row0 * p.N + col;
            if (kCols == 64 && p.direct == 1 && !p.add) {
              store_cols<T>(stage_out, x, reinterpret_cast<T*>(p.out) + to, p.N, p.M - row0, p.N - col);
              continue;
            }
#pragma unroll
            for (int c0 = 0; c0 < kCols; c0 += 32) {
              float v[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = x[c0 + i];
              const int cols = min(32, p.N - col - c0);
              if (cols <= 0) break;
              if (p.direct == 2) store_rows32<float>(stage_out, v, reinterpret_cast<float*>(p.out) + to + c0, p.N, p.M - row0, cols, true, p.add);
              else store_rows32<T>(stage_out, v, reinterpret_cast<T*>(p.out) + to + c0, p.N, p.M - row0, cols, true, p.add);
            }
            continue;
          }
          if constexpr (kCols == 32)
            store_rows32<float>(stage_out, x, reinterpret_cast<float*>(p.out) + ((int64_t)part * p.M + row0) * p.N + col, p.N, p.M - row0, min(32, p.N - col), true,
                                false);
        } else if constexpr (kKeep) {
          if (gone | gone_hi) {
#pragma unroll
            for (int i = 0; i < kCols; ++i)
              if (((i < 32 ? gone : gone_hi) >> (i & 31)) & 1) x[i] = -INFINITY;
          }
          if (at >= 0 && at < kCols) {
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < kCols; ++i) t = i == at ? x[i] : t;
            p.target[row] = t;
          }
          const float ref = m == -INFINITY ? 0.f : m;
          const uint64_t k2 = rb::pack2(k, k), ref2 = rb::pack2(-ref, -ref), scale2 = rb::pack2(kKeepScale, kKeepScale);
          rb::Sums g;
#pragma unroll
          for (int i = 0; i < kCols; i += 2) {
            float u, v;
            rb::unpack2(rb::mul2(rb::add2(rb::pack2(x[i], x[i + 1]), ref2), k2), u, v);
            u = fmaxf(u, -1000.f);
            v = fmaxf(v, -1000.f);
            const uint64_t e = rb::pack2(rb::exp2_fast(u), rb::exp2_fast(v));
            g.s2 = rb::add2(g.s2, e);
            g.w2 = rb::fma2(rb::pack2(u, v), e, g.w2);
            rb::unpack2(rb::mul2(e, scale2), x[i], x[i + 1]);
          }
          s += g.s();
          w += g.w();
          store_cols<__half>(stage_out, x, reinterpret_cast<__half*>(p.out) + (int64_t)row0 * p.ld_out + col, p.ld_out, p.M - row0, p.N - col);
        } else if constexpr (!kBwd) {
          if (gone) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if ((gone >> i) & 1) x[i] = -INFINITY;
          }
          if (at >= 0 && at < 32) {
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) t = i == at ? x[i] : t;
            p.target[row] = t;
          }
          float mc = x[0];
#pragma unroll
          for (int i = 1; i < 32; ++i) mc = rb::max_nan(mc, x[i]);
          if (!(mc <= m)) {
            const float mn = rb::max_nan(m, mc), d = fmaxf((m - mn) * k, -1000.f), f = rb::exp2_fast(d);
            w = f * fmaf(d, s, w);
            s *= f;
            m = mn;
          }
          const float ref = m == -INFINITY ? 0.f : m;
          const uint64_t k2 = rb::pack2(k, k), ref2 = rb::pack2(-ref, -ref);
          rb::Sums g;
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float u, v;
            rb::unpack2(rb::mul2(rb::add2(rb::pack2(x[i], x[i + 1]), ref2), k2), u, v);
            u = fmaxf(u, -1000.f);
            v = fmaxf(v, -1000.f);
            const uint64_t e = rb::pack2(rb::exp2_fast(u), rb::exp2_fast(v));
            g.s2 = rb::add2(g.s2, e);
            g.w2 = rb::fma2(rb::pack2(u, v), e, g.w2);
          }
          s += g.s();
          w += g.w();
        } else {
          const uint64_t c2 = rb::pack2(p.inv_temp, p.inv_temp), l2 = rb::pack2(-lse, -lse), e2 = rb::pack2(rb::kLog2e, rb::kLog2e), g2 = rb::pack2(-ge, -ge),
                         a2 = rb::pack2(a, a);
#pragma unroll
          for (int i = 0; i < kCols; i += 2) {
            float u, v;
            rb::unpack2(rb::fma2(rb::pack2(x[i], x[i + 1]), c2, l2), u, v);
            const uint64_t y = rb::pack2(fmaxf(u, -1000.f), fmaxf(v, -1000.f));
            rb::unpack2(rb::mul2(y, e2), u, v);
            rb::unpack2(rb::mul2(rb::pack2(rb::exp2_fast(u), rb::exp2_fast(v)), rb::fma2(g2, y, a2)), x[i], x[i + 1]);
          }
          if (at >= 0 && at < kCols) {
#pragma unroll
            for (int i = 0; i < kCols; ++i) x[i] += i == at ? gl : 0.f;
          }
          if (p.mask && (gone | gone_hi)) {
#pragma unroll
            for (int i = 0; i < kCols; ++i)
              if (((i < 32 ? gone : gone_hi) >> (i & 31)) & 1) x[i] = lse != lse ? NAN : 0.f;
          }
          if (zero) {
#pragma unroll
            for (int i = 0; i < kCols; ++i) x[i] = 0.f;
          }
          store_cols<T>(stage_out, x, reinterpret_cast<T*>(p.out) + (int64_t)row0 * p.ld_out + col, p.ld_out, p.M - row0, p.N - col);
        }
      }
      if ((kMode == kStats || kKeep) && on) {
        const int64_t to = (int64_t)(2 * nt + half) * p.M + row;
        p.part_m[to] = m;
        p.part_s[to] = s;
        p.part_w[to] = w;
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(ptx::smem_u32(&tmem_empty[as]), 0);
      if (++as == 2) { as = 0; aphase ^= 1; }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  rb::report_given_up(&dead, p.status);
  ptx::cluster_sync();  // neither CTA frees tensor memory or exits while the pair's products or arrivals are under way
  if (warp == 1) {
    ptx::tc_fence_after();
    tmem_dealloc_cg2(tmem_base, 2 * HN);
  }
}

// A row's triples -> its results: 8 rows a block, 32 threads a row over the parts in turn, merged in a fixed order (four threads a row of a warp, then the warps).
constexpr int kMergeRows = 8, kMergeSlices = 32;
__global__ void __launch_bounds__(kMergeRows* kMergeSlices) head_merge_kernel(const HeadParams p, int parts, float* __restrict__ logp, float* __restrict__ entropy,
                                                                             float* __restrict__ lse) {
  constexpr int kWarps = kMergeRows * kMergeSlices / 32;
  __shared__ float sm[3][kWarps][kMergeRows];
  const int at_row = threadIdx.x % kMergeRows, slice = threadIdx.x / kMergeRows, warp = threadIdx.x >> 5, row = blockIdx.x * kMergeRows + at_row;
  const float k = p.inv_temp * rb::kLog2e;
  rb::RowStats st;
  if (row < p.M) {
    constexpr int U = 8;
    for (int t0 = slice; t0 < parts; t0 += U * kMergeSlices) {
      float m[U], s[U], w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * kMergeSlices;
        const int64_t at = (int64_t)t * p.M + row;
        m[u] = t < parts ? p.part_m[at] : -INFINITY;
        s[u] = t < parts ? p.part_s[at] : 0.f;
        w[u] = t < parts ? p.part_w[at] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (t0 + u * kMergeSlices < parts) st.add(m[u], s[u], w[u], k);
    }
  }
#pragma unroll
  for (int o = kMergeRows; o < 32; o <<= 1) {
    const float m = __shfl_xor_sync(0xffffffffu, st.m, o), s = __shfl_xor_sync(0xffffffffu, st.s, o), w = __shfl_xor_sync(0xffffffffu, st.w, o);
    st.add(m, s, w, k);
  }
  if ((threadIdx.x & 31) < kMergeRows) {
    sm[0][warp][at_row] = st.m;
    sm[1][warp][at_row] = st.s;
    sm[2][warp][at_row] = st.w;
  }
  __syncthreads();
  if (threadIdx.x < kMergeRows && row < p.M) {
#pragma unroll
    for (int i = 1; i < kWarps; ++i) st.add(sm[0][i][at_row], sm[1][i][at_row], sm[2][i][at_row], k);
    const rb::RowResult r(st, p.inv_temp);
    lse[row] = r.lse;
    entropy[row] = r.entropy;
    const int64_t label = p.labels[row];
    float l;
    if (label < 0) l = 0.f;
    else if (label >= p.N || r.lse != r.lse) l = NAN;
    else if (r.lse == -INFINITY) l = -INFINITY;
    else l = fmaf(p.target[row], p.inv_temp, -r.lse);
    logp[row] = l;
  }
}

// d logits from kept weights: rows of `kept` belong to rows row0, row0 + 1, ... of the forward pass; in segments of a row
constexpr int kGradThreads = 128, kGradPieces = 4;
template <typename T>
__global__ void __launch_bounds__(kGradThreads) head_grad_kernel(const __half* __restrict__ kept, int64_t ld_kept, const HeadParams p, int row0, int all_rows, int segs) {
  const int row = blockIdx.x / segs, seg = blockIdx.x - row * segs, whole = row0 + row;
  const float lse = p.lse[whole], H = p.entropy[whole];
  const int64_t given = p.labels[whole];
  float ge = p.g_entropy ? p.g_entropy[whole] * p.inv_temp : 0.f;
  float gl = p.g_logp && given >= 0 ? p.g_logp[whole] * p.inv_temp : 0.f;
  if (gl != 0.f && given >= p.N) gl = NAN;
  if constexpr (std::is_same_v<T, __half>) {
    const float up = p.peak ? rb::grad_scale(*p.peak) : 1.f;
    gl *= up;
    ge *= up;
  }
  const bool zero = (gl == 0.f && ge == 0.f) || lse == -INFINITY;
  const bool gone = p.mask && given >= 0 && given < p.N && (p.mask[whole * p.mask_stride + (given >> 3)] >> (given & 7)) & 1;
  const int label = given >= 0 && given < p.N && !gone ? (int)given : -1;
  const float a = -(gl + ge * H);
  const int pieces = RB_CEIL_DIV(p.N, 8);
  const int4* in = reinterpret_cast<const int4*>(kept + row * ld_kept);
  int4* out = reinterpret_cast<int4*>(reinterpret_cast<T*>(p.out) + row * p.ld_out);
  const int i0 = seg * kGradPieces * kGradThreads + threadIdx.x;
  int4 v[kGradPieces];
  const bool plain = zero || lse != lse;
  constexpr int kPartPieces = HN / 2 / 8;                   // pieces of 128 columns
  __shared__ float2 factor[kGradPieces * kGradThreads / kPartPieces];   // of the segment's parts: log-probability of a kept number of 1, and it itself
#pragma unroll
  for (int u = 0; u < kGradPieces; ++u) {
    const int i = i0 + u * kGradThreads;
    if (i < pieces && !plain) {
      v[u] = rb::ld_once(in + i);
    }
  }
  {
    const int part = seg * (kGradPieces * kGradThreads / kPartPieces) + threadIdx.x;
    if (threadIdx.x < kGradPieces * kGradThreads / kPartPieces && part * kPartPieces < pieces) {
      const float m = p.part_m[(int64_t)part * all_rows + whole], y = m == -INFINITY ? 0.f : fmaf(m, p.inv_temp, -lse) - 15.f * rb::kLn2;
      factor[threadIdx.x] = make_float2(y, rb::exp2_fast(y * rb::kLog2e));
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < kGradPieces; ++u) {
    const int i = i0 + u * kGradThreads;
    if (i >= pieces) continue;
    float d[8];
    if (plain) {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = zero ? 0.f : NAN;
    } else {
      const __half2* h = reinterpret_cast<const __half2*>(&v[u]);
      const float2 fac = factor[(u * kGradThreads + threadIdx.x) / kPartPieces];
      const float y1 = fac.x, f = fac.y;
      const uint64_t f2 = rb::pack2(f, f), ln2 = rb::pack2(rb::kLn2, rb::kLn2), y2 = rb::pack2(y1, y1), g2 = rb::pack2(-ge, -ge), a2 = rb::pack2(a, a);
      if (ge != 0.f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = __half22float2(h[e]);
          // y = ln x + y1; a weight of 0 is 0 whatever its logarithm
          const uint64_t y = rb::fma2(rb::pack2(fmaxf(__log2f(x.x), -100.f), fmaxf(__log2f(x.y), -100.f)), ln2, y2);
          rb::unpack2(rb::mul2(rb::mul2(rb::pack2(x.x, x.y), f2), rb::fma2(g2, y, a2)), d[2 * e], d[2 * e + 1]);
        }
      } else {
        const uint64_t af = rb::mul2(f2, a2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = __half22float2(h[e]);
          rb::unpack2(rb::mul2(rb::pack2(x.x, x.y), af), d[2 * e], d[2 * e + 1]);
        }
      }
      const int at = label - i * 8;
      if (at >= 0 && at < 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] += e == at ? gl : 0.f;
      }
    }
    rb::Pack<T, 8> o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o.v[e] = rb::from_f<T>(d[e]);
    if (i * 8 + 8 <= p.N) {
      out[i] = *reinterpret_cast<const int4*>(&o);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i * 8 + e < p.N) reinterpret_cast<T*>(out + i)[e] = o.v[e];
    }
  }
}

// A bound of a row's d logits, c (|g_logp| (1 - p) + |g_entropy| p |y + H|) with p |y| <= 1 / e, into the peak of all rows.
__global__ void __launch_bounds__(256) head_grad_peak_kernel(const int64_t* __restrict__ labels, const float* __restrict__ entropy, const float* __restrict__ g_logp,
                                                             const float* __restrict__ g_entropy, uint32_t* peak, int rows, float inv_temp) {
  const int row = blockIdx.x * 256 + threadIdx.x;
  float v = 0.f;
  if (row < rows) {
    if (g_logp && labels[row] >= 0) v = fabsf(g_logp[row]);
    if (g_entropy && g_entropy[row] != 0.f) v += fabsf(g_entropy[row]) * (entropy[row] + 0.37f);
  }
  rb::raise_peak(peak, v * inv_temp);
}

// parts [splits, n] -> their sum, rounded once; n a multiple of 8; peak: taken back from the scale of d logits
template <typename T> __global__ void __launch_bounds__(256) head_sum_kernel(const float* __restrict__ parts, const uint32_t* __restrict__ peak, T* __restrict__ out, int splits,
                                                                             int64_t n) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i >= n) return;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float4 u = *reinterpret_cast<const float4*>(parts + s * n + i), v = *reinterpret_cast<const float4*>(parts + s * n + i + 4);
    a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
    b.x += v.x; b.y += v.y; b.z += v.z; b.w += v.w;
  }
  if (peak) {
    const float down = rb::grad_unscale(*peak);
    a.x *= down; a.y *= down; a.z *= down; a.w *= down;
    b.x *= down; b.y *= down; b.z *= down; b.w *= down;
  }
  rb::Pack<T, 8> o;
  o.v[0] = rb::from_f<T>(a.x); o.v[1] = rb::from_f<T>(a.y); o.v[2] = rb::from_f<T>(a.z); o.v[3] = rb::from_f<T>(a.w);
  o.v[4] = rb::from_f<T>(b.x); o.v[5] = rb::from_f<T>(b.y); o.v[6] = rb::from_f<T>(b.z); o.v[7] = rb::from_f<T>(b.w);
  *reinterpret_cast<rb::Pack<T, 8>*>(out + i) = o;
}

template <typename T, int kFmt, HeadMode kMode, bool kRound = false> int launch_head(const CUtensorMap& ta, const CUtensorMap& tb, const HeadParams& p, int num_sms, cudaStream_t s) {
  auto kern = head_stats_kernel<T, kFmt, kMode, kRound>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeadSmem) != cudaSuccess) return -2;
  const int tiles = RB_CEIL_DIV(p.M, 2 * BM) * RB_CEIL_DIV(p.N, HN) * (kMode == kHiddenGrad ? p.splits : 1), pairs = num_sms / 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * (tiles < pairs ? tiles : pairs));
  cfg.blockDim = dim3(kHeadThreads);
  cfg.dynamicSmemBytes = kHeadSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, ta, tb, p) != cudaSuccess) return -3;
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// bf16 or fp16, logits as they are or rounded
template <HeadMode kMode> int launch_logits(const CUtensorMap& ta, const CUtensorMap& tb, const HeadParams& p, int in_dt, bool rounded, int num_sms, cudaStream_t s) {
  if (in_dt == 1)
    return rounded ? launch_head<__nv_bfloat16, 1, kMode, true>(ta, tb, p, num_sms, s) : launch_head<__nv_bfloat16, 1, kMode>(ta, tb, p, num_sms, s);
  return rounded ? launch_head<__half, 0, kMode, true>(ta, tb, p, num_sms, s) : launch_head<__half, 0, kMode>(ta, tb, p, num_sms, s);
}

int head_maps(const void* h, const void* w, int64_t ld_h, int64_t ld_w, int M, int N, int K, int in_dt, CUtensorMap& ta, CUtensorMap& tb) {
  if (in_dt != 1 && in_dt != 2) return -10;
  if (K % 8 || ld_h % 8 || ld_w % 8 || (reinterpret_cast<uintptr_t>(h) & 15) || (reinterpret_cast<uintptr_t>(w) & 15)) return -11;
  if (!make_tmap(&ta, h, in_dt == 1, (uint64_t)M, (uint64_t)K, (uint64_t)ld_h, BK, (uint32_t)BM)) return -13;
  if (!make_tmap(&tb, w, in_dt == 1, (uint64_t)N, (uint64_t)K, (uint64_t)ld_w, BK, (uint32_t)(HN / 2))) return -13;
  return 0;
}

}  // namespace

extern "C" {

// fp32 numbers a row that the forward pass leaves beside its results
int64_t rb_head_stats_scratch(int N) { return 6LL * RB_CEIL_DIV(N, HN) + 1; }

// h [M, K], w [N, K], in_dt 1 bf16 / 2 fp16, rows 16-byte aligned; labels [M]; scratch: fp32 [rb_head_stats_scratch(N) * M]; its first M * ceil(N / 256) * 2 numbers are the
// maxima of 128 columns.  kept: fp16 [M, N] for the weights, rows ld_kept apart (a multiple of 8), or null.
int rb_head_stats(const void* h, const void* w, int64_t ld_h, int64_t ld_w, const int64_t* labels, const uint8_t* mask, int64_t mask_stride, float* scratch,
                  void* kept, int64_t ld_kept, float* logp, float* entropy, float* lse, int M, int N, int K, float inv_temp, int rounded, int in_dt, int num_sms,
                  cudaStream_t s) {
  if (M <= 0) return 0;
  CUtensorMap ta, tb;
  if (const int rc = head_maps(h, w, ld_h, ld_w, M, N, K, in_dt, ta, tb)) return rc;
  const int tiles_n = RB_CEIL_DIV(N, HN);
  HeadParams p{};
  p.M = M; p.N = N; p.K = K;
  p.inv_temp = inv_temp;
  p.labels = labels; p.mask = mask; p.mask_stride = mask_stride;
  p.part_m = scratch;
  p.part_s = scratch + 2LL * tiles_n * M;
  p.part_w = scratch + 4LL * tiles_n * M;
  p.target = scratch + 6LL * tiles_n * M;
  p.status = rb_attn_status();
  if (p.status == nullptr) return -14;
  if (kept && (ld_kept % 8 || (reinterpret_cast<uintptr_t>(kept) & 15))) return -12;
  p.out = kept;
  p.ld_out = ld_kept;
  const int rc = kept ? launch_logits<kStatsKeep>(ta, tb, p, in_dt, rounded, num_sms, s) : launch_logits<kStats>(ta, tb, p, in_dt, rounded, num_sms, s);
  if (rc) return rc;
  head_merge_kernel<<<RB_CEIL_DIV(M, kMergeRows), kMergeRows * kMergeSlices, 0, s>>>(p, 2 * tiles_n, logp, entropy, lse);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// peak (zeroed before): a bound of the rows' d logits, for grad_scale; g_logp, g_entropy may be null
int rb_head_grad_peak(const int64_t* labels, const float* entropy, const float* g_logp, const float* g_entropy, uint32_t* peak, int rows, float inv_temp, cudaStream_t s) {
  if (rows <= 0) return 0;
  head_grad_peak_kernel<<<RB_CEIL_DIV(rows, 256), 256, 0, s>>>(labels, entropy, g_logp, g_entropy, peak, rows, inv_temp);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// out: d logits [M, N] of the operands' type, rows ld_out apart (a multiple of 8), 16-byte aligned; peak: see HeadParams
int rb_head_stats_bwd(const void* h, const void* w, int64_t ld_h, int64_t ld_w, const int64_t* labels, const uint8_t* mask, int64_t mask_stride, const float* lse,
                      const float* entropy, const float* g_logp, const float* g_entropy, const uint32_t* peak, void* out, int64_t ld_out, int M, int N, int K, float inv_temp,
                      int rounded, int in_dt, int num_sms, cudaStream_t s) {
  if (M <= 0) return 0;
  if (peak && in_dt != 2) return -10;
  if (ld_out % 8 || (reinterpret_cast<uintptr_t>(out) & 15)) return -12;
  CUtensorMap ta, tb;
  if (const int rc = head_maps(h, w, ld_h, ld_w, M, N, K, in_dt, ta, tb)) return rc;
  HeadParams p{};
  p.M = M; p.N = N; p.K = K;
  p.inv_temp = inv_temp;
  p.labels = labels; p.mask = mask; p.mask_stride = mask_stride;
  p.lse = lse; p.entropy = entropy; p.g_logp = g_logp; p.g_entropy = g_entropy; p.peak = peak;
  p.out = out; p.ld_out = ld_out;
  p.status = rb_attn_status();
  if (p.status == nullptr) return -14;
  return launch_logits<kLogitGrad>(ta, tb, p, in_dt, rounded, num_sms, s);
}

// d logits [rows, N] of rows row0 .. of a forward pass over all_rows rows, from what it kept (`kept`: these rows; part_m, labels, mask and values a row: all rows); out as above
int rb_head_grad(const void* kept, int64_t ld_kept, const float* part_m, const int64_t* labels, const uint8_t* mask, int64_t mask_stride, const float* lse,
                 const float* entropy, const float* g_logp, const float* g_entropy, const uint32_t* peak, void* out, int64_t ld_out, int row0, int rows, int all_rows, int N,
                 float inv_temp, int dt, cudaStream_t s) {
  if (rows <= 0) return 0;
  if (peak && dt != 2) return -10;
  if (ld_out % 8 || ld_kept % 8 || ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(kept)) & 15) || row0 < 0 || row0 + rows > all_rows) return -12;
  HeadParams p{};
  p.M = rows; p.N = N;
  p.inv_temp = inv_temp;
  p.labels = labels; p.mask = mask; p.mask_stride = mask_stride;
  p.part_m = const_cast<float*>(part_m);
  p.lse = lse; p.entropy = entropy; p.g_logp = g_logp; p.g_entropy = g_entropy; p.peak = peak;
  p.out = out; p.ld_out = ld_out;
  const int64_t segs = RB_CEIL_DIV(RB_CEIL_DIV(N, 8), kGradThreads * kGradPieces);
  if (rows * segs > 0x7fffffffLL) return -3;
  if (dt == 1) head_grad_kernel<__nv_bfloat16><<<(unsigned)(rows * segs), kGradThreads, 0, s>>>((const __half*)kept, ld_kept, p, row0, all_rows, (int)segs);
  else if (dt == 2) head_grad_kernel<__half><<<(unsigned)(rows * segs), kGradThreads, 0, s>>>((const __half*)kept, ld_kept, p, row0, all_rows, (int)segs);
  else return -10;
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// How many parts the sum over the vocabulary is cut into for d h = d logits W, [M, V] x [V, N]: 1 where the tiles of d h fill the GPU (or nearly), so that the general product
// takes them.  A k-block of a tile takes 0.28 us; a part costs its fp32 tile once out and once in.
int rb_head_dhidden_splits(int M, int N, int V, int num_sms) {
  const int pairs = num_sms / 2, tiles = RB_CEIL_DIV(M, 2 * BM) * RB_CEIL_DIV(N, HN), kb = RB_CEIL_DIV(V, BK);
  if (tiles * 10 >= pairs * 7) return 1;
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= 64 && s * 4 <= kb; ++s) {
    const double t = (double)RB_CEIL_DIV(tiles * s, pairs) * RB_CEIL_DIV(kb, s) * 0.28 + (double)s * M * N * 8 / 5e6;
    if (t < least) { least = t; best = s; }
  }
  return best;
}

// d [M, V] (rows ld_d apart, a multiple of 8), w [V, N], parts: fp32 [splits, M, N] (one split: null), out [M, N] contiguous; N a multiple of 8.  peak: that d is scaled by, or
// null.
int rb_head_dhidden(const void* d, const void* w, int64_t ld_d, int64_t ld_w, const uint32_t* peak, float* parts, void* out, int M, int N, int V, int splits, int in_dt,
                    int num_sms, cudaStream_t s) {
  if (M <= 0) return 0;
  if (in_dt != 1 && in_dt != 2) return -10;
  if (N % 8 || ld_d % 8 || ld_w % 8 || ((reinterpret_cast<uintptr_t>(d) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out)) & 15)) return -11;
  if (splits < 1 || splits > RB_CEIL_DIV(V, BK)) return -12;
  CUtensorMap ta, tb;
  if (!make_tmap(&ta, d, in_dt == 1, (uint64_t)M, (uint64_t)V, (uint64_t)ld_d, BK, (uint32_t)BM)) return -13;
  if (!make_tmap(&tb, w, in_dt == 1, (uint64_t)V, (uint64_t)N, (uint64_t)ld_w, 64, BK)) return -13;
  HeadParams p{};
  p.M = M; p.N = N; p.K = V;
  p.out = splits > 1 ? parts : out;
  p.splits = splits;
  p.direct = splits == 1;
  p.peak = peak;
  p.status = rb_attn_status();
  if (p.status == nullptr) return -14;
  const int rc = in_dt == 1 ? launch_head<__nv_bfloat16, 1, kHiddenGrad>(ta, tb, p, num_sms, s) : launch_head<__half, 0, kHiddenGrad>(ta, tb, p, num_sms, s);
  if (rc || splits == 1) return rc;
  const int64_t n = (int64_t)M * N;
  const unsigned blocks = (unsigned)RB_CEIL_DIV(n, 256 * 8);
  if (in_dt == 1) head_sum_kernel<__nv_bfloat16><<<blocks, 256, 0, s>>>(parts, peak, (__nv_bfloat16*)out, splits, n);
  else head_sum_kernel<__half><<<blocks, 256, 0, s>>>(parts, peak, (__half*)out, splits, n);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// out [V, N] contiguous, of the operands' type or fp32 (out_dt 0), = or add: += d^T h over the scale of d; d [M, V] (rows ld_d apart), h [M, N], in fp16 (the general product takes
// what has no scale)
int rb_head_dweight(const void* d, const void* h, int64_t ld_d, int64_t ld_h, const uint32_t* peak, void* out, int M, int N, int V, int in_dt, int out_dt, int add, int num_sms,
                    cudaStream_t s) {
  if (M <= 0) return 0;
  if (in_dt != 2 || (out_dt != 0 && out_dt != in_dt)) return -10;
  if (N % 8 || ld_d % 8 || ld_h % 8 || ((reinterpret_cast<uintptr_t>(d) | reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(out)) & 15)) return -11;
  CUtensorMap ta, tb;
  if (!make_tmap(&ta, d, false, (uint64_t)M, (uint64_t)V, (uint64_t)ld_d, 64, BK)) return -13;
  if (!make_tmap(&tb, h, false, (uint64_t)M, (uint64_t)N, (uint64_t)ld_h, 64, BK)) return -13;
  HeadParams p{};
  p.M = V; p.N = N; p.K = M;
  p.out = out;
  p.splits = 1;
  p.direct = out_dt == 0 ? 2 : 1;
  p.add = add;
  p.peak = peak;
  p.status = rb_attn_status();
  if (p.status == nullptr) return -14;
  return launch_head<__half, 0, kWeightGrad>(ta, tb, p, num_sms, s);
}

}  // extern "C"
