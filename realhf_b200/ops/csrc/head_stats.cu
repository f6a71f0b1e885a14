// Language-model head with token statistics in its epilogue: logits X = h W^T (h [T, H], W [V, H], 16 bits, fp32 accumulators) never leave the chip.
//
// Forward: a CTA pair forms a 256 x 256 tile of X (tcgen05.mma.cta_group::2, operands by TMA, two accumulators in tensor memory); while the next tile is multiplied, four
// warps a CTA read theirs, a lane a row, and leave three numbers a row and tile: maximum, sum and weighted sum (vocab_rows.cuh).  A second kernel merges a row's V / 256
// triples.  Logits are what fp32 accumulators hold; stored in 16 bits they would move a log-probability by up to 2^-9 of the logit.
// Backward: the product again, d logits formed in the epilogue from the row's log-sum-exp and entropy and stored in 16 bits (rounded once), as operand of the
// products for d h and d W.
// An epilogue takes 32768 exponentials a CTA, 2048 cycles at least, beside 8 H cycles of products: it hides behind them from H = 512 on.
#include "attn_common.cuh"
#include "cta_pair.cuh"
#include "vocab_rows.cuh"

namespace {

constexpr int HN = 256;                                     // logits of a tile
constexpr int kHeadStages = 6;
constexpr int kHeadA = BM * BK * 2, kHeadB = HN / 2 * BK * 2, kHeadStage = kHeadA + kHeadB;
constexpr int kHeadOut = kHeadStages * kHeadStage, kHeadBars = kHeadOut + 4 * 4096, kHeadSmem = kHeadBars + 1024 + 256;
constexpr int kHeadBand = 8;                                // row tiles walked together, so that the tiles in flight share operands in L2

struct HeadParams {
  int M, N, K;
  float inv_temp;
  const int64_t* labels;
  const uint8_t* mask;
  int64_t mask_stride;
  // forward: [tiles_n, M] each, and the label's logit [M]
  float *part_m, *part_s, *part_w, *target;
  // backward
  const float *lse, *entropy, *g_logp, *g_entropy;
  void* out;
  int64_t ld_out;
  int* status;
};

RB_DEVICE void head_tile(int tile, int tiles_m, int tiles_n, int& mt, int& nt) {
  const int per = kHeadBand * tiles_n, band = tile / per, within = tile - band * per, m0 = band * kHeadBand, size = min(kHeadBand, tiles_m - m0);
  mt = m0 + within % size;
  nt = within / size;
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

template <typename T, int kFmt, bool kBwd>
__global__ void __launch_bounds__(kThreads, 1) head_stats_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                                                                 const HeadParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint32_t dead;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *smem_a = smem, *smem_b = smem + kHeadStages * kHeadA;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kHeadBars);
  uint64_t *full_bar = bars, *empty_bar = bars + kHeadStages, *tmem_full = bars + 2 * kHeadStages, *tmem_empty = tmem_full + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int tiles_m = RB_CEIL_DIV(p.M, 2 * BM), tiles_n = RB_CEIL_DIV(p.N, HN), num_tiles = tiles_m * tiles_n, num_kb = RB_CEIL_DIV(p.K, BK);

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
      ptx::mbar_init(ptx::smem_u32(&tmem_empty[i]), 8);
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
        int mt, nt;
        head_tile(tile, tiles_m, tiles_n, mt, nt);
        const int m0 = mt * 2 * BM + (int)rank * BM, n0 = nt * HN + (int)rank * (HN / 2);
        for (int kb = 0; kb < num_kb; ++kb) {
          bounded_wait(ptx::smem_u32(&empty_bar[stage]), phase ^ 1, &dead);
          const uint32_t fb_local = ptx::smem_u32(&full_bar[stage]);
          if (leader) ptx::mbar_arrive_expect_tx(fb_local, 2 * kHeadStage);
          const uint32_t fb = mapa_u32(fb_local, 0);
          tma_load_2d_cg2(ptx::smem_u32(smem_a + stage * kHeadA), &tma_a, fb, kb * BK, m0);
          tma_load_2d_cg2(ptx::smem_u32(smem_b + stage * kHeadB), &tma_b, fb, kb * BK, n0);
          if (++stage == kHeadStages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (leader) {      // the warp runs converged, one elected lane issues
      constexpr uint32_t idesc = ptx::make_idesc_f16(kFmt, 2 * BM, HN, 0, 0);
      const uint32_t tm = (uint32_t)ptx::uniform((int)tmem_base);
      int stage = 0, as = 0;
      uint32_t phase = 0, aphase = 0;
      for (int tile = pair; tile < num_tiles; tile += num_pairs) {
        bounded_wait(ptx::smem_u32(&tmem_empty[as]), aphase ^ 1, &dead);
        __syncwarp();
        ptx::tc_fence_after();
        const uint32_t d_tmem = tm + as * HN;
        for (int kb = 0; kb < num_kb; ++kb) {
          bounded_wait(ptx::smem_u32(&full_bar[stage]), phase, &dead);
          __syncwarp();
          ptx::tc_fence_after();
          const uint64_t da = ptx::make_smem_desc_sw128(ptx::smem_u32(smem_a + stage * kHeadA), 16, 1024);
          const uint64_t db = ptx::make_smem_desc_sw128(ptx::smem_u32(smem_b + stage * kHeadB), 16, 1024);
          if (ptx::elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) tc_mma_f16_cg2(d_tmem, da + k * 2, db + k * 2, idesc, (kb | k) != 0 ? 1u : 0u);
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
    const int quad = warp & 3;
    const uint32_t stage_out = ptx::smem_u32(smem + kHeadOut + quad * 4096);
    const float k = p.inv_temp * rb::kLog2e;
    int as = 0;
    uint32_t aphase = 0;
    for (int tile = pair; tile < num_tiles; tile += num_pairs) {
      int mt, nt;
      head_tile(tile, tiles_m, tiles_n, mt, nt);
      const int n0 = nt * HN, row0 = mt * 2 * BM + (int)rank * BM + quad * 32, row = row0 + lane;
      const bool on = row < p.M;
      const int64_t given = on ? p.labels[row] : -1;
      const uint8_t* mr = p.mask && on ? p.mask + row * p.mask_stride : nullptr;
      const int label = given >= n0 && given < min(p.N, n0 + HN) ? (int)(given - n0) : -1;       // within this tile
      float lse = 0.f, H = 0.f, gl = 0.f, ge = 0.f;
      if (kBwd && on) {
        lse = p.lse[row];
        H = p.entropy[row];
        if (p.g_logp && given >= 0) gl = p.g_logp[row] * p.inv_temp;
        if (p.g_entropy) ge = p.g_entropy[row] * p.inv_temp;
        if (gl != 0.f && given >= p.N) gl = NAN;
      }
      const bool zero = (gl == 0.f && ge == 0.f) || lse == -INFINITY;
      const float a = -(gl + ge * H);
      bounded_wait(ptx::smem_u32(&tmem_full[as]), aphase, &dead);
      __syncwarp();
      ptx::tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + as * HN;
      float m = -INFINITY, s = 0.f, w = 0.f;
#pragma unroll 1
      for (int c = 0; c < HN; c += 32) {
        uint32_t r[32];
        __syncwarp();
        ptx::tc_ld_32x32(taddr + c, r);
        const int col = n0 + c;
        uint32_t gone = 0;
        if (p.mask || col + 32 > p.N) gone = gone32(mr, p.mask_stride, col, p.N);
        __syncwarp();
        ptx::tc_wait_ld();
        if (row0 >= p.M || col >= p.N) continue;
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]);
        const int at = label - c;
        if constexpr (!kBwd) {
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
          for (int i = 0; i < 32; i += 2) {
            float u, v;
            rb::unpack2(rb::fma2(rb::pack2(x[i], x[i + 1]), c2, l2), u, v);
            const uint64_t y = rb::pack2(fmaxf(u, -1000.f), fmaxf(v, -1000.f));
            rb::unpack2(rb::mul2(y, e2), u, v);
            rb::unpack2(rb::mul2(rb::pack2(rb::exp2_fast(u), rb::exp2_fast(v)), rb::fma2(g2, y, a2)), x[i], x[i + 1]);
          }
          if (at >= 0 && at < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] += i == at ? gl : 0.f;
          }
          if (p.mask && gone) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if ((gone >> i) & 1) x[i] = lse != lse ? NAN : 0.f;
          }
          if (zero) {
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = 0.f;
          }
          store_rows32<T>(stage_out, x, reinterpret_cast<T*>(p.out) + (int64_t)row0 * p.ld_out + col, p.ld_out, p.M - row0, min(32, p.N - col), true, false);
        }
      }
      if (!kBwd && on) {
        const int64_t to = (int64_t)nt * p.M + row;
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

// A row's triples -> its results: 32 rows a block, 16 threads a row over the tiles in turn, merged in a fixed order.
constexpr int kMergeSlices = 16;
__global__ void __launch_bounds__(32 * kMergeSlices) head_merge_kernel(const HeadParams p, int tiles_n, float* __restrict__ logp, float* __restrict__ entropy,
                                                                      float* __restrict__ lse) {
  __shared__ float sm[3][kMergeSlices][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, row = blockIdx.x * 32 + lane;
  const float k = p.inv_temp * rb::kLog2e;
  rb::RowStats st;
  if (row < p.M) {
#pragma unroll 4
    for (int t = slice; t < tiles_n; t += kMergeSlices) {
      const int64_t at = (int64_t)t * p.M + row;
      st.add(p.part_m[at], p.part_s[at], p.part_w[at], k);
    }
  }
  sm[0][slice][lane] = st.m;
  sm[1][slice][lane] = st.s;
  sm[2][slice][lane] = st.w;
  __syncthreads();
  if (slice == 0 && row < p.M) {
#pragma unroll
    for (int i = 1; i < kMergeSlices; ++i) st.add(sm[0][i][lane], sm[1][i][lane], sm[2][i][lane], k);
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

template <typename T, int kFmt, bool kBwd> int launch_head(const CUtensorMap& ta, const CUtensorMap& tb, const HeadParams& p, int num_sms, cudaStream_t s) {
  auto kern = head_stats_kernel<T, kFmt, kBwd>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeadSmem) != cudaSuccess) return -2;
  const int tiles = RB_CEIL_DIV(p.M, 2 * BM) * RB_CEIL_DIV(p.N, HN), pairs = num_sms / 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * (tiles < pairs ? tiles : pairs));
  cfg.blockDim = dim3(kThreads);
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
int64_t rb_head_stats_scratch(int N) { return 3LL * RB_CEIL_DIV(N, HN) + 1; }

// h [M, K], w [N, K], in_dt 1 bf16 / 2 fp16, rows 16-byte aligned; labels [M]; scratch: fp32 [rb_head_stats_scratch(N) * M].
int rb_head_stats(const void* h, const void* w, int64_t ld_h, int64_t ld_w, const int64_t* labels, const uint8_t* mask, int64_t mask_stride, float* scratch,
                  float* logp, float* entropy, float* lse, int M, int N, int K, float inv_temp, int in_dt, int num_sms, cudaStream_t s) {
  if (M <= 0) return 0;
  CUtensorMap ta, tb;
  if (const int rc = head_maps(h, w, ld_h, ld_w, M, N, K, in_dt, ta, tb)) return rc;
  const int tiles_n = RB_CEIL_DIV(N, HN);
  HeadParams p{};
  p.M = M; p.N = N; p.K = K;
  p.inv_temp = inv_temp;
  p.labels = labels; p.mask = mask; p.mask_stride = mask_stride;
  p.part_m = scratch;
  p.part_s = scratch + (int64_t)tiles_n * M;
  p.part_w = scratch + 2LL * tiles_n * M;
  p.target = scratch + 3LL * tiles_n * M;
  p.status = rb_attn_status();
  if (p.status == nullptr) return -14;
  const int rc = in_dt == 1 ? launch_head<__nv_bfloat16, 1, false>(ta, tb, p, num_sms, s) : launch_head<__half, 0, false>(ta, tb, p, num_sms, s);
  if (rc) return rc;
  head_merge_kernel<<<RB_CEIL_DIV(M, 32), 32 * kMergeSlices, 0, s>>>(p, tiles_n, logp, entropy, lse);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// out: d logits [M, N] of the operands' type, rows ld_out apart (a multiple of 8), 16-byte aligned
int rb_head_stats_bwd(const void* h, const void* w, int64_t ld_h, int64_t ld_w, const int64_t* labels, const uint8_t* mask, int64_t mask_stride, const float* lse,
                      const float* entropy, const float* g_logp, const float* g_entropy, void* out, int64_t ld_out, int M, int N, int K, float inv_temp, int in_dt,
                      int num_sms, cudaStream_t s) {
  if (M <= 0) return 0;
  if (ld_out % 8 || (reinterpret_cast<uintptr_t>(out) & 15)) return -12;
  CUtensorMap ta, tb;
  if (const int rc = head_maps(h, w, ld_h, ld_w, M, N, K, in_dt, ta, tb)) return rc;
  HeadParams p{};
  p.M = M; p.N = N; p.K = K;
  p.inv_temp = inv_temp;
  p.labels = labels; p.mask = mask; p.mask_stride = mask_stride;
  p.lse = lse; p.entropy = entropy; p.g_logp = g_logp; p.g_entropy = g_entropy;
  p.out = out; p.ld_out = ld_out;
  p.status = rb_attn_status();
  if (p.status == nullptr) return -14;
  return in_dt == 1 ? launch_head<__nv_bfloat16, 1, true>(ta, tb, p, num_sms, s) : launch_head<__half, 0, true>(ta, tb, p, num_sms, s);
}

}  // extern "C"
