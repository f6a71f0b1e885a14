// Log-probability of a given token and entropy of its distribution from logits [rows, V], forward and backward.
//
// Forward: one read of the row, statistics as in vocab_rows.cuh, one block a row.
// Backward, with y = x inv_temp - lse and p = e^y:   dx_j = inv_temp (g_logp (1[j = label] - p_j) - g_entropy p_j (y_j + H))
// element by element, in segments of a row.
//
// Both are bound by memory: 8192 x 32000 bf16 forward 95 us (5.5 TB/s: the ends of rows of 64 KB), 8192 x 131072 340 (6.3); backward 156 .. 160 and 636 .. 650 (6.6 TB/s) with all loads of a
// thread ahead of the first use, streaming stores and f32x2 arithmetic (189 and 721 with a piece after the other).
#include "vocab_rows.cuh"

namespace {

constexpr int kBwdThreads = 64, kBwdVecs = 4;

template <typename T, bool kMask, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) token_stats_kernel(const T* __restrict__ logits, int64_t row_stride,
                                                                                const int64_t* __restrict__ labels, const uint8_t* __restrict__ mask,
                                                                                int64_t mask_stride, float* __restrict__ logp, float* __restrict__ entropy,
                                                                                float* __restrict__ lse, int V, float inv_temp) {
  constexpr int VEC = rb::RowSpan<T>::VEC;
  __shared__ float red[96];
  const int64_t row = blockIdx.x;
  const T* lr = logits + row * row_stride;
  const uint8_t* mr = kMask ? mask + row * mask_stride : nullptr;
  const float k = inv_temp * rb::kLog2e;
  const rb::RowSpan<T> span(lr, V);
  rb::RunningStats<T, true> run;
  auto bits = [&](int i) { return rb::mask_bits<VEC>(mr, mask_stride, span.head + i * VEC); };
  rb::walk_groups<T, kThreads, rb::kPieces, kMask>(lr + span.head, span.nvec, bits, [&](const int4 (&raw)[rb::kPieces], int, bool whole) { run.add(raw, k, kMask || !whole); });
  if (run.again()) {
    run.sums = rb::Sums();
    rb::walk_groups<T, kThreads, rb::kPieces, kMask>(lr + span.head, span.nvec, bits,
                                 [&](const int4 (&raw)[rb::kPieces], int, bool) { rb::group_add<T, true, true>(raw, run.m, k, run.sums); });
  }
  rb::RowStats st = run.stats();
  const int j = span.edge(threadIdx.x, V);
  if (j >= 0 && !(kMask && (mr[j >> 3] >> (j & 7)) & 1)) st.one(rb::to_f(lr[j]), k);
  st = rb::block_stats(st, k, red);
  if (threadIdx.x == 0) {
    const rb::RowResult r(st, inv_temp);
    lse[row] = r.lse;
    entropy[row] = r.entropy;
    logp[row] = rb::label_logp(lr, labels[row], mr, V, inv_temp, r.lse);
  }
}

template <typename T, bool kMask>
__global__ void __launch_bounds__(kBwdThreads) token_stats_bwd_kernel(const T* logits, int64_t row_stride, const int64_t* __restrict__ labels,
                                                                      const uint8_t* __restrict__ mask, int64_t mask_stride, const float* __restrict__ lse_in,
                                                                      const float* __restrict__ entropy, const float* __restrict__ g_logp,
                                                                      const float* __restrict__ g_entropy, T* out, int64_t out_stride, int V, float inv_temp,
                                                                      int segs) {
  constexpr int VEC = rb::RowSpan<T>::VEC;
  const int64_t row = blockIdx.x / segs;
  const int seg = blockIdx.x - (int)(row * segs);
  const T* lr = logits + row * row_stride;
  T* orow = out + row * out_stride;
  const uint8_t* mr = kMask ? mask + row * mask_stride : nullptr;
  const float lse = lse_in[row], H = entropy[row];
  const int64_t given = labels[row];
  const float ge = g_entropy ? g_entropy[row] * inv_temp : 0.f;
  float gl = g_logp && given >= 0 ? g_logp[row] * inv_temp : 0.f;
  if (gl != 0.f && given >= V) gl = NAN;
  const bool zero = (gl == 0.f && ge == 0.f) || lse == -INFINITY;   // nothing asked of the row, or no token in it
  const bool kept = given >= 0 && given < V && !(kMask && (mr[given >> 3] >> (given & 7)) & 1);
  const int label = kept ? (int)given : -1;
  const float a = -(gl + ge * H);
  // a p - ge p y; a weight of 0 is 0 however low its logit
  auto grad = [&](float x) {
    const float y = fmaxf(fmaf(x, inv_temp, -lse), -1000.f);
    return zero ? 0.f : rb::exp2_fast(y * rb::kLog2e) * fmaf(-ge, y, a);
  };
  auto edge = [&](int j) {
    const float d = kMask && (mr[j >> 3] >> (j & 7)) & 1 ? (lse != lse && !zero ? NAN : 0.f) : grad(rb::to_f(lr[j]));
    return rb::from_f<T>(j == label && !zero ? d + gl : d);
  };
  const rb::RowSpan<T> span(lr, V);
  const bool same = ((reinterpret_cast<uintptr_t>(lr) ^ reinterpret_cast<uintptr_t>(orow)) & 15) == 0;
  if (same) {
    const int4* vecs = reinterpret_cast<const int4*>(lr + span.head);
    int4* outs = reinterpret_cast<int4*>(orow + span.head);
    int4 p[kBwdVecs];                        // all loads before the first use
    const int i0 = seg * kBwdVecs * kBwdThreads + threadIdx.x;
    if (zero) {
#pragma unroll
      for (int u = 0; u < kBwdVecs; ++u)
        if (i0 + u * kBwdThreads < span.nvec) __stcs(outs + i0 + u * kBwdThreads, make_int4(0, 0, 0, 0));
    } else {
      uint32_t gone[kBwdVecs];
#pragma unroll
      for (int u = 0; u < kBwdVecs; ++u) {
        const int i = i0 + u * kBwdThreads;
        if (i < span.nvec) {
          p[u] = rb::ld_once(vecs + i);
          if (kMask) gone[u] = rb::mask_bits<VEC>(mr, mask_stride, span.head + i * VEC);
        }
      }
      const uint64_t c2 = rb::pack2(inv_temp, inv_temp), l2 = rb::pack2(-lse, -lse), e2 = rb::pack2(rb::kLog2e, rb::kLog2e), g2 = rb::pack2(-ge, -ge),
                     a2 = rb::pack2(a, a);
#pragma unroll
      for (int u = 0; u < kBwdVecs; ++u) {
        const int i = i0 + u * kBwdThreads;
        if (i < span.nvec) {
          if (kMask) p[u] = rb::mask_piece<T>(p[u], gone[u]);
          T* v = reinterpret_cast<T*>(&p[u]);
          float d[VEC];
#pragma unroll
          for (int e = 0; e < VEC; e += 2) {
            float x0, x1;
            rb::unpack2(rb::fma2(rb::pack2(rb::to_f(v[e]), rb::to_f(v[e + 1])), c2, l2), x0, x1);
            const uint64_t y = rb::pack2(fmaxf(x0, -1000.f), fmaxf(x1, -1000.f));
            rb::unpack2(rb::mul2(y, e2), x0, x1);
            rb::unpack2(rb::mul2(rb::pack2(rb::exp2_fast(x0), rb::exp2_fast(x1)), rb::fma2(g2, y, a2)), d[e], d[e + 1]);
          }
          const int at = label - (span.head + i * VEC);
          if (at >= 0 && at < VEC) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[e] += e == at ? gl : 0.f;
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[e] = rb::from_f<T>(d[e]);
          __stcs(outs + i, p[u]);
        }
      }
    }
    if (seg == 0) {
      const int j = span.edge(threadIdx.x, V);
      if (j >= 0) orow[j] = edge(j);
    }
  } else {
    constexpr int per = kBwdThreads * kBwdVecs * VEC;
    const int j1 = seg == segs - 1 ? V : min(V, (seg + 1) * per);
    for (int j = seg * per + threadIdx.x; j < j1; j += kBwdThreads) orow[j] = edge(j);
  }
}

}  // namespace

extern "C" {

// dt: 0 fp32, 1 bf16, 2 fp16.  mask may be null; labels, logp, entropy, lse: [rows].
int rb_token_stats(const void* logits, int64_t row_stride, const int64_t* labels, const uint8_t* mask, int64_t mask_stride, float* logp, float* entropy,
                   float* lse, int64_t rows, int V, float inv_temp, int dt, cudaStream_t s) {
  if (rows == 0) return 0;
  const int nt = rb::row_threads(rows, V / (dt == 0 ? 4 : 8));
#define RB_L3(T, M, NT) token_stats_kernel<T, M, NT><<<(unsigned)rows, NT, 0, s>>>((const T*)logits, row_stride, labels, mask, mask_stride, logp, entropy, lse, V, inv_temp);
#define RB_L2(T, M) if (nt == 32) RB_L3(T, M, 32) else if (nt == 128) RB_L3(T, M, 128) else if (nt == 256) RB_L3(T, M, 256) else RB_L3(T, M, 512)
#define RB_L(T) if (mask) { RB_L2(T, true) } else { RB_L2(T, false) }
  if (dt == 0) { RB_L(float); } else if (dt == 1) { RB_L(__nv_bfloat16); } else if (dt == 2) { RB_L(__half); } else return -1;
#undef RB_L
#undef RB_L2
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

// g_logp / g_entropy: [rows] or null; out: [rows, V], may be the logits themselves.
int rb_token_stats_bwd(const void* logits, int64_t row_stride, const int64_t* labels, const uint8_t* mask, int64_t mask_stride, const float* lse,
                       const float* entropy, const float* g_logp, const float* g_entropy, void* out, int64_t out_stride, int64_t rows, int V, float inv_temp,
                       int dt, cudaStream_t s) {
  if (rows == 0) return 0;
  const int per = kBwdThreads * kBwdVecs * (dt == 0 ? 4 : 8);
  const int64_t segs = RB_CEIL_DIV((int64_t)V, per);
  if (rows * segs > 0x7fffffffLL) return -3;
#define RB_L2(T, M)                                                                                                                                        \
  token_stats_bwd_kernel<T, M><<<(unsigned)(rows * segs), kBwdThreads, 0, s>>>((const T*)logits, row_stride, labels, mask, mask_stride, lse, entropy, g_logp, \
                                                                               g_entropy, (T*)out, out_stride, V, inv_temp, (int)segs)
#define RB_L(T) if (mask) RB_L2(T, true); else RB_L2(T, false)
  if (dt == 0) { RB_L(float); } else if (dt == 1) { RB_L(__nv_bfloat16); } else if (dt == 2) { RB_L(__half); } else return -1;
#undef RB_L
#undef RB_L2
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // extern "C"
