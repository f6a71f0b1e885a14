// Log-probability of a given token and entropy of its distribution from logits [rows, V], forward and backward.
//
// Forward: one read of the row, statistics as in vocab_rows.cuh, one block a row.
// Backward, with y = x inv_temp - lse and p = e^y:   dx_j = inv_temp (g_logp (1[j = label] - p_j) - g_entropy p_j (y_j + H))
// element by element, in segments of a row.
#include "vocab_rows.cuh"

namespace {

constexpr int kBwdThreads = 256, kBwdVecs = 4;

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
  auto adjust = [&](int4 v, int i) { return kMask && i < span.nvec ? rb::mask_piece<T>(v, rb::mask8(mr, mask_stride, span.head + i * VEC)) : v; };
  rb::walk_groups<T, kThreads>(lr + span.head, span.nvec, adjust, [&](const int4 (&raw)[rb::kPieces], int, bool whole) { run.add(raw, k, kMask || !whole); });
  if (run.again()) {
    run.sums = rb::Sums();
    rb::walk_groups<T, kThreads>(lr + span.head, span.nvec, adjust,
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
  const int64_t label = labels[row];
  const float ge = g_entropy ? g_entropy[row] * inv_temp : 0.f;
  float gl = g_logp && label >= 0 ? g_logp[row] * inv_temp : 0.f;
  if (gl != 0.f && label >= V) gl = NAN;
  const bool zero = (gl == 0.f && ge == 0.f) || lse == -INFINITY;   // nothing asked of the row, or no token in it
  const float a = -(gl + ge * H);
  auto grad = [&](float x, int j, bool gone) {
    // d = a p - ge p y (+ gl at the label); a weight of 0 is 0 however low its logit
    const float y = fmaf(x, inv_temp, -lse);
    const float p = rb::exp2_fast(y * rb::kLog2e);
    float d = p == 0.f ? 0.f : p * fmaf(-ge, y, a);
    if (j == label) d += gl;
    return zero || gone ? 0.f : d;
  };
  const rb::RowSpan<T> span(lr, V);
  const bool same = ((reinterpret_cast<uintptr_t>(lr) ^ reinterpret_cast<uintptr_t>(orow)) & 15) == 0;
  if (same) {
    const rb::Pack<T, VEC>* vecs = reinterpret_cast<const rb::Pack<T, VEC>*>(lr + span.head);
    rb::Pack<T, VEC>* outs = reinterpret_cast<rb::Pack<T, VEC>*>(orow + span.head);
#pragma unroll
    for (int u = 0; u < kBwdVecs; ++u) {
      const int i = (seg * kBwdVecs + u) * kBwdThreads + threadIdx.x;
      if (i >= span.nvec) break;
      rb::Pack<T, VEC> p = vecs[i];
      const int j0 = span.head + i * VEC;
      const uint32_t gone = kMask ? rb::mask8(mr, mask_stride, j0) : 0u;
#pragma unroll
      for (int e = 0; e < VEC; ++e) p.v[e] = rb::from_f<T>(grad(rb::to_f(p.v[e]), j0 + e, (gone >> e) & 1));
      outs[i] = p;
    }
    if (seg == 0) {
      const int j = span.edge(threadIdx.x, V);
      if (j >= 0) orow[j] = rb::from_f<T>(grad(rb::to_f(lr[j]), j, kMask && (mr[j >> 3] >> (j & 7)) & 1));
    }
  } else {
    constexpr int per = kBwdThreads * kBwdVecs * VEC;
    const int j1 = seg == segs - 1 ? V : min(V, (seg + 1) * per);
    for (int j = seg * per + threadIdx.x; j < j1; j += kBwdThreads) orow[j] = rb::from_f<T>(grad(rb::to_f(lr[j]), j, kMask && (mr[j >> 3] >> (j & 7)) & 1));
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
