// Kullback-Leibler divergence between a teacher known by some tokens' log-probabilities and a student's logits, forward and backward.
//
// Outcomes b: the listed tokens one by one and, as one more, all tokens that are not listed.  Teacher: t_b, p_b = e^{t_b}; student, from
// y_j = x_j inv_temp - lse: y_b = y_id, y_rest = lse over the unlisted tokens - lse, q_b = e^{y_b}.
//   forward  L = sum_b p_b (t_b - y_b)     d L / d z_b = P q_b - p_b,       P = sum_b p_b
//   reverse  L = sum_b q_b (y_b - t_b)     d L / d z_b = q_b (y_b - t_b - L)
// and an unlisted token has the rest's times its share e^{x_j inv_temp - lse_rest} of it (a share is at most 1: dividing by q_rest could overflow).
// Without a rest the teacher is renormalised over its tokens and p_rest = 0 (forward only).
// The rest's mass is summed over the tokens it consists of, from a bitmap of the listed ones: 1 - sum q_b would cancel.
// A negative id is an unused place; an id given again counts where it stands first; an id beyond the vocabulary makes the row's loss NaN.
// p_b = 0 and q_b = 0 contribute 0.
//
// Bound by memory, one read forward and one read and write backward: 8192 x 32000 bf16 with 64 tokens 101 and 165 .. 170 us (5.2 and 6.2 TB/s).  The forward pass leaves what a row's gradient
// needs beside its logits: the listed tokens' own gradients, the rest's and its log-sum-exp.
#include "vocab_rows.cuh"

#include <type_traits>

namespace {

constexpr int kMaxListed = 1024, kMaxVocab = 1 << 20;
constexpr int kBwdThreads = 256, kBwdVecs = 4;

__host__ __device__ constexpr int bitmap_words(int V) { return (V + 16 + 31) / 32; }

struct DistillShared {
  float red[96];
  int dup;
  int ids[kMaxListed];
  float y[kMaxListed], t[kMaxListed];
};

RB_DEVICE float block_sum(float v, float* red) { return rb::block_reduce<false>(v, red); }

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) distill_fwd_kernel(const T* __restrict__ logits, int64_t row_stride, const int64_t* __restrict__ ids,
                                                               const float* __restrict__ top_logp, const float* __restrict__ rest_logp, int reverse,
                                                               float* __restrict__ loss, float* __restrict__ lse_rest_out, float* __restrict__ grad_rest,
                                                               float* __restrict__ grad_listed, int* __restrict__ ids_out, int V, int k, float inv_temp) {
  __shared__ DistillShared sh;
  constexpr int VEC = rb::RowSpan<T>::VEC;
  extern __shared__ uint32_t listed[];                  // a bit a token: bit 8 + j - head, so that a 16-byte piece's bits lie in one byte
  const int64_t row = blockIdx.x;
  const T* lr = logits + row * row_stride;
  const float kk = inv_temp * rb::kLog2e;
  const rb::RowSpan<T> span(lr, V);
  for (int i = threadIdx.x; i < bitmap_words(V); i += kThreads) listed[i] = 0;
  if (threadIdx.x == 0) sh.dup = 0;
  __syncthreads();
  bool beyond = false;
  for (int i = threadIdx.x; i < k; i += kThreads) {
    const int64_t id = ids[row * k + i];
    const bool ok = id >= 0 && id < V;
    beyond |= id >= V;
    sh.ids[i] = ok ? (int)id : -1;
    sh.t[i] = ok ? top_logp[row * k + i] : -INFINITY;
    sh.y[i] = ok ? rb::to_f(lr[id]) * inv_temp : -INFINITY;
    const int bit = ok ? 8 + (int)id - span.head : 0;
    if (ok && (atomicOr(&listed[bit >> 5], 1u << (bit & 31)) >> (bit & 31)) & 1) sh.dup = 1;
  }
  beyond = __syncthreads_or(beyond);
  if (sh.dup) {                                         // the first place of an id stands
    for (int i = threadIdx.x; i < k; i += kThreads) {
      bool again = false;
      const int id = sh.ids[i];
      for (int e = 0; e < i && id >= 0; ++e) again |= ids[row * k + e] == id;
      if (again) { sh.ids[i] = -1; sh.t[i] = -INFINITY; sh.y[i] = -INFINITY; }
    }
    __syncthreads();
  }
  // the row: every unlisted token's part of the rest
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(listed);
  rb::RunningStats<T, false> run;
  rb::walk_groups<T, kThreads, rb::kPieces, true>(
      lr + span.head, span.nvec, [&](int i) -> uint32_t { return VEC == 8 ? bytes[1 + i] : bytes[1 + (i >> 1)] >> ((i & 1) * 4) & 15; },
      [&](const int4 (&raw)[rb::kPieces], int, bool) { run.add(raw, kk, false); });
  rb::RowStats others = run.stats();
  const int ej = span.edge(threadIdx.x, V);
  if (ej >= 0 && !((listed[(8 + ej - span.head) >> 5] >> ((8 + ej - span.head) & 31)) & 1)) others.one(rb::to_f(lr[ej]), kk);
  others = rb::block_stats(others, kk, sh.red);
  const bool rest_empty = others.m == -INFINITY;
  const float lse_rest = others.m < INFINITY ? (rest_empty ? -INFINITY : fmaf(others.m, inv_temp, logf(others.s))) : NAN;
  // lse over the listed tokens and the rest; the teacher's over its listed ones where it is to be renormalised
  rb::RowStats all, teach;
  for (int i = threadIdx.x; i < k; i += kThreads) {
    all.one(sh.y[i], rb::kLog2e);
    teach.one(sh.t[i], rb::kLog2e);
  }
  if (threadIdx.x == 0) all.one(lse_rest, rb::kLog2e);
  all = rb::block_stats(all, rb::kLog2e, sh.red);
  const float lse = all.m < INFINITY ? (all.m == -INFINITY ? -INFINITY : all.m + logf(all.s)) : NAN;
  float tr = -INFINITY, shift = 0.f;
  if (rest_logp) {
    tr = rest_logp[row];
  } else {
    teach = rb::block_stats(teach, rb::kLog2e, sh.red);
    shift = teach.m == -INFINITY ? 0.f : teach.m + logf(teach.s);
  }
  const float base = lse == -INFINITY ? 0.f : lse;      // a row without a token: every y is -inf
  const float yr = lse_rest - base;
  float part = 0.f, mass = 0.f;
  for (int i = threadIdx.x; i <= k; i += kThreads) {
    const float y = i < k ? sh.y[i] - base : yr, t = i < k ? sh.t[i] - shift : tr;
    const float w = expf(reverse ? y : t);
    const float f = reverse ? y - t : t - y;
    if (w != 0.f) part += w * f;                        // (NaN included)
    mass += w;
  }
  float L = block_sum(part, sh.red);
  const float P = block_sum(mass, sh.red);
  if (beyond || lse != lse) L = NAN;
  auto grad = [&](float y, float t) {
    const float q = expf(y);
    if (!reverse) return P * q - expf(t);
    return q == 0.f ? 0.f : q * (y - t - L);
  };
  if (threadIdx.x == 0) {
    loss[row] = L;
    if (grad_rest) {
      lse_rest_out[row] = lse_rest;
      grad_rest[row] = L != L ? NAN : (rest_empty ? 0.f : grad(yr, tr));
    }
  }
  if (grad_rest)
    for (int i = threadIdx.x; i < k; i += kThreads) {
      ids_out[row * k + i] = sh.ids[i];
      grad_listed[row * k + i] = L != L ? NAN : grad(sh.y[i] - base, sh.t[i] - shift);
    }
}

// a piece of a row: as many elements of the gradient's type as 16 bytes of logits
RB_DEVICE void store_once(void* p, const int4& v) { __stcs(reinterpret_cast<int4*>(p), v); }
RB_DEVICE void store_once(void* p, const int2& v) { __stcs(reinterpret_cast<int2*>(p), v); }

// O: the gradient's type, the logits' own or, of fp32 logits, a 16-bit one
template <typename T, typename O>
__global__ void __launch_bounds__(kBwdThreads) distill_bwd_kernel(const T* logits, int64_t row_stride, const float* __restrict__ lse_rest_in,
                                                                  const float* __restrict__ grad_rest, const float* __restrict__ grad_listed,
                                                                  const int* __restrict__ ids, const float* __restrict__ g_loss,
                                                                  const uint32_t* __restrict__ peak, O* out, int64_t out_stride, int V, int k, float inv_temp,
                                                                  int segs) {
  constexpr int VEC = rb::RowSpan<T>::VEC, kPer = kBwdThreads * kBwdVecs * VEC;
  using Raw = std::conditional_t<sizeof(O) == sizeof(T), int4, int2>;
  const int64_t row = blockIdx.x / segs;
  const int seg = blockIdx.x - (int)(row * segs);
  const T* lr = logits + row * row_stride;
  O* orow = out + row * out_stride;
  const float g = g_loss[row] * inv_temp;
  float up = 1.f;                                       // (of products with g, which the peak bounds: g times it may leave fp32)
  if constexpr (std::is_same_v<T, float> && std::is_same_v<O, __half>) up = peak ? rb::grad_scale(*peak) : 1.f;
  const bool zero = g == 0.f;
  const int id0 = threadIdx.x < k ? ids[row * k + threadIdx.x] : -1;         // (asked for beside the logits, as the block ends with them)
  const float listed0 = threadIdx.x < k ? grad_listed[row * k + threadIdx.x] : 0.f;
  const float a = zero ? 0.f : g * grad_rest[row] * up, lr_rest = lse_rest_in[row];
  const float ref = lr_rest == -INFINITY ? 0.f : lr_rest;
  auto grad = [&](float x) {
    const float e = rb::exp2_fast(fmaf(x, inv_temp, -ref) * rb::kLog2e);
    return zero ? 0.f : a * e;
  };
  const rb::RowSpan<T> span(lr, V);
  const bool same = (reinterpret_cast<uintptr_t>(orow + span.head) & (sizeof(Raw) - 1)) == 0;
  int lo, hi;                                           // the elements of this block
  if (same) {
    const rb::Pack<T, VEC>* vecs = reinterpret_cast<const rb::Pack<T, VEC>*>(lr + span.head);
    Raw* outs = reinterpret_cast<Raw*>(orow + span.head);
    lo = seg == 0 ? 0 : span.head + seg * kPer;
    hi = seg == segs - 1 ? V : min(V, span.head + (seg + 1) * kPer);
    rb::Pack<T, VEC> p[kBwdVecs];                       // all loads before the first use
    const uint64_t c2 = rb::pack2(inv_temp, inv_temp), r2 = rb::pack2(-ref, -ref), e2 = rb::pack2(rb::kLog2e, rb::kLog2e), a2 = rb::pack2(a, a);
    const int i0 = seg * kBwdVecs * kBwdThreads + threadIdx.x;
#pragma unroll
    for (int u = 0; u < kBwdVecs; ++u)
      if (i0 + u * kBwdThreads < span.nvec) {
        const int4 v = rb::ld_once(reinterpret_cast<const int4*>(vecs + i0 + u * kBwdThreads));
        p[u] = *reinterpret_cast<const rb::Pack<T, VEC>*>(&v);
      }
#pragma unroll
    for (int u = 0; u < kBwdVecs; ++u) {
      const int i = i0 + u * kBwdThreads;
      if (zero && i < span.nvec) {
        store_once(outs + i, Raw{});
      } else if (i < span.nvec) {
        [[maybe_unused]] rb::Pack<O, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
          float x0, x1;
          rb::unpack2(rb::mul2(rb::fma2(rb::pack2(rb::to_f(p[u].v[e]), rb::to_f(p[u].v[e + 1])), c2, r2), e2), x0, x1);
          rb::unpack2(rb::mul2(rb::pack2(rb::exp2_fast(x0), rb::exp2_fast(x1)), a2), x0, x1);
          if constexpr (std::is_same_v<T, O>) {         // in the logits' registers: 8192 x 131072 656 us, 704 in others
            p[u].v[e] = rb::from_f<O>(x0);
            p[u].v[e + 1] = rb::from_f<O>(x1);
          } else {
            o.v[e] = rb::from_f<O>(x0);
            o.v[e + 1] = rb::from_f<O>(x1);
          }
        }
        store_once(outs + i, std::is_same_v<T, O> ? *reinterpret_cast<const Raw*>(&p[u]) : *reinterpret_cast<const Raw*>(&o));
      }
    }
    const int j = span.edge(threadIdx.x, V);
    if (j >= lo && j < hi) orow[j] = rb::from_f<O>(grad(rb::to_f(lr[j])));
  } else {
    lo = seg * kPer;
    hi = seg == segs - 1 ? V : min(V, (seg + 1) * kPer);
    for (int j = lo + threadIdx.x; j < hi; j += kBwdThreads) orow[j] = rb::from_f<O>(grad(rb::to_f(lr[j])));
  }
  __syncthreads();                                      // the listed tokens over what was just written
  if (id0 >= lo && id0 < hi) orow[id0] = rb::from_f<O>(zero ? 0.f : g * listed0 * up);
  for (int i = threadIdx.x + kBwdThreads; i < k; i += kBwdThreads) {
    const int id = ids[row * k + i];
    if (id >= lo && id < hi) orow[id] = rb::from_f<O>(zero ? 0.f : g * grad_listed[row * k + i] * up);
  }
}

// The largest gradient of a row's logits into the peak of all rows, a warp a row: an unlisted token's is at most the rest's.
__global__ void __launch_bounds__(128) distill_peak_kernel(const float* __restrict__ grad_rest, const float* __restrict__ grad_listed, const float* __restrict__ g_loss,
                                                           uint32_t* peak, int64_t rows, int k, float inv_temp) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const float g = fabsf(g_loss[row]) * inv_temp;
  float v = 0.f;
  for (int i = (threadIdx.x & 31) - 1; i < k; i += 32) {
    const float x = g * fabsf(i < 0 ? grad_rest[row] : grad_listed[row * k + i]);
    if (x < INFINITY) v = fmaxf(v, x);
  }
  rb::raise_peak(peak, v);
}

}  // namespace

extern "C" {

int rb_distill_max_listed() { return kMaxListed; }
int64_t rb_distill_max_vocab() { return kMaxVocab; }

// grad_rest null: no gradient asked for (then lse_rest, grad_listed and ids_out are null too).
int rb_distill_fwd(const void* logits, int64_t row_stride, const int64_t* ids, const float* top_logp, const float* rest_logp, int reverse, float* loss,
                   float* lse_rest, float* grad_rest, float* grad_listed, int* ids_out, int64_t rows, int V, int k, float inv_temp, int dt, cudaStream_t s) {
  if (rows == 0) return 0;
  if (k < 0 || k > kMaxListed || V > rb_distill_max_vocab() || (reverse && !rest_logp)) return -1;
  const int smem = bitmap_words(V) * 4;
  const int nt = rb::row_threads(rows, V / (dt == 0 ? 4 : 8));
#define RB_L2(T, NT)                                                                                                                                       \
  {                                                                                                                                                        \
    if (smem > 32768 && /* the most of any vocabulary: the limit is the process's, and another thread may be about to launch */                              \
        cudaFuncSetAttribute(distill_fwd_kernel<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, bitmap_words(kMaxVocab) * 4) != cudaSuccess)           \
      return -2;                                                                                                                                           \
    distill_fwd_kernel<T, NT><<<(unsigned)rows, NT, smem, s>>>((const T*)logits, row_stride, ids, top_logp, rest_logp, reverse, loss, lse_rest, grad_rest,  \
                                                               grad_listed, ids_out, V, k, inv_temp);                                                       \
  }
#define RB_L(T) if (nt == 32) RB_L2(T, 32) else if (nt == 128) RB_L2(T, 128) else if (nt == 256) RB_L2(T, 256) else RB_L2(T, 512)
  if (dt == 0) { RB_L(float) } else if (dt == 1) { RB_L(__nv_bfloat16) } else if (dt == 2) { RB_L(__half) } else return -1;
#undef RB_L
#undef RB_L2
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

// peak (zeroed before): a bound of all rows' gradients, for grad_scale
int rb_distill_peak(const float* grad_rest, const float* grad_listed, const float* g_loss, uint32_t* peak, int64_t rows, int k, float inv_temp, cudaStream_t s) {
  if (rows == 0) return 0;
  distill_peak_kernel<<<(unsigned)RB_CEIL_DIV(rows, 4), 128, 0, s>>>(grad_rest, grad_listed, g_loss, peak, rows, k, inv_temp);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

// out: [rows, V] of type out_dt (dt, or a 16-bit one for fp32 logits), may be the logits themselves; peak (fp32 logits, fp16 gradients): they leave times grad_scale of it, or null
int rb_distill_bwd(const void* logits, int64_t row_stride, const float* lse_rest, const float* grad_rest, const float* grad_listed, const int* ids,
                   const float* g_loss, const uint32_t* peak, void* out, int64_t out_stride, int64_t rows, int V, int k, float inv_temp, int dt, int out_dt,
                   cudaStream_t s) {
  if (rows == 0) return 0;
  const int per = kBwdThreads * kBwdVecs * (dt == 0 ? 4 : 8);
  const int64_t segs = RB_CEIL_DIV((int64_t)V, per);
  if (rows * segs > 0x7fffffffLL) return -3;
#define RB_L(T, O)                                                                                                                                     \
  distill_bwd_kernel<T, O><<<(unsigned)(rows * segs), kBwdThreads, 0, s>>>((const T*)logits, row_stride, lse_rest, grad_rest, grad_listed, ids, g_loss, peak,  \
                                                                           (O*)out, out_stride, V, k, inv_temp, (int)segs)
  if (peak && !(dt == 0 && out_dt == 2)) return -1;
  if (dt == 0 && out_dt == 0) RB_L(float, float);
  else if (dt == 0 && out_dt == 1) RB_L(float, __nv_bfloat16);
  else if (dt == 0 && out_dt == 2) RB_L(float, __half);
  else if (dt == 1 && out_dt == 1) RB_L(__nv_bfloat16, __nv_bfloat16);
  else if (dt == 2 && out_dt == 2) RB_L(__half, __half);
  else return -1;
#undef RB_L
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // extern "C"
