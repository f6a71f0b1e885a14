// Rows of logits [rows, V]: how a block walks one, and the softmax statistics it gathers on the way.
//
// With k = inv_temp * log2(e) a row's statistics are M = max x, S = sum 2^((x - M) k) and W = sum (x - M) k 2^((x - M) k); from them
//   log-sum-exp  lse = M inv_temp + ln S          entropy  H = ln S - ln 2 * W / S
// S >= 1 and W <= 0, so the entropy is a sum of two terms >= 0 and nothing cancels (lse - sum p x would).  All in fp32.
// A masked token and a logit of -inf weigh nothing.  A row that holds a NaN or +inf has no softmax: its statistics are NaN.
#pragma once
#include "common.cuh"

namespace rb {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

RB_DEVICE float exp2_fast(float x) {  // 2 ulp; flushes below 2^-126, which is nothing beside a sum >= 1
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
RB_DEVICE float max_nan(float a, float b) {  // a NaN wins
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Where the 16-byte pieces of a row lie: `head` elements before the first 16-byte boundary, `nvec` whole pieces, then the tail.
template <typename T> struct RowSpan {
  static constexpr int VEC = 16 / sizeof(T);
  int head, nvec, tail0;  // tail0: first element behind the last whole piece
  RB_DEVICE RowSpan(const T* row, int V) {
    head = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T)));
    nvec = (V - head) / VEC;
    tail0 = head + nvec * VEC;
  }
  // the element outside the pieces that thread t takes, or -1 (at most 2 (VEC - 1) <= 14 of them)
  RB_DEVICE int edge(int t, int V) const {
    if (t < head) return t;
    const int j = tail0 + t - 16;
    return t >= 16 && j < V ? j : -1;
  }
};

// bits [j, j + 8) of a packed mask row of `bytes` bytes
RB_DEVICE uint32_t mask8(const uint8_t* m, int64_t bytes, int j) {
  uint32_t b = m[j >> 3];
  if ((j & 7) && (j >> 3) + 1 < bytes) b |= (uint32_t)m[(j >> 3) + 1] << 8;
  return b >> (j & 7);
}

struct RowStats {
  float m = -INFINITY, s = 0.f, w = 0.f;
  // merge another part of the same row; an empty part has s == 0
  RB_DEVICE void add(float m2, float s2, float w2, float k) {
    const float mn = max_nan(m, m2);
    const float d1 = m == mn ? 0.f : fmaxf((m - mn) * k, -1000.f), d2 = m2 == mn ? 0.f : fmaxf((m2 - mn) * k, -1000.f);
    const float f1 = exp2_fast(d1), f2 = exp2_fast(d2);
    w = f1 * fmaf(d1, s, w) + f2 * fmaf(d2, s2, w2);
    s = f1 * s + f2 * s2;
    m = mn;
  }
  RB_DEVICE void one(float x, float k) { if (x != -INFINITY) add(x, 1.f, 0.f, k); }
};

// N values of one thread at once: their maximum, then the sums against it
template <int N> RB_DEVICE void group_stats(const float (&x)[N], float k, float& m, float& s, float& w) {
  m = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = max_nan(m, x[i]);
  const float ref = m == -INFINITY ? 0.f : m;
  s = 0.f; w = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    // the difference first: the largest token weighs exactly 1, a row of one token has an entropy of 0.  (-inf: weight 2^-1000 = 0, and 0 times a finite d)
    const float d = fmaxf((x[i] - ref) * k, -1000.f);
    const float e = exp2_fast(d);
    s += e;
    w = fmaf(d, e, w);
  }
}

// all threads' parts, in a fixed order, to every thread; red: 3 * 32 floats
RB_DEVICE RowStats block_stats(RowStats a, float k, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m = __shfl_xor_sync(0xffffffffu, a.m, o), s = __shfl_xor_sync(0xffffffffu, a.s, o), w = __shfl_xor_sync(0xffffffffu, a.w, o);
    a.add(m, s, w, k);
  }
  __syncthreads();
  if (lane == 0) { red[warp] = a.m; red[32 + warp] = a.s; red[64 + warp] = a.w; }
  __syncthreads();
  RowStats r;
  if (lane < nwarp) { r.m = red[lane]; r.s = red[32 + lane]; r.w = red[64 + lane]; }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m = __shfl_xor_sync(0xffffffffu, r.m, o), s = __shfl_xor_sync(0xffffffffu, r.s, o), w = __shfl_xor_sync(0xffffffffu, r.w, o);
    r.add(m, s, w, k);
  }
  return r;
}

// What a row's statistics come to.  `lse`, `entropy`: NaN for a row without a softmax, -inf and 0 for one that keeps no token.
struct RowResult {
  float lse, entropy;
  RB_DEVICE RowResult(const RowStats& r, float inv_temp) {
    const bool bad = !(r.m < INFINITY);
    const float ls = logf(r.s);
    lse = bad ? NAN : (r.m == -INFINITY ? -INFINITY : fmaf(r.m, inv_temp, ls));
    entropy = bad ? NAN : (r.m == -INFINITY ? 0.f : ls - kLn2 * (r.w / r.s));
  }
};

// log-probability of a label: 0 for a negative one (no token), NaN for one beyond the vocabulary
template <typename T> RB_DEVICE float label_logp(const T* row, int64_t label, const uint8_t* mask, int V, float inv_temp, float lse) {
  if (label < 0) return 0.f;
  if (label >= V || lse != lse) return NAN;
  if (lse == -INFINITY || (mask && (mask[label >> 3] >> (label & 7)) & 1)) return -INFINITY;
  return fmaf(to_f(row[label]), inv_temp, -lse);
}

}  // namespace rb
