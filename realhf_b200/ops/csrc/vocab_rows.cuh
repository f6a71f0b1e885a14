// Rows of logits [rows, V]: how a block walks one, and the softmax statistics it gathers on the way.
//
// With k = inv_temp * log2(e) a row's statistics are M = max x, S = sum 2^((x - M) k) and W = sum (x - M) k 2^((x - M) k); from them
//   log-sum-exp  lse = M inv_temp + ln S          entropy  H = ln S - ln 2 * W / S
// S >= 1 and W <= 0, so the entropy is a sum of two terms >= 0 and nothing cancels (lse - sum p x would).  All in fp32.
// A masked token and a logit of -inf weigh nothing.  A row that holds a NaN or +inf has no softmax: its statistics are NaN.
//
// A thread takes the row in groups of four 16-byte pieces (32 16-bit or 16 fp32 logits), the next group's loads on their way while one is worked on.
// Per 16-bit logit: half an instruction for the maximum (two at once), one to unpack, half each for difference, scale and the two sums (f32x2), one exponential.
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
RB_DEVICE float warp_max_nan(float v) {
  float y;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(v));
  return y;
}

// two fp32 numbers in one instruction
RB_DEVICE uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
RB_DEVICE void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
RB_DEVICE uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
RB_DEVICE uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
RB_DEVICE uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// A 32-bit word of a row: two 16-bit logits, or one fp32.
template <typename T> struct Word;
template <> struct Word<__nv_bfloat16> {
  static constexpr int N = 2;
  static constexpr uint32_t kNone = 0xff80ff80u;  // -inf twice
  RB_DEVICE static uint32_t max(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  RB_DEVICE static void values(uint32_t a, float& lo, float& hi) { lo = __uint_as_float(a << 16); hi = __uint_as_float(a & 0xffff0000u); }
};
template <> struct Word<__half> {
  static constexpr int N = 2;
  static constexpr uint32_t kNone = 0xfc00fc00u;
  RB_DEVICE static uint32_t max(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  RB_DEVICE static void values(uint32_t a, float& lo, float& hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a));
    lo = f.x;
    hi = f.y;
  }
};
template <> struct Word<float> {
  static constexpr int N = 1;
  static constexpr uint32_t kNone = 0xff800000u;
};

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

// bits [j, j + N) of a packed mask row of `bytes` bytes, N <= 8
template <int N> RB_DEVICE uint32_t mask_bits(const uint8_t* m, int64_t bytes, int j) {
  uint32_t b = m[j >> 3];
  if ((j & 7) + N > 8 && (j >> 3) + 1 < bytes) b |= (uint32_t)m[(j >> 3) + 1] << 8;
  return b >> (j & 7);
}

// a piece that is read once; not through the read-only path, as gradients may take the logits' place
RB_DEVICE int4 ld_once(const int4* p) { return __ldcs(p); }

// a 16-byte piece whose elements with a bit set in `gone` become -inf
template <typename T> RB_DEVICE int4 mask_piece(int4 v, uint32_t gone) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Word<T>::N == 1) {
      if ((gone >> i) & 1) w[i] = Word<T>::kNone;
    } else {                                 // one half at a time (a mask built from two bits took twice the instructions)
      if ((gone >> (2 * i)) & 1) w[i] = __byte_perm(w[i], Word<T>::kNone, 0x3254);
      if ((gone >> (2 * i + 1)) & 1) w[i] = __byte_perm(w[i], Word<T>::kNone, 0x7610);
    }
  }
  return v;
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
  // bring the sums to another maximum `mn` >= m
  RB_DEVICE void to(float mn, float k) {
    const float d = m == mn ? 0.f : fmaxf((m - mn) * k, -1000.f), f = exp2_fast(d);
    w = f * fmaf(d, s, w);
    s *= f;
    m = mn;
  }
};

constexpr int kPieces = 4;  // 16-byte pieces of a group (the functions below take any number)

template <typename T, int P> RB_DEVICE float group_max(const int4 (&raw)[P]) {
  constexpr int NW = P * 4;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
  if constexpr (Word<T>::N == 2) {
    uint32_t m = w[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) m = Word<T>::max(m, w[i]);
    float a, b;
    Word<T>::values(m, a, b);
    return max_nan(a, b);
  } else {
    float m = __uint_as_float(w[0]);
#pragma unroll
    for (int i = 1; i < NW; ++i) m = max_nan(m, __uint_as_float(w[i]));
    return m;
  }
}

// A thread's sums against a reference, two at a time.
struct Sums {
  uint64_t s2 = 0, w2 = 0;
  RB_DEVICE float s() const { float a, b; unpack2(s2, a, b); return a + b; }
  RB_DEVICE float w() const { float a, b; unpack2(w2, a, b); return a + b; }
};

// Adds a group to sums against `ref`.  The difference comes before the scale: the largest token weighs exactly 1, and a row of one token has an
// entropy of 0.  Unless differences are clamped, a logit of -inf (or one further from the reference than fp32 reaches) adds nothing to S and makes W a NaN.
template <typename T, bool kEntropy, bool kClamp, int P> RB_DEVICE void group_add(const int4 (&raw)[P], float ref, float k, Sums& to) {
  constexpr int NW = P * 4, STEP = Word<T>::N == 2 ? 1 : 2;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
  const uint64_t k2 = pack2(k, k), ref2 = pack2(-ref, -ref);
#pragma unroll
  for (int i = 0; i < NW; i += STEP) {
    float a, b;
    if constexpr (Word<T>::N == 2) Word<T>::values(w[i], a, b);
    else { a = __uint_as_float(w[i]); b = __uint_as_float(w[i + 1]); }
    uint64_t d = mul2(add2(pack2(a, b), ref2), k2);
    unpack2(d, a, b);
    if (kClamp) {
      a = fmaxf(a, -1000.f);
      b = fmaxf(b, -1000.f);
      d = pack2(a, b);
    }
    const uint64_t e = pack2(exp2_fast(a), exp2_fast(b));
    to.s2 = add2(to.s2, e);
    if (kEntropy) to.w2 = fma2(d, e, to.w2);
  }
}

// A thread's statistics over groups: the sums run against the largest value so far (a merge of each group's own statistics cost 20 instructions a group).
template <typename T, bool kEntropy> struct RunningStats {
  float m = -INFINITY;
  Sums sums;
  RB_DEVICE float reference() const { return m == -INFINITY ? 0.f : m; }
  // make room for a group with the maximum mg
  RB_DEVICE void raise(float mg, float k) {
    if (!(mg <= m)) {
      const float mn = max_nan(m, mg), d = fmaxf((m - mn) * k, -1000.f), f = exp2_fast(d);
      const uint64_t f2 = pack2(f, f);
      if (kEntropy) sums.w2 = mul2(f2, fma2(pack2(d, d), sums.s2, sums.w2));
      sums.s2 = mul2(f2, sums.s2);
      m = mn;
    }
  }
  // `clamp`: the group may hold -inf
  template <int P> RB_DEVICE void add(const int4 (&raw)[P], float k, bool clamp) {
    raise(group_max<T>(raw), k);
    if (kEntropy && clamp) group_add<T, kEntropy, true>(raw, reference(), k, sums);
    else group_add<T, kEntropy, false>(raw, reference(), k, sums);
  }
  // W met a -inf: the row again, clamped
  RB_DEVICE bool again() const { const float w = sums.w(); return kEntropy && w != w && m < INFINITY; }
  RB_DEVICE RowStats stats() const {
    RowStats r;
    r.m = m;
    r.s = sums.s();
    r.w = sums.w();
    return r;
  }
};

// A row group by group.  `use(raw, i0, whole)` gets the group whose first piece is i0 (the others are i0 + n threads, ...); in a group that is not whole, pieces
// behind the row's end are -inf.  kBits: `bits(i)` gives the elements of piece i that become -inf.
template <typename T, int kThreads, int P, bool kBits, typename Bits, typename Use> RB_DEVICE void walk_groups(const T* aligned, int nvec, Bits bits, Use use) {
  const int4* v = reinterpret_cast<const int4*>(aligned);
  int4 raw[P], next[P];
  uint32_t gone[P], gone_next[P];
  constexpr int none = (int)Word<T>::kNone;
  auto fetch = [&](int4 (&r)[P], uint32_t (&g)[P], int i0) {
    if (i0 + (P - 1) * kThreads < nvec) {
#pragma unroll
      for (int u = 0; u < P; ++u) {
        r[u] = ld_stream(v + i0 + u * kThreads);
        if (kBits) g[u] = bits(i0 + u * kThreads);
      }
    } else {
#pragma unroll
      for (int u = 0; u < P; ++u) {
        const int i = i0 + u * kThreads;
        r[u] = i < nvec ? ld_stream(v + i) : make_int4(none, none, none, none);
        if (kBits) g[u] = i < nvec ? bits(i) : 0u;
      }
    }
  };
  int i0 = threadIdx.x;
  if (i0 < nvec) fetch(raw, gone, i0);
  while (i0 < nvec) {
    const int i1 = i0 + P * kThreads;
    if (i1 < nvec) fetch(next, gone_next, i1);
    if (kBits) {
#pragma unroll
      for (int u = 0; u < P; ++u) raw[u] = mask_piece<T>(raw[u], gone[u]);
    }
    use(raw, i0, i0 + (P - 1) * kThreads < nvec);
#pragma unroll
    for (int u = 0; u < P; ++u) {
      raw[u] = next[u];
      if (kBits) gone[u] = gone_next[u];
    }
    i0 = i1;
  }
}

// all threads' parts, in a fixed order, to every thread; red: 3 * 32 floats
RB_DEVICE RowStats block_stats(RowStats a, float k, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
  const float wm = warp_max_nan(a.m);
  a.to(wm, k);
  a.s = warp_sum(a.s);
  a.w = warp_sum(a.w);
  __syncthreads();
  if (lane == 0) { red[warp] = wm; red[32 + warp] = a.s; red[64 + warp] = a.w; }
  __syncthreads();
  RowStats r;
  if (lane < nwarp) { r.m = red[lane]; r.s = red[32 + lane]; r.w = red[64 + lane]; }
  r.to(warp_max_nan(r.m), k);
  r.s = warp_sum(r.s);
  r.w = warp_sum(r.w);
  return r;
}

// What a row's statistics come to.  `lse`, `entropy`: NaN for a row without a softmax, -inf and 0 for one that keeps no token.
struct RowResult {
  float lse, entropy;
  RB_DEVICE RowResult(const RowStats& r, float inv_temp) {
    const float top = r.m * inv_temp, ls = logf(r.s);       // (may leave fp32's range by its scale)
    const bool bad = !(top < INFINITY), none = top == -INFINITY;
    lse = bad ? NAN : (none ? -INFINITY : fmaf(r.m, inv_temp, ls));
    entropy = bad ? NAN : (none ? 0.f : ls - kLn2 * (r.w / r.s));
  }
};

// Threads a row.  Small blocks overlap the rows' ends, large ones shorten a row.  us, 16-bit logits, 128 / 256 / 512 threads: 8192 x 32000 94 / 100 / 115,
// 2048 x 131072 100 / 96 / 102, 300 x 32000 11.1 / 11.0 / 10.9, 1 x 131072 20.7 / 14.5 / 11.4 (launch included); 8192 x 2048 20.7 / 36.4 / 60.3: a group a thread.
inline int row_threads(int64_t rows, int64_t pieces) {
  if (pieces <= 256) return 32;
  if (pieces <= 1024 || rows >= 16 * kNumSMs) return 128;
  return rows >= 4 * kNumSMs ? 256 : 512;
}

// log-probability of a label: 0 for a negative one (no token), NaN for one beyond the vocabulary
template <typename T> RB_DEVICE float label_logp(const T* row, int64_t label, const uint8_t* mask, int V, float inv_temp, float lse) {
  if (label < 0) return 0.f;
  if (label >= V || lse != lse) return NAN;
  if (lse == -INFINITY || (mask && (mask[label >> 3] >> (label & 7)) & 1)) return -INFINITY;
  return fmaf(to_f(row[label]), inv_temp, -lse);
}

// The power of two that brings `peak` (the bits of a finite fp32 number >= 0, a bound of all gradients of logits) into [2^14, 2^15), 1 for a peak of 0.  Of the type fp16 the
// gradients of a mean over thousands of rows, a probability over thousands of tokens each, lie below the smallest number; scaled they keep 11 bits down to 2^-29 of the
// largest.  Exact to apply and to take back: both it and its reciprocal are normal numbers.
RB_DEVICE float grad_scale(uint32_t peak) {
  const int e = peak ? min(max(268 - (int)(peak >> 23), 1), 253) : 127;
  return __uint_as_float((uint32_t)e << 23);
}
RB_DEVICE float grad_unscale(uint32_t peak) { return __uint_as_float((254u << 23) - __float_as_uint(grad_scale(peak))); }
// a gradient's size into the peak of all of them; one that is no number takes no part (its row is NaN whatever the scale)
RB_DEVICE void raise_peak(uint32_t* peak, float v) {
  const float most = warp_max(v < INFINITY ? v : 0.f);
  if ((threadIdx.x & 31) == 0 && most > 0.f) atomicMax(peak, __float_as_uint(most));
}

}  // namespace rb
