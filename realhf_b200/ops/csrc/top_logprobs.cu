// The k most likely tokens of every row of logits [rows, V] with their log-probabilities, the log of the mass of all other tokens, the log-probability
// of a given token and the entropy of the row.
//
// Order: larger logits first, equal ones by the lower index (-0 equals 0); a masked token and a logit of -inf are no alternatives, and a place that no
// token fills holds id -1 and -inf.  The rest's mass is summed over the tokens it consists of: 1 - sum of the chosen would cancel where they
// hold nearly all of it.
//
// The row is read once.  Every thread keeps, for each of its groups (vocab_rows.cuh), the maxima of its two halves (fp32: of the group) and its sum in shared
// memory.  The k-th largest of the maxima of 512 shares of the row, to 16 bits, is a lower bound of the k-th largest logit: k shares hold an element at least as large;
// only some k .. 2 k elements reach it.  The halves whose maximum does are read again, a lane a half, and give the candidates; the mass of the rest is the groups'
// sums less their candidates', or, where candidates are more than 64 times what is left, the group's other elements added up again.  (With whole groups read
// again, pieces of 64 bytes in memory that the cache had dropped, 256 alternatives of 8192 x 32000 read 1.6 times the logits.)  A candidate's place is the number of
// candidates before it in the order: counted among all of them where they are few, else among those of its bucket, 512 equal intervals of the value (a bitonic sort of
// 128, a barrier for each of its 28 stages, took 7400 cycles; counting among 400 by 128 threads 28000).
// More than 256 alternatives, or nearly as many as the row has pieces: room for 2048 candidates, and the bound from the halves' own maxima, counted by all threads bit by bit.
// (300 of 4096 x 32000: 182 us, 1000: 373; the descent took 1080 and 1210.)
// More candidates or halves than there is room for (ties) and rows of more than 12288 groups take a radix descent instead: the k-th largest value by its bits
// (digits of 8 bits, a histogram in shared memory each: two in bf16, three in fp16, four in fp32), the elements above it in any order, of those equal to it the first in
// index order.
// Sums have a fixed order whichever way candidates arrive.
//
// A row of equal logits: 4096 x 32000 in 457 us, 896 before the descent left the digits out that a 16-bit type does not have.
//
// bf16, us: 8192 x 32000 with 20 / 64 / 256 alternatives 130 / 146 / 205, 4096 x 131072 with 64 212 .. 224 (4.8 .. 5.1 TB/s); the statistics alone take 95 and 170 .. 185.  Bound by issue slots (66 %):
// ten instructions a logit, a fifth of them for bound, candidates and order.
#include "vocab_rows.cuh"

#include <algorithm>

namespace {

constexpr int kMaxTop = 1024;
constexpr int kShares = 512;

RB_DEVICE uint32_t order_key(float x) {  // order-preserving float -> uint, -0 as 0
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
RB_DEVICE float key_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
constexpr uint32_t kKeyNone = 0x007fffffu;  // order_key(-inf)

constexpr int kFastTop = 256, kMaxRecords = 12288, kCountAll = 128;
constexpr int kCap = 1024, kBigCap = 2048;   // candidates of a block
constexpr int kMaxSmem = kMaxRecords * 8;    // dynamic shared memory at most: records, later the candidates by buckets
static_assert(kMaxSmem >= kBigCap * 8);

template <int kCand> struct TopShared {
  static constexpr int kHalves = kCand == kCap ? 768 : kCand;
  float red[96];
  uint32_t warp_n[32];
  uint32_t digit, above, count, selected, kth;
  int last;
  int reach[16];
  alignas(16) uint64_t list[kCand];   // key << 32 | ~index: descending order is the order wanted
  union {                               // one after the other
    uint32_t keys[kShares];
    struct {
      uint32_t half[kHalves];           // halves to look at again: 2 * group + which, groups numbered step * threads + thread
      float hit_sum[kHalves];           // their candidates' sums
    };
    uint32_t hist[kShares];
    float after[kCountAll * 2];
  };
};

// What a group's record says of its maxima: of 16-bit types those of the first and the second half of its pieces, side by side; of fp32 the whole group's.  Returns the
// group's maximum.
template <typename T, int P> constexpr int kHalfPieces = rb::Word<T>::N == 2 && P > 1 ? P / 2 : P;
template <typename T, int P> RB_DEVICE float half_maxima(const int4 (&raw)[P], uint32_t& halves) {
  if constexpr (rb::Word<T>::N == 1) {
    const float m = rb::group_max<T>(raw);
    halves = __float_as_uint(m);
    return m;
  } else {
    constexpr int NW = P * 4, HW = kHalfPieces<T, P> * 4;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
    uint32_t a = w[0], b = HW == NW ? rb::Word<T>::kNone : w[HW % NW];
#pragma unroll
    for (int i = 1; i < HW; ++i) a = rb::Word<T>::max(a, w[i]);
#pragma unroll
    for (int i = HW + 1; i < NW; ++i) b = rb::Word<T>::max(b, w[i]);
    halves = rb::Word<T>::max(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
    float lo, hi;
    rb::Word<T>::values(halves, lo, hi);
    return rb::max_nan(lo, hi);
  }
}
template <typename T> RB_DEVICE void half_values(uint32_t halves, float& lo, float& hi) {
  if constexpr (rb::Word<T>::N == 2) {
    rb::Word<T>::values(halves, lo, hi);
  } else {
    lo = __uint_as_float(halves);
    hi = -INFINITY;
  }
}

template <typename T> struct TopRow {
  const T* lr;
  const uint8_t* mr;
  int64_t mask_row;
  int V;
  RB_DEVICE float at(int j) const { return mr && (mr[j >> 3] >> (j & 7)) & 1 ? -INFINITY : rb::to_f(lr[j]); }
};

// f(logit, index) for every element of the row, whole pieces a thread
template <int kThreads, typename T, typename F> RB_DEVICE void for_each(const TopRow<T>& r, F f) {
  constexpr int VEC = rb::RowSpan<T>::VEC;
  const rb::RowSpan<T> span(r.lr, r.V);
  const int4* v = reinterpret_cast<const int4*>(r.lr + span.head);
  const int ej = span.edge(threadIdx.x, r.V);
  if (ej >= 0) f(r.at(ej), ej);
  for (int i = threadIdx.x; i < span.nvec; i += kThreads) {
    int4 raw = __ldg(v + i);
    const int j0 = span.head + i * VEC;
    if (r.mr) raw = rb::mask_piece<T>(raw, rb::mask_bits<VEC>(r.mr, r.mask_row, j0));
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int c = 0; c < VEC; ++c) f(rb::to_f(e[c]), j0 + c);
  }
}

// The k largest (key, ~index) of the row -> sh.list in any order; returns how many there are (less than k where the row keeps fewer tokens), and in
// sh.kth the k-th largest value's key.
template <int kThreads, typename T, typename Shared> RB_DEVICE int select_radix(const TopRow<T>& r, int k, Shared& sh) {
  constexpr int kDigits = sizeof(T) == 4 ? 4 : rb::Word<T>::kNone == 0xfc00fc00u ? 3 : 2;      // the digits that differ: as fp32, 16-bit types end in zeros
  uint32_t prefix = 0, want = k;      // the want-th largest among the elements whose high digits are `prefix`
  for (int shift = 24; shift >= 32 - 8 * kDigits; shift -= 8) {
    for (int b = threadIdx.x; b < 256; b += kThreads) sh.hist[b] = 0;
    __syncthreads();
    uint32_t same = 0, run = 0;       // a thread's equal digits in a row: one addition
    for_each<kThreads>(r, [&](float x, int) {
      const uint32_t key = order_key(x), digit = (key >> shift) & 255;
      if (shift == 24 || (key >> (shift + 8)) == prefix) {
        if (digit != same) {
          if (run) atomicAdd(&sh.hist[same], run);
          same = digit;
          run = 0;
        }
        ++run;
      }
    });
    if (run) atomicAdd(&sh.hist[same], run);
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t left = want;
      int b = 255;
      while (b > 0 && sh.hist[b] < left) left -= sh.hist[b--];
      sh.digit = b;
      sh.above = left;
    }
    __syncthreads();
    prefix = prefix << 8 | sh.digit;
    want = sh.above;
    __syncthreads();
  }
  if constexpr (kDigits < 4) {        // (a negative number's key is its complement: ends in ones)
    const bool positive = (prefix >> (8 * kDigits - 1)) & 1;
    prefix = prefix << (32 - 8 * kDigits) | (positive ? 0u : (1u << (32 - 8 * kDigits)) - 1u);
  }
  const uint32_t kth = prefix;
  if (threadIdx.x == 0) {
    sh.count = 0;
    sh.kth = max(kth, kKeyNone);
  }
  __syncthreads();
  for_each<kThreads>(r, [&](float x, int j) {
    const uint32_t key = order_key(x);
    if (key > kth && key > kKeyNone) sh.list[atomicAdd(&sh.count, 1u)] = (uint64_t)key << 32 | (uint32_t)~j;
  });
  __syncthreads();
  const int above = sh.count, need = kth > kKeyNone ? k - above : 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int found = 0;
  for (int j0 = 0; j0 < r.V && found < need; j0 += kThreads) {
    const int j = j0 + threadIdx.x;
    const bool hit = j < r.V && order_key(r.at(j)) == kth;
    const uint32_t b = __ballot_sync(0xffffffffu, hit);
    if (lane == 0) sh.warp_n[warp] = __popc(b);
    __syncthreads();
    int at = found, all = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
      const int n = sh.warp_n[i];
      if (i < warp) at += n;
      all += n;
    }
    at += __popc(b & ((1u << lane) - 1u));
    if (hit && at < need) sh.list[above + at] = (uint64_t)kth << 32 | (uint32_t)~j;
    found += all;
    __syncthreads();
  }
  return above + need;
}

// The largest t, to the upper 16 bits of a key, that at least k of the shares' keys reach; by warp 0, N keys a lane (kShares / 32 / N shares taken together:
// k of the fewer and larger ones bound as well while k is a quarter of them at most).  Only the bits in which the keys differ are searched.
template <int N> RB_DEVICE uint32_t bound_of(int k, const uint32_t* keys) {
  uint32_t key[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    key[i] = 0;
#pragma unroll
    for (int e = 0; e < kShares / 32 / N; ++e) key[i] = max(key[i], keys[(e * N + i) * 32 + threadIdx.x] >> 16);
  }
  uint32_t hi = 0, lo = ~0u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    hi = max(hi, key[i]);
    lo = min(lo, key[i]);
  }
  hi = __reduce_max_sync(0xffffffffu, hi);
  lo = __reduce_min_sync(0xffffffffu, lo);
  const int bits = 32 - __clz(hi ^ lo);
  uint32_t t = hi >> bits << bits;
#pragma unroll 1
  for (int bit = bits - 1; bit >= 0; --bit) {
    const uint32_t c = t | 1u << bit;
    int n[2] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) n[i & 1] += key[i] >= c;
    if (__reduce_add_sync(0xffffffffu, n[0] + n[1]) >= k) t = c;
  }
  return t << 16;
}

// how many of list[0, n) are larger than `mine`; the list is padded with zeros to an even number
RB_DEVICE int larger_than(uint64_t mine, const uint64_t* list, int n) {
  int rank = 0;
#pragma unroll 4
  for (int i = 0; i < n; i += 2) {
    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(list + i);
    rank += v.x > mine;
    rank += v.y > mine;
  }
  return rank;
}

template <typename T, bool kMask, int kThreads, int P, int kCand>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) top_logprobs_kernel(const T* __restrict__ logits, int64_t row_stride,
                                                                                 const int64_t* __restrict__ labels, const uint8_t* __restrict__ mask,
                                                                                 int64_t mask_stride, float* __restrict__ logp, float* __restrict__ entropy,
                                                                                 float* __restrict__ top_logp, int64_t* __restrict__ top_ids,
                                                                                 float* __restrict__ rest, int V, int k, float inv_temp, int records) {
  constexpr int VEC = rb::RowSpan<T>::VEC, kStep = P * kThreads;
  constexpr int kHalves = TopShared<kCand>::kHalves;
  __shared__ TopShared<kCand> sh;
  extern __shared__ uint2 rec[];            // [step][thread]: maxima of a group's halves, its sum; later the list by buckets
  const int64_t row = blockIdx.x;
  const TopRow<T> r{logits + row * row_stride, kMask ? mask + row * mask_stride : nullptr, mask_stride, V};
  const float kk = inv_temp * rb::kLog2e;
  const rb::RowSpan<T> span(r.lr, V);
  const int lane = threadIdx.x & 31;
  const bool fast = records > 0;
  constexpr int B = kShares / kThreads;
  float share[B];                           // maxima of the thread's shares: every so many-th group each, the edge with the first
#pragma unroll
  for (int b = 0; b < B; ++b) share[b] = -INFINITY;
  rb::RunningStats<T, true> run;
  auto bits = [&](int i) { return rb::mask_bits<VEC>(r.mr, mask_stride, span.head + i * VEC); };
  rb::walk_groups<T, kThreads, P, kMask>(r.lr + span.head, span.nvec, bits, [&](const int4 (&raw)[P], int i0, bool whole) {
    uint32_t halves;
    const float mg = half_maxima<T>(raw, halves);
    run.raise(mg, kk);
    rb::Sums g;
    if (kMask || !whole) rb::group_add<T, true, true>(raw, run.reference(), kk, g);
    else rb::group_add<T, true, false>(raw, run.reference(), kk, g);
    run.sums.s2 = rb::add2(run.sums.s2, g.s2);
    run.sums.w2 = rb::add2(run.sums.w2, g.w2);
    if (fast) {
      const int step = i0 / kStep;
      rec[step * kThreads + threadIdx.x] = make_uint2(halves, __float_as_uint(g.s()));
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (step % B == b) share[b] = fmaxf(share[b], mg);
    }
  });
  if (run.again()) {
    run.sums.w2 = 0;
    rb::walk_groups<T, kThreads, P, kMask>(r.lr + span.head, span.nvec, bits, [&](const int4 (&raw)[P], int, bool) {
      rb::Sums g;
      rb::group_add<T, true, true>(raw, run.m, kk, g);
      run.sums.w2 = rb::add2(run.sums.w2, g.w2);
    });
  }
  rb::RowStats st = run.stats();
  const int ej = span.edge(threadIdx.x, V);
  const float ex = ej >= 0 ? r.at(ej) : -INFINITY;
  st.one(ex, kk);
  const int groups = RB_CEIL_DIV(max(0, span.nvec - (int)threadIdx.x), kStep);
  st = rb::block_stats(st, kk, sh.red);
  const rb::RowResult res(st, inv_temp);
  if (threadIdx.x == 0) {
    entropy[row] = res.entropy;
    if (logp) logp[row] = rb::label_logp(r.lr, labels[row], r.mr, V, inv_temp, res.lse);
    sh.count = sh.selected = 0;
    sh.kth = kKeyNone;      // where fewer than k tokens are kept there is no rest
    sh.last = V;
  }
  if (!(fabsf(res.lse) < INFINITY)) {     // no softmax, or no token
    for (int i = threadIdx.x; i < k; i += kThreads) {
      top_logp[row * k + i] = res.lse;
      top_ids[row * k + i] = -1;
    }
    if (threadIdx.x == 0) rest[row] = res.lse;
    return;
  }
  float left = 0.f;                         // the rest's sum against the row's maximum
  int n = kCand + 1;
  float lowest = 0.f;                       // no candidate lies below
  if (fast) {
    if constexpr (kCand == kCap) {
#pragma unroll
      for (int b = 0; b < B; ++b) sh.keys[b * kThreads + threadIdx.x] = order_key(b == 0 ? fmaxf(share[0], ex) : share[b]);
    } else {
      if (threadIdx.x < 16) sh.reach[threadIdx.x] = 0;
    }
    // a group's sum was taken against the thread's largest value so far: bring it to the row's
    float so_far = -INFINITY;
    for (int g = 0; g < groups; ++g) {
      uint2& v = rec[g * kThreads + threadIdx.x];
      float lo, hi;
      half_values<T>(v.x, lo, hi);
      so_far = fmaxf(so_far, fmaxf(lo, hi));
      v.y = __float_as_uint(__uint_as_float(v.y) * rb::exp2_fast(fmaxf((so_far - st.m) * kk, -1000.f)));
    }
    __syncthreads();
    uint32_t bound = 0;
    if constexpr (kCand == kCap) {
      if (threadIdx.x < 32) {
        const uint32_t t = k <= 32 ? bound_of<4>(k, sh.keys) : k <= 64 ? bound_of<8>(k, sh.keys) : bound_of<kShares / 32>(k, sh.keys);
        if (threadIdx.x == 0) sh.digit = t;
      }
      __syncthreads();
      bound = sh.digit;
    } else {
      for (int bit = 15; bit >= 0; --bit) {   // (below -inf there are NaNs, which nothing reaches: the bound stays at 0)
        const uint32_t c = bound | 1u << (16 + bit);
        const float x = key_value(c);
        int reach = ex >= x;
        for (int g = 0; g < groups; ++g) {
          float lo, hi;
          half_values<T>(rec[g * kThreads + threadIdx.x].x, lo, hi);
          reach += (lo >= x) + (hi >= x);
        }
        reach = __reduce_add_sync(0xffffffffu, reach);
        if (lane == 0 && reach) atomicAdd(&sh.reach[bit], reach);
        __syncthreads();
        if (sh.reach[bit] >= k) bound = c;
      }
    }
    bound = max(bound, kKeyNone + 1);
    const float bound_x = lowest = key_value(bound);
    // places in `half` or `list` for the bits set in a lane's mask: one addition a warp
    auto places = [&](uint32_t hits, uint32_t& count) {
      const int mine = __popc(hits);
      int before = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      uint32_t at = 0;
      if (lane == 31 && before) at = atomicAdd(&count, (uint32_t)before);
      return __shfl_sync(0xffffffffu, at, 31) + before - mine;
    };
    const int all_groups = RB_CEIL_DIV(span.nvec, kStep);
    for (int g0 = 0; g0 < all_groups; g0 += 16) {
      uint32_t hits = 0;
      for (int g = g0; g < min(groups, g0 + 16); ++g) {
        float lo, hi;
        half_values<T>(rec[g * kThreads + threadIdx.x].x, lo, hi);
        hits |= ((uint32_t)(lo >= bound_x) | (uint32_t)(hi >= bound_x) << 1) << (2 * (g - g0));
      }
      uint32_t at = places(hits, sh.selected);
      for (; hits; hits &= hits - 1, ++at) {
        const int b = __ffs(hits) - 1;
        if (at < kHalves) sh.half[at] = 2 * ((g0 + b / 2) * kThreads + threadIdx.x) + (b & 1);
      }
    }
    if (threadIdx.x < 32) {
      const uint32_t at = places(ex >= bound_x, sh.count);
      if (ex >= bound_x) sh.list[at] = (uint64_t)order_key(ex) << 32 | (uint32_t)~ej;
    }
    __syncthreads();
    const int selected = sh.selected;
    if (selected <= kHalves) {
      constexpr int HP = kHalfPieces<T, P>;
      const int4* v = reinterpret_cast<const int4*>(r.lr + span.head);
      auto piece_of = [&](int id) { return id / kThreads * kStep + id % kThreads; };
      auto fetch = [&](int i) {
        constexpr int none = (int)rb::Word<T>::kNone;
        int4 raw = i < span.nvec ? __ldg(v + i) : make_int4(none, none, none, none);
        if (kMask && i < span.nvec) raw = rb::mask_piece<T>(raw, rb::mask_bits<VEC>(r.mr, mask_stride, span.head + i * VEC));
        return raw;
      };
      for (int q0 = 0; q0 < selected; q0 += kThreads) {
        const int q = q0 + threadIdx.x;
        const bool on = q < selected;
        const int what = on ? sh.half[q] : 0, first = piece_of(what >> 1) + (what & 1) * HP * kThreads;
        int4 raw[HP];
#pragma unroll
        for (int u = 0; u < HP; ++u) raw[u] = fetch(on ? first + u * kThreads : span.nvec);
        uint32_t hits = 0;
        float s = 0.f;
#pragma unroll
        for (int u = 0; u < HP; ++u) {
          const T* e = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
          for (int c = 0; c < VEC; ++c) {
            const float x = rb::to_f(e[c]);
            if (x >= bound_x) {
              hits |= 1u << (u * VEC + c);
              s += rb::exp2_fast((x - st.m) * kk);
            }
          }
        }
        if (on) sh.hit_sum[q] = s;
        uint32_t at = places(hits, sh.count);
        for (; hits; hits &= hits - 1, ++at) {
          const int b = __ffs(hits) - 1, j = span.head + (first + b / VEC * kThreads) * VEC + b % VEC;
          if (at < kCand) sh.list[at] = (uint64_t)order_key(rb::to_f(r.lr[j])) << 32 | (uint32_t)~j;
        }
      }
      __syncthreads();
      n = sh.count;
      // the groups' sums without their candidates; a group's halves lie side by side in the list
      for (int q = threadIdx.x; q < selected; q += kThreads) {
        const int id = sh.half[q] >> 1;
        if (q > 0 && (int)(sh.half[q - 1] >> 1) == id) continue;
        const float h = sh.hit_sum[q] + (q + 1 < selected && (int)(sh.half[q + 1] >> 1) == id ? sh.hit_sum[q + 1] : 0.f);
        float s = __uint_as_float(rec[id].y) - h;
        if (!(s * 64.f >= h)) {
          s = 0.f;
#pragma unroll
          for (int u = 0; u < P; ++u) {
            const int4 raw = fetch(piece_of(id) + u * kThreads);
            const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
              const float x = rb::to_f(e[c]);
              s += x >= bound_x ? 0.f : rb::exp2_fast(fmaxf((x - st.m) * kk, -1000.f));
            }
          }
        }
        rec[id].y = __float_as_uint(s);
      }
      __syncthreads();
    }
    if (n <= kCand) {
      for (int g = 0; g < groups; ++g) left += __uint_as_float(rec[g * kThreads + threadIdx.x].y);
      if (ex != -INFINITY && !(ex >= bound_x)) left += rb::exp2_fast((ex - st.m) * kk);
    }
  }
  const bool listed = n <= kCand;
  if (!listed) {
    __syncthreads();
    n = select_radix<kThreads>(r, k, sh);
    lowest = key_value(sh.kth);
    __syncthreads();
  }
  uint64_t* ordered = reinterpret_cast<uint64_t*>(rec);
  auto place = [&](uint64_t c, int at, float* after) {
    const float x = key_value((uint32_t)(c >> 32));
    const int j = (int)~(uint32_t)c;
    if (at < k) {
      top_logp[row * k + at] = fmaf(x, inv_temp, -res.lse);
      top_ids[row * k + at] = j;
      if (at == k - 1) { sh.kth = (uint32_t)(c >> 32); sh.last = j; }
    } else {
      after[at - k] = x;
    }
  };
  float* after;                             // candidates that are not chosen, in order
  if (n <= kCountAll) {
    after = sh.after;
    if (threadIdx.x == 0 && (n & 1)) sh.list[n] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) place(sh.list[i], larger_than(sh.list[i], sh.list, n), after);
  } else {
    after = reinterpret_cast<float*>(sh.list);
    if (lowest <= key_value(kKeyNone + 1)) {  // every token: the buckets begin at the smallest one there is
      __syncthreads();
      float m = -INFINITY;
      for (int i = threadIdx.x; i < n; i += kThreads) m = fmaxf(m, -key_value((uint32_t)(sh.list[i] >> 32)));
      lowest = -rb::block_reduce<true>(m, sh.red);
    }
    const float width = st.m - lowest, scale = width > 0.f && width < INFINITY ? (kShares - 1) / width : 0.f;
    auto bucket = [&](uint64_t c) { return min(kShares - 1, (int)((st.m - key_value((uint32_t)(c >> 32))) * scale)); };
    for (int b = threadIdx.x; b < kShares; b += kThreads) sh.hist[b] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) atomicAdd(&sh.hist[bucket(sh.list[i])], 1u);
    __syncthreads();
    if (threadIdx.x < 32) {                 // counts -> where the buckets begin
      uint32_t c[kShares / 32], sum = 0;
#pragma unroll
      for (int i = 0; i < kShares / 32; ++i) {
        c[i] = sh.hist[lane * (kShares / 32) + i];
        sum += c[i];
      }
      uint32_t before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      before -= sum;
#pragma unroll
      for (int i = 0; i < kShares / 32; ++i) {
        sh.hist[lane * (kShares / 32) + i] = before;
        before += c[i];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) ordered[atomicAdd(&sh.hist[bucket(sh.list[i])], 1u)] = sh.list[i];
    __syncthreads();                        // hist: where the buckets end
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t c = ordered[i];
      const int b = bucket(c), begin = b > 0 ? sh.hist[b - 1] : 0, end = sh.hist[b];
      int at = begin;
      for (int e = begin; e < end; ++e) at += ordered[e] > c;
      place(c, at, after);
    }
  }
  for (int i = n + threadIdx.x; i < k; i += kThreads) {
    top_logp[row * k + i] = -INFINITY;
    top_ids[row * k + i] = -1;
  }
  __syncthreads();
  // the others: below the k-th value, or equal to it behind the last chosen index
  const uint32_t kth = sh.kth;
  const int last = sh.last;
  auto other = [&](float x, int j) {
    const uint32_t key = order_key(x);
    return key < kth || (key == kth && j > last);
  };
  if (listed) {
    for (int i = threadIdx.x; i < n - k; i += kThreads) left += rb::exp2_fast(fmaxf((after[i] - st.m) * kk, -1000.f));
  } else {
    for_each<kThreads>(r, [&](float x, int j) { left += other(x, j) ? rb::exp2_fast(fmaxf((x - st.m) * kk, -1000.f)) : 0.f; });
  }
  left = rb::block_reduce<false>(left, sh.red);
  if (left > 1e-18f) {
    if (threadIdx.x == 0) rest[row] = logf(left) - logf(st.s);
    return;
  }
  // too small beside the largest logit to be summed against it: against their own
  rb::RowStats others;
  for_each<kThreads>(r, [&](float x, int j) {
    if (other(x, j)) others.one(x, kk);
  });
  others = rb::block_stats(others, kk, sh.red);
  if (threadIdx.x == 0) rest[row] = rb::RowResult(others, inv_temp).lse - res.lse;
}

}  // namespace

extern "C" {

int rb_top_logprobs_max() { return kMaxTop; }

// labels and logp may be null together; 1 <= k <= min(V, kMaxTop).
int rb_top_logprobs(const void* logits, int64_t row_stride, const int64_t* labels, const uint8_t* mask, int64_t mask_stride, float* logp, float* entropy,
                    float* top_logp, int64_t* top_ids, float* rest, int64_t rows, int V, int k, float inv_temp, int dt, cudaStream_t s) {
  if (rows == 0) return 0;
  if (k < 1 || k > kMaxTop || k > V) return -1;
  const int vec = V / (dt == 0 ? 4 : 8);
  const bool big = k > kFastTop || (V > kCap && vec < k + k / 8);
  // pieces a group: one where groups of four (halves of them) are too few to bound the k-th logit
  const int p = vec >= (!big ? 8 : dt == 0 ? 10 : 5) * k ? 4 : 1;
  // threads: as for the statistics, but no fewer than keep 1024 resident beside what a block has in shared memory
  const int64_t bytes = sizeof(TopShared<kCap>) + 1024 + std::max<int64_t>((int64_t)vec / p * 8, kCap * 8);
  const int nt = big ? 256 : rows < 4 * rb::kNumSMs ? 512 : rows >= 16 * rb::kNumSMs && bytes <= 45 << 10 ? 128 : 256;
#define RB_L4(T, M, NT, P, C)                                                                                                                              \
  {                                                                                                                                                        \
    const int groups = RB_CEIL_DIV(vec, P * NT);                                                                                                           \
    const bool fast = groups * NT <= kMaxRecords;                                                                                                          \
    const int smem = std::max(fast ? groups * NT * (int)sizeof(uint2) : 0, C * 8);                                                                         \
    if (smem + (int)sizeof(TopShared<C>) > 48 << 10 && /* the most of any length: the limit is the process's, and another thread may be about to launch */     \
        cudaFuncSetAttribute(top_logprobs_kernel<T, M, NT, P, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem) != cudaSuccess)                    \
      return -2;                                                                                                                                           \
    top_logprobs_kernel<T, M, NT, P, C><<<(unsigned)rows, NT, smem, s>>>((const T*)logits, row_stride, labels, mask, mask_stride, logp, entropy, top_logp,  \
                                                                         top_ids, rest, V, k, inv_temp, fast ? groups : 0);                                 \
  }
#define RB_L3(T, M, NT, C) if (p == 4) RB_L4(T, M, NT, 4, C) else RB_L4(T, M, NT, 1, C)
#define RB_L2(T, M) \
  if (big) { RB_L3(T, M, 256, kBigCap) } else if (nt == 128) { RB_L3(T, M, 128, kCap) } else if (nt == 256) { RB_L3(T, M, 256, kCap) } else { RB_L3(T, M, 512, kCap) }
#define RB_L(T) if (mask) { RB_L2(T, true) } else { RB_L2(T, false) }
  if (dt == 0) { RB_L(float) } else if (dt == 1) { RB_L(__nv_bfloat16) } else if (dt == 2) { RB_L(__half) } else return -1;
#undef RB_L
#undef RB_L2
#undef RB_L3
#undef RB_L4
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // extern "C"
