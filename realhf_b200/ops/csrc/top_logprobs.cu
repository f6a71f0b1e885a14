// The k most likely tokens of every row of logits [rows, V] with their log-probabilities, the log of the mass of all other tokens, the log-probability
// of a given token and the entropy of the row.
//
// Order: larger logits first, equal ones by the lower index (-0 equals 0); a masked token and a logit of -inf are no alternatives, and a place that no
// token fills holds id -1 and -inf.  The rest's mass is summed over the tokens it consists of: 1 - sum of the chosen would cancel where they
// hold nearly all of it.
//
// The k-th largest value by a radix descent over its bits (four digits of 8 bits, a histogram in shared memory each), the elements above it in any order, of
// those equal to it the first in index order, sorted by (value, index).
#include "vocab_rows.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kMaxTop = 1024;

RB_DEVICE uint32_t order_key(float x) {  // order-preserving float -> uint, -0 as 0
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
RB_DEVICE float key_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
constexpr uint32_t kKeyNone = 0x007fffffu;  // order_key(-inf)

struct TopShared {
  float red[96];
  uint32_t hist[256];
  uint32_t warp_n[kThreads / 32];
  uint32_t digit, above, count;
  uint64_t list[kMaxTop];   // key << 32 | ~index: descending order is the order wanted
};

template <typename T> struct TopRow {
  const T* lr;
  const uint8_t* mr;
  int V;
  RB_DEVICE float at(int j) const { return mr && (mr[j >> 3] >> (j & 7)) & 1 ? -INFINITY : rb::to_f(lr[j]); }
};

// The k largest (key, ~index) of the row -> sh.list in any order; returns how many there are (less than k where the row keeps fewer tokens), and in
// `kth` / `last` the smallest chosen value's key and the highest index that is chosen among those equal to it.
template <typename T> RB_DEVICE int select_radix(const TopRow<T>& r, int k, TopShared& sh, uint32_t& kth, int& last) {
  uint32_t prefix = 0, want = k;      // the want-th largest among the elements whose high digits are `prefix`
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int b = threadIdx.x; b < 256; b += kThreads) sh.hist[b] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < r.V; j += kThreads) {
      const uint32_t key = order_key(r.at(j));
      if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&sh.hist[(key >> shift) & 255], 1u);
    }
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
  kth = prefix;
  last = -1;
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  for (int j = threadIdx.x; j < r.V; j += kThreads) {
    const uint32_t key = order_key(r.at(j));
    if (key > kth && key > kKeyNone) sh.list[atomicAdd(&sh.count, 1u)] = (uint64_t)key << 32 | (uint32_t)~j;
  }
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
    if (hit && at < need) {
      sh.list[above + at] = (uint64_t)kth << 32 | (uint32_t)~j;
      if (at == need - 1) sh.digit = j;
    }
    found += all;
    __syncthreads();
  }
  if (need > 0) last = (int)sh.digit;
  return above + need;
}

template <typename T, bool kMask>
__global__ void __launch_bounds__(kThreads) top_logprobs_kernel(const T* __restrict__ logits, int64_t row_stride, const int64_t* __restrict__ labels,
                                                                const uint8_t* __restrict__ mask, int64_t mask_stride, float* __restrict__ logp,
                                                                float* __restrict__ entropy, float* __restrict__ top_logp, int64_t* __restrict__ top_ids,
                                                                float* __restrict__ rest, int V, int k, float inv_temp) {
  __shared__ TopShared sh;
  const int64_t row = blockIdx.x;
  const TopRow<T> r{logits + row * row_stride, kMask ? mask + row * mask_stride : nullptr, V};
  const float kk = inv_temp * rb::kLog2e;
  rb::RowStats st;
  for (int j = threadIdx.x; j < V; j += kThreads) st.one(r.at(j), kk);
  st = rb::block_stats(st, kk, sh.red);
  const rb::RowResult res(st, inv_temp);
  if (threadIdx.x == 0) {
    entropy[row] = res.entropy;
    if (logp) logp[row] = rb::label_logp(r.lr, labels[row], r.mr, V, inv_temp, res.lse);
  }
  if (!(fabsf(res.lse) < INFINITY)) {     // no softmax, or no token
    for (int i = threadIdx.x; i < k; i += kThreads) {
      top_logp[row * k + i] = res.lse;
      top_ids[row * k + i] = -1;
    }
    if (threadIdx.x == 0) rest[row] = res.lse;
    return;
  }
  uint32_t kth;
  int last;
  const int n = select_radix(r, k, sh, kth, last);
  int size = 1;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kThreads) sh.list[i] = 0;
  __syncthreads();
  for (int len = 2; len <= size; len <<= 1)
    for (int d = len >> 1; d > 0; d >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += kThreads) {
        const int lo = 2 * d * (i / d) + i % d, hi = lo + d;
        const uint64_t a = sh.list[lo], b = sh.list[hi];
        if ((a < b) == ((lo & len) == 0)) { sh.list[lo] = b; sh.list[hi] = a; }
      }
      __syncthreads();
    }
  for (int i = threadIdx.x; i < k; i += kThreads) {
    const uint64_t c = i < n ? sh.list[i] : 0;
    top_logp[row * k + i] = i < n ? fmaf(key_value((uint32_t)(c >> 32)), inv_temp, -res.lse) : -INFINITY;
    top_ids[row * k + i] = i < n ? (int64_t)(int)~(uint32_t)c : -1;
  }
  // the others: below the k-th value, or equal to it behind the last chosen index
  rb::RowStats others;
  for (int j = threadIdx.x; j < V; j += kThreads) {
    const float x = r.at(j);
    const uint32_t key = order_key(x);
    if (key < kth || (key == kth && j > last)) others.one(x, kk);
  }
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
#define RB_L2(T, M) top_logprobs_kernel<T, M><<<(unsigned)rows, kThreads, 0, s>>>((const T*)logits, row_stride, labels, mask, mask_stride, logp, entropy, top_logp, top_ids, rest, V, k, inv_temp)
#define RB_L(T) if (mask) RB_L2(T, true); else RB_L2(T, false)
  if (dt == 0) { RB_L(float); } else if (dt == 1) { RB_L(__nv_bfloat16); } else if (dt == 2) { RB_L(__half); } else return -1;
#undef RB_L
#undef RB_L2
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // extern "C"
