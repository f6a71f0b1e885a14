// Products of a few rows with a weight held in 4 bits: y[m, n] = sum_k x[m, k] w[n, k] (+ bias[n]), w ~ scale c + low by groups of 32, 64 or 128 along K (int4.cuh).
//
// A weight is tiles of 16 output rows x 128 channels, the tiles of 16 rows one behind the other along K: weight words [row][t][j] of 128 channels,
// then the group words [row][group].  Rows beyond N and channels beyond K hold codes, scales and lowest values of 0.
//
// One warp per output row: its lanes walk along K, eight rows of x at a time.
#include "int4.cuh"

namespace {

constexpr int kThreads = 128;

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

template <typename T, int G>
__global__ void __launch_bounds__(kThreads) linear_kernel(const T* __restrict__ x, const uint32_t* __restrict__ q, const T* __restrict__ bias, T* __restrict__ y, int M, int N,
                                                          int K, int64_t ldx, int64_t ldy) {
  const int n = blockIdx.x * (kThreads / 32) + threadIdx.x / 32, lane = threadIdx.x & 31, kblocks = RB_CEIL_DIV(K, 128);
  rb::pdl_trigger();
  rb::pdl_wait();
  if (n >= N) return;
  for (int m0 = 0; m0 < M; m0 += 8) {
    float acc[8] = {};
    for (int kw = lane; kw * 8 < K; kw += 32) {
      const uint32_t* at = q + ((int64_t)(n / 16) * kblocks + kw / 16) * WTile<G>::kWords;
      const uint32_t g = at[256 + n % 16 * WTile<G>::kGroups + kw % 16 / (G / 8)];
      float w[8];
      q4::unpack8<q4::kWeight>(at[n % 16 * 16 + q4::word_place<4>(kw % 16)], q4::scale_of<T>(g), q4::low_of<T>(g), w);
      for (int m = 0; m < 8 && m0 + m < M; ++m)
        for (int i = 0; i < 8; ++i) acc[m] = fmaf(rb::to_f(x[(m0 + m) * ldx + kw * 8 + i]), w[i], acc[m]);
    }
    for (int m = 0; m < 8 && m0 + m < M; ++m) {
      const float s = rb::warp_sum(acc[m]);
      if (lane == 0) y[(m0 + m) * ldy + n] = rb::from_f<T>(s + (bias ? rb::to_f(bias[n]) : 0.f));
    }
  }
}

template <typename T, int G> int run(const void* x, const void* q, const void* bias, void* y, int M, int N, int K, int64_t ldx, int64_t ldy, cudaStream_t s) {
  return rb::launch_pdl(linear_kernel<T, G>, dim3(RB_CEIL_DIV(N, kThreads / 32)), dim3(kThreads), 0, s, (const T*)x, (const uint32_t*)q, (const T*)bias, (T*)y, M, N, K, ldx,
                        ldy) == cudaSuccess ? 0 : -3;
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
