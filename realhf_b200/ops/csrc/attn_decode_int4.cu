// Single-token decode attention over a 4-bit cache (layout and rule: int4.cuh): the new token's query and key heads are rotated, its key (rounded to the model's type,
// as a 16-bit cache would hold it) and value are quantised and appended, and the queries attend to rows [0, position] as the cache holds them.
//
// One block of four warps per (sequence, kv head, 8 query heads of its group); a warp takes every fourth row, a lane every 32nd channel.
#include "int4.cuh"

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32, kHeads = 8;

struct Params {
  const void* qkv;          // [B, (nq + 2 nkv) * D]
  uint32_t* cache;          // [B, nkv, tiles, Tile<D>::kWords]
  const int* lens;          // [B]
  void* out;                // [B, nq * D]
  const float *cos, *sin;   // [room or more, rot_dim / 2] or null
  int64_t qkv_stride;
  int nq, nkv, room, tiles, rot_dim, interleaved;
  float scale;              // times log2 e
};

// The eight channels 8 sub .. of a head at `x`, rotated: products and sums rounded one by one, as elementary operations on tensors are.
template <typename T> RB_DEVICE void rotated8(const T* x, int sub, const Params& p, int pos, float (&y)[8]) {
  const int half = p.rot_dim / 2;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = sub * 8 + i;
    y[i] = rb::to_f(x[c]);
    if (p.cos == nullptr || c >= p.rot_dim) continue;
    const bool first = p.interleaved ? c % 2 == 0 : c < half;
    const int pair = p.interleaved ? c / 2 : (first ? c : c - half), other = p.interleaved ? c ^ 1 : (first ? c + half : c - half);
    const float co = p.cos[(int64_t)pos * half + pair], si = p.sin[(int64_t)pos * half + pair];
    const float a = __fmul_rn(y[i], co), b = __fmul_rn(rb::to_f(x[other]), si);
    y[i] = first ? __fsub_rn(a, b) : __fadd_rn(a, b);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) decode_int4_kernel(Params p) {
  using Tl = q4::Tile<D>;
  constexpr int E = D / 32;
  __shared__ float sq[kHeads][D], sm_m[kWarps][kHeads], sm_l[kWarps][kHeads], sm_o[kWarps][kHeads][D];
  rb::pdl_trigger();
  rb::pdl_wait();
  const int b = blockIdx.x, hkv = blockIdx.y, h0 = blockIdx.z * kHeads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rep = p.nq / p.nkv, heads = min(kHeads, rep - h0), pos = p.lens[b];
  T* out = reinterpret_cast<T*>(p.out) + (int64_t)b * p.nq * D + (int64_t)(hkv * rep + h0) * D;
  if (pos < 0 || pos >= p.room) {
    for (int i = threadIdx.x; i < heads * D; i += kThreads) out[i] = rb::from_f<T>(0.f);
    return;
  }
  const T* qkv = reinterpret_cast<const T*>(p.qkv) + b * p.qkv_stride;
  uint32_t* cache = p.cache + ((int64_t)b * p.nkv + hkv) * p.tiles * Tl::kWords;
  for (int i = threadIdx.x; i < heads * Tl::W; i += kThreads) {
    float y[8];
    rotated8(qkv + (int64_t)(hkv * rep + h0 + i / Tl::W) * D, i % Tl::W, p, pos, y);
    for (int e = 0; e < 8; ++e) sq[i / Tl::W][i % Tl::W * 8 + e] = y[e] * p.scale;
  }
  // every block of the group writes the same words
  if (warp == 0) {
    uint32_t* at = cache + (int64_t)(pos / 16) * Tl::kWords;
    const int r = pos % 16, sub = lane % Tl::W;
    float y[8], lo, hi;
    rotated8(qkv + (int64_t)(p.nq + hkv) * D, sub, p, pos, y);
    for (int e = 0; e < 8; ++e) y[e] = rb::to_f(rb::from_f<T>(y[e]));
    q4::extremes<4>(y, lo, hi);
    const uint32_t kg = q4::group_word<T>(lo, hi);
    at[r * Tl::W + q4::word_place<Tl::J>(sub)] = q4::pack8(y, q4::scale_of<T>(kg), lo);
    at[Tl::kKeyScales + r * Tl::J + sub / 4] = kg;
    for (int e = 0; e < 8; ++e) y[e] = rb::to_f(qkv[(int64_t)(p.nq + p.nkv + hkv) * D + sub * 8 + e]);
    q4::extremes<8>(y, lo, hi);
    const uint32_t vg = q4::group_word<T>(lo, hi);
    at[Tl::kValues + sub * 16 + q4::place_of(r)] = q4::pack8(y, q4::scale_of<T>(vg), lo);
    at[Tl::kValueScales + r * Tl::H + sub / 8] = vg;
  }
  __syncthreads();
  float m[kHeads], l[kHeads], o[kHeads][E];
  for (int h = 0; h < kHeads; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
    for (int e = 0; e < E; ++e) o[h][e] = 0.f;
  }
  for (int row = warp; row <= pos; row += kWarps) {
    const uint32_t* at = cache + (int64_t)(row / 16) * Tl::kWords;
    const int r = row % 16;
    float k[E], v[E];
    for (int e = 0; e < E; ++e) {
      const int c = e * 32 + lane, w = c / 8, bit = 4 * (c % 8 >> 1) + 16 * (c & 1);
      const uint32_t kg = at[Tl::kKeyScales + r * Tl::J + c / 32], vg = at[Tl::kValueScales + r * Tl::H + c / 64];
      k[e] = fmaf(q4::scale_of<T>(kg), (float)(at[r * Tl::W + q4::word_place<Tl::J>(w)] >> bit & 15u), q4::low_of<T>(kg));
      v[e] = fmaf(q4::scale_of<T>(vg), (float)(at[Tl::kValues + w * 16 + q4::place_of(r)] >> bit & 15u), q4::low_of<T>(vg));
    }
    for (int h = 0; h < heads; ++h) {
      float s = 0.f;
      for (int e = 0; e < E; ++e) s = fmaf(sq[h][e * 32 + lane], k[e], s);
      s = rb::warp_sum(s);
      const float mx = q4::max_nan(m[h], s), zero = mx == -INFINITY ? 0.f : mx, corr = exp2f(m[h] - zero), w = exp2f(s - zero);
      m[h] = mx;
      l[h] = fmaf(l[h], corr, w);
      for (int e = 0; e < E; ++e) o[h][e] = fmaf(o[h][e], corr, w * v[e]);
    }
  }
  for (int h = 0; h < heads; ++h) {
    if (lane == 0) {
      sm_m[warp][h] = m[h];
      sm_l[warp][h] = l[h];
    }
    for (int e = 0; e < E; ++e) sm_o[warp][h][e * 32 + lane] = o[h][e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * D; i += kThreads) {
    const int h = i / D;
    float mx = -INFINITY, ls = 0.f, acc = 0.f;
    for (int w = 0; w < kWarps; ++w) mx = q4::max_nan(mx, sm_m[w][h]);
    for (int w = 0; w < kWarps; ++w) {
      const float c = sm_m[w][h] == -INFINITY ? 0.f : exp2f(sm_m[w][h] - mx);
      ls = fmaf(sm_l[w][h], c, ls);
      acc = fmaf(sm_o[w][h][i % D], c, acc);
    }
    out[i] = rb::from_f<T>(acc / ls);
  }
}

template <typename T, int D> int launch(const Params& p, int B, cudaStream_t s) {
  return rb::launch_pdl(decode_int4_kernel<T, D>, dim3(B, p.nkv, RB_CEIL_DIV(p.nq / p.nkv, kHeads)), dim3(kThreads), 0, s, p) == cudaSuccess ? 0 : -3;
}

}  // namespace

extern "C" int rb_decode_attention_int4(const void* qkv, void* cache, const int* lens, void* out, const float* cos, const float* sin, int64_t qkv_stride, int B, int nq,
                                        int nkv, int hd, int room, int rot_dim, int interleaved, float scale, int dt, cudaStream_t s) {
  if (B == 0) return 0;
  const Params p{qkv, reinterpret_cast<uint32_t*>(cache), lens, out, cos, sin, qkv_stride, nq, nkv, room, (room + 15) / 16, rot_dim, interleaved,
                 scale * 1.4426950408889634f};
  if (dt == 1 && hd == 128) return launch<__nv_bfloat16, 128>(p, B, s);
  if (dt == 1 && hd == 64) return launch<__nv_bfloat16, 64>(p, B, s);
  if (dt == 2 && hd == 128) return launch<__half, 128>(p, B, s);
  if (dt == 2 && hd == 64) return launch<__half, 64>(p, B, s);
  return -2;
}
