// Single-token decode attention over a 4-bit cache (layout and rule: int4.cuh): the new token's query and key heads are rotated, its key (rounded to the model's type,
// as a 16-bit cache would hold it) and value are quantised and appended, and the queries attend to rows [0, position] as the cache holds them.
//
// One CTA of four warps per (sequence, kv head, up to 8 query heads of its group, split).  A warp takes a tile of 16 rows a step, which is one copy of 2432 bytes (heads
// of 64 channels: 1216) into a ring of its own, and multiplies the codes themselves on the tensor cores, as the fp16 subnormals that they are in the low bits of a
// half-word: scores as codes [16 keys x D] times q [D x 8 columns], sums as codes^T [D x 16 keys] times weights [16 keys x 8 columns].  Scale and lowest value
// stay out of the products: a group's partial score is scaled in fp32 when its 32 channels are through (scale * (q . c) + low * sum q), and a row's weight is taken times its
// value group's scale before it becomes an operand, the lowest values are summed beside.  So nothing is converted and nothing is rounded on the way from the cache to the product.
// Queries and scaled weights are sums of two fp16 parts (22 bits), (part, head) pairs in the 8 columns, brought into fp16's range by powers of two: a query by its largest
// element, weights by the largest scale that the warp has met (a running power of two, as a softmax's maximum is).
#include "attn_common.cuh"
#include "int4.cuh"

#include <atomic>

namespace {

constexpr int kWarps = 4, kDecThreads = kWarps * 32;
constexpr int ctas_of(int rep) { return rep <= 4 ? 4 : 3; }                       // CTAs an SM
template <int D> constexpr int slots_of() { return 12160 / q4::Tile<D>::kBytes; }  // tiles of a warp's ring: 5 or 10
constexpr size_t kRing = 12160, kSmem = kWarps * kRing;
constexpr int kMaxSplits = 8;                                                     // CTAs of a portable cluster

struct StepParams {
  const void* qkv;          // [B, (nq + 2 nkv) * D]
  uint32_t* cache;          // [B, nkv, tiles, Tile<D>::kWords]
  const int* lens;          // [B]
  void* out;                // [B, nq * D]
  const float *cos, *sin;   // [room or more, rot_dim / 2] or null
  int64_t qkv_stride;
  int nq, nkv, room, tiles, rot_dim, interleaved, splits;
  float scale;              // times log2 e
  int* status;              // rb_attn_status()
};

RB_DEVICE void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The codes in nibble i of both halves of a word, in bits 4 .. 7: 2^-20 times the codes.
RB_DEVICE uint32_t nibbles(uint32_t w, int i) { return (i == 0 ? w << 4 : w >> (4 * i - 4)) & 0x00f000f0u; }
template <int N> RB_DEVICE void ld_words(uint32_t (&w)[N], uint32_t addr) {
  static_assert(N == 2 || N == 4, "");
  if constexpr (N == 4)
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
  else
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr) : "memory");
}
RB_DEVICE float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }   // 2^x, 2 ulp
RB_DEVICE float2 unpack_half2(uint32_t r) { return __half22float2(*reinterpret_cast<const __half2*>(&r)); }
RB_DEVICE float power2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // e = -126 .. 127

template <typename T> RB_DEVICE void load8(const T* p, float (&f)[8]) {
  const rb::Pack<T, 8> v = *reinterpret_cast<const rb::Pack<T, 8>*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = rb::to_f(v.v[i]);
}

// The cosines and sines of the 8 channels a lane holds of a head (4 pairs if interleaved), read ahead of their use.
struct Turn { float c[8], s[8]; };
RB_DEVICE void load_turn(Turn& t, int sub, const StepParams& p, int pos) {
  const int half = p.rot_dim / 2, d0 = sub * 8;
  if (d0 >= p.rot_dim) return;
  const int64_t at = (int64_t)pos * half + (p.interleaved ? d0 / 2 : (d0 < half ? d0 : d0 - half));
  const int n = p.interleaved ? min(4, (p.rot_dim - d0) / 2) : 8;
  if (half % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.cos) | reinterpret_cast<uintptr_t>(p.sin)) & 15) == 0) {   // (then n is 4 or 8, and `at` a multiple of 4)
#pragma unroll
    for (int i = 0; i < 8; i += 4)
      if (i < n) {
        const float4 c = *reinterpret_cast<const float4*>(p.cos + at + i), s = *reinterpret_cast<const float4*>(p.sin + at + i);
        t.c[i] = c.x; t.c[i + 1] = c.y; t.c[i + 2] = c.z; t.c[i + 3] = c.w;
        t.s[i] = s.x; t.s[i + 1] = s.y; t.s[i + 2] = s.z; t.s[i + 3] = s.w;
      }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) { t.c[i] = p.cos[at + i]; t.s[i] = p.sin[at + i]; }
  }
}
// Rotates the 8 channels this lane holds of one head; products and sums are rounded one by one, as elementary operations on tensors are.
template <int D> RB_DEVICE void rotate8(float (&x)[8], int sub, const Turn& t, const StepParams& p) {
  const int half = p.rot_dim / 2, d0 = sub * 8;
  if (p.interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d0 + 2 * i < p.rot_dim) {
        const float a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = __fsub_rn(__fmul_rn(a, t.c[i]), __fmul_rn(b, t.s[i]));
        x[2 * i + 1] = __fadd_rn(__fmul_rn(b, t.c[i]), __fmul_rn(a, t.s[i]));
      }
  } else {
    const int off = half / 8;                  // the partner channel is `half` away: so many lanes
    const bool first = d0 < half, active = d0 < p.rot_dim;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float up = __shfl_down_sync(0xffffffffu, x[i], off, D / 8), dn = __shfl_up_sync(0xffffffffu, x[i], off, D / 8);
      if (active) x[i] = first ? __fsub_rn(__fmul_rn(x[i], t.c[i]), __fmul_rn(up, t.s[i])) : __fadd_rn(__fmul_rn(x[i], t.c[i]), __fmul_rn(dn, t.s[i]));
    }
  }
}

template <typename T, int D, int REP>
__global__ void __launch_bounds__(kDecThreads, ctas_of(REP)) decode_int4_kernel(const StepParams p) {
  using Tl = q4::Tile<D>;
  constexpr int LPR = D / 8, J = Tl::J, H = Tl::H, NS = slots_of<D>();
  constexpr int kProd = REP == 8 ? 2 : 1;          // products a tile: (part, head) pairs fill 8 columns, or each part has its own
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ __align__(8) uint64_t bar[kWarps][NS];
  __shared__ uint32_t dead_flag;
  __shared__ __align__(16) float sq[REP][D], sk[D], sv[D];          // the new token: queries (in base-2 units, times a power of two), key and value as the cache holds them
  __shared__ __align__(16) __half sparts[2][REP][D + 8];            // the queries' parts
  __shared__ float s_unit[REP], s_qsum[REP][J];                     // the power of two inverted; sums of the queries over a key group, in base-2 units
  __shared__ float sm_m[kWarps + 1][REP], sm_l[kWarps + 1][REP], sm_z[kWarps][H][REP];
  __shared__ float cta_m[REP], cta_l[REP];
  float(*cta_acc)[D] = sq;                                          // (the queries' place once the warps are done)
  const int groups = RB_CEIL_DIV(p.nq / p.nkv, REP);                // sets of REP query heads of a kv head
  const int b = blockIdx.x, hkv = blockIdx.y / groups, h0 = blockIdx.y % groups * REP, split = blockIdx.z;
  const int rep = p.nq / p.nkv, heads = min(REP, rep - h0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  volatile uint32_t* dead = &dead_flag;
  if (threadIdx.x == 0) *dead = 0;
  if (lane < NS) ptx::mbar_init(ptx::smem_u32(&bar[warp][lane]), 1);
  ptx::fence_barrier_init();
  __syncthreads();
  rb::pdl_trigger();
  rb::pdl_wait();
  const int pos = p.lens[b];
  T* out = reinterpret_cast<T*>(p.out) + (int64_t)b * p.nq * D + (int64_t)(hkv * rep + h0) * D;
  if (pos < 0 || pos >= p.room) {                                   // (all CTAs of the cluster: one sequence)
    if (split == 0)
      for (int i = threadIdx.x; i < heads * D; i += kDecThreads) out[i] = rb::from_f<T>(0.f);
    return;
  }
  // ---- the new token's values are asked for ahead of the tiles.  A group of D / 8 lanes has one of the REP queries or the key.
  const T* qkv = reinterpret_cast<const T*>(p.qkv) + b * p.qkv_stride;
  constexpr int kGroups = kDecThreads / LPR, kTurns = (REP + 1 + kGroups - 1) / kGroups;
  const int sub = threadIdx.x % LPR;
  float xn[kTurns][8], vn[8];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int r = threadIdx.x / LPR + i * kGroups;
    load8(qkv + (int64_t)(r < heads ? hkv * rep + h0 + r : p.nq + hkv) * D + sub * 8, xn[i]);
  }
  load8(qkv + (int64_t)(p.nq + p.nkv + hkv) * D + sub * 8, vn);
  Turn turn;
  if (p.cos) load_turn(turn, sub, p, pos);

  // ---- this split's tiles of the cached rows [0, pos) (the new one is handled from registers); the first of them are asked for
  const int n_tiles = RB_CEIL_DIV(pos, 16), per = RB_CEIL_DIV(n_tiles, p.splits);
  const int lo = min(n_tiles, split * per), hi = min(n_tiles, lo + per);
  uint32_t* cache = p.cache + ((int64_t)b * p.nkv + hkv) * p.tiles * Tl::kWords;
  const uint32_t base = ptx::smem_u32(ring) + warp * (uint32_t)kRing;
  auto fetch = [&](int tile, int slot) {
    if (tile < hi && ptx::elect_one()) {
      const uint32_t full = ptx::smem_u32(&bar[warp][slot]);
      ptx::mbar_arrive_expect_tx(full, Tl::kBytes);
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(base + slot * Tl::kBytes),
                   "l"(cache + (int64_t)tile * Tl::kWords), "r"(Tl::kBytes), "r"(full) : "memory");
    }
  };
#pragma unroll
  for (int n = 0; n < NS; ++n) fetch(lo + warp + n * kWarps, n);

#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int r = threadIdx.x / LPR + i * kGroups;
    if (p.cos) rotate8<D>(xn[i], sub, turn, p);
    // the key (r == REP; the lanes of other rows go along)
    float key[8], klo, khi;
#pragma unroll
    for (int e = 0; e < 8; ++e) key[e] = rb::to_f(rb::from_f<T>(xn[i][e]));
    q4::extremes<4>(key, klo, khi);
    if (r == REP) {
      const uint32_t kg = q4::group_word<T>(klo, khi), kw = q4::pack8(key, q4::scale_of<T>(kg), klo);
      if (split == 0 && h0 == 0) {
        uint32_t* at = cache + (int64_t)(pos / 16) * Tl::kWords;
        at[pos % 16 * Tl::W + q4::word_place<J>(sub)] = kw;
        if (sub % 4 == 0) at[Tl::kKeyScales + pos % 16 * J + sub / 4] = kg;
      }
      q4::unpack8(kw, q4::scale_of<T>(kg), q4::low_of<T>(kg), key);
#pragma unroll
      for (int e = 0; e < 8; e += 4) *reinterpret_cast<float4*>(&sk[sub * 8 + e]) = make_float4(key[e], key[e + 1], key[e + 2], key[e + 3]);
    }
    // a query: its sums over the key groups, then its largest element to 2^14 .. 2^15
    float sum = 0.f, most = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      xn[i][e] = r < heads ? xn[i][e] * p.scale : 0.f;
      sum += xn[i][e];
      most = fmaxf(most, fabsf(xn[i][e]));
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const int up = max(min(14 + 127 - (int)(__float_as_uint(most) >> 23), 100), -100);
    if (r < REP) {
      if (sub % 4 == 0) s_qsum[r][sub / 4] = sum;
      if (sub == 0) s_unit[r] = power2(-up);
      uint32_t part[2][4];
      const float f = power2(up);
#pragma unroll
      for (int e = 0; e < 8; ++e) xn[i][e] *= f;
#pragma unroll
      for (int e = 0; e < 8; e += 4) *reinterpret_cast<float4*>(&sq[r][sub * 8 + e]) = make_float4(xn[i][e], xn[i][e + 1], xn[i][e + 2], xn[i][e + 3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        part[0][e] = pack2<__half>(xn[i][2 * e], xn[i][2 * e + 1]);
        const float2 f0 = unpack_half2(part[0][e]);
        part[1][e] = pack2<__half>(xn[i][2 * e] - f0.x, xn[i][2 * e + 1] - f0.y);
      }
#pragma unroll
      for (int f2 = 0; f2 < 2; ++f2) *reinterpret_cast<uint4*>(&sparts[f2][r][sub * 8]) = make_uint4(part[f2][0], part[f2][1], part[f2][2], part[f2][3]);
    }
  }
  {
    float vlo, vhi;
    q4::extremes<8>(vn, vlo, vhi);
    if (threadIdx.x < LPR) {
      const uint32_t vg = q4::group_word<T>(vlo, vhi), vw = q4::pack8(vn, q4::scale_of<T>(vg), vlo);
      if (split == 0 && h0 == 0) {
        uint32_t* at = cache + (int64_t)(pos / 16) * Tl::kWords;
        at[Tl::kValues + sub * 16 + q4::place_of(pos % 16)] = vw;
        if (sub % 8 == 0) at[Tl::kValueScales + pos % 16 * H + sub / 8] = vg;
      }
      q4::unpack8(vw, q4::scale_of<T>(vg), q4::low_of<T>(vg), vn);
#pragma unroll
      for (int e = 0; e < 8; e += 4) *reinterpret_cast<float4*>(&sv[sub * 8 + e]) = make_float4(vn[e], vn[e + 1], vn[e + 2], vn[e + 3]);
    }
  }
  __syncthreads();

  // ---- the queries as column operands: column g is (part g / REP, head g % REP); columns beyond the parts are never looked at
  const int head = g % REP, part = min(g / REP, 1);
  uint32_t qb[J][kProd][4];
#pragma unroll
  for (int c = 0; c < kProd; ++c)
#pragma unroll
    for (int j = 0; j < J; ++j) ld_words(qb[j][c], ptx::smem_u32(&sparts[REP == 8 ? c : part][head][32 * j + 8 * t]));
  // of the columns 2t, 2t + 1 of a product: the unit (2^20: the codes' subnormals), and the sums of the queries (with the first part alone)
  float unit[2], qs[J][2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int col = 2 * t + i;
    unit[i] = s_unit[col % REP] * 1048576.f;
#pragma unroll
    for (int j = 0; j < J; ++j) qs[j][i] = col < REP ? s_qsum[col % REP][j] : 0.f;
  }
  if (warp == 0 && split == p.splits - 1) {      // the new token: one more set of partial sums
#pragma unroll
    for (int r = 0; r < REP; ++r) {
      float s = 0.f;
#pragma unroll
      for (int d = 0; d < D; d += 32) s = fmaf(sq[r][d + lane], sk[d + lane], s);
      s = rb::warp_sum(s);
      if (lane == 0) {
        sm_m[kWarps][r] = s * s_unit[r];
        sm_l[kWarps][r] = 1.f;
      }
    }
  }

  float o[4 * H][4];
#pragma unroll
  for (int j = 0; j < 4 * H; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m = -INFINITY, l = 0.f, z[H];               // of head `head`, over the lane's keys: maximum, sum of weights, sums of weights times lowest values
#pragma unroll
  for (int h = 0; h < H; ++h) z[h] = 0.f;
  int top = -100;                                   // scaled weights are in units of 2^(top - 14); every scale so far is below 2^top
  uint32_t bound = 0;                               // the group word of that scale
  int slot = 0;
  uint32_t round = 0;                               // parity of the ring's current round
#pragma unroll 1
  for (int tile = lo + warp; tile < hi; tile += kWarps) {
    bounded_wait(ptx::smem_u32(&bar[warp][slot]), round, dead);
    const uint32_t at = base + slot * Tl::kBytes;
    // ---- scores of 16 keys: lane (g, t) gets keys g and g + 8 of columns 2t and 2t + 1
    float v[4];
    {
      uint32_t w0[J], w1[J], s0[J], s1[J];
      ld_words(w0, at + g * (D / 2) + t * (J * 4));
      ld_words(w1, at + (g + 8) * (D / 2) + t * (J * 4));
      ld_words(s0, at + Tl::kKeyScales * 4 + g * (J * 4));
      ld_words(s1, at + Tl::kKeyScales * 4 + (g + 8) * (J * 4));
      float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int f = 0; f < kProd; ++f)
            mma_f16(c, nibbles(w0[j], 2 * e), nibbles(w1[j], 2 * e), nibbles(w0[j], 2 * e + 1), nibbles(w1[j], 2 * e + 1), qb[j][f][2 * e], qb[j][f][2 * e + 1]);
        }
        const float f0 = q4::scale_of<T>(s0[j]), f1 = q4::scale_of<T>(s1[j]), l0 = q4::low_of<T>(s0[j]), l1 = q4::low_of<T>(s1[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = fmaf(i < 2 ? f0 : f1, c[i], x[i]);
          y[i] = fmaf(i < 2 ? l0 : l1, qs[j][i & 1], y[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = fmaf(x[i], unit[i & 1], y[i]);
    }
    // ---- the parts of a head added up, then lane (g, t) takes the keys 2t, 2t + 1, 2t + 8, 2t + 9 of head g % REP
    float s[4];
    if constexpr (REP == 1) { v[0] += v[1]; v[2] += v[3]; }
    if constexpr (REP == 2 || REP == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], REP / 2);
    }
    if constexpr (REP == 8) {
      const int from = 8 * t + (head >> 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float even = __shfl_sync(0xffffffffu, v[(i >> 1) * 2], from + (i & 1) * 4), odd = __shfl_sync(0xffffffffu, v[(i >> 1) * 2 + 1], from + (i & 1) * 4);
        s[i] = head & 1 ? odd : even;
      }
    } else {
      // lanes of a row that hold the same sums offer one head each: t & 1, or for four heads 2 (t & 1) + (t >> 1)
      const bool second = REP == 2 ? t & 1 : (REP == 4 ? t >> 1 : false);
      const float lo8 = second ? v[1] : v[0], hi8 = second ? v[3] : v[2];
      const int from = 8 * t + (REP == 4 ? (head >> 1) | ((head & 1) << 1) : head);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = __shfl_sync(0xffffffffu, i < 2 ? lo8 : hi8, from + (i & 1) * 4);
    }
    // the value groups of those keys
    uint32_t vg[4][H];
    {
      uint32_t a[2 * H], c[2 * H];
      ld_words(a, at + Tl::kValueScales * 4 + 2 * t * (H * 4));
      ld_words(c, at + Tl::kValueScales * 4 + (2 * t + 8) * (H * 4));
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < H; ++h) { vg[i][h] = a[i * H + h]; vg[2 + i][h] = c[i * H + h]; }
    }
    if (tile * 16 + 16 > pos) {                     // rows behind the length may hold anything
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (tile * 16 + 2 * t + (i & 1) + (i >> 1) * 8 >= pos) {
          s[i] = -INFINITY;
#pragma unroll
          for (int h = 0; h < H; ++h) vg[i][h] = 0;
        }
    }
    // ---- running softmax; the accumulators are corrected only where a maximum or the unit moved
    float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)), m);
    const float zero = mx == -INFINITY ? 0.f : mx;
    if (__any_sync(0xffffffffu, mx != m)) {
      const float corr = ex2(m - zero);
      l *= corr;
#pragma unroll
      for (int h = 0; h < H; ++h) z[h] *= corr;
      const float ce = __shfl_sync(0xffffffffu, corr, 8 * t), co = __shfl_sync(0xffffffffu, corr, 8 * t + 4);   // of columns 2t, 2t + 1
#pragma unroll
      for (int j = 0; j < 4 * H; ++j) { o[j][0] *= ce; o[j][1] *= co; o[j][2] *= ce; o[j][3] *= co; }
      m = mx;
    }
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < H; ++h) most = max(most, vg[i][h]);
    if (__any_sync(0xffffffffu, most >= bound)) {
      constexpr uint32_t kNan = std::is_same<T, __half>::value ? 0x7c000000u : 0x7f800000u;   // infinities and NaN: no unit holds them
      most = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < H; ++h) most = max(most, vg[i][h] < kNan ? vg[i][h] : 0u);
      most = __reduce_max_sync(0xffffffffu, most);
      if (most >= bound) {                          // two bits of room, so that it seldom moves
        constexpr int kShift = std::is_same<T, __half>::value ? 26 : 23, kBias = std::is_same<T, __half>::value ? 15 : 127;
        const int ex = min((int)(most >> kShift) + 3, (int)(kNan >> kShift)), was = top;
        top = max(min(ex - kBias, 127), -100);
        bound = (uint32_t)ex << kShift;
        const float f = power2(max(was - top, -126));
#pragma unroll
        for (int j = 0; j < 4 * H; ++j) { o[j][0] *= f; o[j][1] *= f; o[j][2] *= f; o[j][3] *= f; }
      }
    }
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = ex2(s[i] - zero);
    l += (w[0] + w[1]) + (w[2] + w[3]);
    const float into = power2(14 - top);
    uint32_t pb[H][kProd][2];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float a = w[2 * e] * into * q4::scale_of<T>(vg[2 * e][h]), c = w[2 * e + 1] * into * q4::scale_of<T>(vg[2 * e + 1][h]);
        z[h] = fmaf(w[2 * e], q4::low_of<T>(vg[2 * e][h]), z[h]);
        z[h] = fmaf(w[2 * e + 1], q4::low_of<T>(vg[2 * e + 1][h]), z[h]);
        const uint32_t p0 = pack2<__half>(a, c);
        const float2 f0 = unpack_half2(p0);
        const uint32_t p1 = pack2<__half>(a - f0.x, c - f0.y);
        if constexpr (REP == 8) { pb[h][0][e] = p0; pb[h][1][e] = p1; } else pb[h][0][e] = part ? p1 : p0;
      }
    // ---- sums: codes^T times the weights' parts.  Word g of the lane's four keys: rows g are its even channels, rows g + 8 its odd ones.
#pragma unroll
    for (int h = 0; h < H; ++h) {
      uint32_t w4[4];
      ld_words(w4, at + Tl::kValues * 4 + h * 512 + g * 64 + t * 16);
      const uint32_t xl = __byte_perm(w4[0], w4[1], 0x5410), yl = __byte_perm(w4[0], w4[1], 0x7632), xh = __byte_perm(w4[2], w4[3], 0x5410),
                     yh = __byte_perm(w4[2], w4[3], 0x7632);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int f = 0; f < kProd; ++f)
          mma_f16(o[4 * h + i], nibbles(xl, i), nibbles(yl, i), nibbles(xh, i), nibbles(yh, i), pb[h][f][0], pb[h][f][1]);
      }
    }
    __syncwarp();
    fetch(tile + NS * kWarps, slot);
    if (++slot == NS) { slot = 0; round ^= 1; }
  }
  __syncwarp();

  // ---- merge the warps, then the CTAs of the cluster.  A warp's sums take the place of its ring.
  static_assert(kRing >= REP * D * 4, "");
  float* mysum = reinterpret_cast<float*>(ring + warp * kRing);
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
#pragma unroll
  for (int h = 0; h < H; ++h) {
    z[h] += __shfl_xor_sync(0xffffffffu, z[h], 1);
    z[h] += __shfl_xor_sync(0xffffffffu, z[h], 2);
  }
  if (g < REP && t == 0) {
    sm_m[warp][head] = m;
    sm_l[warp][head] = l;
#pragma unroll
    for (int h = 0; h < H; ++h) sm_z[warp][h][head] = z[h];
  }
#pragma unroll
  for (int j = 0; j < 4 * H; ++j) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = o[j][i] * 64.f * power2(top);      // 2^20 of the subnormals, 2^-14 of the weights
    if constexpr (REP == 1) { x[0] += x[1]; x[2] += x[3]; }
    if constexpr (REP == 2 || REP == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], REP / 2);
    }
    const int d = 64 * (j >> 2) + 8 * g + 2 * (j & 3);
    if constexpr (REP == 1) {
      if (t == 0) *reinterpret_cast<float2*>(mysum + d) = make_float2(x[0], x[2]);
    } else if (2 * t < REP) {
      *reinterpret_cast<float2*>(mysum + 2 * t * D + d) = make_float2(x[0], x[2]);
      *reinterpret_cast<float2*>(mysum + (2 * t + 1) * D + d) = make_float2(x[1], x[3]);
    }
  }
  __syncthreads();
  const int sets = split == p.splits - 1 ? kWarps + 1 : kWarps;
  for (int idx = threadIdx.x; idx < heads * D; idx += kDecThreads) {
    const int r = idx / D, d = idx % D;
    float mg = -INFINITY;
    for (int w = 0; w < sets; ++w) mg = fmaxf(mg, sm_m[w][r]);
    float lg = 0.f, ag = 0.f;
#pragma unroll
    for (int w = 0; w <= kWarps; ++w) {
      if (w == sets) break;
      const float c = (sm_m[w][r] == -INFINITY) ? 0.f * sm_l[w][r] : ex2(sm_m[w][r] - mg);
      lg += sm_l[w][r] * c;
      ag += (w < kWarps ? reinterpret_cast<const float*>(ring + w * kRing)[idx] + sm_z[w][d / 64][r] : sv[d]) * c;
    }
    if (p.splits == 1) {
      out[idx] = rb::from_f<T>(ag / lg);
    } else {
      cta_acc[r][d] = ag;
      if (d == 0) { cta_m[r] = mg; cta_l[r] = lg; }
    }
  }
  rb::report_given_up(dead, p.status);
  if (p.splits == 1) return;
  ptx::cluster_sync();
  // the cluster is (1, 1, splits): CTA `split` of it finishes its share of the outputs from everybody's sums
  auto peer = [](const float* x, int cta) {
    uint32_t a;
    float f;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(ptx::smem_u32(x)), "r"(cta));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(a) : "memory");
    return f;
  };
  for (int idx = split * kDecThreads + threadIdx.x; idx < heads * D; idx += p.splits * kDecThreads) {
    const int r = idx / D, d = idx % D;
    float mg = -INFINITY;
    for (int c = 0; c < p.splits; ++c) mg = fmaxf(mg, peer(&cta_m[r], c));
    float lg = 0.f, ag = 0.f;
    for (int c = 0; c < p.splits; ++c) {
      const float mc = peer(&cta_m[r], c), lc = peer(&cta_l[r], c), w = mc == -INFINITY ? 0.f * lc : ex2(mc - mg);
      lg += lc * w;
      ag += peer(&cta_acc[r][d], c) * w;
    }
    out[idx] = rb::from_f<T>(ag / lg);
  }
  ptx::cluster_sync();  // nobody leaves while its sums are being read
}

template <typename T, int D, int REP> int launch_one(const StepParams& p, int B, cudaStream_t s) {
  static std::atomic<uint64_t> opted_in{0};          // the attribute is the kernel's on one device: a bit per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -3;
  if (dev >= 64 || !(opted_in.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(decode_int4_kernel<T, D, REP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem) != cudaSuccess) return -3;
    if (dev < 64) opted_in.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(B, p.nkv * RB_CEIL_DIV(p.nq / p.nkv, REP), p.splits);
  cfg.blockDim = dim3(kDecThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (p.splits > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = p.splits;
  }
  if (rb::pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, decode_int4_kernel<T, D, REP>, p) == cudaSuccess ? 0 : -3;
}

template <typename T, int D> int launch(StepParams p, int B, cudaStream_t s) {
  const int rep = p.nq / p.nkv, wide = rep == 1 ? 1 : rep == 2 ? 2 : rep <= 4 ? 4 : 8;
  // CTAs a (sequence, kv head, set of heads): doubled as long as all of them still fit at once and each keeps two tiles a warp of a full cache
  const int64_t ctas = (int64_t)B * p.nkv * RB_CEIL_DIV(rep, wide);
  p.splits = 1;
  while (p.splits < kMaxSplits && ctas * p.splits * 2 <= rb::kNumSMs * ctas_of(wide) && p.tiles >= 2 * kWarps * p.splits * 2) p.splits *= 2;
  return wide == 1 ? launch_one<T, D, 1>(p, B, s) : wide == 2 ? launch_one<T, D, 2>(p, B, s) : wide == 4 ? launch_one<T, D, 4>(p, B, s) : launch_one<T, D, 8>(p, B, s);
}

}  // namespace

// nkv * ceil(query heads of a kv head / 8) <= 65535; rot_dim a multiple of 16 (interleaved: of 2).  dt: 1 bf16, 2 fp16.
extern "C" int rb_decode_attention_int4(const void* qkv, void* cache, const int* lens, void* out, const float* cos, const float* sin, int64_t qkv_stride, int B, int nq,
                                        int nkv, int hd, int room, int rot_dim, int interleaved, float scale, int dt, cudaStream_t s) {
  if (B == 0) return 0;
  const StepParams p{qkv, reinterpret_cast<uint32_t*>(cache), lens, out, cos, sin, qkv_stride, nq, nkv, room, (room + 15) / 16, rot_dim, interleaved, 1,
                 scale * 1.4426950408889634f, rb_attn_status()};
  if (p.status == nullptr) return -5;
  if (dt == 1 && hd == 128) return launch<__nv_bfloat16, 128>(p, B, s);
  if (dt == 1 && hd == 64) return launch<__nv_bfloat16, 64>(p, B, s);
  if (dt == 2 && hd == 128) return launch<__half, 128>(p, B, s);
  if (dt == 2 && hd == 64) return launch<__half, 64>(p, B, s);
  return -2;
}
