// Single-token decode attention over a 4-bit cache (layout and rule: int4.cuh): the new token's query and key heads are rotated, its key (rounded to the model's type,
// as a 16-bit cache would hold it) and value are quantised and appended, and the queries attend to rows [0, position] as the cache holds them.
//
// A warp works on one (sequence, kv head, set of up to 8 query heads), or with other warps of its block and cluster on shares of its rows.  A step is two tiles of 16 rows, one
// copy of 4864 bytes (heads of 64 channels: 2432) into a ring of its own, and the codes themselves are operands on the tensor cores:
//   scores  codes, as bytes, [16 keys x 32 channels of a group] times q [32 x 8 columns] in whole numbers: a query is a 23-bit whole number (with one power of two a head), three signed
//           bytes, (byte, head) pairs in the columns.  A sum is exact; the group's scale times it, and the lowest value times the query's sum over the group, are added in fp32.
//   sums    codes^T, as small fp16 numbers, [16 channels x 16 keys] times weights [16 x 8 columns]: a row's softmax weight times its value group's scale, two fp16 parts (22 bits) of it,
//           (part, head) pairs in the columns, in units of a power of two above all scales so far (it moves as a softmax's maximum does).  The lowest values are summed beside.
// So nothing is converted on the way from the cache to a product.  The tensor core aligns subnormals as if they were 2^-14 and cuts off some 23 bits below: codes in bits 0 .. 3
// (one shift less for every two operands) left errors of 6e-5 in outputs of size 1.  In bits 7 .. 10, where 8 is 2^-14, nothing of a code is below that (32 x 4095 rows: errors of 5.5e-6
// of the outputs' size before their rounding, in bits 4 .. 7 8.6e-6, 0.5 % less time).
//
// Bound: the bytes of the cache, 152 a row of 128 channels (at the copy's rate 36 us for 128 sequences up to 639 rows of 32 heads, 16 for 32 sequences up to 4095 of 8 heads under 32
// queries).  Taken: 58.6 us (4.05 TB/s; a 16-bit cache 122) and 41.5 (2.5 TB/s; 59): issue slots 66 % and 53 %, the pipe of masks, minima and conversions 55 % and 38 %, and the
// warps that are there do not cover the rest: 128 registers allow an SM 16 (with eight queries 12), and where all blocks begin at once those of short sequences end early (32 sequences of 1300 ..
// 4095 rows: 12 on average, the longest has 16 steps a warp where the mean is 10).  Few sequences are a chain of latencies: 1 x 3900 rows 10.4 us, of which 3 are a launch's.
//
// Precision: queries keep 22 or 23 bits below the largest of a head, softmax weights times steps 22 (two fp16 parts), sums are fp32's.  Errors before the outputs' rounding: 0.4 .. 1.2e-5 of
// their size (fp32 throughout 0.2 .. 0.4e-5); by arithmetic most of it comes from scores, whose codes' part and lowest values' part cancel where keys have channels far larger than others.
#include "attn_common.cuh"
#include "int4.cuh"

#include <atomic>

namespace {

constexpr int kWarps = 4, kDecThreads = kWarps * 32;
constexpr int ctas_of(int rep) { return rep <= 4 ? 4 : 3; }                       // CTAs an SM
template <int D> constexpr int slots_of() { return 9728 / (2 * q4::Tile<D>::kBytes); }   // steps of a warp's ring: 2 or 4
constexpr size_t kRing = 9728, kSmem = kWarps * kRing;
constexpr float kSlack = 4.f;                                                     // how far (in powers of two) a maximum grows before the sums are corrected: weights up to 2^4
constexpr int kMaxSplits = 8;                                                     // CTAs of a portable cluster

struct StepParams {
  const void* qkv;          // [B, (nq + 2 nkv) * D]
  uint32_t* cache;          // [B, nkv, tiles, Tile<D>::kWords]
  const int* lens;          // [B]
  void* out;                // [B, nq * D]
  const float *cos, *sin;   // [room or more, rot_dim / 2] or null
  int64_t qkv_stride;
  int B, nq, nkv, room, tiles, rot_dim, interleaved;
  int longest_first;
  int wide, splits;         // warps of a block, blocks of a cluster that share the rows of one (sequence, kv head, set of query heads)
  float scale;              // times log2 e
  int* status;              // rb_attn_status()
};

RB_DEVICE void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
RB_DEVICE void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, int c) {   // unsigned times signed bytes, plus c
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c));
}
// [16 x 8] times [8 x 8] of the model's type
template <typename T> RB_DEVICE void mma_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};" : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(b));
  else
    asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};" : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(b));
}
// The codes in nibble i of both halves of a word, in bits 7 .. 10: as fp16 2^-17 times the codes (8 is 2^-14, the first normal number, so there is no gap).
RB_DEVICE uint32_t nibbles(uint32_t w, int i) { return (i < 2 ? w << (7 - 4 * i) : w >> (4 * i - 7)) & 0x07800780u; }
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

// The sequence that comes `rank`-th when the longest comes first: lengths in 32 classes, sequences of one class in their order.  A whole warp; B <= kRanked.
constexpr int kRanked = 256;
RB_DEVICE int sequence_of(const int* lens, int B, int room, int rank, int& len) {
  const int lane = threadIdx.x & 31, down = max(27 - __clz(room), 0);      // classes 0 .. 31
  int raw[kRanked / 32], v[kRanked / 32];
#pragma unroll
  for (int j = 0; j < kRanked / 32; ++j) raw[j] = j * 32 + lane < B ? lens[j * 32 + lane] : 0;
#pragma unroll
  for (int j = 0; j < kRanked / 32; ++j) v[j] = j * 32 + lane < B ? min(max(raw[j], 0), room) >> down : -1;
  int cls = 0, before = 0;                          // the class of that sequence: the largest with more than `rank` sequences in it and above
#pragma unroll
  for (int bit = 16; bit > 0; bit >>= 1) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < kRanked / 32; ++j)
      if (j * 32 < B) n += __popc(__ballot_sync(0xffffffffu, v[j] >= cls + bit));
    if (n > rank) cls += bit; else before = n;      // (`before` ends as the number of sequences above the class)
  }
  int left = rank - before, b = 0;
#pragma unroll
  for (int j = 0; j < kRanked / 32; ++j)
    if (j * 32 < B) {
      const uint32_t hit = __ballot_sync(0xffffffffu, v[j] == cls);
      const uint32_t it = __ballot_sync(0xffffffffu, v[j] == cls && __popc(hit & ((1u << lane) - 1)) == left);
      if (it != 0) {
        b = j * 32 + __ffs(it) - 1;
        len = __shfl_sync(0xffffffffu, raw[j], __ffs(it) - 1);
      }
      left -= __popc(hit);
    }
  return b;
}

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
    const int from = !active ? sub : first ? sub + off : sub - off;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl_sync(0xffffffffu, x[i], from, D / 8), a = __fmul_rn(x[i], t.c[i]), b = __fmul_rn(other, t.s[i]);
      if (active) x[i] = first ? __fsub_rn(a, b) : __fadd_rn(a, b);
    }
  }
}

template <typename T, int D, int REP>
__global__ void __launch_bounds__(kDecThreads, ctas_of(REP)) decode_int4_kernel(const StepParams p) {
  using Tl = q4::Tile<D>;
  constexpr int LPR = D / 8, RPT = 32 / LPR, kTurns = (REP + RPT - 1) / RPT;   // lanes of a row, rows a turn of the warp
  constexpr int J = Tl::J, H = Tl::H, NS = slots_of<D>();
  constexpr int kProd = REP == 8 ? 2 : 1;          // products of weights: (part, head) pairs fill 8 columns, or each part has its own
  constexpr int kScores = REP == 8 ? 3 : REP == 4 ? 2 : 1;   // products of queries: (byte, head) pairs
  constexpr int kTogether = REP == 1 ? 1 : 2;      // tiles whose products are added to the sums at once (128 x 639 rows with one query a key head 59.1 us, both at once 59.7; 32 x 4095 with four 42.1, 41.4)
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ __align__(8) uint64_t bar[kWarps][NS];
  __shared__ uint32_t dead_flag;
  __shared__ __align__(16) uint32_t sbytes[kWarps][3][REP][D / 4 + 2];   // the queries' three bytes, lowest first
  __shared__ uint16_t ssums[kWarps][3][REP][J];                     // their sums over a key group in three parts of the model's type
  __shared__ float s_unit[kWarps][REP];                             // the queries' power of two inverted
  __shared__ float sm_m[kWarps][REP], sm_l[kWarps][REP], sm_z[kWarps][H][REP];
  __shared__ uint2 s_new[kWarps][32];                               // the new row: a lane's word and its group's
  __shared__ float cta_m[REP], cta_l[REP];
  __shared__ __align__(16) float cta_acc[REP][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  volatile uint32_t* dead = &dead_flag;
  if (threadIdx.x == 0) *dead = 0;
  if (lane < NS) ptx::mbar_init(ptx::smem_u32(&bar[warp][lane]), 1);
  ptx::fence_barrier_init();
  __syncthreads();
  rb::pdl_trigger();
  rb::pdl_wait();
  // ---- the warp's work: share `share` of `shares` of the rows of one (sequence, kv head, set of REP query heads)
  const int rep = p.nq / p.nkv, sets = RB_CEIL_DIV(rep, REP);
  const unsigned all = (unsigned)p.B * p.nkv * sets, at_work = blockIdx.x * (kWarps / p.wide) + warp / p.wide;
  const unsigned work = min(at_work, all - 1), pair = work / sets, nth = pair / p.nkv;     // (the last block's warps beyond the work go along and store nothing)
  const int hkv = (int)(pair % p.nkv), h0 = (int)(work % sets) * REP, heads = min(REP, rep - h0);
  int b = nth, len;
  if (p.longest_first) b = sequence_of(p.lens, p.B, p.room, nth, len); else len = p.lens[b];
  const int share = blockIdx.y * p.wide + warp % p.wide, shares = p.splits * p.wide;
  const int pos = len < p.room ? len : -1;
  const bool live = pos >= 0 && at_work < all;
  // ---- its queries (a group of D / 8 lanes has one; the warps of a work share them) and the new key and value, asked for ahead of the tiles
  const T* qkv = reinterpret_cast<const T*>(p.qkv) + b * p.qkv_stride;
  const int sub = lane % LPR, wi = warp % p.wide, w0 = warp - wi;
  float xn[kTurns][8], kv[8];
#pragma unroll
  for (int i = 0; i < kTurns; ++i)
    if (i % p.wide == wi) load8(qkv + (int64_t)(hkv * rep + h0 + min(lane / LPR + i * RPT, heads - 1)) * D + sub * 8, xn[i]);
  // steps of two tiles of the rows [0, pos]; who has the last one has the new row: of it lanes of even groups have the key, of odd ones the value
  const int n_tiles = live ? pos / 16 + 1 : 0, n_steps = (n_tiles + 1) / 2;
  const bool fresh = live && (n_steps - 1) % shares == share, of_value = lane / LPR % 2;
  if (fresh) load8(qkv + (int64_t)(p.nq + (of_value ? p.nkv : 0) + hkv) * D + sub * 8, kv);
  Turn turn;
  if (p.cos && live) load_turn(turn, sub, p, pos);
  uint32_t* cache = p.cache + ((int64_t)b * p.nkv + hkv) * p.tiles * Tl::kWords;
  const uint32_t base = ptx::smem_u32(ring) + warp * (uint32_t)kRing;
  auto fetch = [&](int step, int slot) {
    if (step < n_steps && ptx::elect_one()) {
      const uint32_t full = ptx::smem_u32(&bar[warp][slot]), bytes = min(2, n_tiles - 2 * step) * Tl::kBytes;
      ptx::mbar_arrive_expect_tx(full, bytes);
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(base + slot * (2 * Tl::kBytes)),
                   "l"(cache + (int64_t)step * (2 * Tl::kWords)), "r"(bytes), "r"(full) : "memory");
    }
  };
#pragma unroll
  for (int n = 0; n < NS; ++n) fetch(share + n * shares, n);

#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    if (i % p.wide != wi) continue;
    const int r = lane / LPR + i * RPT;
    if (p.cos) rotate8<D>(xn[i], sub, turn, p);
    // sums over the key groups, then whole numbers: the largest element to 2^21 .. 2^22
    float sum = 0.f, most = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      xn[i][e] *= p.scale;
      most = q4::max_nan(most, fabsf(xn[i][e]));
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) most = q4::max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    // (ex is 254 at most in a finite query; the factors below stay normal numbers, and below 2^-105 a query's elements keep fewer bits)
    const int ex = (int)(__float_as_uint(most) >> 23), up = max(min(21 + 127 - ex, 126), 21 + 127 - 254);
    const float down = power2(up - 12);              // 32 numbers below 2^22: their sum, taken by 2^(up - 12), is below 2^15
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(xn[i][e], down, sum);
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (r < REP) {                                   // (heads beyond the set repeat its last one and are not stored)
      if (sub == 0) s_unit[w0][r] = ex == 255 ? __int_as_float(0x7fc00000) : power2(-up);   // (an infinity or a NaN: every score is NaN)
      if (sub % 4 == 0) {
        float rest = sum;
#pragma unroll
        for (int d = 0; d < 3; ++d) {
          const T x = rb::from_f<T>(rest);
          ssums[w0][d][r][sub / 4] = *reinterpret_cast<const uint16_t*>(&x);
          rest -= rb::to_f(x);
        }
      }
      // n = d0 + 256 d1 + 65536 d2 with signed bytes: the bytes of n + 0x808080, each less 128.  n is read off the last bits of 1.5 2^23 + n.
      uint32_t n[8];
      const float f = power2(up);
#pragma unroll
      for (int e = 0; e < 8; ++e) n[e] = __float_as_uint(fmaf(xn[i][e], f, 12582912.f)) + (0x808080u - 0x4b400000u);
      uint32_t bytes[3][2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t a = __byte_perm(n[4 * q], n[4 * q + 1], 0x5140), c = __byte_perm(n[4 * q + 2], n[4 * q + 3], 0x5140);
        bytes[0][q] = __byte_perm(a, c, 0x5410) ^ 0x80808080u;
        bytes[1][q] = __byte_perm(a, c, 0x7632) ^ 0x80808080u;
        bytes[2][q] = __byte_perm(__byte_perm(n[4 * q], n[4 * q + 1], 0x0062), __byte_perm(n[4 * q + 2], n[4 * q + 3], 0x0062), 0x5410) ^ 0x80808080u;
      }
#pragma unroll
      for (int d = 0; d < 3; ++d) *reinterpret_cast<uint2*>(&sbytes[w0][d][r][sub * 2]) = make_uint2(bytes[d][0], bytes[d][1]);
    }
  }
  if (fresh) {                                      // the new row: quantised and written; it goes into the last tile when that has come
    if (p.cos) {
      float turned[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) turned[e] = kv[e];
      rotate8<D>(turned, sub, turn, p);
#pragma unroll
      for (int e = 0; e < 8; ++e) kv[e] = of_value ? kv[e] : rb::to_f(rb::from_f<T>(turned[e]));
    }
    float klo, khi;
    q4::extremes<4>(kv, klo, khi);
    const float vlo = q4::min_nan(klo, __shfl_xor_sync(0xffffffffu, klo, 4)), vhi = q4::max_nan(khi, __shfl_xor_sync(0xffffffffu, khi, 4));
    const uint32_t new_group = q4::group_word<T>(of_value ? vlo : klo, of_value ? vhi : khi);
    uint32_t code[8], new_word = 0;
    q4::codes8(kv, q4::scale_of<T>(new_group), q4::low_of<T>(new_group), code);
#pragma unroll
    for (int e = 0; e < 8; ++e) new_word |= code[e] << (of_value ? q4::bit_of<q4::kValue>(e) : q4::bit_of<q4::kKey>(e));
    s_new[warp][lane] = make_uint2(new_word, new_group);
  }
  auto put_row = [&](uint32_t* tile) {              // the new row's words and groups into its tile, in global or in shared memory
    const int r = pos % 16;
    const uint32_t new_word = s_new[warp][lane].x, new_group = s_new[warp][lane].y;
    if (lane >= 2 * LPR) return;
    if (of_value) {
      uint16_t* halves = reinterpret_cast<uint16_t*>(tile + Tl::kValues) + q4::half_place(sub, r);
      halves[0] = (uint16_t)new_word;
      halves[2] = (uint16_t)(new_word >> 16);
    } else {
      tile[r * Tl::W + q4::word_place<J>(sub)] = new_word;
    }
    if (sub % (of_value ? 8 : 4) == 0) tile[of_value ? Tl::kValueScales + r * H + sub / 8 : Tl::kKeyScales + r * J + sub / 4] = new_group;
  };
  if (fresh && h0 == 0) put_row(cache + (int64_t)(pos / 16) * Tl::kWords);
  if (p.wide == 1) __syncwarp(); else __syncthreads();

  // ---- the queries as column operands: column g of product c is (byte, head g % REP); of the weights, (part g / REP, head g % REP): columns beyond the parts are never looked at
  const int head = g % REP, part = min(g / REP, 1);
  auto byte_of = [](int c, int col) { return min(REP == 8 ? c : REP == 4 ? 2 * c + col / 4 : col / REP, 3); };
  uint32_t qb[J][kScores][2], sb[kScores];          // sb: the sums of group t
  float unit[kScores][2], unit_low[2];              // of the columns 2t, 2t + 1
#pragma unroll
  for (int c = 0; c < kScores; ++c) {
    const int mine = byte_of(c, g);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      ld_words(qb[j][c], ptx::smem_u32(&sbytes[w0][min(mine, 2)][head][8 * j + 2 * t]));
      if (mine > 2) qb[j][c][0] = qb[j][c][1] = 0;
    }
    sb[c] = mine < 3 && t < J ? ssums[w0][mine][head][t % J] : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int byte = byte_of(c, 2 * t + i);
      unit[c][i] = byte < 3 ? s_unit[w0][(2 * t + i) % REP] * (byte == 0 ? 1.f : byte == 1 ? 256.f : 65536.f) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) unit_low[i] = s_unit[w0][(2 * t + i) % REP] * 4096.f;

  float o[4 * H][4];
#pragma unroll
  for (int j = 0; j < 4 * H; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m = -INFINITY, l = 0.f, z[H];               // of head `head`, over the lane's keys: maximum, sum of weights, sums of weights times lowest values
#pragma unroll
  for (int h = 0; h < H; ++h) z[h] = 0.f;
  // Weights are 2^(s - m - kSpare): sums of the type's largest numbers over thousands of rows stay inside fp32, and so do the codes' part and the lowest values' part of a group that spans the
  // whole type, which cancel; numbers of 2^-126 still keep the bits that bf16 has.  A weight goes into the products as `unit_w` times it, so that they are 2^(10 - top) 2^(s - m); every
  // value scale so far is below 2^top.  l and z are free of that factor: a lowest value may be any number of the type where steps are 0, and a factor made for small steps would take
  // it past fp32.
  constexpr int kSpare = 12, kRoom = 14 - (int)kSlack + kSpare;
  float unit_w = power2(kRoom + 100);               // (top = -100)
  uint32_t bound = 0;                               // the group word of 2^top
  int slot = 0;
  uint32_t round = 0;                               // parity of the ring's current round
#pragma unroll 1
  for (int step = share; step < n_steps; step += shares) {
    bounded_wait(ptx::smem_u32(&bar[warp][slot]), round, dead);
    const uint32_t at = base + slot * (2 * Tl::kBytes);
    if (fresh && step == n_steps - 1) {
      put_row(reinterpret_cast<uint32_t*>(ring + warp * kRing + slot * (2 * Tl::kBytes)) + (pos / 16 - 2 * step) * Tl::kWords);
      __syncwarp();
    }
    // ---- scores of 2 x 16 keys: lane (g, t) gets keys g and g + 8 of columns 2t and 2t + 1, then the keys 2t, 2t + 1, 2t + 8, 2t + 9 of head g % REP
    float s[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t w0[J], w1[J], s0[J], s1[J];
      ld_words(w0, at + u * Tl::kBytes + g * (D / 2) + t * (J * 4));
      ld_words(w1, at + u * Tl::kBytes + (g + 8) * (D / 2) + t * (J * 4));
      ld_words(s0, at + u * Tl::kBytes + Tl::kKeyScales * 4 + g * (J * 4));
      ld_words(s1, at + u * Tl::kBytes + Tl::kKeyScales * 4 + (g + 8) * (J * 4));
      float x[kScores][4] = {}, y[4] = {};
      {
        uint32_t a0, a1;                            // the group words as operands: lowest values, and scales that meet zeros
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(a0) : "r"(at + u * Tl::kBytes + Tl::kKeyScales * 4 + g * (J * 4) + t % J * 4) : "memory");
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(a1) : "r"(at + u * Tl::kBytes + Tl::kKeyScales * 4 + (g + 8) * (J * 4) + t % J * 4) : "memory");
#pragma unroll
        for (int c = 0; c < kScores; ++c) mma_k8<T>(y, a0, a1, sb[c]);
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float f0 = q4::scale_of<T>(s0[j]), f1 = q4::scale_of<T>(s1[j]);
        constexpr uint32_t kLow = 0x0f0f0f0fu;
#pragma unroll
        for (int c = 0; c < kScores; ++c) {
          int d[4];                                 // 1.5 2^23 as fp32's bits, plus the sum: a number whose difference from 1.5 2^23 is the sum
          mma_s8(d, w0[j] & kLow, w1[j] & kLow, w0[j] >> 4 & kLow, w1[j] >> 4 & kLow, qb[j][c][0], qb[j][c][1], 0x4b400000);
          float n[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) n[i] = __int_as_float(d[i]);
          add_pair(n[0], n[1], -12582912.f, -12582912.f);
          add_pair(n[2], n[3], -12582912.f, -12582912.f);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[c][i] = fmaf(i < 2 ? f0 : f1, n[i], x[c][i]);
        }
      }
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = fmaf(x[0][i], unit[0][i & 1], y[i] * unit_low[i & 1]);
#pragma unroll
        for (int c = 1; c < kScores; ++c) v[i] = fmaf(x[c][i], unit[c][i & 1], v[i]);
      }
      // the bytes of a head added up: in columns 0 .. 2 (lanes t = 0, 1), in pairs of columns (t = 0 .. 2), in halves of the columns
      if constexpr (REP == 1) { v[0] += v[1]; v[2] += v[3]; }
#pragma unroll
      for (int i = 0; i < 4; i += REP == 1 ? 2 : 1) {
        if constexpr (REP <= 2) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 1);
        if constexpr (REP == 2 || REP == 4) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 2);
      }
      if constexpr (REP == 8) {
        const int from = 8 * t + (head >> 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float even = __shfl_sync(0xffffffffu, v[(i >> 1) * 2], from + (i & 1) * 4), odd = __shfl_sync(0xffffffffu, v[(i >> 1) * 2 + 1], from + (i & 1) * 4);
          s[u][i] = head & 1 ? odd : even;
        }
      } else {
        // lanes of a row that hold the same sums offer one head each: t & 1, or for four heads 2 (t & 1) + (t >> 1)
        const bool second = REP == 2 ? t & 1 : (REP == 4 ? t >> 1 : false);
        const float lo8 = second ? v[1] : v[0], hi8 = second ? v[3] : v[2];
        const int from = 8 * t + (REP == 4 ? (head >> 1) | ((head & 1) << 1) : head);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][i] = __shfl_sync(0xffffffffu, i < 2 ? lo8 : hi8, from + (i & 1) * 4);
      }
    }
    // the value groups of those keys
    uint32_t vg[2][4][H];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t a[2 * H], c[2 * H];
      ld_words(a, at + u * Tl::kBytes + Tl::kValueScales * 4 + 2 * t * (H * 4));
      ld_words(c, at + u * Tl::kBytes + Tl::kValueScales * 4 + (2 * t + 8) * (H * 4));
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < H; ++h) { vg[u][i][h] = a[i * H + h]; vg[u][2 + i][h] = c[i * H + h]; }
    }
    if (step * 32 + 32 > pos + 1) {                    // rows behind the length may hold anything
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (step * 32 + u * 16 + 2 * t + (i & 1) + (i >> 1) * 8 > pos) {
            s[u][i] = -INFINITY;
#pragma unroll
            for (int h = 0; h < H; ++h) vg[u][i][h] = 0;
          }
    }
    // ---- running softmax; the accumulators are corrected only where a maximum has grown by more than kSlack or the unit moved
    float mx = m;
    uint32_t most = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mx = fmaxf(mx, s[u][i]);
#pragma unroll
        for (int h = 0; h < H; ++h) most = max(most, vg[u][i][h]);
      }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    if (__any_sync(0xffffffffu, mx > m + kSlack || most >= bound)) {
      const float corr = ex2(m - (mx == -INFINITY ? 0.f : mx));
      float corr_o = corr;
      m = mx;
      constexpr uint32_t kNan = std::is_same<T, __half>::value ? 0x7c000000u : 0x7f800000u;   // infinities and NaN: no unit holds them
      most = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < H; ++h) most = max(most, vg[u][i][h] < kNan ? vg[u][i][h] : 0u);
      most = __reduce_max_sync(0xffffffffu, most);
      if (most >= bound) {                          // two bits of room, so that it seldom moves
        constexpr int kShift = std::is_same<T, __half>::value ? 26 : 23, kBias = std::is_same<T, __half>::value ? 15 : 127;
        const int ex = min((int)(most >> kShift) + 3, (int)(kNan >> kShift)), was = kRoom + 127 - (int)(__float_as_uint(unit_w) >> 23), top = max(min(ex - kBias, 127), -100);
        unit_w = power2(kRoom - top);
        bound = (uint32_t)ex << kShift;
        corr_o *= power2(max(was - top, -126));
      }
      l *= corr;
#pragma unroll
      for (int h = 0; h < H; ++h) z[h] *= corr;
      const float ce = __shfl_sync(0xffffffffu, corr_o, 8 * t), co = __shfl_sync(0xffffffffu, corr_o, 8 * t + 4);   // of columns 2t, 2t + 1
#pragma unroll
      for (int j = 0; j < 4 * H; ++j) { o[j][0] *= ce; o[j][1] *= co; o[j][2] *= ce; o[j][3] *= co; }
    }
    const float zero = (m == -INFINITY ? 0.f : m) + (float)kSpare;
    // ---- sums: codes^T times the weights' parts.  A lane's eight channels of four keys: rows g are the first quad of channels, rows g + 8 the second.  Products begin at zero and are added
    // to the sums in fp32: the tensor core cuts off what it adds to an accumulator instead of rounding it, and sums of codes, which are all positive, fall behind (128 x 639 rows: errors of 3.8e-5
    // of the outputs' size before their rounding, so 0.9e-5).
#pragma unroll
    for (int u0 = 0; u0 < 2; u0 += kTogether) {
      float w[kTogether][4], wu[kTogether][4];
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[u][i] = ex2(s[u0 + u][i] - zero);
          wu[u][i] = w[u][i] * unit_w;
        }
        l += (w[u][0] + w[u][1]) + (w[u][2] + w[u][3]);
      }
#pragma unroll
      for (int h = 0; h < H; ++h) {
        uint32_t pb[kTogether][kProd][2], w4[kTogether][4];
#pragma unroll
        for (int u = 0; u < kTogether; ++u) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t g0 = vg[u0 + u][2 * e][h], g1 = vg[u0 + u][2 * e + 1][h];
            const float a = wu[u][2 * e] * q4::scale_of<T>(g0), c = wu[u][2 * e + 1] * q4::scale_of<T>(g1);
            z[h] = fmaf(w[u][2 * e], q4::low_of<T>(g0), z[h]);
            z[h] = fmaf(w[u][2 * e + 1], q4::low_of<T>(g1), z[h]);
            const uint32_t p0 = pack2<__half>(a, c);
            const float2 f0 = unpack_half2(p0);
            const uint32_t p1 = pack2<__half>(a - f0.x, c - f0.y);
            if constexpr (REP == 8) { pb[u][0][e] = p0; pb[u][1][e] = p1; } else pb[u][0][e] = part ? p1 : p0;
          }
          ld_words(w4[u], at + (u0 + u) * Tl::kBytes + Tl::kValues * 4 + h * 512 + g * 64 + t * 16);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x[4] = {};
#pragma unroll
          for (int u = 0; u < kTogether; ++u)
#pragma unroll
            for (int f = 0; f < kProd; ++f)
              mma_f16(x, nibbles(w4[u][0], i), nibbles(w4[u][1], i), nibbles(w4[u][2], i), nibbles(w4[u][3], i), pb[u][f][0], pb[u][f][1]);
          float(&to)[4] = o[4 * h + i];
          add_pair(to[0], to[1], x[0], x[1]);
          add_pair(to[2], to[3], x[2], x[3]);
        }
      }
    }
    __syncwarp();
    fetch(step + NS * shares, slot);
    if (++slot == NS) { slot = 0; round ^= 1; }
  }
  __syncwarp();

  // ---- merge the shares of a work: those of the block, then those of the cluster.  A warp's sums take the place of its ring.
  static_assert(kRing >= REP * D * 4, "");
  float* mysum = reinterpret_cast<float*>(ring + warp * kRing);
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
#pragma unroll
  for (int h = 0; h < H; ++h) {
    z[h] += __shfl_xor_sync(0xffffffffu, z[h], 1);
    z[h] += __shfl_xor_sync(0xffffffffu, z[h], 2);
  }
  const float back = power2(127 - (int)(__float_as_uint(unit_w) >> 23));
  if (g < REP && t == 0) {
    sm_m[warp][head] = m;
    sm_l[warp][head] = l;
#pragma unroll
    for (int h = 0; h < H; ++h) sm_z[warp][h][head] = z[h];
  }
#pragma unroll
  for (int h = 0; h < H; ++h) {
    float x[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i][j] = o[4 * h + j][i] * 131072.f * back;   // 2^17 of the codes; apart, since the product of the two can leave fp32
        if constexpr (REP == 2 || REP == 4) x[i][j] += __shfl_xor_sync(0xffffffffu, x[i][j], REP / 2);
      }
      if constexpr (REP == 1) { x[0][j] += x[1][j]; x[2][j] += x[3][j]; }
    }
    // lanes whose columns are heads: channels 64 h + 8 g .. (rows g), and the next four (rows g + 8)
    const int d = 64 * h + 8 * g;
    auto put = [&](int r, const float (&a)[4], const float (&c)[4]) {
      *reinterpret_cast<float4*>(mysum + r * D + d) = make_float4(a[0], a[1], a[2], a[3]);
      *reinterpret_cast<float4*>(mysum + r * D + d + 4) = make_float4(c[0], c[1], c[2], c[3]);
    };
    if (2 * t < REP) {
      put(2 * t, x[0], x[2]);
      if constexpr (REP > 1) put(2 * t + 1, x[1], x[3]);
    }
  }
  if (p.wide == 1) __syncwarp(); else __syncthreads();
  T* out = reinterpret_cast<T*>(p.out) + (int64_t)b * p.nq * D + (int64_t)(hkv * rep + h0) * D;
  auto write4 = [&](int at4, const float (&a)[4], float l4) {
    // (a mean of what the cache holds can lie above T's largest number by the rounding of a step: finite numbers stay finite)
    constexpr float kMost = std::is_same<T, __half>::value ? 65504.f : 3.3895313892515355e38f;
    rb::Pack<T, 4> x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = live ? a[i] / l4 : 0.f;
      x.v[i] = rb::from_f<T>(fabsf(y) <= 3.4028234663852886e38f ? fminf(fmaxf(y, -kMost), kMost) : y);
    }
    *reinterpret_cast<rb::Pack<T, 4>*>(out + at4 * 4) = x;
  };
  for (int c4 = wi * 32 + lane; c4 < heads * (D / 4); c4 += p.wide * 32) {   // four channels a lane
    const int r = c4 / (D / 4), d = c4 % (D / 4) * 4;
    float mg = -INFINITY, lg = 0.f, ag[4] = {};
    for (int w = w0; w < w0 + p.wide; ++w) mg = fmaxf(mg, sm_m[w][r]);
    for (int w = w0; w < w0 + p.wide; ++w) {
      const float c = sm_m[w][r] == -INFINITY ? 0.f : ex2(sm_m[w][r] - mg), zw = sm_z[w][d / 64][r];
      const float4 x = reinterpret_cast<const float4*>(ring + w * kRing)[c4];
      lg = fmaf(sm_l[w][r], c, lg);
      ag[0] = fmaf(x.x + zw, c, ag[0]);
      ag[1] = fmaf(x.y + zw, c, ag[1]);
      ag[2] = fmaf(x.z + zw, c, ag[2]);
      ag[3] = fmaf(x.w + zw, c, ag[3]);
    }
    if (p.splits == 1) {
      if (at_work < all) write4(c4, ag, lg);
    } else {
      *reinterpret_cast<float4*>(&cta_acc[r][d]) = make_float4(ag[0], ag[1], ag[2], ag[3]);
      if (d == 0) { cta_m[r] = mg; cta_l[r] = lg; }
    }
  }
  if (*dead) {
    __syncwarp();
    if (lane == 0) {
      *reinterpret_cast<volatile int*>(p.status) = rb::kStatusGaveUp;
      __threadfence_system();
    }
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  if (p.splits == 1) return;
  ptx::cluster_sync();
  // the cluster is (1, splits) blocks of one work: each finishes its share of the outputs from everybody's sums
  auto peer = [](const float* x, int cta) {
    uint32_t a;
    float f;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(ptx::smem_u32(x)), "r"(cta));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(a) : "memory");
    return f;
  };
  const int each = RB_CEIL_DIV(heads * (D / 4), p.splits);
  for (int i = threadIdx.x; i < each; i += kDecThreads) {
    const int c4 = blockIdx.y * each + i, r = c4 / (D / 4), d = c4 % (D / 4) * 4;
    if (c4 >= heads * (D / 4)) break;
    float mg = -INFINITY, lg = 0.f, ag[4] = {};
#pragma unroll 4
    for (int c = 0; c < p.splits; ++c) mg = fmaxf(mg, peer(&cta_m[r], c));
#pragma unroll 4
    for (int c = 0; c < p.splits; ++c) {
      const float mc = peer(&cta_m[r], c), w = mc == -INFINITY ? 0.f : ex2(mc - mg);
      const float4 x = ptx::ld_cluster_f4(ptx::smem_u32(&cta_acc[r][d]), c);
      lg = fmaf(peer(&cta_l[r], c), w, lg);
      ag[0] = fmaf(x.x, w, ag[0]);
      ag[1] = fmaf(x.y, w, ag[1]);
      ag[2] = fmaf(x.z, w, ag[2]);
      ag[3] = fmaf(x.w, w, ag[3]);
    }
    write4(c4, ag, lg);
  }
  ptx::cluster_sync();  // nobody leaves while its sums are being read
}

template <typename T, int D, int REP> int launch_one(const StepParams& p, cudaStream_t s) {
  static std::atomic<uint64_t> opted_in{0};          // the attribute is the kernel's on one device: a bit per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -3;
  if (dev >= 64 || !(opted_in.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(decode_int4_kernel<T, D, REP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem) != cudaSuccess) return -3;
    if (dev < 64) opted_in.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg{};
  const int64_t works = (int64_t)p.B * p.nkv * RB_CEIL_DIV(p.nq / p.nkv, REP);
  cfg.gridDim = dim3((unsigned)((works * p.wide + kWarps - 1) / kWarps), p.splits);
  cfg.blockDim = dim3(kDecThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (p.splits > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = attr[n].val.clusterDim.z = 1;
    attr[n++].val.clusterDim.y = p.splits;
  }
  if (rb::pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, decode_int4_kernel<T, D, REP>, p) == cudaSuccess ? 0 : -3;
}

template <typename T, int D> int launch(StepParams p, cudaStream_t s) {
  const int rep = p.nq / p.nkv, heads = rep == 1 ? 1 : rep == 2 ? 2 : rep <= 4 ? 4 : 8;
  // Warps a work, then blocks: doubled as long as all of them still fit at once and each keeps two steps of a full cache
  const int64_t works = (int64_t)p.B * p.nkv * RB_CEIL_DIV(rep, heads), places = (int64_t)rb::kNumSMs * ctas_of(heads) * kWarps;
  p.wide = p.splits = 1;
  while (p.wide * p.splits < kWarps * kMaxSplits && works * p.wide * p.splits * 2 <= places && p.tiles >= 8 * p.wide * p.splits) (p.wide < kWarps ? p.wide : p.splits) *= 2;
  // The longest sequences first, where there are more works than places: the last to begin are short ones then (128 x 639 rows of 32 heads 57 us, in the order given 66; where all
  // begin at once the order is only its own cost).
  p.longest_first = p.B > 1 && p.B <= kRanked && works > places;
  if (works * p.wide > 0x7fffffff) return -1;
  return heads == 1 ? launch_one<T, D, 1>(p, s) : heads == 2 ? launch_one<T, D, 2>(p, s) : heads == 4 ? launch_one<T, D, 4>(p, s) : launch_one<T, D, 8>(p, s);
}

}  // namespace

// rot_dim a multiple of 16 (interleaved: of 2).  dt: 1 bf16, 2 fp16.
extern "C" int rb_decode_attention_int4(const void* qkv, void* cache, const int* lens, void* out, const float* cos, const float* sin, int64_t qkv_stride, int B, int nq,
                                        int nkv, int hd, int room, int rot_dim, int interleaved, float scale, int dt, cudaStream_t s) {
  if (B == 0) return 0;
  const StepParams p{qkv, reinterpret_cast<uint32_t*>(cache), lens, out, cos, sin, qkv_stride, B, nq, nkv, room, (room + 15) / 16, rot_dim, interleaved, 0, 1, 1,
                 scale * 1.4426950408889634f, rb_attn_status()};
  if (p.status == nullptr) return -5;
  if (dt == 1 && hd == 128) return launch<__nv_bfloat16, 128>(p, s);
  if (dt == 1 && hd == 64) return launch<__nv_bfloat16, 64>(p, s);
  if (dt == 2 && hd == 128) return launch<__half, 128>(p, s);
  if (dt == 2 && hd == 64) return launch<__half, 64>(p, s);
  return -2;
}
