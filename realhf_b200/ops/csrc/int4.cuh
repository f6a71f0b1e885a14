// Numbers in groups of 4-bit codes: x ~ scale * c + low with low = min x, scale = T((max x - low) / 15), c = 0 .. 15 (T: the 16-bit type of the model).
//
// A group's numbers are one word: scale in its upper half, low in its lower half.  Codes go to matrix instructions as they are, so each kind of operand has the order of
// nibbles that costs the fewest instructions to take apart:
//   key words     eight channels c, at bits 8 (c & 3) + 4 (c >> 2): two masks and a shift leave two operands of four bytes.
//   value halves  four channels c of one row at bits 4 c of a half-word, a row's neighbour in the other half: a shift and a mask leave pairs of neighbouring rows in bits 7 .. 10, where a code
//                 is the fp16 number c 2^-17.
//   weight words  eight channels c, at bits 4 (c >> 1) + 16 (c & 1): pairs of neighbouring channels, which a mask and a larger number's bits make exact 16-bit numbers.
//
// A row of n words (n / 4 = channels / 32 = J) is stored as [t = 0 .. 3][j < J], word (t, j) holding the channels 32 j + 8 t ..: the four lanes of a row in a matrix
// instruction's operand take 16 neighbouring bytes each, and what they take together for step j lies in one group of 32.
//
// A cache is tiles of 16 rows of one head: key words [row][t][j], the values, the keys' group words [row][D / 32], the values' [row][D / 64].  The values of a tile are
// [channels / 8][t = 0 .. 3][row / 8][quad of channels][row & 1] halves, t = (row & 7) / 2: a lane's four rows and eight channels are 16 neighbouring bytes.
#pragma once
#include "common.cuh"

#include <type_traits>

namespace q4 {

constexpr int kRows = 16;            // rows of a tile
constexpr int kKeyGroup = 32, kValueGroup = 64;

template <int D> struct Tile {
  static constexpr int J = D / 32;                       // words a lane takes of a key; key groups
  static constexpr int H = D / kValueGroup;              // value groups
  static constexpr int W = D / 8;                        // words of a row
  static constexpr int kValues = kRows * W, kKeyScales = 2 * kRows * W, kValueScales = kKeyScales + kRows * J;   // offsets in words
  static constexpr int kWords = kValueScales + kRows * H;
  static constexpr int kBytes = kWords * 4;
};

// the first of the two halves (the other is two further) that hold the channels 8 w .. of row r
RB_DEVICE int half_place(int w, int r) { return 32 * w + 8 * ((r & 7) >> 1) + 4 * (r >> 3) + (r & 1); }
// the place of word w (channels 8 w ..) in a row
template <int J> RB_DEVICE int word_place(int w) { return (w & 3) * J + (w >> 2); }

RB_DEVICE float min_nan(float a, float b) { float d; asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b)); return d; }
RB_DEVICE float max_nan(float a, float b) { float d; asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b)); return d; }

template <typename T> RB_DEVICE uint32_t bits16(float x) {
  const T v = rb::from_f<T>(x);
  return *reinterpret_cast<const uint16_t*>(&v);
}
template <typename T> RB_DEVICE float scale_of(uint32_t w) {
  if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) return __uint_as_float(w & 0xffff0000u);   // (bf16: fp32's upper half)
  return __high2float(*reinterpret_cast<const __half2*>(&w));
}
template <typename T> RB_DEVICE float low_of(uint32_t w) {
  if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) return __uint_as_float(w << 16);
  return __low2float(*reinterpret_cast<const __half2*>(&w));
}

// The group word of a group whose extremes are lo and hi; a group that holds an infinity or a NaN is NaN throughout.  Everything is taken by 1/16, an exact factor,
// so that the widest group of bf16 does not leave fp32.
template <typename T> RB_DEVICE uint32_t group_word(float lo, float hi) {
  constexpr float kMost = 3.4028234663852886e38f;
  if (!(fabsf(lo) <= kMost && fabsf(hi) <= kMost)) return bits16<T>(__int_as_float(0x7fc00000)) * 0x10001u;
  return bits16<T>(__fdiv_rn(__fsub_rn(hi * 0.0625f, lo * 0.0625f), 0.9375f)) << 16 | bits16<T>(lo);
}
// (x - low) / scale is taken as (x f - l) / s with an exact factor f that keeps the largest and the smallest groups inside fp32's normal numbers.
struct Grid { float f, s, l; };
RB_DEVICE Grid grid_of(float scale, float low) {
  const float f = scale < 8.67e-19f ? 1.8446744073709552e19f : 0.0625f;    // 2^-60, 2^64
  return {f, scale * f, low * f};
}
// The codes of eight numbers of a group: (x - low) / scale rounded to the nearest whole number, halves to the even one.  The quotient is correctly rounded: a product with the
// correctly rounded reciprocal, corrected once by its remainder (Markstein's theorem), so that ties are ties.
RB_DEVICE void codes8(const float (&x)[8], float scale, float low, uint32_t (&c)[8]) {
  const Grid g = grid_of(scale, low);
  const float r = __frcp_rn(g.s);
  const bool any = scale > 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fmaf(x[i], g.f, -g.l), q = __fmul_rn(a, r), e = fmaf(fmaf(-q, g.s, a), r, q);
    c[i] = any ? __float_as_uint(__fadd_rn(fminf(e, 15.f), 12582912.f)) & 15u : 0u;   // (1.5 2^23: the sum's last bits are the whole number)
  }
}
constexpr int kKey = 0, kValue = 1, kWeight = 2;
template <int kKind> RB_DEVICE constexpr int bit_of(int c) { return kKind == kKey ? 8 * (c & 3) + 4 * (c >> 2) : kKind == kValue ? 4 * c : 4 * (c >> 1) + 16 * (c & 1); }

// two fp32 numbers at once
RB_DEVICE uint64_t both(float a, float b) { uint64_t d; asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b)); return d; }
RB_DEVICE void parts(uint64_t d, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d)); }
RB_DEVICE uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }
RB_DEVICE uint64_t mul2(uint64_t a, uint64_t b) { uint64_t d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
RB_DEVICE uint64_t add2(uint64_t a, uint64_t b) { uint64_t d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }

// two numbers of T in a word as fp32
template <typename T> RB_DEVICE void numbers(uint32_t u, float& a, float& b) {
  if constexpr (std::is_same<T, __half>::value) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    a = f.x, b = f.y;
  } else {
    a = __uint_as_float(u << 16), b = __uint_as_float(u & 0xffff0000u);
  }
}

// a * by + w as one integer multiply-add, which keeps shifts and sums off the pipe that minima, masks and shifts have
RB_DEVICE uint32_t shifted_onto(uint32_t a, uint32_t by, uint32_t w) { uint32_t d; asm("mad.lo.u32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(by), "r"(w)); return d; }

// Eight numbers of T (two a word) of a group with the extremes lo and hi: the group's word and that of the codes.  Where the group is finite and its step not so far below T's
// normal numbers that a quotient could reach 15.5, nothing has to be cut at 15, the factor is 1/16, and two numbers at once take five instructions and an addition each: whole
// numbers in the last bits of 1.5 2^23 + c, added up in their places, less what the sum of the shifted 1.5 2^23s is, modulo 2^32.  All other groups, those of one value among
// them, take the long way.
struct Coded { uint32_t word, group; };
template <typename T, int kKind> __device__ __noinline__ Coded code8_long(uint4 u, float lo, float hi) {
  const uint32_t words[4] = {u.x, u.y, u.z, u.w};
  const uint32_t g = group_word<T>(lo, hi);
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) numbers<T>(words[i], x[2 * i], x[2 * i + 1]);
  uint32_t c[8], w = 0;
  codes8(x, scale_of<T>(g), low_of<T>(g), c);
#pragma unroll
  for (int i = 0; i < 8; ++i) w |= c[i] << bit_of<kKind>(i);
  return {w, g};
}
template <typename T, int kKind> RB_DEVICE Coded code8(const uint4& u, float lo, float hi) {
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr float kLeast = kHalf ? 1.9073486e-6f : 8.8817842e-16f;   // fp16: steps of 2^-19 and more are off by 2^-6 at most (relative); bf16: 2^-50
  const uint32_t words[4] = {u.x, u.y, u.z, u.w};
  const float l = -0.0625f * lo, wide = fmaf(hi, 0.0625f, l);
  if (wide >= kLeast && wide <= 3.4028234663852886e38f) {
    constexpr float kFifteen = 1.f / 0.9375f;
    const float q15 = __fmul_rn(wide, kFifteen), step = fmaf(fmaf(-q15, 0.9375f, wide), kFifteen, q15);
    uint32_t g;
    if constexpr (kHalf) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(g) : "f"(step), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(g) : "f"(step), "f"(lo));
    // The correctly rounded reciprocal: one step from an approximation that is off by an ulp at most (Markstein again; s has 11 bits at most, so is none of the exceptions).
    const float s = scale_of<T>(g) * -0.0625f;                              // (negated, as the products want it)
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(-s));
    r = fmaf(fmaf(s, r, 1.f), r, r);
    const uint64_t f2 = both(0.0625f, 0.0625f), l2 = both(l, l), r2 = both(r, r), s2 = both(s, s), magic = both(12582912.f, 12582912.f);
    uint32_t w = 0, extra = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x, y;
      numbers<T>(words[i], x, y);
      const uint64_t a = fma2(both(x, y), f2, l2), q = mul2(a, r2), e = add2(fma2(fma2(q, s2, a), r2, q), magic);
      w = shifted_onto((uint32_t)e, 1u << bit_of<kKind>(2 * i), w);
      w = shifted_onto((uint32_t)(e >> 32), 1u << bit_of<kKind>(2 * i + 1), w);
      extra += (0x4b400000u << bit_of<kKind>(2 * i)) + (0x4b400000u << bit_of<kKind>(2 * i + 1));
    }
    return {w - extra, g};
  }
  if ((__float_as_uint(lo) | __float_as_uint(hi)) == 0) return {0, 0};      // (zeros: rows of padding)
  return code8_long<T, kKind>(u, lo, hi);
}
// A word's channels as numbers of T, two a word: scale * c is exact, so two roundings, fp32's and T's.  A step that was rounded up can leave 15 steps above T's largest number, which is
// what is read back then (NaN stays NaN).  `magic`: 2^23's bits, as a number that the compiler does not know
// (a mask and a magic number as two immediates are two instructions where an immediate and a register are one).
constexpr uint32_t kWholeMagic = 0x4b000000u;
template <typename T, int kKind> RB_DEVICE uint4 unpack8(uint32_t w, uint32_t g, uint32_t magic) {
  const float scale = scale_of<T>(g), low = low_of<T>(g);
  const uint64_t s2 = both(scale, scale), l2 = both(low, low), less = both(-8388608.f, -8388608.f);
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t c = both(__uint_as_float(w >> bit_of<kKind>(2 * i) & 15u | magic), __uint_as_float(w >> bit_of<kKind>(2 * i + 1) & 15u | magic));
    float a, b;
    parts(fma2(add2(c, less), s2, l2), a, b);
    if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(y[i]) : "f"(b), "f"(a));
    else asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(y[i]) : "f"(b), "f"(a));
  }
  return make_uint4(y[0], y[1], y[2], y[3]);
}

// The least of two pairs of numbers of T, and the largest; NaN where one is.
template <typename T> RB_DEVICE uint32_t min_pair(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (std::is_same<T, __half>::value) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <typename T> RB_DEVICE uint32_t max_pair(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// The extremes over a group that kLanes neighbouring lanes hold, eight numbers of T each: the lowest and the negated highest go through one minimum as a pair.
template <typename T, int kLanes> RB_DEVICE void extremes(const uint4& u, float& lo, float& hi) {
  const uint32_t m = min_pair<T>(min_pair<T>(u.x, u.y), min_pair<T>(u.z, u.w)), x = max_pair<T>(max_pair<T>(u.x, u.y), max_pair<T>(u.z, u.w)) ^ 0x80008000u;
  uint32_t z = min_pair<T>(__byte_perm(m, x, 0x5410), __byte_perm(m, x, 0x7632));
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) z = min_pair<T>(z, __shfl_xor_sync(0xffffffffu, z, o));
  numbers<T>(z, lo, hi);
  hi = -hi;
}

// The extremes over a group that kLanes neighbouring lanes hold, eight channels each.
template <int kLanes> RB_DEVICE void extremes(const float (&x)[8], float& lo, float& hi) {
  lo = hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
}

}  // namespace q4
