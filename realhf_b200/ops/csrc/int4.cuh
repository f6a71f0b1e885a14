// Numbers in groups of 4-bit codes: x ~ scale * c + low with low = min x, scale = T((max x - low) / 15), c = 0 .. 15 (T: the 16-bit type of the model).
//
// A group's numbers are one word: scale in its upper half, low in its lower half.  Codes go to matrix instructions as they are, so each kind of operand has the order of
// nibbles that costs the fewest instructions to take apart:
//   key words     eight channels c, at bits 8 (c & 3) + 4 (c >> 2): two masks and a shift leave two operands of four bytes.
//   value halves  four channels c of one row at bits 4 c of a half-word, a row's neighbour in the other half: masks and one shift leave pairs of neighbouring rows, and in the low
//                 ten bits of an fp16 number a code is a subnormal, c 2^-24 (from bits 0 .. 3) or 16 c 2^-24 (from bits 4 .. 7).
//   weight words  eight channels c, at bits 4 (c >> 1) + 16 (c & 1): pairs of neighbouring channels, as fp16 subnormals too.
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
// The codes of eight numbers of a group: (x - low) / scale rounded to the nearest whole number, halves to the even one.  The quotient is correctly rounded: a product with the
// correctly rounded reciprocal, corrected once by its remainder (Markstein's theorem), so that ties are ties.
RB_DEVICE void codes8(const float (&x)[8], float scale, float low, uint32_t (&c)[8]) {
  const float s = scale * 0.0625f, l = low * 0.0625f, r = __frcp_rn(s);
  const bool any = scale > 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fmaf(x[i], 0.0625f, -l), q = __fmul_rn(a, r), e = fmaf(fmaf(-q, s, a), r, q);
    c[i] = any ? __float_as_uint(__fadd_rn(fminf(e, 15.f), 12582912.f)) & 15u : 0u;   // (1.5 2^23: the sum's last bits are the whole number)
  }
}
constexpr int kKey = 0, kValue = 1, kWeight = 2;
template <int kKind> RB_DEVICE int bit_of(int c) { return kKind == kKey ? 8 * (c & 3) + 4 * (c >> 2) : kKind == kValue ? 4 * c : 4 * (c >> 1) + 16 * (c & 1); }
template <int kKind> RB_DEVICE uint32_t pack8(const float (&x)[8], float scale, float low) {
  uint32_t c[8], w = 0;
  codes8(x, scale, low, c);
#pragma unroll
  for (int i = 0; i < 8; ++i) w |= c[i] << bit_of<kKind>(i);
  return w;
}
// fp32 values of a word's channels: scale * c is exact, one rounding
template <int kKind> RB_DEVICE void unpack8(uint32_t w, float scale, float low, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf(scale, (float)(w >> bit_of<kKind>(i) & 15u), low);
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
