// Numbers in groups of 4-bit codes: x ~ scale * c + low with low = min x, scale = T((max x - low) / 15), c = 0 .. 15 (T: the 16-bit type of the model).
//
// Eight neighbouring channels are one 32-bit word, channel 2i in bits 4i .. 4i + 3, channel 2i + 1 in bits 16 + 4i ..: a mask over both halves of a word leaves
// a pair of neighbouring channels, and in the low 10 bits of an fp16 number a code is a subnormal, c 2^-24 (from bits 0 .. 3) or 16 c 2^-24 (from bits 4 .. 7).
// A matrix instruction multiplies those exactly: no conversion, one shift for four pairs, and the powers of two go where they cost nothing.
// A group's numbers are one word: scale in its upper half, low in its lower half.
//
// A row of n words (n / 4 = channels / 32 = J) is stored as [t = 0 .. 3][j < J], word (t, j) holding the channels 32 j + 8 t ..: the four lanes of a row in a matrix
// instruction's operand take 16 neighbouring bytes each, and what they take together for step j lies in one group of 32.
//
// A cache is tiles of 16 rows of one head: key words [row][t][j], value words [word 0 .. D / 8 - 1][place of the row], the keys' group words [row][D / 32], the
// values' [row][D / 64].  The place of row r, 4 ((r & 7) >> 1) + (r & 1) + 2 (r >> 3), brings the four rows whose weights a lane holds together.
#pragma once
#include "common.cuh"

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

RB_DEVICE int place_of(int r) { return 4 * ((r & 7) >> 1) + (r & 1) + 2 * (r >> 3); }
// the place of word w (channels 8 w ..) in a row
template <int J> RB_DEVICE int word_place(int w) { return (w & 3) * J + (w >> 2); }

RB_DEVICE float min_nan(float a, float b) { float d; asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b)); return d; }
RB_DEVICE float max_nan(float a, float b) { float d; asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b)); return d; }

template <typename T> RB_DEVICE uint32_t bits16(float x) {
  const T v = rb::from_f<T>(x);
  return *reinterpret_cast<const uint16_t*>(&v);
}
template <typename T> RB_DEVICE float from_bits16(uint32_t b) {
  const uint16_t h = (uint16_t)b;
  return rb::to_f(*reinterpret_cast<const T*>(&h));
}
template <typename T> RB_DEVICE float scale_of(uint32_t w) { return from_bits16<T>(w >> 16); }
template <typename T> RB_DEVICE float low_of(uint32_t w) { return from_bits16<T>(w & 0xffffu); }

// The group word of a group whose extremes are lo and hi; a group that holds an infinity or a NaN is NaN throughout.  Everything is taken by 1/16, an exact factor,
// so that the widest group of bf16 does not leave fp32.
template <typename T> RB_DEVICE uint32_t group_word(float lo, float hi) {
  constexpr float kMost = 3.4028234663852886e38f;
  if (!(fabsf(lo) <= kMost && fabsf(hi) <= kMost)) return bits16<T>(__int_as_float(0x7fc00000)) * 0x10001u;
  return bits16<T>(__fdiv_rn(__fsub_rn(hi * 0.0625f, lo * 0.0625f), 0.9375f)) << 16 | bits16<T>(lo);
}
// The code of x in a group with this scale and low: the quotient rounded to the nearest whole number, halves to the even one.
RB_DEVICE uint32_t code_of(float x, float scale, float low) {
  if (!(scale > 0.f)) return 0;
  return (uint32_t)__float2int_rn(fminf(__fdiv_rn(__fsub_rn(x * 0.0625f, low * 0.0625f), scale * 0.0625f), 15.f));
}
RB_DEVICE uint32_t pack8(const float (&x)[8], float scale, float low) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) w |= code_of(x[i], scale, low) << (4 * (i >> 1) + 16 * (i & 1));
  return w;
}
// fp32 values of a word's channels: scale * c is exact, one rounding
RB_DEVICE void unpack8(uint32_t w, float scale, float low, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf(scale, (float)(w >> (4 * (i >> 1) + 16 * (i & 1)) & 15u), low);
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
