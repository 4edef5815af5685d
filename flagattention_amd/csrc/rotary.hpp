// Rows of D values turned in pairs, as the norm and rotation kernels and the cache append hold them: D / 16 lanes per row,
// each with eight values of the first half of the turned part and the eight they are paired with (what is behind the
// turned part is dealt the same way), so that both kinds of pairs are local to a lane.
#pragma once
#include "common.hpp"
#include "params.hpp"

namespace fa {

// The 16 values of a row that one lane holds: eight from `lo` on, eight from `hi` on.
struct RotaryPlace {
  int lo, hi;
  bool turned;   // otherwise they are behind the turned part
};
template <int D>
FA_DEVICE RotaryPlace rotary_place(int lane, int rotary) {
  const int c = 8 * (lane % (D / 16)), half = rotary / 2;
  RotaryPlace r;
  r.turned = c < half;
  r.lo = r.turned ? c : rotary + (c - half);
  r.hi = r.lo + (r.turned ? half : (D - rotary) / 2);
  return r;
}

// Cosines and sines of the lane's eight pairs (halves: of values lo .. lo + 7; interleaved: of four pairs from lo on and
// four from hi on).  A position without a row in the tables turns by NaN.
struct Turn { float c[8], s[8]; };
template <bool INTER>
FA_DEVICE Turn load_turn(const float* cos, const float* sin, int64_t stride, int64_t row, int64_t rows, RotaryPlace at) {
  Turn t;
  const bool there = row >= 0 && row < rows;
  const int64_t base = there ? row * stride : 0;
  // lanes behind the turned part read the row's first values and use none of them
  const int a = !at.turned ? 0 : INTER ? at.lo / 2 : at.lo, b = !at.turned ? 0 : INTER ? at.hi / 2 : at.lo + 4;
  const hw::f32x4 c0 = *(const hw::f32x4*)(cos + base + a), c1 = *(const hw::f32x4*)(cos + base + b);
  const hw::f32x4 s0 = *(const hw::f32x4*)(sin + base + a), s1 = *(const hw::f32x4*)(sin + base + b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t.c[i] = there ? c0[i] : __builtin_nanf("");
    t.s[i] = there ? s0[i] : __builtin_nanf("");
    t.c[4 + i] = there ? c1[i] : __builtin_nanf("");
    t.s[4 + i] = there ? s1[i] : __builtin_nanf("");
  }
  return t;
}

// Turns the lane's values by the angle (SIGN = 1) or back (-1).  x[0..7] are those from lo on, x[8..15] those from hi on.
// Products and sums are rounded one by one, so that a value next to a rounding border of the result (a code of an 8-bit
// cache, a power of two of its scale) falls as it does where fp32 arithmetic is written out.
template <bool INTER, int SIGN>
FA_DEVICE void turn(float* x, const Turn& t, bool turned) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int p = INTER ? 2 * (i & 3) + 8 * (i >> 2) : i, q = INTER ? p + 1 : i + 8;
    const float a = x[p], b = x[q], s = SIGN * t.s[i];
    const float ya = a * t.c[i] - b * s, yb = b * t.c[i] + a * s;
    x[p] = turned ? ya : a;
    x[q] = turned ? yb : b;
  }
}

template <class T>
FA_DEVICE void unpack8(u32x4 raw, float* x) {
  const auto v = hw::as_v8<T>(raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
}
template <class T>
FA_DEVICE u32x4 pack8(const float* x) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = hw::pack2(T{}, x[2 * i], x[2 * i + 1]);
  return r;
}

// A lane's share of a row as it lies in memory.  ONCE: marked non-temporal where each of the two loads takes whole 128-byte
// lines (a line of which another load wants the rest may be gone by then).
struct RawRow { u32x4 lo, hi; };
template <class T, int D, bool ONCE>
FA_DEVICE RawRow load_row(const T* row, RotaryPlace at) {
  if constexpr (D >= 128 && ONCE) return RawRow{hw::load_once<u32x4>(row + at.lo), hw::load_once<u32x4>(row + at.hi)};
  else return RawRow{*(const u32x4*)(row + at.lo), *(const u32x4*)(row + at.hi)};
}
template <class T>
FA_DEVICE void unpack_row(const RawRow& r, float* x) {
  unpack8<T>(r.lo, x);
  unpack8<T>(r.hi, x + 8);
}

}  // namespace fa
