// Host stand-ins for the e4m3 conversions and byte selection of csrc/hw.hpp (test infrastructure, as hw_sim.hpp).
#pragma once
#include "hw_sim.hpp"

namespace hw {

inline uint32_t byte_perm(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r = 0;
  for (int i = 0; i < 4; ++i) {
    const uint32_t s = (sel >> (8 * i)) & 0xff;
    if (s > 7) hwsim::die("byte_perm: selector out of range");
    r |= (((s < 4 ? b : a) >> (8 * (s & 3))) & 0xff) << (8 * i);
  }
  return r;
}
// sign, four bits of exponent (bias 7), three of mantissa; all ones is NaN, there is no infinity
inline float e4m3_value(uint8_t c) {
  const int e = (c >> 3) & 15, m = c & 7;
  float v = e == 15 && m == 7 ? NAN : e ? ldexpf(1.f + m / 8.f, e - 7) : ldexpf((float)m, -9);
  return c & 0x80 ? -v : v;
}
inline uint8_t e4m3_code(float x) {
  const uint8_t sign = signbit(x) ? 0x80 : 0;
  const float a = fabsf(x);
  if (!(a <= 448.f)) {
    if (a > 448.f) hwsim::die("to_e4m3: magnitude above 448");
    return sign | 0x7f;
  }
  if (a == 0.f) return sign;
  int e = 0;
  frexpf(a, &e);
  e = e - 1 < -6 ? -6 : e - 1;
  const float steps = nearbyintf(ldexpf(a, 3 - e));   // round to nearest even
  int code = (int)steps + ((e + 6) << 3);             // steps 8..16 carry into the exponent by themselves
  return sign | (uint8_t)code;
}
inline f32x4 from_e4m3(uint32_t codes) {
  f32x4 r;
  for (int i = 0; i < 4; ++i) r[i] = e4m3_value((uint8_t)(codes >> (8 * i)));
  return r;
}
template <bool HIGH, class T> inline uint32_t from_e4m3(T t, uint32_t codes) {
  const f32x4 v = from_e4m3(codes);
  return pack2(t, v[HIGH ? 2 : 0], v[HIGH ? 3 : 1]);
}
inline uint32_t to_e4m3(f32x4 x) {
  uint32_t r = 0;
  for (int i = 0; i < 4; ++i) r |= (uint32_t)e4m3_code(x[i]) << (8 * i);
  return r;
}
template <class V> inline V load_once(const void* p) { return *(const V*)p; }
template <class V> inline void store_once(void* p, V v) { *(V*)p = v; }
inline float rsqrt_fast(float x) { return 1.f / sqrtf(x); }

}  // namespace hw
