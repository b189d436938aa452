// The CPU emulation's counterpart of csrc/fp4.hpp: the conversions and the products of 4-bit numbers from their
// definition.
#pragma once

#include "matrix.hpp"

namespace rw {

constexpr int kShared = 32;
constexpr uint32_t kNanScale = 255;
template <typename T> constexpr int kMostScale = 252;
template <> constexpr int kMostScale<F16> = 140;

inline int scale_of(uint32_t most, int limit) {
  if (most >= 0x7f800000u) return (int)kNanScale;
  const int e = (int)((most + 0x200000u) >> 23) - 2;
  return e < 1 ? 1 : e > limit ? limit : e;
}
inline float power_of(uint32_t scale) { return __builtin_bit_cast(float, scale << 23); }
inline uint32_t scale_in(uint32_t byte) { return byte > 252u ? kNanScale : byte; }

namespace emu_fp4 {
// 2^(byte - 127) of the exponent field; NaN where it is full
inline double power(float scale) {
  const uint32_t byte = __builtin_bit_cast(uint32_t, scale) >> 23 & 255u;
  return byte == 255u ? (double)NAN : std::ldexp(1.0, (int)byte - 127);
}
inline double value(uint32_t code) {
  static const double v[8] = {0, 0.5, 1, 1.5, 2, 3, 4, 6};
  return code & 8u ? -v[code & 7u] : v[code & 7u];
}
inline uint32_t code(double x) {
  const double y = std::fabs(x);
  const uint32_t c = (y > 0.25) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0);
  return c | (std::signbit(x) ? 8u : 0u);
}
inline double e4m3(uint32_t b) {
  const int e = b >> 3 & 15, m = b & 7;
  const double v = e == 15 && m == 7 ? (double)NAN : e ? std::ldexp(1 + m / 8.0, e - 7) : std::ldexp(m / 8.0, -6);
  return b & 0x80u ? -v : v;
}
inline uint32_t nearest_e4m3(double x) {
  uint32_t best = 0;
  double far = INFINITY;
  for (uint32_t b = 0; b < 0x7f; ++b) {
    const double d = std::fabs(std::fabs(x) - e4m3(b));
    if (d < far || (d == far && !(b & 1u))) best = b, far = d;
  }
  return best | (std::signbit(x) ? 0x80u : 0u);
}
}  // namespace emu_fp4

template <typename T> inline u32x4 widen4(uint32_t codes, float scale) {
  float f[8];
  for (int i = 0; i < 8; ++i) f[i] = (float)(emu_fp4::value(codes >> (4 * i) & 15u) * emu_fp4::power(scale));
  return pack<T>(f);
}
template <typename T> inline uint32_t narrow4(const u32x4& x, float scale) {
  float f[8];
  unpack<T>(x, f);
  uint32_t r = 0;
  for (int i = 0; i < 8; ++i) r |= emu_fp4::code((double)f[i] / emu_fp4::power(scale)) << (4 * i);
  return r;
}

struct Eights {
  u32x4 lo, hi;
};
namespace emu_fp4 {
struct State {
  u32x4 a[16][64];
  Eights b[16][64];
  uint32_t sa[16][64], sb[16][64];
};
inline State& S() {
  static thread_local State s;
  return s;
}
}  // namespace emu_fp4
inline f32x4 product_fp4(const u32x4& a, const Eights& b, const f32x4& c, uint32_t scale_a, uint32_t scale_b) {
  auto& s = emu_fp4::S();
  const int w = emu::wid(), l = emu::lid();
  s.a[w][l] = a, s.b[w][l] = b, s.sa[w][l] = scale_a, s.sb[w][l] = scale_b;
  emu::wave_sync(__LINE__);
  f32x4 r = c;
  for (int i = 0; i < 4; ++i) {
    const int row = 4 * (l / 16) + i, col = l % 16;
    double sum = 0.0;
    for (int k = 0; k < 128; ++k) {
      const int la = row + 16 * (k / 32), n = k % 32, lb = col + 16 * (k / 16 % 4), m = k % 16;
      const u32x4& half = k < 64 ? s.b[w][lb].lo : s.b[w][lb].hi;
      sum += emu_fp4::value(s.a[w][la][n / 8] >> (4 * (n % 8)) & 15u) *
             emu_fp4::power(power_of(s.sa[w][la])) * emu_fp4::e4m3(half[m / 4] >> (8 * (m % 4)) & 255u) *
             emu_fp4::power(power_of(s.sb[w][col + 16 * (k / 32)]));
    }
    r[i] += (float)sum;
  }
  emu::wave_sync(__LINE__);
  return r;
}
inline uint32_t take_e4m3(float* x) {
  uint32_t r = 0;
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = emu_fp4::nearest_e4m3(x[i]);
    r |= b << (8 * i);
    x[i] = (x[i] - (float)emu_fp4::e4m3(b)) * 16.0f;
  }
  return r;
}

}  // namespace rw
