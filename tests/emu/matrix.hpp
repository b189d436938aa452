// The CPU emulation's counterpart of csrc/matrix.hpp, put in its place when a kernel source that uses it is built for
// the host: matrix products and transposing LDS reads as exchanges between the wave's lanes, and loads to LDS that are
// held back until the lane waits for them (a read before the wait sees what was there).
#pragma once

#include "rowwise.hpp"

inline unsigned __umulhi(unsigned a, unsigned b) { return (unsigned)((unsigned long long)a * b >> 32); }

namespace rw {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

namespace emu_matrix {
struct Load {
  const void* from;
  char* to;
  int bytes;
};
struct State {
  u32x4 a[16][64], b[16][64];
  const char* at[16][64];
  std::vector<Load> loads[16][64];
};
inline State& S() {
  static thread_local State s;
  return s;
}
template <typename T> inline float element(const u32x4& v, int e) {
  const uint16_t x = (uint16_t)(v[e / 2] >> (16 * (e % 2)));
  return load_elem<T>(&x, 0);
}
}  // namespace emu_matrix

template <typename T>
inline f32x16 product32(const u32x4& a, const u32x4& b, const f32x16& c) {
  auto& s = emu_matrix::S();
  const int w = emu::wid(), l = emu::lid();
  s.a[w][l] = a;
  s.b[w][l] = b;
  emu::wave_sync(__LINE__);
  f32x16 r = c;
  for (int i = 0; i < 16; ++i) {
    const int row = 8 * (i / 4) + 4 * (l / 32) + i % 4;
    float sum = 0.0f;
    for (int h = 0; h < 2; ++h)
      for (int e = 0; e < 8; ++e)
        sum += emu_matrix::element<T>(s.a[w][row + 32 * h], e) * emu_matrix::element<T>(s.b[w][l % 32 + 32 * h], e);
    r[i] += sum;
  }
  emu::wave_sync(__LINE__);
  return r;
}

inline f32x4 product16(const u32x4& a, const u32x4& b, const f32x4& c) {
  auto& s = emu_matrix::S();
  const int w = emu::wid(), l = emu::lid();
  s.a[w][l] = a;
  s.b[w][l] = b;
  emu::wave_sync(__LINE__);
  f32x4 r = c;
  for (int i = 0; i < 4; ++i) {
    float sum = 0.0f;
    for (int h = 0; h < 4; ++h)
      for (int e = 0; e < 8; ++e)
        sum += emu_matrix::element<BF16>(s.a[w][4 * (l / 16) + i + 16 * h], e) *
               emu_matrix::element<BF16>(s.b[w][l % 16 + 16 * h], e);
    r[i] += sum;
  }
  emu::wave_sync(__LINE__);
  return r;
}

typedef char* lds_ptr;
inline lds_ptr in_lds(char* p) { return p; }
inline lds_ptr own(lds_ptr p) { return p; }
inline u32x4 lds_vector(lds_ptr at) { return *reinterpret_cast<const u32x4*>(at); }
inline void settle(uint32_t&) {}
inline void settle(float&) {}
inline void settle(int&) {}
inline void settle(const char*&) {}
inline u32x2 lds_column(lds_ptr at) {
  auto& s = emu_matrix::S();
  const int w = emu::wid(), l = emu::lid(), i = l % 16;
  s.at[w][l] = at;
  emu::wave_sync(__LINE__);
  uint16_t v[4];
  for (int e = 0; e < 4; ++e) std::memcpy(&v[e], s.at[w][(l & ~15) + 4 * e + i / 4] + 2 * (i % 4), 2);
  emu::wave_sync(__LINE__);
  return (u32x2){v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16};
}

// (an inactive lane's load counts in its wave, and moves nothing)
inline void load_to_lds(const void* from, char* at, bool active) {
  emu_matrix::S().loads[emu::wid()][emu::lid()].push_back({from, at + 16 * emu::lid(), active ? 16 : 0});
}
inline void load_to_lds_at(const char* base, uint32_t offset, char* at, bool active) {
  load_to_lds(base + offset, at, active);
}
inline void stream_to_lds(const void* from, char* at, bool active) { load_to_lds(from, at, active); }
inline void load_word_to_lds(const void* from, char* at) {
  emu_matrix::S().loads[emu::wid()][emu::lid()].push_back({from, at + 4 * emu::lid(), 4});
}
template <int newer = 0>
inline void wait_loads() {
  auto& q = emu_matrix::S().loads[emu::wid()][emu::lid()];
  const size_t n = q.size() > (size_t)newer ? q.size() - newer : 0;
  for (size_t i = 0; i < n; ++i) std::memcpy(q[i].to, q[i].from, q[i].bytes);
  q.erase(q.begin(), q.begin() + n);
  emu::wave_sync(__LINE__);
}
inline void wait_lds() { emu::wave_sync(__LINE__); }
inline void order_lds() {}
inline void keep_order() {}
inline void meet() { emu::block_sync(__LINE__); }

inline int from_lane(int v, int from) { return (int)(uint32_t)emu::read_from((uint32_t)v, from, __LINE__); }
template <int D> inline uint32_t across(uint32_t v) { return (uint32_t)from_lane((int)v, emu::lid() ^ D); }
inline float other_half(float v) {
  return __builtin_bit_cast(float, from_lane(__builtin_bit_cast(int, v), emu::lid() ^ 32));
}
inline float max_of_halves(float v) { return fmaxf(v, other_half(v)); }
inline float sum_of_halves(float v) { return emu::lid() < 32 ? v + other_half(v) : other_half(v) + v; }

inline float next_quarter(float v) {
  return __builtin_bit_cast(float, from_lane(__builtin_bit_cast(int, v), emu::lid() ^ 16));
}
inline float max_of_quarters(float v) { return max_of_halves(fmaxf(v, next_quarter(v))); }
inline float sum_of_quarters(float v) {
  return sum_of_halves(emu::lid() & 16 ? next_quarter(v) + v : v + next_quarter(v));
}

template <typename T>
inline float add_pair(uint32_t pair, float sum) {
  const u32x4 v = {pair, 0, 0, 0};
  return sum + emu_matrix::element<T>(v, 0) + emu_matrix::element<T>(v, 1);
}
template <typename T> inline uint32_t pack2(float a, float b);
template <> inline uint32_t pack2<BF16>(float a, float b) { return pack_bf16x2(a, b); }
template <> inline uint32_t pack2<F16>(float a, float b) { return pack_f16x2(a, b); }

}  // namespace rw

// A buffer between pages that cannot be touched.
extern "C" __attribute__((visibility("default"))) void* emu_guarded(size_t n) { return emu::guarded_alloc(n); }
