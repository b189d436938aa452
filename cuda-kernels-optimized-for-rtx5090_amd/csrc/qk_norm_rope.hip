// RMS norm of every query and key head, its weight, and the rotary embedding in one pass, optionally with the append of
// keys and values to a paged cache (include/qk_norm_rope.h has the formulas). fp32 between one load and one store of
// each element: run as two operators, the norm's output would be written, read and rounded once more.
//
// Vector kernel. A lane holds P rotation pairs of a head, their halves in two vectors of P elements: 8 pairs where
// head_dim and rotary_dim are multiples of 16 and all is aligned to 16 bytes, else 4 (multiples of 8, 8 bytes). A head
// is LPH lanes (head_dim / 2 P rounded up to 4, 8 or 16; lanes past the head idle), a step is 64 / LPH heads and a
// wave does up to STEPS steps of ONE token. So the sum of squares stays within a 16-lane row (DPP, no barrier), and
// since a lane has the same pairs in every head of its token, it keeps their sines and cosines, times the weights, in
// registers. A token's sines and cosines are formed once by the wave, one or two pairs to a lane, and handed round
// through LDS while its loads are in flight. All loads and stores of heads are non-temporal: nothing is read twice.
//
// Bound by memory where there is enough to do: 4 x 4096 tokens of 32 + 8 heads of 128 in bf16 (335 MB in and out) take
// 59 us, 5.7 TB/s; 2 x 1024 tokens of a 256-wide grouped head with the append 11 us. Small calls are a launch and one
// trip to memory: 64 tokens with the append 3.8 us in a graph, 6 us from Python.
#include <climits>

#include "host.hpp"
#include "rowwise.hpp"

#pragma clang fp contract(off)

using namespace rw;

namespace {

struct Tensor {
  const void* p;
  long long sb, ss, sh;  // element strides: batch, seq, head
};

struct Args {
  Tensor in[3];   // q, k, v
  Tensor out[3];  // q_out, k_out, v_cache; a cache's token stride is its row
  const void* w[2];
  const float* inv_freq;
  const long long* ids;
  const long long* slots;  // slot_mapping, or null: outputs at the token
  long long n_slots;
  long long tokens, seq;
  int heads[3];  // q_heads, kv_heads, kv_heads (the cache's values) or 0
  int head_dim, rotary;
  float inverse_dim, eps;
};

// cos and sin of pos * f: the product in fp64 (exact up to positions of 2^29), less the nearest multiple of pi/2 (in
// two parts, so that the difference is good to 2^-53 of the angle or 2^-25, whichever is more), then the Taylor
// polynomials of an argument within pi/4: their first dropped terms are 2e-9 and 1e-10.
__device__ __forceinline__ float2 angle_trig(double pos, float f) {
  constexpr double kHigh = 1.57079632679489661923, kLow = 6.123233995736766036e-17;  // pi/2
  const double a = pos * (double)f;
  const double n = __builtin_rint(a * 0.63661977236758134308);
  const float x = (float)__builtin_fma(-n, kLow, __builtin_fma(-n, kHigh, a));
  const float z = x * x;
  float s = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = __builtin_fmaf(z, s, 8.3333333e-3f);
  s = __builtin_fmaf(z, s, -1.6666667e-1f);
  s = __builtin_fmaf(x * z, s, x);
  float c = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = __builtin_fmaf(z, c, -1.3888889e-3f);
  c = __builtin_fmaf(z, c, 4.1666667e-2f);
  c = __builtin_fmaf(z, c, -0.5f);
  c = __builtin_fmaf(z, c, 1.0f);
  const int quarter = (int)(n - 4.0 * __builtin_floor(0.25 * n));
  const float cs = (quarter & 1) ? s : c, sn = (quarter & 1) ? c : s;
  return make_float2((quarter == 1 || quarter == 2) ? -cs : cs, (quarter & 2) ? -sn : sn);
}

template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
  v += dpp<kDppXor1>(v);
  v += dpp<kDppXor2>(v);
  if constexpr (LPH > 4) v += dpp<kDppHalfMirror>(v);
  if constexpr (LPH > 8) v += dpp<kDppMirror>(v);
  return v;
}

// 1 / sqrt(mean + eps) of a head's sum of squares. v_rsq_f32 is good to an ulp but takes subnormal numbers for 0.
__device__ __forceinline__ float inverse_rms(float sum, const Args& a) {
  const float m = __builtin_fmaf(sum, a.inverse_dim, a.eps);
  const bool tiny = m < 0x1p-100f;
  return __builtin_amdgcn_rsqf(tiny ? m * 0x1p64f : m) * (tiny ? 0x1p32f : 1.0f);
}

// Which tensor head h of a token is in (0 q, 1 k, 2 v) and its number there.
__device__ __forceinline__ int head_kind(const Args& a, int h, int& at) {
  const int kind = h < a.heads[0] ? 0 : h < a.heads[0] + a.heads[1] ? 1 : 2;
  at = h - (kind > 0 ? a.heads[0] : 0) - (kind > 1 ? a.heads[1] : 0);
  return kind;
}

__device__ __forceinline__ Tensor pick(const Tensor* t, int kind) { return kind == 0 ? t[0] : kind == 1 ? t[1] : t[2]; }

// The element offset of a head in its output; false where a token's slot takes nothing.
__device__ __forceinline__ bool head_out(const Args& a, const Tensor& t, int kind, int at, long long b, long long s,
                                         long long slot, long long& o) {
  if (kind > 0 && a.slots) {
    o = slot * t.ss + at * t.sh;
    return slot >= 0 && slot < a.n_slots;
  }
  o = b * t.sb + s * t.ss + at * t.sh;
  return true;
}

// What a lane holds of a head: the elements of P pairs, each half of them adjacent.
template <typename T, int P>
struct Pairs {
  typedef uint32_t Half __attribute__((ext_vector_type(P / 2)));
  Half a, b;
  template <bool NT>
  __device__ __forceinline__ void load(const void* p, long long at_a, long long at_b) {
    const auto* x = reinterpret_cast<const Half*>(static_cast<const char*>(p) + 2 * at_a);
    const auto* y = reinterpret_cast<const Half*>(static_cast<const char*>(p) + 2 * at_b);
    a = NT ? __builtin_nontemporal_load(x) : *x;
    b = NT ? __builtin_nontemporal_load(y) : *y;
  }
  __device__ __forceinline__ void store(void* p, long long at_a, long long at_b) const {
    __builtin_nontemporal_store(a, reinterpret_cast<Half*>(static_cast<char*>(p) + 2 * at_a));
    __builtin_nontemporal_store(b, reinterpret_cast<Half*>(static_cast<char*>(p) + 2 * at_b));
  }
  __device__ __forceinline__ void get(float* f, float* g) const {
    if constexpr (P == 8) {
      unpack<T>(a, f);
      unpack<T>(b, g);
    } else {
      float both[8];
      unpack<T>((u32x4){a.x, a.y, b.x, b.y}, both);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = both[e], g[e] = both[e + 4];
    }
  }
  __device__ __forceinline__ void set(const float* f, const float* g) {
    if constexpr (P == 8) {
      a = pack<T>(f);
      b = pack<T>(g);
    } else {
      const float both[8] = {f[0], f[1], f[2], f[3], g[0], g[1], g[2], g[3]};
      const u32x4 r = pack<T>(both);
      a = (Half){r.x, r.y};
      b = (Half){r.z, r.w};
    }
  }
};

// A lane's weights folded into the cosines and sines of its pairs.
template <typename T, int P>
struct Turns {
  float aa[P], ab[P], ba[P], bb[P];  // out a = aa f - ab g, out b = bb g + ba f
  __device__ __forceinline__ void set(const void* w, int ea, int eb, const float2* cs, bool turns) {
    float p[P], r[P];
#pragma unroll
    for (int e = 0; e < P; ++e) p[e] = r[e] = 1.0f;
    if (w) {
      Pairs<T, P> x;
      x.template load<false>(w, ea, eb);
      x.get(p, r);
    }
#pragma unroll
    for (int e = 0; e < P; ++e) {
      const float c = turns ? cs[e].x : 1.0f, s = turns ? cs[e].y : 0.0f;
      aa[e] = p[e] * c;
      ab[e] = r[e] * s;
      ba[e] = p[e] * s;
      bb[e] = r[e] * c;
    }
  }
};

// MIXED: a step's heads may be of several kinds, so that few heads make fewer steps.
template <typename T, int P, int LPH, int STEPS, bool MIXED>
__global__ void __launch_bounds__(256) norm_rope_vec(Args a, int groups, int q_steps, int kv_steps) {
  constexpr int HPW = kWave / LPH;
  __shared__ float2 trig[4][128];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  const long long unit = rw_host::workgroup() * 4 + wave;
  const long long token = unit / groups;
  if (token >= a.tokens) return;
  const int first = (int)(unit - token * groups) * STEPS, steps = q_steps + kv_steps * (a.slots ? 2 : 1);
  const long long b = token / a.seq, s = token - b * a.seq;
  const int c = lane % LPH, pairs = a.rotary / (2 * P);  // lanes with rotation pairs
  const bool mine = c < a.head_dim / (2 * P);
  const bool turns = c < pairs;
  // the lane's elements of a head: P pairs, or 2 P elements behind the rotated part
  const int ea = turns ? P * c : a.rotary + 2 * P * (c - pairs), eb = turns ? ea + (a.rotary >> 1) : ea + P;

  // the kind of this lane's head in step t, and the head (-1: none)
  auto head_of = [&](int t, int& h) {
    int kind;
    if constexpr (MIXED) {
      const int g = t * HPW + lane / LPH;
      kind = head_kind(a, g, h);
      if (!mine || g >= a.heads[0] + a.heads[1] + a.heads[2]) h = -1;
    } else {
      kind = t < q_steps ? 0 : t < q_steps + kv_steps ? 1 : 2;
      h = (t - (kind > 0 ? q_steps : 0) - (kind > 1 ? kv_steps : 0)) * HPW + lane / LPH;
      if (!mine || t >= steps || h >= a.heads[kind]) h = -1;
    }
    return kind;
  };
  Pairs<T, P> x[STEPS];
#pragma unroll
  for (int u = 0; u < STEPS; ++u) {
    int h;
    const int kind = head_of(first + u, h);
    x[u].a = x[u].b = (typename Pairs<T, P>::Half)(0u);
    if (h >= 0) {
      const Tensor t = pick(a.in, kind);
      const long long o = b * t.sb + s * t.ss + h * t.sh;
      x[u].template load<true>(t.p, o + ea, o + eb);
    }
  }
  const long long slot = a.slots ? a.slots[token] : 0;
  const double pos = (double)a.ids[token];
  for (int i = lane; i < P * pairs; i += kWave) trig[wave][i] = angle_trig(pos, a.inv_freq[i]);
  wave_lds_sync();
  const float2* cs = trig[wave] + P * (turns ? c : 0);
  Turns<T, P> turn;
  int set = -1;  // the kind that it is for
#pragma unroll
  for (int u = 0; u < STEPS; ++u) {
    int h;
    const int kind = head_of(first + u, h);
    const Tensor t = pick(a.out, kind);
    if (MIXED || kind < 2) {
      if (kind != set && mine && kind < 2) turn.set(kind ? a.w[1] : a.w[0], ea, eb, cs, turns), set = kind;
      float f[P], g[P];
      x[u].get(f, g);
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < P; ++e) sum = __builtin_fmaf(f[e], f[e], sum);
#pragma unroll
      for (int e = 0; e < P; ++e) sum = __builtin_fmaf(g[e], g[e], sum);
      const float inv = inverse_rms(head_sum<LPH>(sum), a);  // every lane: the sum crosses lanes
      if (!MIXED || kind < 2) {
        float p[P], r[P];
#pragma unroll
        for (int e = 0; e < P; ++e) {
          p[e] = __builtin_fmaf(f[e], turn.aa[e], -(g[e] * turn.ab[e])) * inv;
          r[e] = __builtin_fmaf(g[e], turn.bb[e], f[e] * turn.ba[e]) * inv;
        }
        x[u].set(p, r);
      }
    }  // values are copied as they are
    long long o;
    if (h < 0 || !head_out(a, t, kind, h, b, s, slot, o)) continue;
    x[u].store(const_cast<void*>(t.p), o + ea, o + eb);
  }
}

// Few heads: a step is all heads of `per` tokens (at least two, at most 256 pairs in all).
template <typename T, int P, int LPH>
__global__ void __launch_bounds__(256) norm_rope_few(Args a, int per) {
  __shared__ float2 trig[4][256];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  const long long begin = (rw_host::workgroup() * 4 + wave) * per;  // the wave's first token
  if (begin >= a.tokens) return;
  const int left = a.tokens - begin < per ? (int)(a.tokens - begin) : per;
  const int heads = a.heads[0] + a.heads[1] + a.heads[2];
  const int c = lane % LPH, pairs = a.rotary / (2 * P);
  const bool turns = c < pairs;
  const int ea = turns ? P * c : a.rotary + 2 * P * (c - pairs), eb = turns ? ea + (a.rotary >> 1) : ea + P;
  const int mine = lane / LPH / heads;  // this lane's token
  int at;
  const int kind = head_kind(a, lane / LPH - mine * heads, at);
  const bool there = mine < left && c < a.head_dim / (2 * P);
  const unsigned token = (unsigned)begin + (unsigned)(mine < left ? mine : 0);  // tokens < 2^31
  const unsigned b = token / (unsigned)a.seq, s = token - b * (unsigned)a.seq;
  Pairs<T, P> x;
  x.a = x.b = (typename Pairs<T, P>::Half)(0u);
  if (there) {
    const Tensor t = pick(a.in, kind);
    const long long o = b * t.sb + s * t.ss + at * t.sh;
    x.template load<true>(t.p, o + ea, o + eb);
  }
  const long long slot = a.slots ? a.slots[token] : 0;
  const int angles = P * pairs;
  for (int i = lane; i < angles * left; i += kWave) {
    const int t = i / angles;
    trig[wave][i] = angle_trig((double)a.ids[begin + t], a.inv_freq[i - t * angles]);
  }
  wave_lds_sync();
  float f[P], g[P], sum = 0.0f;
  x.get(f, g);
#pragma unroll
  for (int e = 0; e < P; ++e) sum = __builtin_fmaf(f[e], f[e], sum);
#pragma unroll
  for (int e = 0; e < P; ++e) sum = __builtin_fmaf(g[e], g[e], sum);
  const float inv = inverse_rms(head_sum<LPH>(sum), a);  // every lane: the sum crosses lanes
  if (!there) return;
  if (kind < 2) {
    Turns<T, P> turn;
    turn.set(kind ? a.w[1] : a.w[0], ea, eb, trig[wave] + mine * angles + P * (turns ? c : 0), turns);
    float p[P], r[P];
#pragma unroll
    for (int e = 0; e < P; ++e) {
      p[e] = __builtin_fmaf(f[e], turn.aa[e], -(g[e] * turn.ab[e])) * inv;
      r[e] = __builtin_fmaf(g[e], turn.bb[e], f[e] * turn.ba[e]) * inv;
    }
    x.set(p, r);
  }
  const Tensor t = pick(a.out, kind);
  long long o;
  if (head_out(a, t, kind, at, b, s, slot, o)) x.store(const_cast<void*>(t.p), o + ea, o + eb);
}

// Any head_dim, rotary_dim, alignment and stride: a wave per head, an element or a pair per lane and turn. Both passes
// read the head (the second from the caches), so nothing of it is kept and its length is free.
template <typename T>
__global__ void __launch_bounds__(256) norm_rope_any(Args a) {
  const int lane = lane_id(), total = a.heads[0] + a.heads[1] + a.heads[2];
  const long long unit = rw_host::workgroup() * 4 + __builtin_amdgcn_readfirstlane(wave_id());
  const long long token = unit / total;
  if (token >= a.tokens) return;
  const long long b = token / a.seq, s = token - b * a.seq;
  int at;
  const int kind = head_kind(a, (int)(unit - token * total), at);
  const Tensor t = pick(a.in, kind), to = pick(a.out, kind);
  const long long i0 = b * t.sb + s * t.ss + at * t.sh;
  long long o0;
  if (!head_out(a, to, kind, at, b, s, a.slots ? a.slots[token] : 0, o0)) return;
  void* out = const_cast<void*>(to.p);
  if (kind == 2) {
    for (int e = lane; e < a.head_dim; e += kWave) store_elem<T>(out, o0 + e, load_elem<T>(t.p, i0 + e));
    return;
  }
  float sum = 0.0f;
  for (int e = lane; e < a.head_dim; e += kWave) {
    const float v = load_elem<T>(t.p, i0 + e);
    sum = __builtin_fmaf(v, v, sum);
  }
  const float inv = inverse_rms(wave_sum(sum), a);
  const void* w = kind ? a.w[1] : a.w[0];
  auto normed = [&](int e) {
    const float v = load_elem<T>(t.p, i0 + e) * inv;
    return w ? v * load_elem<T>(w, e) : v;
  };
  const int half = a.rotary >> 1;
  const double pos = (double)a.ids[token];
  for (int e = lane; e < a.head_dim - half; e += kWave) {  // a pair, or an element behind the rotated part
    if (e < half) {
      const float f = normed(e), g = normed(e + half);
      const float2 v = angle_trig(pos, a.inv_freq[e]);
      store_elem<T>(out, o0 + e, __builtin_fmaf(f, v.x, -(g * v.y)));
      store_elem<T>(out, o0 + e + half, __builtin_fmaf(g, v.x, f * v.y));
    } else {
      store_elem<T>(out, o0 + e + half, normed(e + half));
    }
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------

enum { kTuneSteps = 0, kTuneScalar = 1, kTuneFew = 2 };
constexpr long long kMostHeads = 1LL << 38;  // of all tokens, a wave each: a quarter as many workgroups fit a grid
static_assert(kMostHeads / 4 <= rw_host::kMostGroups, "");

template <typename K, typename... A>
int launch_waves(K kern, long long waves, hipStream_t stream, A... args) {
  hipLaunchKernelGGL(kern, rw_host::grid_of((waves + 3) / 4), dim3(256), 0, stream, args...);
  return (int)hipGetLastError();
}

template <typename T, int P, int LPH, bool MIXED>
int launch_steps(const Args& a, int per_token, int q_steps, int kv_steps, hipStream_t stream) {
  int steps = rw_host::tune_get(kTuneSteps);
  if (steps <= 0) {
    // A wave's sines serve all its steps, but steps of one wave wait for each other's loads: up to four steps, as long
    // as four waves are left to each SIMD. Measured at 1, 2 and 4 steps: 81920 steps 68, 63 and 60.6 us, 14336 steps
    // 14.3, 11.4 and 11.0, 6309 steps 5.2, 6.4 and 6.7, 448 steps 3.8, 4.5 and 5.8. Five and more steps take over 128
    // registers and more time (83 us of the first).
    const long long want = a.tokens * per_token / (16LL * rw_host::device_cus());
    steps = want < 2 ? 1 : want < 4 ? 2 : 4;
  }
  auto go = [&](auto kern, int n) {
    const int groups = (per_token + n - 1) / n;
    return launch_waves(kern, a.tokens * groups, stream, a, groups, q_steps, kv_steps);
  };
  if (steps <= 1 || per_token == 1) return go(norm_rope_vec<T, P, LPH, 1, MIXED>, 1);
  if (steps <= 2 || per_token == 2) return go(norm_rope_vec<T, P, LPH, 2, MIXED>, 2);
  return go(norm_rope_vec<T, P, LPH, 4, MIXED>, 4);
}

template <typename T, int P, int LPH>
int launch_lph(const Args& a, hipStream_t stream) {
  constexpr int HPW = kWave / LPH;
  const int q_steps = (a.heads[0] + HPW - 1) / HPW, kv_steps = (a.heads[1] + HPW - 1) / HPW;
  const int apart = q_steps + kv_steps * (a.slots ? 2 : 1);
  const int heads = a.heads[0] + a.heads[1] + a.heads[2], mixed = (heads + HPW - 1) / HPW;
  // several tokens to a wave where they leave waves enough: 60000 tokens of 1 + 1 heads of 64 take 32.7 us one by one
  // and 13.1 so, of 2 + 1 heads of 128 39.3 and 28.6; 4096 of them 5.0 and 4.9, 5.2 and 5.0; 1024 of them 4.4 and 4.7,
  // 4.3 and 4.4
  const int per = HPW / heads;
  const int few = rw_host::tune_get(kTuneFew);
  if (per > 1 && (few ? few == 1 : a.tokens >= 16LL * rw_host::device_cus()))
    return launch_waves(norm_rope_few<T, P, LPH>, (a.tokens + per - 1) / per, stream, a, per);
  if (mixed < apart) return launch_steps<T, P, LPH, true>(a, mixed, q_steps, kv_steps, stream);
  return launch_steps<T, P, LPH, false>(a, apart, q_steps, kv_steps, stream);
}

// Whether lanes of `pairs` pairs cover heads in whole vectors.
bool in_vectors(const Args& a, int pairs) {
  const auto fits = [&](const Tensor& t) {
    return (uintptr_t)t.p % (2 * pairs) == 0 && t.sb % pairs == 0 && t.ss % pairs == 0 && t.sh % pairs == 0;
  };
  bool all = a.head_dim % (2 * pairs) == 0 && a.rotary % (2 * pairs) == 0;
  for (int i = 0; i < (a.slots ? 3 : 2); ++i) all = all && fits(a.in[i]) && fits(a.out[i]);
  for (int i = 0; i < 2; ++i) all = all && (uintptr_t)a.w[i] % (2 * pairs) == 0;
  return all;
}

template <typename T>
int launch_type(const Args& a, hipStream_t stream) {
  if (rw_host::tune_get(kTuneScalar) != 1) {
    if (a.head_dim >= 48 && a.head_dim <= 256 && in_vectors(a, 8)) {
      if (a.head_dim <= 64) return launch_lph<T, 8, 4>(a, stream);
      if (a.head_dim <= 128) return launch_lph<T, 8, 8>(a, stream);
      return launch_lph<T, 8, 16>(a, stream);
    }
    if (a.head_dim <= 128 && in_vectors(a, 4)) {
      if (a.head_dim <= 64) return launch_lph<T, 4, 8>(a, stream);
      return launch_lph<T, 4, 16>(a, stream);
    }
  }
  return launch_waves(norm_rope_any<T>, a.tokens * (a.heads[0] + a.heads[1] + a.heads[2]), stream, a);
}

int run(Args& a, long long batch, int dtype, hipStream_t stream) {
  if (a.seq > INT_MAX || batch > INT_MAX / a.seq || a.heads[0] <= 0 || a.heads[1] <= 0 || a.heads[0] > (1 << 20) ||
      a.heads[1] > (1 << 20) || a.head_dim < 1 || a.head_dim > 65536 || a.rotary < 0 || a.rotary % 2 ||
      a.rotary > a.head_dim || (a.rotary && !a.inv_freq) || !a.ids || (dtype != 1 && dtype != 2))
    return rw_host::kInvalid;
  for (int i = 0; i < (a.slots ? 3 : 2); ++i)
    if (!a.in[i].p || (!a.out[i].p && (i == 0 || !a.slots || a.n_slots))) return rw_host::kInvalid;
  a.tokens = batch * a.seq;
  if (a.tokens * (a.heads[0] + a.heads[1] + a.heads[2]) > kMostHeads) return rw_host::kInvalid;
  a.inverse_dim = 1.0f / (float)a.head_dim;
  return dtype == 1 ? launch_type<BF16>(a, stream) : launch_type<F16>(a, stream);
}

// (a dimension of one element has a stride that is not used and may be anything: 0 here, so that it decides nothing)
Tensor tensor(const void* p, const long long* strides, int i, long long batch, long long seq, int heads, int head_dim) {
  if (strides)
    return Tensor{p, batch == 1 ? 0 : strides[3 * i], seq == 1 ? 0 : strides[3 * i + 1],
                  heads == 1 ? 0 : strides[3 * i + 2]};
  return Tensor{p, seq * heads * head_dim, (long long)heads * head_dim, head_dim};
}

}  // namespace

extern "C" int qk_norm_rope_launch(const void* q, const void* k, const void* ids, const float* inv_freq,
                                   const void* q_weight, const void* k_weight, void* q_out, void* k_out,
                                   const long long* strides, long long batch, long long seq, int q_heads, int kv_heads,
                                   int head_dim, int rotary_dim, int dtype, float eps, hipStream_t stream) {
  if (batch <= 0 || seq <= 0) return rw_host::kOk;
  Args a{};
  a.in[0] = tensor(q, strides, 0, batch, seq, q_heads, head_dim);
  a.in[1] = tensor(k, strides, 1, batch, seq, kv_heads, head_dim);
  a.out[0] = tensor(q_out, strides, 2, batch, seq, q_heads, head_dim);
  a.out[1] = tensor(k_out, strides, 3, batch, seq, kv_heads, head_dim);
  a.w[0] = q_weight;
  a.w[1] = k_weight;
  a.inv_freq = inv_freq;
  a.ids = (const long long*)ids;
  a.seq = seq;
  a.heads[0] = q_heads;
  a.heads[1] = kv_heads;
  a.head_dim = head_dim;
  a.rotary = rotary_dim;
  a.eps = eps;
  return run(a, batch, dtype, stream);
}

extern "C" int qk_norm_rope_kv_launch(const void* q, const void* k, const void* v, const void* ids,
                                      const float* inv_freq, const void* q_weight, const void* k_weight, void* q_out,
                                      void* k_cache, void* v_cache, const void* slot_mapping, const long long* strides,
                                      long long batch, long long seq, long long slots, int q_heads, int kv_heads,
                                      int head_dim, int rotary_dim, int dtype, float eps, hipStream_t stream) {
  if (batch <= 0 || seq <= 0) return rw_host::kOk;
  if (!slot_mapping || slots < 0) return rw_host::kInvalid;
  Args a{};
  a.in[0] = tensor(q, strides, 0, batch, seq, q_heads, head_dim);
  a.in[1] = tensor(k, strides, 1, batch, seq, kv_heads, head_dim);
  a.in[2] = tensor(v, strides, 2, batch, seq, kv_heads, head_dim);
  a.out[0] = tensor(q_out, strides, 3, batch, seq, q_heads, head_dim);
  a.out[1] = tensor(k_cache, nullptr, 0, batch, seq, kv_heads, head_dim);
  a.out[2] = tensor(v_cache, nullptr, 0, batch, seq, kv_heads, head_dim);
  a.w[0] = q_weight;
  a.w[1] = k_weight;
  a.inv_freq = inv_freq;
  a.ids = (const long long*)ids;
  a.slots = (const long long*)slot_mapping;
  a.n_slots = slots;
  a.seq = seq;
  a.heads[0] = q_heads;
  a.heads[1] = a.heads[2] = kv_heads;
  a.head_dim = head_dim;
  a.rotary = rotary_dim;
  a.eps = eps;
  return run(a, batch, dtype, stream);
}

extern "C" int qk_norm_rope_tune(int slot, int value) { return rw_host::tune_set(slot, value); }
