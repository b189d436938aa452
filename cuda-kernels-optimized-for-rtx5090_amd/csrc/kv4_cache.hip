// Keys and values written into a paged cache of 4-bit codes, and read back (include/kv4_cache.h has the format).
//
// Both are bound by memory: appending reads 2 bytes an element and writes half a byte and a 32nd of one, reading the
// reverse. A lane takes 8 elements (16 bytes in 16 bits, 4 bytes of codes), so that both sides of the wave's accesses
// are whole pieces of a head's row; a group of 32 is 4 neighbouring lanes, and their largest magnitude two exchanges in
// the quad. A workgroup is 32 tokens of one head: their codes lie side by side in a page, which holds a head's tokens
// one behind the other. A lane has two tokens 16 apart, so that their trips to memory overlap.
//
// 16384 tokens of 8 heads of 128 (67 MB in 16 bits, 18 MB of codes and scales) appended and read in 36 us, 4.7 TB/s; with
// a token to a lane in 40.5 us, with four in 36.4. Appending alone takes 18.7 us to slots one behind the other or to whole
// pages, and 21.3 to scattered slots (counted: 68 MB read, 18 and 21 written).
#include <climits>

#include "divide.hpp"
#include "fp4.hpp"
#include "host.hpp"

#pragma clang fp contract(off)

using namespace rw;

namespace {

constexpr int kTokens = 16, kUnroll = 2;  // tokens that a workgroup takes at once, and times

struct Args {
  const void* in[2];         // keys, values: to write
  void* out[2];              // read
  uint8_t* codes[2];
  uint8_t* scales[2];
  const long long* slots;
  long long token[2], head[2];  // strides of `in`
  long long tokens;
  int kv_heads, block_size;
  unsigned most;             // slots of the cache
  Divisor by_heads, by_block;
};

// A lane's tokens, head and 8 elements.
template <int D> struct Place {
  long long token;           // of the call: the first, each next one kTokens further
  long long row[kUnroll];    // of the cache's rows, -1 where a token has none
  int head, chunk;
  bool values;
  __device__ __forceinline__ Place(const Args& a) {
    constexpr int chunks = D / 8;
    unsigned rest = (unsigned)rw_host::workgroup();  // fewer than 2^31: the host's check
    head = a.by_heads.take(rest);
    values = rest & 1u;
    token = (long long)(rest >> 1) * kTokens * kUnroll + threadIdx.x / chunks;
    chunk = (int)(threadIdx.x % chunks);
    long long slot[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const long long t = token + u * kTokens;
      slot[u] = a.slots[t < a.tokens ? t : a.tokens - 1];
      if (t >= a.tokens) slot[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      unsigned page = (unsigned)slot[u];
      const int at = a.by_block.take(page);
      const bool none = slot[u] < 0 || slot[u] >= (long long)a.most;
      row[u] = none ? -1 : ((long long)page * a.kv_heads + head) * a.block_size + at;
    }
  }
};

// The magnitudes of two packed elements as fp32 bits: the larger.
template <typename T> __device__ __forceinline__ uint32_t magnitude(uint32_t pair);
template <> __device__ __forceinline__ uint32_t magnitude<BF16>(uint32_t pair) {
  const uint32_t a = pair << 16 & 0x7fffffffu, b = pair & 0x7fff0000u;
  return a > b ? a : b;
}
template <> __device__ __forceinline__ uint32_t magnitude<F16>(uint32_t pair) {
  const f32x2 v = unpack_f16x2(pair & 0x7fff7fffu);
  const float x = v.x, y = v.y;
  const uint32_t a = __builtin_bit_cast(uint32_t, x), b = __builtin_bit_cast(uint32_t, y);
  return a > b ? a : b;
}
// The largest of the quad's (a group's 4 lanes: of one token, so all of them are there).
template <int CTRL> __device__ __forceinline__ uint32_t larger_of(uint32_t v) {
  const uint32_t u = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
  return u > v ? u : v;
}

template <typename T, int D>
__global__ void __launch_bounds__(kTokens* D / 8) append(Args a) {
  constexpr int U = kUnroll;
  const Place<D> p(a);
  const int n = p.values;
  u32x4 x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    x[u] = u32x4{0u, 0u, 0u, 0u};
    if (p.row[u] >= 0)
      x[u] = load16<true>(static_cast<const char*>(a.in[n]) +
                          2 * ((p.token + u * kTokens) * a.token[n] + p.head * a.head[n]), p.chunk);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    uint32_t most = magnitude<T>(x[u][0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      const uint32_t m = magnitude<T>(x[u][i]);
      most = m > most ? m : most;
    }
    most = larger_of<kDppXor2>(larger_of<kDppXor1>(most));
    if (p.row[u] < 0) continue;
    const uint32_t scale = (uint32_t)scale_of(most, kMostScale<T>);
    const uint32_t codes = scale == kNanScale ? 0u : narrow4<T>(x[u], power_of(scale));
    *reinterpret_cast<uint32_t*>(a.codes[n] + p.row[u] * (D / 2) + 4 * p.chunk) = codes;
    if (p.chunk % 4 == 0) a.scales[n][p.row[u] * (D / kShared) + p.chunk / 4] = (uint8_t)scale;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kTokens* D / 8) read(Args a) {
  const Place<D> p(a);
  const int n = p.values;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const long long token = p.token + u * kTokens;
    if (token >= a.tokens) return;
    u32x4 x = {0u, 0u, 0u, 0u};
    if (p.row[u] >= 0) {
      const uint32_t codes = *reinterpret_cast<const uint32_t*>(a.codes[n] + p.row[u] * (D / 2) + 4 * p.chunk);
      const uint32_t scale = a.scales[n][p.row[u] * (D / kShared) + p.chunk / 4];
      x = widen4<T>(codes, power_of(scale_in(scale)));
    }
    store16<false>(static_cast<char*>(a.out[n]) + 2 * ((token * a.kv_heads + p.head) * D), p.chunk, x);
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------

bool sizes_ok(long long tokens, long long pages, int kv_heads, int head_dim, int block_size, int dtype) {
  const bool dim = head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 192 || head_dim == 256;
  return dim && kv_heads >= 1 && kv_heads <= 65536 && block_size >= 1 && pages >= 0 && pages <= INT_MAX / block_size &&
         tokens <= (long long)(INT_MAX - 2 * kv_heads) / (2 * kv_heads) * kTokens && (dtype == 1 || dtype == 2);
}

Args sized(long long tokens, long long pages, int kv_heads, int block_size) {
  Args a{};
  a.tokens = tokens;
  a.kv_heads = kv_heads;
  a.block_size = block_size;
  a.most = (unsigned)(pages * block_size);
  a.by_heads = divisor(kv_heads);
  a.by_block = divisor(block_size);
  return a;
}

template <typename T, int D>
int launch_dim(const Args& a, bool writes, hipStream_t stream) {
  constexpr int tokens = kTokens * kUnroll;
  const dim3 grid = rw_host::grid_of((a.tokens + tokens - 1) / tokens * 2 * a.kv_heads), threads(kTokens * D / 8);
  if (writes) hipLaunchKernelGGL((append<T, D>), grid, threads, 0, stream, a);
  else hipLaunchKernelGGL((read<T, D>), grid, threads, 0, stream, a);
  return (int)hipGetLastError();
}
template <typename T>
int launch_type(const Args& a, int head_dim, bool writes, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_dim<T, 64>(a, writes, stream);
    case 96: return launch_dim<T, 96>(a, writes, stream);
    case 128: return launch_dim<T, 128>(a, writes, stream);
    case 192: return launch_dim<T, 192>(a, writes, stream);
    default: return launch_dim<T, 256>(a, writes, stream);
  }
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace

extern "C" int kv4_append_launch(const void* k, const void* v, void* k_codes, void* k_scales, void* v_codes,
                                 void* v_scales, const void* slot_mapping, const long long* strides, long long tokens,
                                 long long pages, int kv_heads, int head_dim, int block_size, int dtype,
                                 hipStream_t stream) {
  using rw_host::aligned16;
  if (tokens <= 0) return rw_host::kOk;
  if (!sizes_ok(tokens, pages, kv_heads, head_dim, block_size, dtype) || !k || !v || !aligned16(k) || !aligned16(v) ||
      !slot_mapping || (pages && (!k_codes || !k_scales || !v_codes || !v_scales)) || !aligned4(k_codes) ||
      !aligned4(v_codes))
    return rw_host::kInvalid;
  Args a = sized(tokens, pages, kv_heads, block_size);
  for (int n = 0; n < 2; ++n) {
    a.token[n] = strides ? strides[2 * n] : (long long)kv_heads * head_dim;
    a.head[n] = strides ? strides[2 * n + 1] : head_dim;
    // the stride of a single token or head decides nothing
    if (tokens == 1) a.token[n] = 0;
    if (kv_heads == 1) a.head[n] = 0;
    if (a.token[n] % 8 || a.head[n] % 8) return rw_host::kInvalid;
  }
  a.in[0] = k, a.in[1] = v;
  a.codes[0] = static_cast<uint8_t*>(k_codes), a.codes[1] = static_cast<uint8_t*>(v_codes);
  a.scales[0] = static_cast<uint8_t*>(k_scales), a.scales[1] = static_cast<uint8_t*>(v_scales);
  a.slots = static_cast<const long long*>(slot_mapping);
  return dtype == 1 ? launch_type<BF16>(a, head_dim, true, stream) : launch_type<F16>(a, head_dim, true, stream);
}

extern "C" int kv4_read_launch(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                               const void* slots, void* k, void* v, long long tokens, long long pages, int kv_heads,
                               int head_dim, int block_size, int dtype, hipStream_t stream) {
  using rw_host::aligned16;
  if (tokens <= 0) return rw_host::kOk;
  if (!sizes_ok(tokens, pages, kv_heads, head_dim, block_size, dtype) || !k || !v || !aligned16(k) || !aligned16(v) ||
      !slots || (pages && (!k_codes || !k_scales || !v_codes || !v_scales)) || !aligned4(k_codes) || !aligned4(v_codes))
    return rw_host::kInvalid;
  Args a = sized(tokens, pages, kv_heads, block_size);
  a.out[0] = k, a.out[1] = v;
  a.codes[0] = static_cast<uint8_t*>(const_cast<void*>(k_codes));
  a.codes[1] = static_cast<uint8_t*>(const_cast<void*>(v_codes));
  a.scales[0] = static_cast<uint8_t*>(const_cast<void*>(k_scales));
  a.scales[1] = static_cast<uint8_t*>(const_cast<void*>(v_scales));
  a.slots = static_cast<const long long*>(slots);
  return dtype == 1 ? launch_type<BF16>(a, head_dim, false, stream) : launch_type<F16>(a, head_dim, false, stream);
}
