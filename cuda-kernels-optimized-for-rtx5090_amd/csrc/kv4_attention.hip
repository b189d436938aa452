// Attention over paged keys and values held in 4 bits (include/kv4_attention.h has the formula, include/kv4_cache.h the
// cache).
//
// A sequence's rows of a kv head (its tokens' query heads) are 16 or 32 columns of the products; a wave goes over slices
// of 32 keys:
//   - S^T = K Q^T by the products of 4-bit and 8-bit numbers, whose left operand is a lane's 16 bytes of codes and their
//     scale as they lie in the cache: nothing is converted. A query becomes two numbers of e4m3 (three of fp16), each
//     with 4 of its bits, and the row's power of two: they add up to the query as it is, down to 2^-18 of the row's
//     largest (a second product's operands then cost 16 registers of 128 elements, and no rounding).
//   - weights in base 2, a lane's own 8 keys; the reference point moves only when a row's maximum has grown by 2^8, so
//     that the rows' lanes exchange it only then.
//   - O^T = V^T P^T in bf16, which holds every value of the cache: the codes are widened two to an instruction, written
//     to LDS, and read transposed. fp16 rows' weights are two bf16 numbers, a high and a low part, in two products.
// The next two slices are in registers or on their way.
//
// The work is cut evenly: all sequences' slices one behind the other are dealt out in equal runs, one to each of a fixed
// number of workgroups to a kv head, whose 4 waves take a run's slices in turn. A run that crosses from one sequence to
// the next leaves a part for each; part w + b is run w's of sequence b (along the runs and the sequences one of the two
// grows at every border, so no two parts have a number in common). A second launch joins a row's parts. The lengths
// are on the device, and so is the dealing: a wave adds the slices of 64 sequences at a time.
#include <climits>

#include "divide.hpp"
#include "fp4.hpp"
#include "host.hpp"

#pragma clang fp contract(off)

using namespace rw;

namespace {

constexpr int kRows = 16, kKeys = 32, kWaves = 4;
constexpr float kGrow = 8.0f, kNone = -3.0e38f;  // kNone: the reference point of a row that has met no key

struct Args {
  const void* q;
  const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  const int *tables, *lens;
  void* out;
  float* sums;    // [kv heads][tiles][runs + batch][rows][head_dim]
  float2* stats;  // [kv heads][tiles][runs + batch][rows]: reference point (base 2), sum of weights
  long long qb, qs, qh;
  int batch, seq, q_heads, kv_heads, group, blocks, block_size, pages;
  int tiles, tile_rows, runs;  // runs 0: a workgroup to a sequence, nothing to join
  Divisor by_tiles, by_heads, by_group, by_block;
  float scale;                 // times log2(e)
};

__device__ uint8_t g_zeros[16] __attribute__((aligned(16)));  // an absent key

template <int D> struct Dims {
  static constexpr int wide = (D + 127) / 128;          // 128-element parts of a row
  static constexpr int shared = D / kShared;            // scales of a row
  static constexpr int blocks = D / 16;                 // of the sums
  static constexpr int pieces = D <= 64 ? 8 : D <= 128 ? 16 : 32;  // 16-byte places of a widened row in LDS
  static constexpr int row = 16 * pieces;
  static constexpr int slice = kKeys * row;
};
// Terms of a query, and of a weight.
template <typename T> constexpr int kTerms = 2;
template <> constexpr int kTerms<F16> = 3;

__device__ __forceinline__ int keys_of(const Args& a, int b) {
  const int most = a.blocks * a.block_size, n = a.lens[b];
  return n < 0 ? 0 : n < most ? n : most;
}
__device__ __forceinline__ int slices_of(int keys) { return (keys + kKeys - 1) / kKeys; }

// The sum over lanes 0 .. l.
__device__ __forceinline__ int sum_to(int v, int lane) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int below = from_lane(v, lane - d < 0 ? lane : lane - d);
    if (lane >= d) v += below;
  }
  return v;
}
// All sequences' slices; and the sequence that slice `at` of them lies in, with the slices before it.
__device__ __forceinline__ long long all_slices(const Args& a, int lane) {
  long long total = 0;
  for (int first = 0; first < a.batch; first += kWave) {
    const int b = first + lane;
    total += __builtin_amdgcn_readlane(sum_to(b < a.batch ? slices_of(keys_of(a, b)) : 0, lane), kWave - 1);
  }
  return total;
}
__device__ __forceinline__ int sequence_at(const Args& a, long long at, long long& before, int lane) {
  before = 0;
  for (int first = 0; first < a.batch; first += kWave) {
    const int b = first + lane, n = b < a.batch ? slices_of(keys_of(a, b)) : 0, sum = sum_to(n, lane);
    const uint64_t past = __ballot(before + sum > at);
    if (past) {
      const int l = __builtin_ctzll(past);
      before += __builtin_amdgcn_readlane(sum - n, l);
      return first + l;
    }
    before += __builtin_amdgcn_readlane(sum, kWave - 1);
  }
  return a.batch;
}

// Where 16-byte piece c of key r of a widened slice lies: XORed with the key, so that the pieces that lanes write
// together (of 16 keys, 4 pieces apart) and the pairs of pieces that they read together (of 4 keys) meet all banks.
template <int D> __device__ __forceinline__ int place(int r, int c) {
  const int turn = (Dims<D>::pieces == 8 ? r & 6 : 2 * r & 14) | (r >> 3 & 1);
  return r * Dims<D>::row + (c ^ turn) * 16;
}

// A lane's share of 32 keys: of key r and of key 16 + r the codes at 32 h ... and their scales.
template <int D> struct Slice {
  u32x4 k[2][Dims<D>::wide], v[2][Dims<D>::wide];
  uint32_t k_scale[2][Dims<D>::wide], v_scale[2][Dims<D>::wide];
  uint32_t present;  // a bit to a key
};

// 16 rows of a wave.
template <typename T, int D> struct Tile {
  Eights q[kTerms<T>][Dims<D>::wide];
  uint32_t q_scale;
  f32x4 o[Dims<D>::blocks];
  float m, l;        // reference point; sum of weights over this lane's keys
  int at, limit;     // the row's place in the outputs, or -1; the last key it sees
  uint32_t poison;   // a bit to a group of 32 elements: it has met a NaN there
};

template <typename T, int D>
__device__ __forceinline__ void start(Tile<T, D>& t, const Args& a, int b, int head, int i, int keys, int h) {
  unsigned token = (unsigned)i;
  const int g = a.by_group.take(token), s = (int)token;
  t.at = -1;
  t.limit = -1;
  u32x4 x[Dims<D>::wide][4];
#pragma unroll
  for (int w = 0; w < Dims<D>::wide; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j) x[w][j] = (u32x4){0u, 0u, 0u, 0u};
  if (s < a.seq) {
    t.at = (b * a.seq + s) * a.q_heads + head * a.group + g;
    t.limit = keys - a.seq + s;
    const char* q = static_cast<const char*>(a.q) + 2 * (b * a.qb + s * a.qs + (head * a.group + g) * a.qh);
#pragma unroll
    for (int w = 0; w < Dims<D>::wide; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // elements 128 w + 64 (j / 2) + 16 h + 8 (j % 2) ...
        const int c = 16 * w + 8 * (j / 2) + 2 * h + j % 2;
        if (c < D / 8) x[w][j] = load16<false>(q, c);
      }
  }
  float y[Dims<D>::wide][4][8], most = 0.0f;
  bool wild = false;
#pragma unroll
  for (int w = 0; w < Dims<D>::wide; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      unpack<T>(x[w][j], y[w][j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        most = fmaxf(most, fabsf(y[w][j][e]));
        wild = wild || !(fabsf(y[w][j][e]) <= 3.4e38f);
      }
    }
  most = max_of_quarters(wild ? INFINITY : most);
  // the row's largest to [2^7, 2^8) of e4m3's 448; the terms after the first are 2^4 down each
  const int exponent = (int)(__builtin_bit_cast(uint32_t, most) >> 23) - 7, up = exponent < 9 ? 9 : exponent;
  t.q_scale = most > 3.4e38f ? kNanScale : (uint32_t)up;
  const float by = power_of((uint32_t)(254 - up));
#pragma unroll
  for (int w = 0; w < Dims<D>::wide; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) y[w][j][e] = t.q_scale == kNanScale ? 0.0f : y[w][j][e] * by;
#pragma unroll
  for (int n = 0; n < kTerms<T>; ++n)
#pragma unroll
    for (int w = 0; w < Dims<D>::wide; ++w)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        t.q[n][w].lo[2 * j] = take_e4m3(y[w][j]);
        t.q[n][w].lo[2 * j + 1] = take_e4m3(y[w][j] + 4);
        t.q[n][w].hi[2 * j] = take_e4m3(y[w][2 + j]);
        t.q[n][w].hi[2 * j + 1] = take_e4m3(y[w][2 + j] + 4);
      }
#pragma unroll
  for (int d = 0; d < Dims<D>::blocks; ++d) t.o[d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  t.m = kNone;
  t.l = 0.0f;
  t.poison = 0u;
}

// A lane's two rows of a slice: where they lie in the cache, or -1.
struct Rows {
  long long of[2];
};

template <typename T, int D, int TILES>
__device__ __forceinline__ void attend_run(Tile<T, D> (&t)[TILES], const Args& a, int b, int head, int keys, int all_see,
                                           int first, int stop, char* lds, int wave, int lane) {
  constexpr int W = Dims<D>::wide;
  const int r = lane & 15, h = lane >> 4;
  const int* table = a.tables + (long long)b * a.blocks;
  const int page_rows = a.kv_heads * a.block_size, head_rows = head * a.block_size;
  auto entry = [&](int s, int j) {
    const int t = s * kKeys + 16 * j + r, page = (int)a.by_block.of((unsigned)(t < keys ? t : 0));
    return table[page];
  };
  auto row = [&](int block, int s, int j) -> long long {
    unsigned page = (unsigned)(s * kKeys + 16 * j + r);
    const bool there = (int)page < keys && (unsigned)block < (unsigned)a.pages;
    const int at = a.by_block.take(page);
    return there ? (long long)block * page_rows + (head_rows + at) : -1;
  };
  auto load = [&](Slice<D>& x, const long long (&at)[2]) {
    x.present = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      x.present |= (uint32_t)(__ballot(at[j] >= 0) & 0xffffu) << (16 * j);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int c = 4 * w + h;
        const bool mine = at[j] >= 0 && (Dims<D>::shared == 4 * W || c < Dims<D>::shared);
        const uint64_t codes = (uint64_t)at[j] * (D / 2) + 16 * c, scales = (uint64_t)at[j] * (D / kShared) + c;
        x.k[j][w] = load16<true>(mine ? a.k_codes + codes : g_zeros, 0);
        x.v[j][w] = load16<true>(mine ? a.v_codes + codes : g_zeros, 0);
        x.k_scale[j][w] = mine ? a.k_scales[scales] : 0u;
        x.v_scale[j][w] = mine ? a.v_scales[scales] : 0u;
      }
    }
  };
  lds_ptr at_lo[Dims<D>::blocks];
#pragma unroll
  for (int d = 0; d < Dims<D>::blocks; ++d)
    at_lo[d] = in_lds(lds) + place<D>(4 * h + (r >> 2), 2 * d + ((r & 3) >> 1)) + 8 * (r & 1);

  auto step = [&](Slice<D>& x, int s) {
    f32x4 score[TILES][2];
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        score[n][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int e = 0; e < kTerms<T>; ++e)
            score[n][j] = product_fp4(x.k[j][w], t[n].q[e][w], score[n][j], scale_in(x.k_scale[j][w]),
                                      t[n].q_scale == kNanScale ? kNanScale : t[n].q_scale - 4 * e);
      }
    // values that are NaN leave the products (0 times NaN is NaN) and mark the rows that see their key
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int w = 0; w < W; ++w) most = x.v_scale[j][w] > most ? x.v_scale[j][w] : most;
    if (__ballot(most > 252u)) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int w = 0; w < W; ++w) {
          uint64_t bad = __ballot(x.v_scale[j][w] > 252u);
          if (x.v_scale[j][w] > 252u) x.v_scale[j][w] = 0u, x.v[j][w] = (u32x4){0u, 0u, 0u, 0u};
          for (; bad; bad &= bad - 1) {
            const int l = __builtin_ctzll(bad), key = s * kKeys + 16 * j + (l & 15);
#pragma unroll
            for (int n = 0; n < TILES; ++n)
              if (key <= t[n].limit) t[n].poison |= 1u << (4 * w + (l >> 4));
          }
        }
    }
    order_lds();
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int c = 4 * w + h;
        const float power = power_of(x.v_scale[j][w]);
        if (Dims<D>::shared == 4 * W || c < Dims<D>::shared) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<u32x4*>(lds + place<D>(16 * j + r, 4 * c + e)) = widen4<BF16>(x.v[j][w][e], power);
        }
      }
    order_lds();
    if (x.present != ~0u || s * kKeys + kKeys - 1 > all_see) {
      const uint32_t present = x.present >> (4 * h);
#pragma unroll
      for (int n = 0; n < TILES; ++n) {
        const int limit = t[n].limit - s * kKeys - 4 * h;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!(present >> (16 * j + i) & 1u) || 16 * j + i > limit) score[n][j][i] = -INFINITY;
      }
    }
    u32x4 p[TILES], p_low[TILES];
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
      float top = fmaxf(score[n][0][0], score[n][1][0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) top = fmaxf(top, fmaxf(score[n][0][i], score[n][1][i]));
      top *= a.scale;
      if (__ballot(top > t[n].m + kGrow)) {
        top = max_of_quarters(top);
        const float m = top > t[n].m + kGrow ? top : t[n].m, f = __builtin_amdgcn_exp2f(t[n].m - m);
        t[n].m = m;
        t[n].l *= f;
#pragma unroll
        for (int d = 0; d < Dims<D>::blocks; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) t[n].o[d][i] *= f;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(score[n][j][i], a.scale, -t[n].m));
          const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(score[n][j][i + 1], a.scale, -t[n].m));
          const uint32_t two = pack2<BF16>(x0, x1);
          p[n][2 * j + i / 2] = two;
          if constexpr (kTerms<T> == 2) {
            t[n].l = add_pair<BF16>(two, t[n].l);
          } else {
            p_low[n][2 * j + i / 2] = pack2<BF16>(x0 - bf16_lo(two), x1 - bf16_hi(two));
            t[n].l += x0 + x1;
          }
        }
    }
#pragma unroll
    for (int d = 0; d < Dims<D>::blocks; ++d) {
      const u32x2 lo = lds_column(at_lo[d]), hi = lds_column(at_lo[d] + 16 * Dims<D>::row);
      const u32x4 v = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
      for (int n = 0; n < TILES; ++n) {
        t[n].o[d] = product16(v, p[n], t[n].o[d]);
        if constexpr (kTerms<T> == 3) t[n].o[d] = product16(v, p_low[n], t[n].o[d]);
      }
    }
  };

  // slices first + wave, first + wave + 4, ...: this one and the next in registers, the pages of the one after
  const int begin = first + wave;
  if (begin >= stop) return;
  Slice<D> x[2];
  int next[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int s = begin + n * kWaves;
    long long at[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) at[j] = s < stop ? row(entry(s, j), s, j) : -1;
    load(x[n], at);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) next[j] = entry(begin + 2 * kWaves, j);
  for (int s = begin; s < stop; s += 2 * kWaves) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int now = s + n * kWaves;
      if (now >= stop) break;
      step(x[n], now);
      const int then = now + 2 * kWaves;
      long long at[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        at[j] = then < stop ? row(next[j], then, j) : -1;
        next[j] = entry(then + kWaves, j);
      }
      if (then < stop) load(x[n], at);
    }
  }
}

// The waves' sums over the same 16 rows joined through LDS, and the part, or the result where there is no other,
// written. part < 0: the result.
template <typename T, int D>
__device__ __forceinline__ void finish(Tile<T, D>& t, const Args& a, long long part, int n, char* lds, float2* stats,
                                       int wave, int lane) {
  constexpr int quads = D / 4;
  static_assert(kRows * D * 4 <= Dims<D>::slice, "a tile's sums fit its wave's slice");
  const int r = lane & 15, h = lane >> 4;
  const float l = sum_of_quarters(t.l);
  __syncthreads();  // all waves are done with what is overwritten
  if (lane < kRows) stats[wave * kRows + lane] = make_float2(t.m, l);
  __syncthreads();
  float m = kNone;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, stats[w * kRows + r].x);
  const float f = __builtin_amdgcn_exp2f(t.m - m);
  float4* mine = reinterpret_cast<float4*>(lds + wave * Dims<D>::slice);
#pragma unroll
  for (int d = 0; d < Dims<D>::blocks; ++d) {
    const float by = t.poison >> (d / 2) & 1u ? __builtin_nanf("") : f;
    mine[r * quads + ((4 * d + h) ^ (r & 7))] = make_float4(t.o[d][0] * by, t.o[d][1] * by, t.o[d][2] * by,
                                                            t.o[d][3] * by);
  }
  // the rows' places, for the lanes that write them
  int* places = reinterpret_cast<int*>(stats + kWaves * kRows);
  if (wave == 0 && lane < kRows) places[lane] = t.at;
  __syncthreads();
  for (int i = wave * kWave + lane; i < kRows * quads; i += kWaves * kWave) {
    const int row = i / quads, c = i % quads;
    const long long at = places[row];
    if (at < 0) continue;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float top = kNone, total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w * kRows + row].x);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float4 y = reinterpret_cast<const float4*>(lds + w * Dims<D>::slice)[row * quads + (c ^ (row & 7))];
      sum.x += y.x, sum.y += y.y, sum.z += y.z, sum.w += y.w;
      const float2 s = stats[w * kRows + row];
      total += s.y * __builtin_amdgcn_exp2f(s.x - top);
    }
    if (part < 0) {
      const float by = total > 0.0f || total != total ? 1.0f / total : 0.0f;  // a row that sees no key: 0
      *reinterpret_cast<u32x2*>(static_cast<char*>(a.out) + 2 * (at * D + 4 * c)) =
          (u32x2){pack2<T>(sum.x * by, sum.y * by), pack2<T>(sum.z * by, sum.w * by)};
    } else {
      const long long to = part * a.tile_rows + n * kRows + row;
      *reinterpret_cast<float4*>(a.sums + to * D + 4 * c) = sum;
      if (c == 0) a.stats[to] = make_float2(top, total);
    }
  }
}

// TILES: 16 or 32 rows.
template <typename T, int D, int TILES>
__global__ void __launch_bounds__(kWaves* kWave, D <= 128 ? 2 : 1) attend(Args a) {
  __shared__ __align__(16) char lds[kWaves * Dims<D>::slice];
  __shared__ float2 stats[kWaves * kRows + kRows / 2];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  unsigned u = (unsigned)rw_host::workgroup();
  const int tile = a.by_tiles.take(u), head = a.by_heads.take(u);
  int b = (int)u;
  long long at = 0, end = 0, before = 0;  // of all slices
  if (a.runs) {
    if (b >= a.runs) return;
    const long long total = all_slices(a, lane), each = (total + a.runs - 1) / a.runs;
    at = b * each;
    end = at + each < total ? at + each : total;
    if (at >= end) return;
    b = sequence_at(a, at, before, lane);
  } else if (b >= a.batch) {
    return;
  }
  for (;;) {
    const int keys = __builtin_amdgcn_readfirstlane(keys_of(a, b)), n = slices_of(keys);
    const int first = (int)(at - before), stop = a.runs && end - before < n ? (int)(end - before) : n;
    if (!a.runs || stop > first) {
      Tile<T, D> t[TILES];
      const int row = tile * TILES * kRows + (lane & 15);
#pragma unroll
      for (int i = 0; i < TILES; ++i) start(t[i], a, b, head, row + i * kRows, keys, lane >> 4);
      const int all_see = keys - a.seq + (int)a.by_group.of((unsigned)(tile * TILES * kRows));  // its first token
      attend_run<T, D, TILES>(t, a, b, head, keys, all_see, first, stop, lds + wave * Dims<D>::slice, wave, lane);
      const long long run = (long long)u + b;
      const long long part = a.runs ? ((long long)head * a.tiles + tile) * (a.runs + a.batch) + run : -1;
#pragma unroll
      for (int i = 0; i < TILES; ++i) finish(t[i], a, part, i, lds, stats, wave, lane);
    }
    if (!a.runs) return;
    at = before + stop;
    if (at >= end) return;
    before += n;
    ++b;
    __syncthreads();  // the next part's values go over this one's sums
  }
}

// A row's parts joined: a wave to a row (a workgroup: heads 4 y ... of token x, and of 2^21 z more).
template <typename T, int D>
__global__ void __launch_bounds__(256) join(Args a) {
  constexpr int E = D <= 64 ? 1 : D <= 128 ? 2 : 4, batch = 8;  // elements of a lane; parts to a trip to memory
  const int lane = lane_id(), token = (int)(blockIdx.z << rw_host::kGridShift | blockIdx.x);
  const int q_head = (int)blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(wave_id());
  if (q_head >= a.q_heads || token >= a.batch * a.seq) return;
  const int b = token / a.seq, s = token % a.seq, head = (int)a.by_group.of((unsigned)q_head);
  const int i = s * a.group + q_head - head * a.group, tile = i / a.tile_rows;
  const long long row = i % a.tile_rows, total = all_slices(a, lane);
  const int each = (int)((total + a.runs - 1) / a.runs), keys = keys_of(a, b), n = slices_of(keys);
  float o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
  float sum = 0.0f;
  const bool mine = lane * E < D;
  if (n > 0 && keys - a.seq + s >= 0) {
    long long before = 0;
    for (int first = 0; first < b; first += kWave) {
      const int x = first + lane;
      before += __builtin_amdgcn_readlane(sum_to(x < b ? slices_of(keys_of(a, x)) : 0, lane), kWave - 1);
    }
    const int from = (int)(before / each), parts = (int)((before + n - 1) / each) - from + 1;
    const long long first = ((long long)head * a.tiles + tile) * (a.runs + a.batch) + from + b;
    const float2* stats = a.stats + first * a.tile_rows + row;
    const float* sums = a.sums + (first * a.tile_rows + row) * D + lane * E;
    const long long step = a.tile_rows;
    float m = kNone;
    for (int p = lane; p < parts; p += kWave) m = fmaxf(m, stats[p * step].x);
    m = wave_max(m);
    for (int p0 = 0; p0 < parts; p0 += kWave) {
      float w = 0.0f, l = 0.0f;
      if (p0 + lane < parts) {
        const float2 stat = stats[(p0 + lane) * step];
        w = __builtin_amdgcn_exp2f(stat.x - m);
        l = stat.y * w;
      }
      sum += wave_sum(l);
      const int some = least(parts - p0, kWave);
      for (int p1 = 0; p1 < some; p1 += batch) {
        float x[batch][E];
#pragma unroll
        for (int p = 0; p < batch; ++p)
#pragma unroll
          for (int e = 0; e < E; ++e) x[p][e] = mine && p1 + p < some ? sums[(p0 + p1 + p) * step * D + e] : 0.0f;
#pragma unroll
        for (int p = 0; p < batch; ++p) {
          const float by = readlane(w, least(p1 + p, kWave - 1));
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += x[p][e] * by;
        }
      }
    }
  }
  const float inverse = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
  if (mine) {
    const long long at = (long long)token * a.q_heads + q_head;
#pragma unroll
    for (int e = 0; e < E; ++e) store_elem<T>(a.out, at * D + lane * E + e, o[e] * inverse);
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------

enum { kTuneRuns = 0, kTuneTiles = 1 };
constexpr long long kMostKeys = 1 << 30;  // of a table

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

bool sizes_ok(long long batch, long long seq, int q_heads, int kv_heads, int head_dim, long long blocks,
              long long block_size) {
  const bool dim = head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 192 || head_dim == 256;
  return dim && kv_heads >= 1 && q_heads >= kv_heads && q_heads <= 65536 && q_heads % kv_heads == 0 &&
         block_size >= 1 && block_size <= kMostKeys && blocks >= 0 && blocks <= kMostKeys / block_size &&
         seq <= INT_MAX / 2 / q_heads && batch <= INT_MAX / 2 / (seq * q_heads);
}

Args sized(long long batch, long long seq, int q_heads, int kv_heads, long long blocks, long long block_size) {
  Args a{};
  a.batch = (int)batch, a.seq = (int)seq;
  a.q_heads = q_heads, a.kv_heads = kv_heads, a.group = q_heads / kv_heads;
  a.blocks = (int)blocks, a.block_size = (int)block_size;
  const long long rows = seq * a.group;
  const int tiles = rw_host::tune_get(kTuneTiles);
  a.tile_rows = tiles == 1 || (tiles != 2 && rows <= kRows) ? kRows : 2 * kRows;
  a.tiles = (int)ceil_div(rows, a.tile_rows);
  // Two workgroups to a CU, of 4 slices to a wave at least; nothing is cut where a sequence is no longer than that.
  const long long slices = ceil_div(blocks * block_size, kKeys), share = 4 * kWaves;
  const long long units = (long long)kv_heads * a.tiles, most = ceil_div(2LL * rw_host::device_cus(), units);
  long long runs = slices <= share ? 0 : most < ceil_div(batch * slices, share) ? most : ceil_div(batch * slices, share);
  if (rw_host::tune_get(kTuneRuns)) runs = rw_host::tune_get(kTuneRuns) < 0 ? 0 : rw_host::tune_get(kTuneRuns);
  a.runs = (int)runs;
  return a;
}

// Rows of parts; workgroups.
long long part_rows(const Args& a) {
  return a.runs ? (long long)a.kv_heads * a.tiles * (a.runs + a.batch) * a.tile_rows : 0;
}
constexpr long long kMostGroups = (1LL << 30) - (1LL << rw_host::kGridShift);
long long groups_of(const Args& a) { return (long long)a.kv_heads * a.tiles * (a.runs ? a.runs : a.batch); }

template <typename T, int D>
int launch_dim(const Args& a, hipStream_t stream) {
  const dim3 grid = rw_host::grid_of(groups_of(a)), threads(kWaves * kWave);
  if (a.tile_rows == kRows) hipLaunchKernelGGL((attend<T, D, 1>), grid, threads, 0, stream, a);
  else hipLaunchKernelGGL((attend<T, D, 2>), grid, threads, 0, stream, a);
  const int err = (int)hipGetLastError();
  if (err || a.runs == 0) return err;
  dim3 tokens = rw_host::grid_of((long long)a.batch * a.seq);
  tokens.z = tokens.y, tokens.y = (unsigned)ceil_div(a.q_heads, 4);
  hipLaunchKernelGGL((join<T, D>), tokens, dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}
template <typename T>
int launch_type(const Args& a, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_dim<T, 64>(a, stream);
    case 96: return launch_dim<T, 96>(a, stream);
    case 128: return launch_dim<T, 128>(a, stream);
    case 192: return launch_dim<T, 192>(a, stream);
    default: return launch_dim<T, 256>(a, stream);
  }
}

}  // namespace

extern "C" long long kv4_attention_work(long long batch, long long seq, int q_heads, int kv_heads, int head_dim,
                                        long long blocks, long long block_size) {
  if (batch <= 0 || seq <= 0) return 0;
  if (!sizes_ok(batch, seq, q_heads, kv_heads, head_dim, blocks, block_size)) return -1;
  const Args a = sized(batch, seq, q_heads, kv_heads, blocks, block_size);
  return groups_of(a) > kMostGroups ? -1 : part_rows(a) * (4LL * head_dim + 8);
}

extern "C" int kv4_attention_launch(const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                                    const void* v_scales, const void* block_tables, const void* seq_lens, void* out,
                                    void* work, long long work_bytes, const long long* strides, long long batch,
                                    long long seq, long long pages, int q_heads, int kv_heads, int head_dim,
                                    long long blocks, long long block_size, float scale, int dtype,
                                    hipStream_t stream) {
  using rw_host::aligned16;
  if (batch <= 0 || seq <= 0) return rw_host::kOk;
  if (!sizes_ok(batch, seq, q_heads, kv_heads, head_dim, blocks, block_size) || pages < 0 ||
      pages > INT_MAX / block_size || (dtype != 1 && dtype != 2) || !q || !aligned16(q) || !out || !aligned16(out) ||
      !seq_lens || (pages && (!k_codes || !k_scales || !v_codes || !v_scales)) || !aligned16(k_codes) ||
      !aligned16(v_codes) || (blocks && !block_tables) || !(scale >= 1.0e-30f && scale <= 1.0e30f))
    return rw_host::kInvalid;
  Args a = sized(batch, seq, q_heads, kv_heads, blocks, block_size);
  if (groups_of(a) > kMostGroups) return rw_host::kInvalid;
  const long long rows = part_rows(a);
  if (rows && (!work || !aligned16(work) || work_bytes < rows * (4LL * head_dim + 8))) return rw_host::kInvalid;
  const long long token = (long long)q_heads * head_dim;
  a.qb = batch == 1 ? 0 : strides ? strides[0] : seq * token;
  a.qs = seq == 1 ? 0 : strides ? strides[1] : token;
  a.qh = q_heads == 1 ? 0 : strides ? strides[2] : head_dim;
  if (a.qb % 8 || a.qs % 8 || a.qh % 8) return rw_host::kInvalid;
  a.q = q, a.out = out;
  a.k_codes = static_cast<const uint8_t*>(k_codes), a.k_scales = static_cast<const uint8_t*>(k_scales);
  a.v_codes = static_cast<const uint8_t*>(v_codes), a.v_scales = static_cast<const uint8_t*>(v_scales);
  a.tables = static_cast<const int*>(block_tables), a.lens = static_cast<const int*>(seq_lens);
  a.sums = static_cast<float*>(work);
  a.stats = reinterpret_cast<float2*>(a.sums + rows * head_dim);
  a.pages = (int)pages;
  a.by_tiles = divisor(a.tiles), a.by_heads = divisor(kv_heads), a.by_group = divisor(a.group);
  a.by_block = divisor(block_size);
  a.scale = scale * 1.44269504088896341f;
  return dtype == 1 ? launch_type<BF16>(a, head_dim, stream) : launch_type<F16>(a, head_dim, stream);
}

extern "C" int kv4_attention_tune(int slot, int value) { return rw_host::tune_set(slot, value); }
