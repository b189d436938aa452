// Attention over paged keys and values held in 4 bits (include/kv4_attention.h has the formula, include/kv4_cache.h the
// cache).
//
// A sequence's rows of a kv head (its tokens' query heads) are 16 or 32 columns of the products; a wave goes over slices
// of 32 keys:
//   - S^T = K Q^T and O^T = V^T P^T by the products of bf16, which holds every value of the cache: codes are widened two to
//     an instruction. A lane's 16 bytes of a key are the left operand's as they lie in the cache (the order of the
//     contraction is free); values are written to LDS and read transposed. fp16 queries and all weights are two bf16
//     numbers, a high and a low part, in two products. (The products of 4-bit and 8-bit numbers would take the codes as they
//     are, but keep some 18 bits of the largest product of a sum: with one of 120 in a score weights were off by 1% and more.)
//   - weights in base 2, a lane's own 8 keys, against the largest score of the wave's first slice.
// The next two slices are on their way (three of the smaller tiles).
//
// The work is cut evenly: all sequences' slices one behind the other are dealt out in equal runs, one to each of a fixed
// number of workgroups to a kv head, whose 4 waves take a run's slices in turn. A run that crosses from one sequence to
// the next leaves a part for each; part w + b is run w's of sequence b (along the runs and the sequences one of the two
// grows at every border, so no two parts have a number in common). A second launch joins a row's parts. The lengths
// are on the device, and so is the dealing: a wave adds the slices of 64 sequences at a time.
//
// Bound by memory: 64 tokens of 32/8 heads of 128 behind 2048 to 8192 keys in 69 us with one set of inputs, in 70 to 75 with
// two in turn, 360 MB at 4.8 to 5.2 TB/s; one token behind 32768 keys in 16.2 us, of which the 36 MB are 6 and the join 4.
#include <climits>
#include <type_traits>

#include "divide.hpp"
#include "fp4.hpp"
#include "host.hpp"

#pragma clang fp contract(off)

using namespace rw;

namespace {

constexpr int kRows = 16, kKeys = 32, kWaves = 4;
constexpr float kNone = -3.0e38f;  // the reference point of a row that has met no key

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

template <int D> struct Dims {
  static constexpr int wide = (D + 127) / 128;          // 128-element parts of a row
  static constexpr int shared = D / kShared;            // scales of a row
  static constexpr int blocks = D / 16;                 // of the sums
  static constexpr int pieces = D <= 64 ? 8 : D <= 128 ? 16 : 32;  // 16-byte places of a widened row in LDS
  static constexpr int row = 16 * pieces;
  static constexpr int slice = kKeys * row;
};
// Terms of a query.
template <typename T> constexpr int kTerms = 1;
template <> constexpr int kTerms<F16> = 2;

__device__ __forceinline__ int keys_of(const Args& a, int b) {
  const int most = a.blocks * a.block_size, n = a.lens[b];
  return n < 0 ? 0 : n < most ? n : most;
}
__device__ __forceinline__ int slices_of(int keys) { return (keys + kKeys - 1) / kKeys; }

// The sum over lanes 0 .. l, of 2^25 slices each at most; and lane l's.
__device__ __forceinline__ uint32_t sum_to(uint32_t v, int lane) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint32_t below = (uint32_t)from_lane((int)v, lane - d < 0 ? lane : lane - d);
    if (lane >= d) v += below;
  }
  return v;
}
__device__ __forceinline__ uint32_t sum_of(uint32_t sum, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)sum, l); }
// All sequences' slices; and the sequence that slice `at` of them lies in, with the slices before it.
__device__ __forceinline__ long long all_slices(const Args& a, int lane) {
  long long total = 0;
  for (int first = 0; first < a.batch; first += kWave) {
    const int b = first + lane;
    total += sum_of(sum_to(b < a.batch ? slices_of(keys_of(a, b)) : 0, lane), kWave - 1);
  }
  return total;
}
__device__ __forceinline__ int sequence_at(const Args& a, long long at, long long& before, int lane) {
  before = 0;
  for (int first = 0; first < a.batch; first += kWave) {
    const int b = first + lane;
    const uint32_t n = b < a.batch ? slices_of(keys_of(a, b)) : 0, sum = sum_to(n, lane);
    const uint64_t past = __ballot(before + sum > at);
    if (past) {
      const int l = __builtin_ctzll(past);
      before += sum_of(sum - n, l);
      return first + l;
    }
    before += sum_of(sum, kWave - 1);
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

// How many slices of a wave are on their way or in registers, within what its sums leave of them.
template <int D, int TILES> constexpr int kAhead = D <= 128 ? (TILES == 1 ? 3 : 2) : 2;

// 16 rows of a wave.
template <typename T, int D> struct Tile {
  u32x4 q[kTerms<T>][Dims<D>::wide][4];
  f32x4 o[Dims<D>::blocks];
  float m, l;        // reference point; sum of weights over this lane's keys
  int at, limit;     // the row's place in the outputs, or -1; the last key it sees
  uint32_t poison;   // a bit to a group of 32 elements: it has met a NaN there
};

// A row's query as it is loaded: elements 128 w + 32 h + 8 j ..., as a word of the lane's codes has them.
template <int D> struct Query {
  u32x4 x[Dims<D>::wide][4];
};
template <typename T, int D>
__device__ __forceinline__ void find(Tile<T, D>& t, Query<D>& q, const Args& a, int b, int head, int i, int keys, int h) {
  unsigned token = (unsigned)i;
  const int g = a.by_group.take(token), s = (int)token;
  t.at = -1;
  t.limit = -1;
#pragma unroll
  for (int w = 0; w < Dims<D>::wide; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j) q.x[w][j] = (u32x4){0u, 0u, 0u, 0u};
  if (s < a.seq) {
    t.at = (b * a.seq + s) * a.q_heads + head * a.group + g;
    t.limit = keys - a.seq + s;
    const char* from = static_cast<const char*>(a.q) + 2 * (b * a.qb + s * a.qs + (head * a.group + g) * a.qh);
#pragma unroll
    for (int w = 0; w < Dims<D>::wide; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 16 * w + 4 * h + j;
        if (c < D / 8) q.x[w][j] = load16<false>(from, c);
      }
  }
}
template <typename T, int D>
__device__ __forceinline__ void start(Tile<T, D>& t, const Query<D>& q) {
  // a row with a NaN or an infinity is NaN altogether (the largest is NaN where one is; as it is, a packed pair is the second
  // of the two with some bits more)
  float most = 0.0f;
#pragma unroll
  for (int w = 0; w < Dims<D>::wide; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t two = q.x[w][j][i];
        float x0 = bf16_lo(two), x1 = __builtin_bit_cast(float, two);
        t.q[0][w][j][i] = two;
        if constexpr (kTerms<T> == 2) {
          const f32x2 y = unpack_f16x2(two);
          x0 = y.x, x1 = y.y;
          const uint32_t high = pack2<BF16>(x0, x1);
          t.q[0][w][j][i] = high;
          t.q[1][w][j][i] = pack2<BF16>(x0 - bf16_lo(high), x1 - bf16_hi(high));  // (of 3 bits)
        }
        most = __builtin_elementwise_maximum(most, __builtin_elementwise_maximum(fabsf(x0), fabsf(x1)));
      }
  const bool bad = max_of_quarters(most < INFINITY ? 0.0f : 1.0f) > 0.0f;
#pragma unroll
  for (int w = 0; w < Dims<D>::wide; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) t.q[0][w][j][i] = bad ? 0x7fc07fc0u : t.q[0][w][j][i];
#pragma unroll
  for (int d = 0; d < Dims<D>::blocks; ++d) t.o[d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  t.m = kNone;
  t.l = 0.0f;
  t.poison = 0u;
}

// The reference point of a row's weights is the largest score of the wave's first slice, and stays: weights are floating
// point, and the sums have room for 2^60 times as many. Where a row's scores grow by more than that, or its sums are not
// finite, the run is done again with a point that follows the largest (kFollow). So the loop has no branch that touches the
// sums: for one that moved the point there, the compiler copied them at every slice, 18 to 39 of 150 instructions.
constexpr float kMostSum = 0x1p60f;
enum Point { kFirst, kKept, kFollow };

// The weights of a lane's 8 scores as two bf16 numbers each, `low` what rounding took from the first; their sum. In one
// number, and summed as rounded, outputs of bf16 were off by 0.0023 from the formula in 64 bits where their own rounding
// alone is 0.0017; the second product costs 3% of the time (one token behind 32768 keys) to 13% (33 x 5 tokens of 32/8 heads
// of 128 behind up to 1801).
__device__ __forceinline__ float weigh(const f32x4 (&score)[2], float scale, float m, u32x4& p, u32x4& low) {
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(score[j][i], scale, -m));
      const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(score[j][i + 1], scale, -m));
      const uint32_t two = pack2<BF16>(x0, x1);
      p[2 * j + i / 2] = two;
      low[2 * j + i / 2] = pack2<BF16>(x0 - bf16_lo(two), x1 - bf16_hi(two));
      sum += x0 + x1;
    }
  return sum;
}

// A slice of 32 keys: its scores, weights and values.
template <typename T, int D, int TILES, Point POINT>
__device__ __forceinline__ void step(Tile<T, D> (&t)[TILES], Slice<D>& x, const Args& a, int s, int all_see, char* lds,
                                     const lds_ptr (&columns)[Dims<D>::blocks], int lane) {
  constexpr int W = Dims<D>::wide;
  const int r = lane & 15, h = lane >> 4;
  // scales that stand for NaN: keys' products become NaN; values leave the products (0 times NaN is NaN) and mark the
  // rows that see their key
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int w = 0; w < W; ++w) {
      most = x.k_scale[j][w] > most ? x.k_scale[j][w] : most;
      most = x.v_scale[j][w] > most ? x.v_scale[j][w] : most;
    }
  if (__builtin_expect(__ballot(most > 252u) != 0, 0)) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        x.k_scale[j][w] = scale_in(x.k_scale[j][w]);
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
  f32x4 score[TILES][2];
#pragma unroll
  for (int n = 0; n < TILES; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) score[n][j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const u32x4 k = widen4<BF16>(x.k[j][w][c], power_of(x.k_scale[j][w]));
#pragma unroll
        for (int n = 0; n < TILES; ++n)
#pragma unroll
          for (int e = 0; e < kTerms<T>; ++e) score[n][j] = product16(k, t[n].q[e][w][c], score[n][j]);
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
  if (__builtin_expect(x.present != ~0u || s * kKeys + kKeys - 1 > all_see, 0)) {
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
  u32x4 p[TILES], low[TILES];
#pragma unroll
  for (int n = 0; n < TILES; ++n) {
    if constexpr (POINT != kKept) {
      float top = fmaxf(score[n][0][0], score[n][1][0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) top = fmaxf(top, fmaxf(score[n][0][i], score[n][1][i]));
      const float m = fmaxf(t[n].m, max_of_quarters(top) * a.scale);
      if constexpr (POINT == kFollow) {
        const float f = __builtin_amdgcn_exp2f(t[n].m - m);
        t[n].l *= f;
#pragma unroll
        for (int d = 0; d < Dims<D>::blocks; ++d) t[n].o[d] = t[n].o[d] * f;
      }
      t[n].m = m;
    }
    t[n].l += weigh(score[n], a.scale, t[n].m, p[n], low[n]);
  }
#pragma unroll
  for (int d = 0; d < Dims<D>::blocks; ++d) {
    const u32x2 first = lds_column(columns[d]), second = lds_column(columns[d] + 16 * Dims<D>::row);
    const u32x4 v = {first.x, first.y, second.x, second.y};
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
      t[n].o[d] = product16(v, p[n], t[n].o[d]);
      t[n].o[d] = product16(v, low[n], t[n].o[d]);
    }
  }
}

// A wave's slices first + wave, first + wave + 4, ... of a run. WHOLE: pages of whole slices, so a slice lies in one: its
// address is the wave's, and the pages of the next 64 slices are in the lanes of a register.
// Returns whether it is to be done again. AGAIN: slice by slice, with a reference point that follows the largest score.
template <typename T, int D, int TILES, bool WHOLE, bool AGAIN>
__device__ __forceinline__ bool attend_run(Tile<T, D> (&t)[TILES], const Query<D> (&q)[TILES], const Args& a, int b,
                                           int head, int keys, int all_see, int first, int stop, char* lds, int wave,
                                           int lane) {
  constexpr int W = Dims<D>::wide, ahead = kAhead<D, TILES>;
  const int r = lane & 15, h = lane >> 4, begin = first + wave;
  if (begin >= stop) {
#pragma unroll
    for (int i = 0; i < TILES; ++i) start(t[i], q[i]);
    return false;
  }
  const int* table = a.tables + (long long)b * a.blocks;
  const int page_rows = a.kv_heads * a.block_size, head_rows = head * a.block_size;
  lds_ptr columns[Dims<D>::blocks];
#pragma unroll
  for (int d = 0; d < Dims<D>::blocks; ++d)
    columns[d] = in_lds(lds) + place<D>(4 * h + (r >> 2), 2 * d + ((r & 3) >> 1)) + 8 * (r & 1);
  // A lane's part of a row: where the row is shorter than the lanes, the first again (its codes meet zeros of the query,
  // and its values are not written). Loads are issued without a branch, and behind the last slice they load it again:
  // where one path to a wait had fewer of them under way than another, the wait would be for all.
  const auto part = [&](int w) {
    return Dims<D>::shared == 4 * W || 4 * w + h < Dims<D>::shared ? 4 * w + h : 0;
  };
  const int last = begin + (stop - 1 - begin) / kWaves * kWaves;

  int pages = 0;  // WHOLE: lane i's is that of slice fetched + 4 i
  auto fetch = [&](int s) {
    const unsigned t = (unsigned)(s + lane * kWaves) * (unsigned)kKeys;
    pages = table[a.by_block.of(t < (unsigned)keys ? t : 0u)];
    settle(pages);  // waited for here, and not at every slice
  };
  auto load_whole = [&](Slice<D>& x, int s) {
    if (__builtin_expect((unsigned)(s - begin) / kWaves % kWave == 0, 0)) fetch(s);
    const int block = __builtin_amdgcn_readlane(pages, (unsigned)(s - begin) / kWaves % kWave);
    unsigned page = (unsigned)(s * kKeys);
    const int at = a.by_block.take(page);
    const bool there = (unsigned)block < (unsigned)a.pages;
    const long long row = (long long)(there ? block : 0) * page_rows + (head_rows + at);
    const uint8_t *kc = a.k_codes + row * (D / 2), *vc = a.v_codes + row * (D / 2);
    const uint8_t *ks = a.k_scales + row * (D / kShared), *vs = a.v_scales + row * (D / kShared);
    const int left = keys - s * kKeys;
    x.present = !there ? 0u : left >= kKeys ? ~0u : (1u << left) - 1u;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t codes = (uint32_t)((16 * j + r) * (D / 2) + 16 * part(w));
        const uint32_t scales = (uint32_t)((16 * j + r) * (D / kShared) + part(w));
        x.k[j][w] = load16<true>(kc + codes, 0);
        x.v[j][w] = load16<true>(vc + codes, 0);
        x.k_scale[j][w] = ks[scales];
        x.v_scale[j][w] = vs[scales];
      }
  };

  int next[2];
  auto entry = [&](int s, int j) {
    const unsigned t = (unsigned)(s * kKeys + 16 * j + r);
    return table[a.by_block.of(t < (unsigned)keys ? t : 0u)];
  };
  auto load_rows = [&](Slice<D>& x, int s) {
    // the next slice's pages are asked for before this one's keys: loads return in order
    const int now[2] = {next[0], next[1]};
#pragma unroll
    for (int j = 0; j < 2; ++j) next[j] = entry(least(s + kWaves, last), j);
    x.present = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      unsigned page = (unsigned)(s * kKeys + 16 * j + r);
      const bool there = page < (unsigned)keys && (unsigned)now[j] < (unsigned)a.pages;
      const int in_page = a.by_block.take(page);
      const long long row = there ? (long long)now[j] * page_rows + (head_rows + in_page) : 0;
      x.present |= (uint32_t)(__ballot(there) & 0xffffu) << (16 * j);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int c = part(w);
        x.k[j][w] = load16<true>(a.k_codes + row * (D / 2), c);
        x.v[j][w] = load16<true>(a.v_codes + row * (D / 2), c);
        x.k_scale[j][w] = a.k_scales[row * (D / kShared) + c];
        x.v_scale[j][w] = a.v_scales[row * (D / kShared) + c];
      }
    }
  };
  auto load = [&](Slice<D>& x, int s) {
    s = least(s, last);
    if constexpr (WHOLE) load_whole(x, s);
    else load_rows(x, s);
  };
  // what lies behind the last key, and where there is no page, is not read into the result
  auto cut = [&](Slice<D>& x) {
    if (__builtin_expect(x.present == ~0u, 1)) return;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (!(x.present >> (16 * j + r) & 1u)) x.k_scale[j][w] = x.v_scale[j][w] = 0u;
  };

  auto take = [&](Slice<D>& x, int s, auto point) {
    cut(x);
    step<T, D, TILES, decltype(point)::value>(t, x, a, s, all_see, lds, columns, lane);
  };
  using Kept = std::integral_constant<Point, kKept>;
  if constexpr (!WHOLE) {
#pragma unroll
    for (int j = 0; j < 2; ++j) next[j] = entry(begin, j);
  }
  if constexpr (AGAIN) {
#pragma unroll
    for (int i = 0; i < TILES; ++i) start(t[i], q[i]);
    for (int s = begin; s < stop; s += kWaves) {
      Slice<D> x;
      load(x, s);
      take(x, s, std::integral_constant<Point, kFollow>{});
    }
    return false;
  } else {
    Slice<D> x[ahead];
#pragma unroll
    for (int n = 0; n < ahead; ++n) load(x[n], begin + n * kWaves);
#pragma unroll
    for (int i = 0; i < TILES; ++i) start(t[i], q[i]);
    take(x[0], begin, std::integral_constant<Point, kFirst>{});
    load(x[0], begin + ahead * kWaves);
    // slice s + 4 n is in place n + 1
    int s = begin + kWaves;
    for (; s + (ahead - 1) * kWaves < stop; s += ahead * kWaves) {
#pragma unroll
      for (int n = 0; n < ahead; ++n) {
        const int now = s + n * kWaves;
        take(x[(n + 1) % ahead], now, Kept{});
        load(x[(n + 1) % ahead], now + ahead * kWaves);
      }
    }
    // (apart from the loop: left in its middle, it would wait for the last loads at its every turn)
#pragma unroll
    for (int n = 0; n + 1 < ahead; ++n)
      if (s + n * kWaves < stop) take(x[(n + 1) % ahead], s + n * kWaves, Kept{});
    bool wild = false;
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      wild = wild || !(t[i].l < kMostSum);
#pragma unroll
      for (int d = 0; d < Dims<D>::blocks; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) wild = wild || !(fabsf(t[i].o[d][e]) < INFINITY);
    }
    return __ballot(wild) != 0;
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
template <typename T, int D, int TILES, bool WHOLE>
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
      Query<D> q[TILES];
      int row = tile * TILES * kRows + (lane & 15);
#pragma unroll
      for (int i = 0; i < TILES; ++i) find(t[i], q[i], a, b, head, row + i * kRows, keys, lane >> 4);
      const int all_see = keys - a.seq + (int)a.by_group.of((unsigned)(tile * TILES * kRows));  // its first token
      char* mine = lds + wave * Dims<D>::slice;
      if (attend_run<T, D, TILES, WHOLE, false>(t, q, a, b, head, keys, all_see, first, stop, mine, wave, lane)) {
        settle(row);  // the queries' addresses are computed again, and not kept until here
#pragma unroll
        for (int i = 0; i < TILES; ++i) {  // (16 rows at a time: both would take registers that the other form has)
          Tile<T, D>(&one)[1] = reinterpret_cast<Tile<T, D>(&)[1]>(t[i]);
          Query<D>(&its)[1] = reinterpret_cast<Query<D>(&)[1]>(q[i]);
          find(one[0], its[0], a, b, head, row + i * kRows, keys, lane >> 4);
          attend_run<T, D, 1, WHOLE, true>(one, its, a, b, head, keys, all_see, first, stop, mine, wave, lane);
        }
      }
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

// A row's parts: where they are and how many; none where the row sees no key.
struct Parts {
  const float2* stats;
  const float* sums;
  int n;
};
template <int D> __device__ __forceinline__ Parts parts_of(const Args& a, int token, int q_head, int lane) {
  const int b = token / a.seq, s = token % a.seq, head = (int)a.by_group.of((unsigned)q_head);
  const int i = s * a.group + q_head - head * a.group, tile = i / a.tile_rows, row = i % a.tile_rows;
  long long total = 0, before = 0;  // slices of all sequences, of those before this one
  int n = 0, keys = 0;
  for (int first = 0; first < a.batch; first += kWave) {
    const int x = first + lane, k = x < a.batch ? keys_of(a, x) : 0;
    const uint32_t sum = sum_to(slices_of(k), lane);
    if (first <= b && b < first + kWave) {
      keys = __builtin_amdgcn_readlane(k, b - first);
      n = slices_of(keys);
      before = total + sum_of(sum, b - first) - n;
    }
    total += sum_of(sum, kWave - 1);
  }
  if (n == 0 || keys - a.seq + s < 0) return {nullptr, nullptr, 0};
  const long long each = (total + a.runs - 1) / a.runs;
  const int from = (int)(before / each), parts = (int)((before + n - 1) / each) - from + 1;
  const long long at = (((long long)head * a.tiles + tile) * (a.runs + a.batch) + from + b) * a.tile_rows + row;
  return {a.stats + at, a.sums + at * D, parts};
}
// Their largest reference point, and the sum of their weights against it.
__device__ __forceinline__ float2 point_of(const Args& a, const Parts& p, int lane) {
  float m = kNone, l = 0.0f;
  for (int i = lane; i < p.n; i += kWave) m = fmaxf(m, p.stats[(long long)i * a.tile_rows].x);
  m = wave_max(m);
  for (int i = lane; i < p.n; i += kWave) {
    const float2 stat = p.stats[(long long)i * a.tile_rows];
    l += stat.y * __builtin_amdgcn_exp2f(stat.x - m);
  }
  return make_float2(m, wave_sum(l));
}
__device__ __forceinline__ float inverse_of(float l) { return l > 0.0f || l != l ? 1.0f / l : 0.0f; }

// Few parts of a row joined: a wave to a row (a workgroup: heads 4 y ... of token x, and of 2^21 z more).
template <typename T, int D>
__global__ void __launch_bounds__(256) join_few(Args a) {
  constexpr int E = D <= 64 ? 1 : D <= 128 ? 2 : 4;  // elements of a lane
  const int lane = lane_id(), token = (int)(blockIdx.z << rw_host::kGridShift | blockIdx.x);
  const int q_head = (int)blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(wave_id());
  if (q_head >= a.q_heads || token >= a.batch * a.seq) return;
  const Parts p = parts_of<D>(a, token, q_head, lane);
  const float2 point = point_of(a, p, lane);
  float o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
  const bool mine = lane * E < D;
#pragma unroll 4
  for (int i = 0; i < p.n; ++i) {
    const float by = __builtin_amdgcn_exp2f(p.stats[(long long)i * a.tile_rows].x - point.x);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (mine) o[e] += p.sums[(long long)i * a.tile_rows * D + lane * E + e] * by;
  }
  const float by = inverse_of(point.y);
  if (mine) {
    const long long at = (long long)token * a.q_heads + q_head;
#pragma unroll
    for (int e = 0; e < E; ++e) store_elem<T>(a.out, at * D + lane * E + e, o[e] * by);
  }
}

// Many: a workgroup to a row, D / 4 threads to a part, as many parts at a time as there are such teams (64 parts of 32 rows
// 4.4 us, by a wave 8.3; 3 parts of 4620 rows 12 us, by a wave 5.8). Head y of token x, and of 2^21 z more.
template <typename T, int D>
__global__ void __launch_bounds__(256) join_many(Args a) {
  constexpr int team = D / 4, teams = 256 / team;
  __shared__ float4 sums[teams * team];
  const int lane = lane_id(), token = (int)(blockIdx.z << rw_host::kGridShift | blockIdx.x), q_head = (int)blockIdx.y;
  if (token >= a.batch * a.seq) return;
  const int mine = (int)threadIdx.x / team, c = (int)threadIdx.x % team;
  const Parts p = parts_of<D>(a, token, q_head, lane);
  const float2 point = point_of(a, p, lane);
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (mine < teams) {
#pragma unroll 4
    for (int i = mine; i < p.n; i += teams) {
      const float4 x = reinterpret_cast<const float4*>(p.sums + (long long)i * a.tile_rows * D)[c];
      const float by = __builtin_amdgcn_exp2f(p.stats[(long long)i * a.tile_rows].x - point.x);
      o.x += x.x * by, o.y += x.y * by, o.z += x.z * by, o.w += x.w * by;
    }
    sums[mine * team + c] = o;
  }
  __syncthreads();
  if (mine) return;
  for (int i = 1; i < teams; ++i) {
    const float4 x = sums[i * team + c];
    o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
  }
  const float by = inverse_of(point.y);
  *reinterpret_cast<u32x2*>(static_cast<char*>(a.out) + 2 * (((long long)token * a.q_heads + q_head) * D + 4 * c)) =
      (u32x2){pack2<T>(o.x * by, o.y * by), pack2<T>(o.z * by, o.w * by)};
}

// ---- host side ------------------------------------------------------------------------------------------------------

enum { kTuneRuns = 0, kTuneTiles = 1 };
constexpr long long kMostKeys = 1 << 30;  // of a table

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

bool sizes_ok(long long batch, long long seq, int q_heads, int kv_heads, int head_dim, long long blocks,
              long long block_size) {
  const bool dim = head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 192 || head_dim == 256;
  return dim && kv_heads >= 1 && q_heads >= kv_heads && q_heads <= 65536 && q_heads % kv_heads == 0 &&
         block_size >= 1 && block_size <= kMostKeys && kv_heads <= INT_MAX / block_size && blocks >= 0 &&
         blocks <= kMostKeys / block_size && seq <= INT_MAX / 2 / q_heads &&
         batch <= INT_MAX / 2 / (seq * q_heads);
}

Args sized(long long batch, long long seq, int q_heads, int kv_heads, long long blocks, long long block_size) {
  Args a{};
  a.batch = (int)batch, a.seq = (int)seq;
  a.q_heads = q_heads, a.kv_heads = kv_heads, a.group = q_heads / kv_heads;
  a.blocks = (int)blocks, a.block_size = (int)block_size;
  const long long rows = seq * a.group, slots = 2LL * rw_host::device_cus();
  // Tiles of 32 rows read the cache half as often, and are the longer chain: 33 x 5 tokens of 28/4 heads of 64 behind up to
  // 1801 keys 17.6 us in tiles of 16, 22.1 in tiles of 32; 64 x 8 of 32/8 heads of 128 behind 2048 to 8192 127 and 104. So
  // of 16 while all of them are on the CUs at once.
  const int tiles = rw_host::tune_get(kTuneTiles);
  const bool narrow = rows <= kRows || batch * kv_heads * ceil_div(rows, kRows) <= slots;
  a.tile_rows = tiles ? kRows * (tiles == 1 ? 1 : 2) : narrow ? kRows : 2 * kRows;
  a.tiles = (int)ceil_div(rows, a.tile_rows);
  // Runs of a slice to a wave at least. One to a CU where that leaves them no more than 48 slices each (0.6 of a table taken
  // for its keys), else two: one token of 32/8 heads of 128 behind 32768 keys 16.3 us with 32 runs of a kv head, 17.1 with
  // 64; 64 tokens behind 2048 to 8192 86 and 70. A second part's beginning and end and the join take about 9 us, in which a
  // workgroup does 45 slices: a workgroup to a sequence where a table's slices are fewer than a run's and those: 256 tokens
  // behind 1024 to 4096 take 119 us so, with runs 148, 128 behind 2048 to 8192 116 and 130, 33 x 5 of 28/4 heads of 64 behind
  // up to 1801 17.6 and 32, one token behind 32768 195. The longest sequence then bounds the launch, which 0.2 us a slice make
  // dear in wide tables: one of 8192 keys among 127 of up to 500 takes 53 us, with runs 35, one of 32768 198 and 44. So no
  // more than 256 and those 45 (128 behind 4096 to 16384 take 235 us with runs, 223 without), but for batches of so many
  // sequences that their parts would outnumber the runs by far.
  const long long slices = ceil_div(blocks * block_size, kKeys), share = kWaves, all = batch * slices;
  const long long units = (long long)kv_heads * a.tiles, some = batch > 1 ? 5 * all / 8 : all;
  long long most = slots / 2 < units ? 1 : slots / 2 / units;
  if (some > 48 * most) most = slots < units ? 1 : slots / units;
  long long runs = most < ceil_div(all, share) ? most : ceil_div(all, share);
  const long long each = runs ? some / runs : 0;
  if (slices <= (each < share ? share : each) + 45 && (slices <= 256 + 45 || batch > 4 * runs)) runs = 0;
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
  const bool whole = a.block_size % kKeys == 0;
  if (a.tile_rows == kRows) {
    if (whole) hipLaunchKernelGGL((attend<T, D, 1, true>), grid, threads, 0, stream, a);
    else hipLaunchKernelGGL((attend<T, D, 1, false>), grid, threads, 0, stream, a);
  } else {
    if (whole) hipLaunchKernelGGL((attend<T, D, 2, true>), grid, threads, 0, stream, a);
    else hipLaunchKernelGGL((attend<T, D, 2, false>), grid, threads, 0, stream, a);
  }
  const int err = (int)hipGetLastError();
  if (err || a.runs == 0) return err;
  dim3 tokens = rw_host::grid_of((long long)a.batch * a.seq);
  tokens.z = tokens.y, tokens.y = (unsigned)a.q_heads;
  if (a.runs > 8LL * a.batch && a.q_heads <= 65535) {
    hipLaunchKernelGGL((join_many<T, D>), tokens, dim3(256), 0, stream, a);
  } else {
    tokens.y = (unsigned)ceil_div(a.q_heads, 4);
    hipLaunchKernelGGL((join_few<T, D>), tokens, dim3(256), 0, stream, a);
  }
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
  if (pages == 0) a.blocks = 0;  // no keys, and nothing that could be read in their place
  a.by_tiles = divisor(a.tiles), a.by_heads = divisor(kv_heads), a.by_group = divisor(a.group);
  a.by_block = divisor(block_size);
  a.scale = scale * 1.44269504088896341f;
  return dtype == 1 ? launch_type<BF16>(a, head_dim, stream) : launch_type<F16>(a, head_dim, stream);
}

extern "C" int kv4_attention_tune(int slot, int value) { return rw_host::tune_set(slot, value); }
