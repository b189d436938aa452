// Attention over a paged prefix that a batch shares and over each sequence's own paged keys
// (include/shared_prefix_attention.h has the formula).
//
// A query row is one token's one head. The rows that meet the same keys are a matrix: all of the batch's rows of a kv
// head over the prefix, a sequence's rows of a kv head over its own keys. Both are cut into tiles of rows and, over the
// keys, into splits; a workgroup does one (tile, split) and leaves, for each row, the weighted sum of values, the
// running maximum and the sum of the weights; a second launch joins a row's parts.
//
// The products are transposed, so that a lane keeps one row throughout: S^T = K Q^T has a key per matrix row and a query
// per column, its result puts 16 keys of one query into a lane, and these are, packed in pairs, the B operand of O^T =
// V^T P^T without a move between lanes (the order of the 16 keys of a product is free, and V's transposing LDS read
// takes them in the same order). So maximum, sum and rescaling are a lane's own, but for one exchange of the two halves
// of the wave. Softmax in base 2 with the scale folded into the exponent; the reference point moves only when a row's
// maximum has grown by 2^8 (no result depends on it but for rounding, and the sum of values is rescaled only then).
#include <climits>
#include <cmath>
#include <type_traits>

#include "host.hpp"
#include "matrix.hpp"

#pragma clang fp contract(off)

using namespace rw;

namespace {

constexpr int kRows = 32;   // query rows of a wave: the columns of a product
constexpr int kKeys = 32;   // keys of a slice: the rows of a product
constexpr float kGrow = 8.0f;
constexpr int kMix = 7;

// 2^kBias is the weight of a row's reference point: fp16 weights start 2^7 up, so that those down to 2^-21 of the
// largest stay normal numbers; at most 2^(7 + 8).
template <typename T> constexpr float kBias = 0.0f;
template <> constexpr float kBias<F16> = 7.0f;

struct Args {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const int* prefix_table;
  const int* prefix_len;
  const int* block_tables;
  const int* seq_lens;
  float* sums;    // [rows][parts][head_dim]: a part's weighted sum of values
  float2* stats;  // [rows][parts]: its reference point (base 2) and sum of weights
  long long qb, qs, qh;
  int batch, seq, q_heads, kv_heads, group, slots, block_size;
  int prefix_blocks, own_blocks;
  int prefix_splits, own_splits;  // parts of a row: first the prefix's, then its own keys'
  int prefix_tiles, own_tiles;    // row tiles of a kv head: over the batch, of a sequence
  unsigned prefix_groups;         // workgroups over the prefix
  int waves;                      // of a workgroup
  bool wide;                      // the prefix's tiles: 32 rows to each wave, or to the workgroup
  bool near;                      // the caches' bytes are within 32 bits
  int shift;                      // log2 of the page size, or -1
  float scale;                    // times log2(e)
};

__device__ char g_zeros[512] __attribute__((aligned(16)));  // what an absent key's row reads

template <int D> struct Dims {
  static constexpr int chunks = D <= 64 ? 8 : D <= 128 ? 16 : 32;  // 16-byte places of a row in LDS
  static constexpr int used = D / 8;                               // of these hold the row
  static constexpr int row = chunks * 16;
  static constexpr int slice = kKeys * row;                        // bytes of a slice of K or V
  static constexpr int steps = D / 16;                             // products of a slice's scores
  static constexpr int blocks = (D + 31) / 32;                     // 32-wide blocks of the values
};

// How many keys a table holds (at most 2^30), and each split's run of 32-key slices: as even as it gets in whole pairs,
// but not below four slices (one per wave).
__device__ __forceinline__ int keys_of(int len, int blocks, int block_size) {
  const int most = blocks * block_size;
  return len < 0 ? 0 : len < most ? len : most;
}
__device__ __forceinline__ int slices_of(int keys) { return (keys + kKeys - 1) / kKeys; }
__device__ __forceinline__ int slices_per_split(int keys, int splits) {
  const int per = ((slices_of(keys) + splits - 1) / splits + 1) & ~1;
  return per < 4 ? 4 : per;
}

// A wave's rows: per lane (its column's row) the place of the row in the outputs, or -1; the last own key it sees.
struct Row {
  int at;
  int limit;
};

// 32 rows of a wave.
template <typename T, int D>
struct Tile {
  u32x4 q[Dims<D>::steps];
  f32x16 o[Dims<D>::blocks];
  float m, l;  // reference point; sum of weights over this lane's half of the keys
};
constexpr float kNone = -3.0e38f;  // the reference point of a row that has met no key

template <typename T, int D>
__device__ __forceinline__ void start_tile(Tile<T, D>& t, const Args& a, const Row& row, int lane) {
  const int h = lane >> 5;
  const char* p = nullptr;
  if (row.at >= 0) {
    const int token = row.at / a.q_heads, head = row.at - token * a.q_heads, b = token / a.seq, s = token - b * a.seq;
    p = static_cast<const char*>(a.q) + 2 * (b * a.qb + s * a.qs + head * a.qh);
  }
#pragma unroll
  for (int c = 0; c < Dims<D>::steps; ++c) {
    t.q[c] = (u32x4){0u, 0u, 0u, 0u};
    if (p) t.q[c] = load16<false>(p, 2 * c + h);
  }
#pragma unroll
  for (int d = 0; d < Dims<D>::blocks; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) t.o[d][i] = 0.0f;
  t.m = kNone;
  t.l = 0.0f;
}

// Where chunk c of row r of a slice lies: XORed with the row, so that the lanes of a read (8 rows' same chunk for K, 4
// rows' same pair of chunks for V) meet different banks.
template <int D> __device__ __forceinline__ int k_place(int r, int c) {
  return r * Dims<D>::row + ((c ^ r) & (Dims<D>::chunks - 1)) * 16;
}
template <int D> __device__ __forceinline__ int v_place(int r, int c) {
  return r * Dims<D>::row + ((c ^ (2 * r)) & (Dims<D>::chunks - 1)) * 16;
}

// A slice's keys from LDS as the scores' left operands.
template <int D>
__device__ __forceinline__ void read_keys(u32x4* kf, const char* k, int lane) {
#pragma unroll
  for (int c = 0; c < Dims<D>::steps; ++c)
    kf[c] = *reinterpret_cast<const u32x4*>(k + k_place<D>(lane & 31, 2 * c + (lane >> 5)));
}

// The scores of a slice of 32 keys, 16 of them in each lane.
template <typename T, int D>
__device__ __forceinline__ f32x16 scores(const Tile<T, D>& t, const u32x4* kf) {
  f32x16 s;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
  for (int c = 0; c < Dims<D>::steps; ++c) s = product32<T>(kf[c], t.q[c], s);
  return s;
}

// -inf for the keys that are absent (`present` has a bit per key) or past the row's limit (counted from the slice).
__device__ __forceinline__ void hide(f32x16& s, uint32_t present, int limit, int lane) {
  const int h = 4 * (lane >> 5);  // taken off here, so that what is left of a key's number is a constant
  present >>= h;
  limit -= h;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int key = 8 * (i / 4) + i % 4;
    if (!(present & (1u << key)) || key > limit) s[i] = -INFINITY;
  }
}

// The scores of N slices to weights in pairs. Returns what the row's sum of values so far is to be multiplied by.
template <typename T, int D, int N>
__device__ __forceinline__ float soften(Tile<T, D>& t, const f32x16* s, float scale, u32x4* p) {
  float top = s[0][0];
#pragma unroll
  for (int i = 1; i < 16 * N; ++i) top = fmaxf(top, s[i / 16][i % 16]);
  top = max_of_halves(top) * scale - kBias<T>;
  const float m = top > t.m + kGrow ? top : t.m, f = __builtin_amdgcn_exp2f(t.m - m);
  t.m = m;
  t.l *= f;
#pragma unroll
  for (int i = 0; i < 8 * N; ++i) {
    const float x = s[i / 8][2 * i % 16], y = s[i / 8][2 * i % 16 + 1];
    const uint32_t two = pack2<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(x, scale, -m)),
                                  __builtin_amdgcn_exp2f(__builtin_fmaf(y, scale, -m)));
    t.l = add_pair<T>(two, t.l);
    p[i / 4][i % 4] = two;
  }
  return f;
}

template <typename T, int D>
__device__ __forceinline__ void rescale(Tile<T, D>& t, float f) {
  if (__ballot(f != 1.0f) == 0) return;
#pragma unroll
  for (int d = 0; d < Dims<D>::blocks; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) t.o[d][i] *= f;
}

// Which values the 16 rows n (0 or 1) of block d of the sums are: for 128 values and more the two are half the row apart,
// so that the 32 lanes of a read meet all banks (with neighbours they met half of them twice).
template <int D> __device__ __forceinline__ int value_of(int d, int n) {
  return D % 128 == 0 ? 16 * d + D / 2 * n : 32 * d + 16 * n;
}

// A slice's values from LDS, transposed, as the left operands of the weighted sums: keys 16 j ..., block d.
template <int D>
__device__ __forceinline__ void read_values(u32x4* vf, char* v, int lane) {
  const int i16 = lane & 15, n = (lane >> 4) & 1;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int d = 0; d < Dims<D>::blocks; ++d) {
      const int chunk = value_of<D>(d, n) / 8 + ((i16 & 3) >> 1), at = 16 * j + 4 * (lane >> 5) + (i16 >> 2);
      const u32x2 lo = lds_column(v + v_place<D>(at, chunk) + 8 * (lane & 1));
      const u32x2 hi = lds_column(v + v_place<D>(at + 8, chunk) + 8 * (lane & 1));
      vf[j * Dims<D>::blocks + d] = (u32x4){lo.x, lo.y, hi.x, hi.y};
    }
}

template <typename T, int D>
__device__ __forceinline__ void add_values(Tile<T, D>& t, const u32x4* p, const u32x4* vf) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int d = 0; d < Dims<D>::blocks; ++d) t.o[d] = product32<T>(vf[j * Dims<D>::blocks + d], p[j], t.o[d]);
}

// The slot of key t of a table, or -1.
__device__ __forceinline__ int slot_of(const int* table, int t, int keys, const Args& a) {
  if (t >= keys) return -1;
  const unsigned page = a.shift >= 0 ? (unsigned)t >> a.shift : (unsigned)t / (unsigned)a.block_size;
  const long long slot = (long long)table[page] * a.block_size + (int)((unsigned)t - page * (unsigned)a.block_size);
  return slot >= 0 && slot < a.slots ? (int)slot : -1;
}

// Starts the loads of ROWS rows of K or V (`base`: the kv head's first row; K's or V's order of chunks) from row r0 on
// (lane l holds the slot of row l) into LDS at `to`, row r0's place. `plain`: no row is absent, and all are within 32 bits.
template <int D, int ROWS, bool KEYS>
__device__ __forceinline__ void load_rows(const Args& a, const char* base, int slot, bool plain, int r0, char* to,
                                          int lane) {
  constexpr int C = Dims<D>::chunks, rows = kWave / C;
  const uint32_t row_bytes = (uint32_t)(2 * D) * (uint32_t)a.kv_heads;
#pragma unroll
  for (int i = 0; i < ROWS / rows; ++i) {
    const int r = r0 + i * rows + lane / C, place = lane & (C - 1);
    const int c = (place ^ (KEYS ? r : 2 * r)) & (C - 1);
    const int at = from_lane(slot, r);
    const bool mine = Dims<D>::used == C || c < Dims<D>::used;
    char* dst = to + i * kWave * 16;
    if (plain) {
      load_to_lds(base, (uint32_t)at * row_bytes + 16u * c, dst, mine);
    } else {
      load_to_lds((at < 0 ? g_zeros : base + (long long)at * row_bytes) + 16 * c, dst, mine);
    }
  }
}

// Where lane (r, h)'s four sums i of block d start among the values.
template <int D> __device__ __forceinline__ int sums_at(int d, int i, int h) {
  return value_of<D>(d, i / 2) + 8 * (i % 2) + 4 * h;
}

// The waves' tiles over the same rows joined through LDS (each wave's own 2 slices of it), and the part, or the result
// where it is the only one, written.
template <typename T, int D, int WAVES>
__device__ __forceinline__ void finish(Tile<T, D>& t, const Args& a, const Row& row, int part, int parts, char* lds,
                                       float2* stats, int wave, int lane) {
  constexpr int B = Dims<D>::blocks, per_row = 2 * WAVES;  // lanes
  static_assert(kRows * 32 * B * 4 <= 2 * Dims<D>::slice, "a tile's sums fit its wave's slices");
  t.l = sum_of_halves(t.l);
  if (lane < 32) stats[wave * kRows + lane] = make_float2(t.m, t.l);
  __syncthreads();
  const int r = lane & 31, h = lane >> 5;
  float m = kNone, l = 0.0f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) m = fmaxf(m, stats[w * kRows + r].x);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const float2 s = stats[w * kRows + r];
    l += s.y * __builtin_amdgcn_exp2f(s.x - m);
  }
  const float f = __builtin_amdgcn_exp2f(t.m - m);
  // the wave's sums, row r's 4 values from d on at chunk d / 4, XORed with the row
  float4* mine = reinterpret_cast<float4*>(lds + wave * 2 * Dims<D>::slice);
#pragma unroll
  for (int d = 0; d < B; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = sums_at<D>(d, i, h) / 4;
      mine[r * 8 * B + (c ^ (r & 7))] = make_float4(t.o[d][4 * i] * f, t.o[d][4 * i + 1] * f, t.o[d][4 * i + 2] * f,
                                                    t.o[d][4 * i + 3] * f);
    }
  __syncthreads();
  const int mr = (wave * kWave + lane) / per_row;
  const long long at = from_lane(row.at, mr);
  const float rl = __builtin_bit_cast(float, from_lane(__builtin_bit_cast(int, l), mr));
  const float rm = __builtin_bit_cast(float, from_lane(__builtin_bit_cast(int, m), mr));
  if (at < 0) return;
  const float inverse = rl > 0.0f || rl != rl ? 1.0f / rl : 0.0f;
#pragma unroll
  for (int c = lane % per_row; c < D / 4; c += per_row) {
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float4 y = reinterpret_cast<const float4*>(lds + w * 2 * Dims<D>::slice)[mr * 8 * B + (c ^ (mr & 7))];
      x[0] += y.x, x[1] += y.y, x[2] += y.z, x[3] += y.w;
    }
    if (parts == 1) {
      *reinterpret_cast<u32x2*>(static_cast<char*>(a.out) + 2 * (at * D + 4 * c)) =
          (u32x2){pack2<T>(x[0] * inverse, x[1] * inverse), pack2<T>(x[2] * inverse, x[3] * inverse)};
    } else {
      *reinterpret_cast<float4*>(a.sums + (at * parts + part) * D + 4 * c) = make_float4(x[0], x[1], x[2], x[3]);
    }
  }
  if (parts > 1 && lane % per_row == 0) a.stats[at * parts + part] = make_float2(rm, rl);
}

// One split over 256 rows: 8 waves with 32 of their own, and the keys in pairs of slices that all share, kRing pairs of K
// and of V in LDS. A wave goes from pair to pair in two phases:
//   products: pair n's scores and pair n - 1's values, a slice's operands read from LDS under the products before them;
//   weights: pair n's weights, and the loads to LDS of K's pair n + kRing - 1 and V's pair n + kRing - 2.
// Four waves are in the one phase while the other four, on the same SIMDs, are in the other (a barrier stands between
// phases), so that matrix cores and vector units work at the same time: 32 products take 1024 cycles with 128 values, and
// the weights of 64 keys about as many. (Slice by slice, with twice the phases, the barriers and the chain from the scores
// to the first exponential took a third of the time.)
//
// In weights phase n, the first four waves may not overwrite what the others read in products phase n at the same time
// (K's pair n, V's n - 1), so the places of K's pair n - 1 and V's n - 2 are filled. At its end all loads but its own
// have to be there; they are read one to one and a half pairs later. The page of a key comes to LDS the same way, so that
// no wave ever waits for a single load.
constexpr int kRing = 4;

template <typename T, int D>
__device__ __forceinline__ void attend_wide(const Args& a, const int* table, int keys, int split, int splits, int part,
                                            int kv_head, const Row& row, char* lds, int wave, int lane) {
  constexpr int slice = Dims<D>::slice, pair = 2 * slice, C = Dims<D>::chunks, rows = kWave / C;
  constexpr int loads = 64 / rows / 8;  // of a wave, of K's pair; row r of the pair is at r * row in LDS
  const int parts = a.prefix_splits + a.own_splits;
  const int per = slices_per_split(keys, splits), from = split * per;
  const int n = (least(per, slices_of(keys) - from) + 1) / 2;  // pairs
  char* kt = lds;
  char* vt = lds + kRing * pair;
  char* pages = lds + 2 * kRing * pair + wave * kRing * (kWave * 4);  // this wave's
  const char* kb = static_cast<const char*>(a.k) + 2 * kv_head * D;
  const char* vb = static_cast<const char*>(a.v) + 2 * kv_head * D;
  const uint32_t row_bytes = (uint32_t)(2 * D) * (uint32_t)a.kv_heads;
  const int key = from * kKeys + lane;  // this lane's key of the first pair
  const int end = least(keys, from * kKeys + n * 64);
  // this lane's row of a load and its place in it, the same in each of the wave's loads
  const int r0 = wave * rows + lane / C, place = lane & (C - 1);
  const uint32_t ck = 16u * ((place ^ r0) & (C - 1)), cv = 16u * ((place ^ (2 * r0)) & (C - 1));
  const bool kmine = Dims<D>::used == C || ck < 2 * D, vmine = Dims<D>::used == C || cv < 2 * D;

  auto page_of = [&](int t) { return a.shift >= 0 ? (unsigned)t >> a.shift : (unsigned)t / (unsigned)a.block_size; };
  auto load_page = [&](int i, char* to) {
    const int t = key + i * 64;
    load_word_to_lds(table + page_of(t < end ? t : 0), to);
  };
  auto slot_from = [&](int entry, int t) {
    const long long slot = (long long)entry * a.block_size + (int)((unsigned)t - page_of(t) * (unsigned)a.block_size);
    return t < end && slot >= 0 && slot < a.slots ? (int)slot : -1;
  };
  struct Slots {
    int of[loads];   // of this lane's rows
    uint64_t there;  // the pair's keys that are there
  };
  auto rows_of = [&](int slot) {
    Slots s;
#pragma unroll
    for (int x = 0; x < loads; ++x) s.of[x] = from_lane(slot, r0 + x * 8 * rows);
    s.there = __ballot(slot >= 0);
    return s;
  };
  auto load = [&](const char* base, const Slots& s, uint32_t c, bool mine, char* to) {
    to += wave * kWave * 16;
    if (a.near && s.there == ~0ull) {
#pragma unroll
      for (int x = 0; x < loads; ++x)
        load_to_lds(base, (uint32_t)s.of[x] * row_bytes + c, to + x * 8 * kWave * 16, mine);
    } else {
#pragma unroll
      for (int x = 0; x < loads; ++x)
        load_to_lds((s.of[x] < 0 ? g_zeros : base + (long long)s.of[x] * row_bytes) + c, to + x * 8 * kWave * 16, mine);
    }
  };

  Tile<T, D> t;
  Slots last;             // of pair n + kRing - 2 at weights phase n
  uint64_t there[kRing];  // the keys that are there, by the pair's place
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) {
    const int x = key + i * 64;
    last = rows_of(x < end ? slot_from(table[page_of(x)], x) : -1);
    there[i] = last.there;
    load(kb, last, ck, kmine, kt + i * pair);
    if (i < kRing - 2) load(vb, last, cv, vmine, vt + i * pair);
  }
  load_page(kRing - 1, pages + (kRing - 1) * (kWave * 4));
  load_page(kRing, pages);
  start_tile<T, D>(t, a, row, lane);
  u32x4 kf[Dims<D>::steps], p[4];
  f32x16 s[2];
  wait_loads();
  meet();
  read_keys<D>(kf, kt, lane);
  wait_lds();
  if (wave >= 4) meet();
  // what the products of pair i, in place i % kRing, share: its scores
  auto score = [&](auto where) {
    u32x4 more[Dims<D>::steps];
    read_keys<D>(more, kt + decltype(where)::value * pair + slice, lane);
    s[0] = scores<T, D>(t, kf);
    keep_order();
    s[1] = scores<T, D>(t, more);
  };
  auto weigh = [&](int i, auto where) {
    constexpr int here = decltype(where)::value, after = (here + 1) % kRing;
    constexpr int before = (here + kRing - 1) % kRing, two_before = (here + kRing - 2) % kRing;
    const int entry = *reinterpret_cast<const int*>(pages + before * (kWave * 4) + 4 * lane);
    read_keys<D>(kf, kt + after * pair, lane);
    const Slots next = rows_of(slot_from(entry, key + (i + kRing - 1) * 64));
    load(kb, next, ck, kmine, kt + before * pair);
    load(vb, last, cv, vmine, vt + two_before * pair);
    load_page(i + kRing + 1, pages + after * (kWave * 4));
    last = next;
    there[before] = next.there;
    if (there[here] != ~0ull) {
      hide(s[0], (uint32_t)there[here], INT_MAX, lane);
      hide(s[1], (uint32_t)(there[here] >> 32), INT_MAX, lane);
    }
    rescale<T, D>(t, soften<T, D, 2>(t, s, a.scale, p));
    wait_lds();
    wait_loads<2 * loads + 1>();
    meet();
  };
  auto step = [&](int i, auto where) {
    constexpr int before = (decltype(where)::value + kRing - 1) % kRing;
    u32x4 more[Dims<D>::steps], vf[2 * Dims<D>::blocks], vg[2 * Dims<D>::blocks];
    read_keys<D>(more, kt + decltype(where)::value * pair + slice, lane);
    s[0] = scores<T, D>(t, kf);
    keep_order();
    read_values<D>(vf, vt + before * pair, lane);
    s[1] = scores<T, D>(t, more);
    keep_order();
    read_values<D>(vg, vt + before * pair + slice, lane);
    add_values<T, D>(t, p, vf);
    keep_order();
    add_values<T, D>(t, p + 2, vg);
    meet();
    weigh(i, where);
  };
  score(std::integral_constant<int, 0>{});
  meet();
  weigh(0, std::integral_constant<int, 0>{});
  for (int i = 1; i < n;) {
    step(i++, std::integral_constant<int, 1>{});
    if (i < n) step(i++, std::integral_constant<int, 2>{});
    if (i < n) step(i++, std::integral_constant<int, 3>{});
    if (i < n) step(i++, std::integral_constant<int, 0>{});
  }
  if (wave < 4) meet();
  {
    u32x4 vf[2 * Dims<D>::blocks];
    char* v = vt + ((n - 1) & (kRing - 1)) * pair;
    read_values<D>(vf, v, lane);
    add_values<T, D>(t, p, vf);
    read_values<D>(vf, v + slice, lane);
    add_values<T, D>(t, p + 2, vf);
  }
  wait_loads();  // none may arrive after the workgroup has gone
  const float l = sum_of_halves(t.l);
  if (row.at < 0) return;
  const long long at = (long long)row.at * parts + part;
  const int h = lane >> 5;
#pragma unroll
  for (int d = 0; d < Dims<D>::blocks; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = sums_at<D>(d, e, h);
      if (c < D)
        *reinterpret_cast<float4*>(a.sums + at * D + c) =
            make_float4(t.o[d][4 * e], t.o[d][4 * e + 1], t.o[d][4 * e + 2], t.o[d][4 * e + 3]);
    }
  if (h == 0) a.stats[at] = make_float2(t.m, l);
}

// One (tile, split). WIDE: the prefix by 256 rows, else by 32. A sequence's own keys always by 32 rows: the waves take
// a split's slices in turn, each through LDS of its own, without barriers.
template <typename T, int D, int WAVES, bool WIDE>
__global__ void __launch_bounds__(WAVES* kWave, D <= 128 ? 2 : 1) attend(Args a) {
  constexpr int narrow = WAVES * 2 * Dims<D>::slice, wide = 4 * kRing * Dims<D>::slice + WAVES * kRing * kWave * 4;
  __shared__ __align__(16) char lds[WIDE && wide > narrow ? wide : narrow];
  __shared__ float2 stats[WAVES * kRows];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  const int parts = a.prefix_splits + a.own_splits;
  const unsigned shared = a.prefix_groups;
  Row row{-1, INT_MAX};
  int part, kv_head, keys, end, splits, split;
  const int* table;
  if (blockIdx.x < shared) {  // the prefix: rows of the whole batch
    // the tiles of one (kv head, split) read the same keys: all to one XCD (workgroups go round the 8 in turn), so that
    // its L2 has them for all
    const unsigned turn = blockIdx.x / 8u, tile = turn % (unsigned)a.prefix_tiles;
    const unsigned u = turn / (unsigned)a.prefix_tiles * 8u + blockIdx.x % 8u;
    if (u >= (unsigned)(a.kv_heads * a.prefix_splits)) return;
    split = (int)(u % (unsigned)a.prefix_splits);
    kv_head = (int)(u / (unsigned)a.prefix_splits);
    part = split;
    splits = a.prefix_splits;
    table = a.prefix_table;
    keys = keys_of(a.prefix_len[0], a.prefix_blocks, a.block_size);
    end = keys;
    auto place = [&](int x) {
      const int token = x / a.group;
      return token < a.batch * a.seq ? token * a.q_heads + kv_head * a.group + x % a.group : -1;
    };
    if constexpr (WIDE) {
      if (split * slices_per_split(keys, splits) >= slices_of(keys)) return;
      row.at = place(((int)tile * WAVES + wave) * kRows + (lane & 31));
      attend_wide<T, D>(a, table, keys, split, splits, part, kv_head, row, lds, wave, lane);
      return;
    }
    row.at = place((int)tile * kRows + (lane & 31));
  } else {  // a sequence's own keys: its rows
    unsigned u = blockIdx.x - shared;
    const int tile = (int)(u % (unsigned)a.own_tiles);
    u /= (unsigned)a.own_tiles;
    split = (int)(u % (unsigned)a.own_splits);
    u /= (unsigned)a.own_splits;
    kv_head = (int)(u % (unsigned)a.kv_heads);
    const int b = (int)(u / (unsigned)a.kv_heads);
    part = a.prefix_splits + split;
    splits = a.own_splits;
    keys = keys_of(a.seq_lens[b], a.own_blocks, a.block_size);
    const int x = tile * kRows + (lane & 31), i = x / a.group;
    if (i < a.seq) {
      row.at = (b * a.seq + i) * a.q_heads + kv_head * a.group + x % a.group;
      row.limit = keys - a.seq + i;
    }
    table = a.block_tables + (long long)b * a.own_blocks;
    const int last = least((tile * kRows + kRows - 1) / a.group, a.seq - 1);  // the tile's last token sees the most keys
    end = keys - a.seq + 1 + last;
    end = end < 0 ? 0 : end;
  }
  const int per = slices_per_split(keys, splits);
  if (split * per >= slices_of(keys) && parts > 1) return;
  const int stop = least(split * per + per, slices_of(end));

  Tile<T, D> t;
  start_tile<T, D>(t, a, row, lane);
  char* k = lds + wave * 2 * Dims<D>::slice;
  char* v = k + Dims<D>::slice;
  const char* kb = static_cast<const char*>(a.k) + 2 * kv_head * D;
  const char* vb = static_cast<const char*>(a.v) + 2 * kv_head * D;
  int s = split * per + wave;
  int slot = s < stop ? slot_of(table, s * kKeys + (lane & 31), keys, a) : -1;
  for (; s < stop; s += WAVES) {
    const uint32_t present = (uint32_t)__ballot(slot >= 0);
    const bool plain = a.near && present == 0xffffffffu;
    wait_lds();  // the slice before has been read
    load_rows<D, kKeys, true>(a, kb, slot, plain, 0, k, lane);
    load_rows<D, kKeys, false>(a, vb, slot, plain, 0, v, lane);
    slot = s + WAVES < stop ? slot_of(table, (s + WAVES) * kKeys + (lane & 31), keys, a) : -1;
    wait_loads();
    u32x4 kf[Dims<D>::steps], vf[2 * Dims<D>::blocks];
    read_keys<D>(kf, k, lane);
    f32x16 x = scores<T, D>(t, kf);
    read_values<D>(vf, v, lane);
    const int first = s * kKeys;
    if (present != 0xffffffffu || __ballot(first + kKeys - 1 > row.limit && row.at >= 0))
      hide(x, present, row.limit - first, lane);
    u32x4 p[2];
    rescale<T, D>(t, soften<T, D, 1>(t, &x, a.scale, p));
    add_values<T, D>(t, p, vf);
  }
  __syncthreads();  // finish() reuses the waves' LDS
  finish<T, D, WAVES>(t, a, row, part, parts, lds, stats, wave, lane);
}

// A row's parts joined: a wave per row.
template <typename T, int D>
__global__ void __launch_bounds__(256) join(Args a) {
  constexpr int E = D <= 64 ? 1 : D <= 128 ? 2 : 4;  // values per lane
  const int lane = lane_id();
  const long long at = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(wave_id());
  if (at >= (long long)a.batch * a.seq * a.q_heads) return;
  const int token = (int)at / a.q_heads, b = token / a.seq;
  const int own = keys_of(a.seq_lens[b], a.own_blocks, a.block_size);
  const int parts = a.prefix_splits + a.own_splits;
  float o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
  float total = 0.0f;
  if (own - a.seq + (token - b * a.seq) >= 0) {
    const int prefix = a.prefix_splits ? keys_of(a.prefix_len[0], a.prefix_blocks, a.block_size) : 0;
    // the parts that have been written: those whose split has slices
    auto written = [&](int p) {
      const bool shared = p < a.prefix_splits;
      const int keys = shared ? prefix : own, split = shared ? p : p - a.prefix_splits;
      return p < parts &&
             split * slices_per_split(keys, shared ? a.prefix_splits : a.own_splits) < slices_of(keys);
    };
    float m = kNone;
    for (int p = lane; p < parts; p += kWave)
      if (written(p)) m = fmaxf(m, a.stats[at * parts + p].x);
    m = wave_max(m);
    for (int p0 = 0; p0 < parts; p0 += kWave) {
      float w = 0.0f, l = 0.0f;
      if (written(p0 + lane)) {
        const float2 s = a.stats[at * parts + p0 + lane];
        w = __builtin_amdgcn_exp2f(s.x - m);
        l = s.y * w;
      }
      total += wave_sum(l);
      for (uint64_t left = __ballot(w != 0.0f); left; left &= left - 1) {  // NaN is not zero
        const int p = __builtin_ctzll(left);
        const float f = readlane(w, p);
        const float* x = a.sums + (at * parts + p0 + p) * D + lane * E;
        if (lane * E < D) {
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += x[e] * f;
        }
      }
    }
  }
  const float inverse = total > 0.0f || total != total ? 1.0f / total : 0.0f;
  if (lane * E < D) {
#pragma unroll
    for (int e = 0; e < E; ++e) store_elem<T>(a.out, at * D + lane * E + e, o[e] * inverse);
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------

enum { kTunePrefix = 0, kTuneOwn = 1, kTuneWide = 2 };
constexpr long long kMostKeys = 1 << 30;  // of a table

bool sizes_ok(long long batch, long long seq, int q_heads, int kv_heads, int head_dim, long long prefix_blocks,
              long long own_blocks, long long block_size) {
  const bool dim = head_dim == 64 || head_dim == 80 || head_dim == 96 || head_dim == 128 || head_dim == 192 ||
                   head_dim == 256;
  return dim && kv_heads >= 1 && q_heads >= kv_heads && q_heads <= 65536 && q_heads % kv_heads == 0 &&
         block_size >= 1 && block_size <= kMostKeys && prefix_blocks >= 0 && prefix_blocks <= kMostKeys / block_size &&
         own_blocks >= 0 && own_blocks <= kMostKeys / block_size && seq <= INT_MAX / 2 / q_heads &&
         batch <= INT_MAX / 2 / (seq * q_heads);
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// The splits: as many as leave each workgroup some slices and the grid some workgroups per CU.
void plan(Args& a, int head_dim) {
  const long long fill = 4LL * rw_host::device_cus();
  auto splits = [&](long long keys, long long tiles, int tuned) -> int {
    if (keys <= 0) return 0;
    const long long most = ceil_div(ceil_div(keys, kKeys), 8);
    long long n = tuned > 0 ? tuned : ceil_div(fill, tiles);
    if (n > most) n = most;
    return (int)(n > 256 ? 256 : n < 1 ? 1 : n);
  };
  const long long rows = (long long)a.batch * a.seq * a.group;
  const int tuned = rw_host::tune_get(kTuneWide);
  a.wide = head_dim <= 128 && (tuned > 0 ? tuned > 1 : rows > 64);
  a.waves = a.wide ? 8 : 4;
  a.prefix_tiles = (int)ceil_div(rows, a.wide ? a.waves * kRows : kRows);
  a.own_tiles = (int)ceil_div((long long)a.seq * a.group, kRows);
  a.prefix_splits = splits((long long)a.prefix_blocks * a.block_size, (long long)a.prefix_tiles * a.kv_heads,
                           rw_host::tune_get(kTunePrefix));
  a.own_splits = splits((long long)a.own_blocks * a.block_size, (long long)a.own_tiles * a.kv_heads * a.batch,
                        rw_host::tune_get(kTuneOwn));
}

long long work_bytes(const Args& a, int head_dim) {
  const long long parts = a.prefix_splits + a.own_splits;
  return parts == 0 || (parts == 1 && a.own_splits) ? 0 : (long long)a.batch * a.seq * a.q_heads * parts * (4LL * head_dim + 8);
}

Args sized(long long batch, long long seq, int q_heads, int kv_heads, int head_dim, long long prefix_blocks,
           long long own_blocks, long long block_size) {
  Args a{};
  a.batch = (int)batch;
  a.seq = (int)seq;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.group = q_heads / kv_heads;
  a.block_size = (int)block_size;
  a.prefix_blocks = (int)prefix_blocks;
  a.own_blocks = (int)own_blocks;
  plan(a, head_dim);
  return a;
}

template <typename T, int D>
int launch_dim(Args a, hipStream_t stream) {
  const long long rows = (long long)a.batch * a.seq * a.q_heads;
  const long long shared = ceil_div((long long)a.kv_heads * a.prefix_splits, 8) * 8 * a.prefix_tiles;
  const long long own = (long long)a.batch * a.kv_heads * a.own_splits * a.own_tiles;
  if (shared + own > INT_MAX) return rw_host::kInvalid;
  a.prefix_groups = (unsigned)shared;
  const dim3 grid((unsigned)(shared + own)), threads(a.waves * kWave);
  if (shared + own) {
    if constexpr (D <= 128) {
      if (a.wide) hipLaunchKernelGGL((attend<T, D, 8, true>), grid, threads, 0, stream, a);
    }
    if (!a.wide) hipLaunchKernelGGL((attend<T, D, 4, false>), grid, threads, 0, stream, a);
  }
  const int err = (int)hipGetLastError();
  if (err || (a.prefix_splits == 0 && a.own_splits == 1)) return err;  // the only part is the result
  hipLaunchKernelGGL((join<T, D>), dim3((unsigned)ceil_div(rows, 4)), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

template <typename T>
int launch_type(const Args& a, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 64: return launch_dim<T, 64>(a, stream);
    case 80: return launch_dim<T, 80>(a, stream);
    case 96: return launch_dim<T, 96>(a, stream);
    case 128: return launch_dim<T, 128>(a, stream);
    case 192: return launch_dim<T, 192>(a, stream);
    default: return launch_dim<T, 256>(a, stream);
  }
}

}  // namespace

extern "C" long long prefix_attention_work(long long batch, long long seq, int q_heads, int kv_heads, int head_dim,
                                           long long prefix_blocks, long long own_blocks, long long block_size) {
  if (batch <= 0 || seq <= 0) return 0;
  if (!sizes_ok(batch, seq, q_heads, kv_heads, head_dim, prefix_blocks, own_blocks, block_size)) return -1;
  return work_bytes(sized(batch, seq, q_heads, kv_heads, head_dim, prefix_blocks, own_blocks, block_size), head_dim);
}

extern "C" int prefix_attention_launch(const void* q, const void* k_cache, const void* v_cache,
                                       const void* prefix_table, const void* prefix_len, const void* block_tables,
                                       const void* seq_lens, void* out, void* work, const long long* strides,
                                       long long batch, long long seq, long long slots, int q_heads, int kv_heads,
                                       int head_dim, long long prefix_blocks, long long own_blocks,
                                       long long block_size, float scale, int dtype, hipStream_t stream) {
  using rw_host::aligned16;
  if (batch <= 0 || seq <= 0) return rw_host::kOk;
  if (!sizes_ok(batch, seq, q_heads, kv_heads, head_dim, prefix_blocks, own_blocks, block_size) || slots < 0 ||
      slots > INT_MAX || (dtype != 1 && dtype != 2) || !q || !aligned16(q) || !out || !aligned16(out) || !seq_lens ||
      (slots && (!k_cache || !v_cache)) || !aligned16(k_cache) || !aligned16(v_cache) ||
      (prefix_blocks && (!prefix_table || !prefix_len)) || (own_blocks && !block_tables) || !(scale >= 1.0e-30f && scale <= 1.0e30f))
    return rw_host::kInvalid;
  Args a = sized(batch, seq, q_heads, kv_heads, head_dim, prefix_blocks, own_blocks, block_size);
  if (work_bytes(a, head_dim) && (!work || !aligned16(work))) return rw_host::kInvalid;
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.out = out;
  a.prefix_table = (const int*)prefix_table;
  a.prefix_len = (const int*)prefix_len;
  a.block_tables = (const int*)block_tables;
  a.seq_lens = (const int*)seq_lens;
  a.sums = (float*)work;
  a.stats = (float2*)((char*)work + (long long)a.batch * a.seq * q_heads * (a.prefix_splits + a.own_splits) * 4 *
                                        head_dim);
  a.qh = head_dim;
  a.qs = (long long)q_heads * head_dim;
  a.qb = seq * a.qs;
  if (strides) a.qb = strides[0], a.qs = strides[1], a.qh = strides[2];
  if (a.qb % 8 || a.qs % 8 || a.qh % 8) return rw_host::kInvalid;
  a.slots = (int)slots;
  a.near = slots * kv_heads * head_dim * 2 < (1LL << 32);
  a.shift = (block_size & (block_size - 1)) ? -1 : __builtin_ctzll(block_size);
  a.scale = scale * 1.44269504088896341f;
  return dtype == 1 ? launch_type<BF16>(a, head_dim, stream) : launch_type<F16>(a, head_dim, stream);
}

extern "C" int prefix_attention_tune(int slot, int value) { return rw_host::tune_set(slot, value); }
