// Attention over a paged prefix that a batch shares and over each sequence's own paged keys
// (include/shared_prefix_attention.h has the formula).
//
// A query row is one token's one head. The rows that meet the same keys are a matrix: all of the batch's rows of a kv
// head over the prefix, a sequence's rows of a kv head over its own keys. Both are cut into tiles of rows and, over the
// keys, into splits; a workgroup does one (tile, split) and leaves, for each row, the weighted sum of values, the
// running maximum and the sum of the weights; a second launch joins a row's parts.
//
// tiles.hpp has the products and the softmax of a wave's rows.
#include <array>
#include <climits>
#include <cmath>
#include <type_traits>

#include "divide.hpp"
#include "host.hpp"
#include "matrix.hpp"
#include "tiles.hpp"

#pragma clang fp contract(off)

using namespace rw;

namespace {

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
  int prefix_per, own_per;        // 32-key slices of a split
  int prefix_team, own_team;      // waves that share a split of a 32-row tile
  int merged;                     // the prefix's slices are the first of each sequence's own
  Divisor by_block, by_seq, by_group, by_kv_heads;
  Divisor by_prefix_tiles, by_prefix_splits, by_own_tiles, by_own_splits;
  int prefix_tiles, own_tiles;    // row tiles of a kv head: over the batch, of a sequence
  unsigned prefix_groups;         // workgroups over the prefix
  int waves;                      // of a workgroup
  bool wide;                      // the prefix's tiles: 32 rows to each wave, or to the workgroup
  int cache_blocks;               // blocks that begin in the cache
  float scale;                    // times log2(e)
};

__device__ char g_zeros[512] __attribute__((aligned(16)));  // what an absent key's row reads

// How many keys a table holds (at most 2^30).
__device__ __forceinline__ int keys_of(int len, int blocks, int block_size) {
  const int most = blocks * block_size;
  return len < 0 ? 0 : len < most ? len : most;
}
__device__ __forceinline__ int slices_of(int keys) { return (keys + kKeys - 1) / kKeys; }

// A wave's rows: per lane (its column's row) the place of the row in the outputs, or -1; the last own key it sees; its
// query.
struct Row {
  int at;
  int limit;
  const char* q;
  __device__ __forceinline__ void place(const Args& a, int b, int s, int head) {
    at = (b * a.seq + s) * a.q_heads + head;
    q = static_cast<const char*>(a.q) + 2 * (b * a.qb + s * a.qs + head * a.qh);
  }
};

template <typename T, int D>
__device__ __forceinline__ void start_tile(Tile<T, D>& t, const Row& row, int lane) {
  const int h = lane >> 5;
#pragma unroll
  for (int c = 0; c < Dims<D>::steps; ++c) {
    t.q[c] = (u32x4){0u, 0u, 0u, 0u};
    if (row.at >= 0) t.q[c] = load16<false>(row.q, 2 * c + h);
  }
#pragma unroll
  for (int d = 0; d < Dims<D>::blocks; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) t.o[d][i] = 0.0f;
  t.m = kNone;
  t.l = 0.0f;
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

__device__ __forceinline__ int page_of(int t, const Args& a) { return (int)a.by_block.of((unsigned)t); }
// The slot of key t, which lies on page `page` of its table, in block `block` of the cache; -1 if it is outside.
__device__ __forceinline__ int slot_in(int block, int page, int t, const Args& a) {
  const unsigned slot = (unsigned)block * (unsigned)a.block_size + (unsigned)(t - page * a.block_size);
  return (unsigned)block < (unsigned)a.cache_blocks && slot < (unsigned)a.slots ? (int)slot : -1;
}

// A slice's slots by this lane's rows in its loads; lane l < 32 holds the slot of row l.
template <int D> struct Slots {
  static constexpr int rows = kWave / Dims<D>::chunks, loads = kKeys / rows;
  int of[loads];
  __device__ __forceinline__ void spread(int slot, int lane) {
#pragma unroll
    for (int i = 0; i < loads; ++i) of[i] = from_lane(slot, i * rows + lane / Dims<D>::chunks);
  }
};

// Starts the loads of a slice's 32 rows of K or V (`base`: the kv head's first row) into LDS. `once`: nobody else reads
// them (16 own contexts of 2048 to 8192 keys: 69.4 us without the distinction, 60.3 with it). A wave alone on its SIMD
// issues an instruction in 8 cycles, so a slice takes what its instructions number: the rows' slots are handed out once
// for K and V, and an absent row's address is chosen, not branched to.
template <int D, bool KEYS>
__device__ __forceinline__ void load_slice(const Args& a, const char* base, const Slots<D>& slots, bool once, char* to,
                                           int lane) {
  constexpr int C = Dims<D>::chunks, rows = Slots<D>::rows, loads = Slots<D>::loads, some = loads < 8 ? loads : 8;
  const uint32_t row_bytes = (uint32_t)(2 * D) * (uint32_t)a.kv_heads;
  const char* zeros = g_zeros + 16 * (lane & (C - 1));
  if constexpr (D > 128) {  // the places in a row are computed anew: kept, they would take the sums' registers
    uint32_t anew = (uint32_t)lane;
    settle(anew);
    lane = (int)anew;
  }
#pragma unroll
  for (int first = 0; first < loads; first += some) {
    const char* from[some];
    bool mine[some];
#pragma unroll
    for (int i = 0; i < some; ++i) {
      const int r = (first + i) * rows + lane / C, c = ((lane & (C - 1)) ^ (KEYS ? r : 2 * r)) & (C - 1);
      const int at = slots.of[first + i];
      const char* p = base + 16 * c + (uint64_t)(uint32_t)at * row_bytes;
      settle(p);
      from[i] = at < 0 ? zeros : p;
      mine[i] = Dims<D>::used == C || c < Dims<D>::used;
    }
    if (once) {
#pragma unroll
      for (int i = 0; i < some; ++i) stream_to_lds(from[i], to + (first + i) * kWave * 16, mine[i]);
    } else {
#pragma unroll
      for (int i = 0; i < some; ++i) load_to_lds(from[i], to + (first + i) * kWave * 16, mine[i]);
    }
  }
}

// A hidden key's weight is 0, but 0 times a NaN or an infinity is NaN. So where a slice's values hold one for a key
// that not all of a tile's rows see, the slice's keys of that kind become zeros in LDS before the product, and
// add_apart() adds them to the rows that see them when the tile is through. Only the last slices of a step of several
// tokens have such keys; looking for a NaN there is a trip or two to LDS (64 x 4 tokens of 32/8 heads of 128 behind 146
// keys, up to 400 own: 31 us, without it 30.1; 33 x 5 of 28/4 heads of 64 behind 4999, up to 701 own: 24.5 both).
template <typename T> constexpr uint32_t kExponent = 0x7f807f80;  // of two elements: all set in infinities and NaN
template <> constexpr uint32_t kExponent<F16> = 0x7c007c00;
template <typename T> constexpr uint32_t kExponentOne = 0x00800080;
template <> constexpr uint32_t kExponentOne<F16> = 0x04000400;

// Whether a value of a slice's keys from ... to - 1 is infinite or NaN; they are zeros then.
template <typename T, int D>
__device__ __forceinline__ bool take_apart(char* v, int from, int to, int lane) {
  constexpr int used = Dims<D>::used;
  const int n = (to - from) * used;
  auto place = [&](int i) { return reinterpret_cast<u32x4*>(v + v_place<D>(from + i / used, i % used)); };
  uint32_t found = 0;  // a sign bit
#pragma unroll 1
  for (int first = lane; first - lane < n; first += 4 * kWave) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u32x4 x = *place(least(first + j * kWave, n - 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) found |= (x[e] & kExponent<T>) + kExponentOne<T>;
    }
  }
  if (__ballot(found & 0x80008000u) == 0) return false;
#pragma unroll 1
  for (int i = lane; i < n; i += kWave) *place(i) = (u32x4){0u, 0u, 0u, 0u};
  wait_lds();
  return true;
}
// Own keys first + j whose bits j are set, weighed anew against the tile's last reference points.
template <typename T, int D>
__device__ __forceinline__ void add_apart(Tile<T, D>& t, const Args& a, const char* kb, const char* vb, uint32_t keys,
                                          int first, int slot, const Row& row, int lane) {
  const int h = lane >> 5;
  const uint64_t row_bytes = (uint64_t)(2 * D) * (uint64_t)a.kv_heads;
  f32x16 s;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
  for (int c = 0; c < Dims<D>::steps; ++c) {
    u32x4 k = {0u, 0u, 0u, 0u};
    if (keys >> (lane & 31) & 1) k = load16<false>(kb + (uint64_t)(uint32_t)slot * row_bytes, 2 * c + h);
    s = product32<T>(k, t.q[c], s);
  }
  for (; keys; keys &= keys - 1) {
    const int key = __builtin_ctz(keys), at = 4 * (key >> 3) + (key & 3);  // of a lane of half key / 4 % 2
    float x = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) x = i == at ? s[i] : x;
    x = __builtin_bit_cast(float, from_lane(__builtin_bit_cast(int, x), (lane & 31) + 32 * (key >> 2 & 1)));
    float w[8];
    unpack<T>((u32x4){pack2<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(x, a.scale, -t.m)), 0.0f), 0u, 0u, 0u}, w);
    const char* v = vb + (uint64_t)(uint32_t)__builtin_amdgcn_readlane(slot, key) * row_bytes;
    const bool seen = first + key <= row.limit;
#pragma unroll
    for (int d = 0; d < Dims<D>::blocks; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int c = value_of<D>(d, i / 8) + 8 * (i / 4 % 2) + 4 * h + i % 4;
        if (seen && c < D) t.o[d][i] = __builtin_fmaf(w[0], load_elem<T>(v, c), t.o[d][i]);
      }
  }
}

// The tiles of a team's waves over the same rows joined through LDS (each wave's own two slices of it), and the part,
// or the result where it is the only one, written.
template <typename T, int D, int WAVES>
__device__ __forceinline__ void finish(Tile<T, D>& t, const Args& a, const Row& row, int part, int parts, int team,
                                       char* lds, float2* stats, int wave, int lane) {
  constexpr int B = Dims<D>::blocks;
  static_assert(kRows * 32 * B * 4 <= 2 * Dims<D>::slice, "a tile's sums fit its wave's slices");
  const int r = lane & 31, h = lane >> 5, leader = wave & ~(team - 1);
  t.l = sum_of_halves(t.l);
  float m = t.m, l = t.l, f = 1.0f;
  if (team > 1) {
    if (lane < 32) stats[wave * kRows + lane] = make_float2(t.m, t.l);
    __syncthreads();
    for (int w = 0; w < team; ++w) m = fmaxf(m, stats[(leader + w) * kRows + r].x);
    l = 0.0f;
    for (int w = 0; w < team; ++w) {
      const float2 s = stats[(leader + w) * kRows + r];
      l += s.y * __builtin_amdgcn_exp2f(s.x - m);
    }
    f = __builtin_amdgcn_exp2f(t.m - m);
  }
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
  if (team > 1) __syncthreads();
  else wave_lds_sync();
  // 8 lanes to a row, the team's waves in turn
  for (int first = 8 * (wave - leader); first < kRows; first += 8 * team) {
    const int mr = first + (lane >> 3);
    const long long at = from_lane(row.at, mr);
    const float rl = __builtin_bit_cast(float, from_lane(__builtin_bit_cast(int, l), mr));
    const float rm = __builtin_bit_cast(float, from_lane(__builtin_bit_cast(int, m), mr));
    if (at < 0) continue;
    const bool none = !(rl > 0.0f) && rl == rl;  // a row that sees no key: 0, whatever its tile's other rows see
    const float inverse = 1.0f / rl;
    for (int c = lane & 7; c < D / 4; c += 8) {
      float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int w = 0; w < team; ++w) {
        const float4 y =
            reinterpret_cast<const float4*>(lds + (leader + w) * 2 * Dims<D>::slice)[mr * 8 * B + (c ^ (mr & 7))];
        x[0] += y.x, x[1] += y.y, x[2] += y.z, x[3] += y.w;
      }
      if (none) x[0] = x[1] = x[2] = x[3] = 0.0f;
      if (parts == 1) {
        const float by = none ? 0.0f : inverse;
        *reinterpret_cast<u32x2*>(static_cast<char*>(a.out) + 2 * (at * D + 4 * c)) =
            (u32x2){pack2<T>(x[0] * by, x[1] * by), pack2<T>(x[2] * by, x[3] * by)};
      } else {
        *reinterpret_cast<float4*>(a.sums + (at * parts + part) * D + 4 * c) = make_float4(x[0], x[1], x[2], x[3]);
      }
    }
    if (parts > 1 && (lane & 7) == 0) a.stats[at * parts + part] = make_float2(rm, rl);
  }
}

// One split over the rows of a workgroup, 32 of its own to a wave, and the keys in groups of slices that all share,
// kRing groups of K and of V in LDS. Up to 128 values 8 waves and pairs of slices; longer rows, whose sums and queries
// take more than half of a SIMD's registers, 4 waves and single slices. Measured, a slice for all the tile's rows: of
// 64 values 0.54 us, of 128 0.72 for a workgroup alone and 0.90 where every CU has one, of 256 1.0 for 128 rows; teams
// over 32 rows take 0.76, 1.0 and 2.2 us. 1008 rows of four kv heads behind 9671 keys of 256 values 124 us by those, 79
// so.
//
// A wave goes from slice to slice, and in the turn of slice i it does three things that do not depend on each other:
// the scores of slice i + 1, the weights of slice i and the values of slice i - 1. They are woven together product by
// product (a score's, a value's, an eighth of the weights), since a wave can issue a vector instruction in 8 cycles and
// a product occupies the matrix core for 32: two waves of a SIMD then fill both. (With the two kinds in phases of their
// own, half of the waves in each, a SIMD's one wave in the weights' phase got a vector instruction in 11 cycles, and
// that phase took 1.7 times the other.) The operands are read from LDS half a turn ahead of their products.
//
// There is a barrier a group. Between those of pairs n and n + 1, K's pairs n and n + 1 and V's n - 1 and n are read;
// K's pair n + 3 and V's n + 2 are loaded, and the pages of the keys of pair n + 5, over what was read before the
// barrier. Of single slices, K's n + 1 and n + 2 and V's n - 1 and n are read, K's n + 4 and V's n + 2 are loaded, and
// the pages of n + 6. What is read was loaded two barriers ago, so that no wave waits for a single load.
constexpr int kRing = 4;
template <int D> struct Wide {
  static constexpr int waves = D <= 128 ? 8 : 4;
  static constexpr int group = D <= 128 ? 2 : 1;          // slices
  static constexpr int lead = group == 2 ? 3 : 4;         // how many groups ahead K is loaded
  static constexpr int bytes = 2 * kRing * group * Dims<D>::slice + waves * kRing * kWave * 4;  // of LDS
};

template <typename T, int D>
__device__ __forceinline__ void attend_wide(const Args& a, int keys, int split, int kv_head, const Row& row, char* lds,
                                            int wave, int lane) {
  constexpr int G = Wide<D>::group, W = Wide<D>::waves, lead = Wide<D>::lead, group_keys = G * kKeys;
  constexpr int slice = Dims<D>::slice, group = G * slice, C = Dims<D>::chunks, rows = kWave / C;
  constexpr int loads = group_keys / rows / W;  // of a wave, of K's group; row r of the group is at r * row in LDS
  const int parts = a.prefix_splits + a.own_splits;
  const int from = split * a.prefix_per, part = split;
  const int n = (least(a.prefix_per, slices_of(keys) - from) + G - 1) / G;  // groups
  const int* table = a.prefix_table;
  char* kt = lds;
  char* vt = lds + kRing * group;
  char* pages = lds + 2 * kRing * group + wave * kRing * (kWave * 4);  // this wave's
  const char* kb = static_cast<const char*>(a.k) + 2 * kv_head * D;
  const char* vb = static_cast<const char*>(a.v) + 2 * kv_head * D;
  const uint32_t row_bytes = (uint32_t)(2 * D) * (uint32_t)a.kv_heads;
  const int key = from * kKeys + lane % group_keys;  // this lane's key of the first group
  const int end = least(keys, from * kKeys + n * group_keys);
  // this lane's row of a load and its place in it: over 16 chunks the same in each of the wave's loads, over 32 not
  const int r0 = wave * rows + lane / C, place = lane & (C - 1);
  constexpr int kinds = C > 16 ? loads : 1;
  const char *kp[kinds], *vp[kinds];
  bool kmine[kinds], vmine[kinds];
#pragma unroll
  for (int x = 0; x < kinds; ++x) {
    const int r = r0 + x * W * rows;
    const uint32_t ck = 16u * ((place ^ r) & (C - 1)), cv = 16u * ((place ^ (2 * r)) & (C - 1));
    kmine[x] = Dims<D>::used == C || ck < 2 * D;
    vmine[x] = Dims<D>::used == C || cv < 2 * D;
    kp[x] = kb + ck;
    vp[x] = vb + cv;
  }
  static_assert(C > 16 || W * rows % 16 == 0, "");
  const char* zeros = g_zeros + 16 * place;

  auto load_page = [&](int i, char* to) {
    const int t = key + i * group_keys;
    load_word_to_lds(table + page_of(t < end ? t : 0, a), to);
  };
  auto slot_from = [&](int block, int t) { return t < end ? slot_in(block, page_of(t, a), t, a) : -1; };
  struct Slots {
    int of[loads];  // of this lane's rows
  };
  auto rows_of = [&](int slot) {
    Slots s;
#pragma unroll
    for (int x = 0; x < loads; ++x) s.of[x] = from_lane(slot, r0 + x * W * rows);
    return s;
  };
  // (no branch: the loads are woven into a turn)
  auto load = [&](const char* const (&base)[kinds], const Slots& s, const bool (&mine)[kinds], char* to) {
#pragma unroll
    for (int x = 0; x < loads; ++x) {
      const char* p = base[x % kinds] + (uint64_t)(uint32_t)s.of[x] * row_bytes;
      settle(p);  // chosen or not, not branched to
      load_to_lds(s.of[x] < 0 ? zeros : p, to + (wave + W * x) * kWave * 16, mine[x % kinds]);
    }
  };

  Tile<T, D> t;
  Slots last[lead - 2];   // at the turn of group n: of groups n + 2 ... n + lead - 1
  uint64_t there[kRing];  // the keys that are there, by the group's place
#pragma unroll
  for (int i = 0; i < lead; ++i) {
    const int x = key + i * group_keys;
    const int slot = x < end ? slot_from(table[page_of(x, a)], x) : -1;
    const Slots of = rows_of(slot);
    there[i] = __ballot(slot >= 0);
    load(kp, of, kmine, kt + i * group);
    if (i < 2) load(vp, of, vmine, vt + i * group);
    else last[i - 2] = of;
  }
  load_page(lead, pages + lead % kRing * (kWave * 4));
  load_page(lead + 1, pages + (lead + 1) % kRing * (kWave * 4));
  start_tile<T, D>(t, row, lane);
  constexpr int S = Dims<D>::steps, V = 2 * Dims<D>::blocks, parts_of = S > V ? S : V, ahead = parts_of / 2;
  u32x4 kf[S], vf[V], p[2];
  f32x16 s;  // the scores of slice i at its turn
  // this lane's places in the first slices; V's of 8 rows on are as many bytes on, but of more than 16 chunks to a row
  constexpr int eight = 8 * Dims<D>::row;
  lds_ptr kl[S], vl[V / 2], vl8[C > 16 ? V / 2 : 1];
#pragma unroll
  for (int c = 0; c < S; ++c) kl[c] = own(keys_at<D>(kt, c, lane));
#pragma unroll
  for (int d = 0; d < V / 2; ++d) {
    vl[d] = own(values_at<D>(vt, 0, d, lane));
    if (C > 16) vl8[d % (C > 16 ? V / 2 : 1)] = own(values_at<D>(vt, 8, d, lane));
  }
  // block d of the values of 16 rows, `at` bytes behind the first
  auto value = [&](int d, int at) {
    const lds_ptr first = vl[d] + at;
    return read_values(first, C > 16 ? vl8[d % (C > 16 ? V / 2 : 1)] + at : first + eight);
  };
  wait_loads();
  meet();
#pragma unroll
  for (int c = 0; c < S; ++c) kf[c] = lds_vector(kl[c]);
  scores<T, D>(s, t, kf);
#pragma unroll
  for (int c = 0; c < ahead && c < S; ++c) kf[c] = lds_vector(kl[c] + slice);
  if (G == 1) {  // the first turn loads over the first slice
    wait_lds();
    meet();
  }

  // The turn of slice i, in place X = i % (G kRing) of its ring; in that of a group's first, the loads behind its
  // barrier.
  auto turn = [&](int i, auto where, uint32_t present, auto begun) {
    constexpr int X = decltype(where)::value, R = G * kRing, here = X / G;
    constexpr int k_place = (here + lead) % kRing, v_place = (here + 2) % kRing, page_place = (here + lead + 2) % kRing;
    int entry = 0, slot = 0;
    Slots next;
    constexpr int k1 = (X + 1) % R * slice, k2 = (X + 2) % R * slice;  // K's slices i + 1, i + 2
    constexpr int v0 = (X + R - 1) % R * slice, v1 = X * slice;         // V's slices i - 1, i
    if (present != ~0u) hide(s, present, INT_MAX, lane);
    f32x16 x;
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0.0f;
    float top = 0.0f, f = 1.0f;
    u32x4 q[2];
#pragma unroll
    for (int c = 0; c < parts_of; ++c) {
      if (c < S) x = product32<T>(kf[c], t.q[c], x);
      if (decltype(begun)::value && c < V)
        t.o[c % (V / 2)] = product32<T>(vf[c], p[c / (V / 2)], t.o[c % (V / 2)]);
      const int n = (c + ahead) % parts_of;
      if (n < S) kf[n] = lds_vector(kl[n] + (c + ahead < parts_of ? k1 : k2));
      if (n < V && (decltype(begun)::value || c + ahead >= parts_of))
        vf[n] = value(n % (V / 2), (c + ahead < parts_of ? v0 : v1) + 2 * eight * (n / (V / 2)));
      if (c == 0) top = largest(s);
      if (c == 1) f = refer<T, D>(t, top, a.scale);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c == 2 + e * (parts_of - 2) / 8) weigh<T, D>(t, s, a.scale, e, q);
      if (X % G == 0) {
        if (c == 0) {
          entry = *reinterpret_cast<const int*>(pages + k_place * (kWave * 4) + 4 * lane);
          load(vp, last[0], vmine, vt + v_place * group);
        }
        if (c == 1) {
          slot = slot_from(entry, key + (i / G + lead) * group_keys);
          there[k_place] = __ballot(slot >= 0);
        }
        if (c == 2) next = rows_of(slot);
        if (c == parts_of - 1) {
          load(kp, next, kmine, kt + k_place * group);
          load_page(i / G + lead + 2, pages + page_place * (kWave * 4));
#pragma unroll
          for (int e = 0; e + 1 < lead - 2; ++e) last[e] = last[e + 1];
          last[lead - 3] = next;
        }
      }
      keep_order();
    }
    s = x;
    p[0] = q[0], p[1] = q[1];
    rescale<T, D>(t, f);
  };
  auto both = [&](int i, auto where, auto begun) {
    constexpr int here = decltype(where)::value;
    const uint64_t now = there[here];
    if (decltype(begun)::value) {
      wait_loads<2 * loads + 1>();
      meet();
    }
    turn(G * i, std::integral_constant<int, G * here>{}, (uint32_t)now, begun);
    if constexpr (G == 2)
      turn(2 * i + 1, std::integral_constant<int, 2 * here + 1>{}, (uint32_t)(now >> 32), std::true_type{});
  };
  both(0, std::integral_constant<int, 0>{}, std::false_type{});
  for (int i = 1; i < n;) {
    both(i++, std::integral_constant<int, 1>{}, std::true_type{});
    if (i < n) both(i++, std::integral_constant<int, 2>{}, std::true_type{});
    if (i < n) both(i++, std::integral_constant<int, 3>{}, std::true_type{});
    if (i < n) both(i++, std::integral_constant<int, 0>{}, std::true_type{});
  }
#pragma unroll
  for (int c = 0; c < V; ++c) {
    const int d = c % (V / 2);
    const u32x4 v = value(d, (G * n - 1) % (G * kRing) * slice + 2 * eight * (c / (V / 2)));
    t.o[d] = product32<T>(v, p[c / (V / 2)], t.o[d]);
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

// A run of keys: the first `keys` of a table of `blocks` blocks.
struct Run {
  const int* table;
  int blocks, keys;
};

// A team of waves over one split of 32 rows: the waves take its slices in turn, each through LDS of its own, without
// barriers. K's and V's next slices are on their way as soon as this slice's are in registers; the page of a key comes
// to LDS a slice before it is needed. The slices before `own_from` are those of `before`, whose keys every row sees
// that sees any; own keys up to `all_see` too. A slice takes a lone wave 0.76 us (64 values), 1.0 (128) and 2.2 (256),
// by its instructions' number; with all waves resident own keys come at 6 TB/s.
template <typename T, int D>
__device__ __forceinline__ void attend_slices(Tile<T, D>& t, const Args& a, const Run& before, const Run& own,
                                              int own_from, int all_see, int first, int stop, int turn, int team,
                                              bool once, int kv_head, const Row& row, char* lds, char* pages,
                                              int lane) {
  constexpr int loads = kKeys / (kWave / Dims<D>::chunks);
  char *k = lds, *v = lds + Dims<D>::slice;
  const char* kb = static_cast<const char*>(a.k) + 2 * kv_head * D;
  const char* vb = static_cast<const char*>(a.v) + 2 * kv_head * D;
  auto entry = [&](int s) {  // of the table, not yet knowing the keys
    const bool early = s < own_from;
    const int page = page_of((s - (early ? 0 : own_from)) * kKeys + (lane & 31), a);
    return (early ? before.table : own.table) + least(page, (early ? before.blocks : own.blocks) - 1);
  };
  auto slot_at = [&](int block, int s) {
    const bool early = s < own_from;
    const int x = (s - (early ? 0 : own_from)) * kKeys + (lane & 31);
    return x < (early ? before.keys : own.keys) ? slot_in(block, page_of(x, a), x, a) : -1;
  };
  int s = first + turn;
  const int block = *entry(s);
  load_word_to_lds(entry(s + team), pages);
  if (s >= stop) {
    wait_loads();
    return;
  }
  int slot = slot_at(block, s);
  uint32_t present = (uint32_t)__ballot(slot >= 0);
  Slots<D> rows;
  rows.spread(slot, lane);
  load_slice<D, true>(a, kb, rows, once, k, lane);
  load_slice<D, false>(a, vb, rows, once, v, lane);
  uint32_t apart = 0;  // of the 32 own keys behind all_see, which lie in slices from mixed_from on
  const int mixed_from = own_from == INT_MAX ? INT_MAX : own_from + (all_see + 1) / kKeys;
  for (;;) {
    const bool more = s + team < stop;
    // operands in batches that leave the sums their registers
    constexpr int S = Dims<D>::steps, V = 2 * Dims<D>::blocks, KB = S <= 8 ? S : S / 2, VB = V <= 8 ? V : V / 2;
    u32x4 p[2];
    f32x16 x;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.0f;
    wait_loads<loads>();  // all but V's slice
    const int next = slot_at(*reinterpret_cast<const int*>(pages + 4 * lane), s + team);
    const uint32_t seen = (uint32_t)__ballot(next >= 0);
    rows.spread(next, lane);
#pragma unroll
    for (int first = 0; first < S; first += KB) {
      u32x4 kf[KB];
#pragma unroll
      for (int c = 0; c < KB; ++c) kf[c] = lds_vector(keys_at<D>(k, first + c, lane));
      if (first + KB == S) {
        wait_lds();
        if (more) {
          load_slice<D, true>(a, kb, rows, once, k, lane);
          load_word_to_lds(entry(s + 2 * team), pages);
        }
      }
#pragma unroll
      for (int c = 0; c < KB; ++c) x = product32<T>(kf[c], t.q[first + c], x);
      if (KB < S) keep_order();
    }
    const int limit = s >= own_from ? row.limit - (s - own_from) * kKeys : row.limit < 0 ? -1 : kKeys;
    if (present != ~0u || __ballot(kKeys - 1 > limit && row.at >= 0)) hide(x, present, limit, lane);
    if (more) wait_loads<loads + 1>();  // all but K's next slice and the page
    else wait_loads();
    if (s >= mixed_from) {
      const int begin = (s - own_from) * kKeys, from = all_see + 1 > begin ? all_see + 1 - begin : 0;
      const int to = 32 - __builtin_clz(present | 1);
      if (from < to && take_apart<T, D>(v, from, to, lane)) apart |= (present >> from) << (begin + from - all_see - 1);
    }
    u32x4 vf[VB];
    auto read = [&](int from_c) {
#pragma unroll
      for (int c = 0; c < VB; ++c) {
        const int first = 16 * ((from_c + c) / (V / 2)), d = (from_c + c) % (V / 2);
        vf[c] = read_values(values_at<D>(v, first, d, lane), values_at<D>(v, first + 8, d, lane));
      }
    };
    read(0);
    const float f = refer<T, D>(t, largest(x), a.scale);
#pragma unroll
    for (int i = 0; i < 8; ++i) weigh<T, D>(t, x, a.scale, i, p);
    rescale<T, D>(t, f);
#pragma unroll
    for (int first = 0; first < V; first += VB) {
      if (first) read(first);
      if (first + VB == V) {
        wait_lds();
        if (more) load_slice<D, false>(a, vb, rows, once, v, lane);
      }
#pragma unroll
      for (int c = 0; c < VB; ++c)
        t.o[(first + c) % (V / 2)] = product32<T>(vf[c], p[(first + c) / (V / 2)], t.o[(first + c) % (V / 2)]);
      if (VB < V) keep_order();
    }
    if (!more) break;
    s += team;
    slot = next;
    present = seen;
  }
  if (apart) {
    const int first = all_see + 1, x = first + (lane & 31);
    const int page = page_of(x, a), block = own.table[least(page, own.blocks - 1)];
    add_apart<T, D>(t, a, kb, vb, apart, first, x < own.keys ? slot_in(block, page, x, a) : -1, row, lane);
  }
}

// WIDE: the prefix by 256 rows and a workgroup to a (tile, split), else by 32 rows and a team of waves. A sequence's
// own keys always by 32 rows.
template <typename T, int D, int WAVES, bool WIDE>
__global__ void __launch_bounds__(WAVES* kWave, D <= 128 ? 2 : 1) attend(Args a) {
  constexpr int narrow = WAVES * (2 * Dims<D>::slice + kWave * 4);
  constexpr int wide = Wide<D>::bytes;
  __shared__ __align__(16) char lds[WIDE && wide > narrow ? wide : narrow];
  __shared__ float2 stats[WAVES * kRows];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  const int parts = a.prefix_splits + a.own_splits;
  Row row{-1, INT_MAX, nullptr};
  const unsigned workgroup = (unsigned)rw_host::workgroup();
  auto place = [&](int x, int kv_head) {  // the row x of all the batch's of a kv head
    unsigned token = (unsigned)x;
    const int g = a.by_group.take(token);
    if ((int)token >= a.batch * a.seq) return;
    unsigned b = token;
    const int s = a.by_seq.take(b);
    row.place(a, (int)b, s, kv_head * a.group + g);
  };
  if constexpr (WIDE) {
    if (workgroup < a.prefix_groups) {
      // the tiles of one (kv head, split) read the same keys: all to one XCD (workgroups go round the 8 in turn), so
      // that its L2 has them for all
      unsigned turn = workgroup / 8u;
      const int tile = a.by_prefix_tiles.take(turn);
      unsigned u = turn * 8u + workgroup % 8u;
      if (u >= (unsigned)(a.kv_heads * a.prefix_splits)) return;
      const int split = a.by_prefix_splits.take(u), kv_head = (int)u;
      const int keys = keys_of(a.prefix_len[0], a.prefix_blocks, a.block_size);
      if (split * a.prefix_per >= slices_of(keys)) return;
      place((tile * WAVES + wave) * kRows + (lane & 31), kv_head);
      attend_wide<T, D>(a, keys, split, kv_head, row, lds, wave, lane);
      return;
    }
  }
  const bool shared = !WIDE && workgroup < a.prefix_groups;
  const int team = shared ? a.prefix_team : a.own_team, log_team = __builtin_ctz((unsigned)team);
  const unsigned group = workgroup - (shared ? 0u : a.prefix_groups);
  unsigned u = group * (unsigned)(WAVES >> log_team) + (unsigned)(wave >> log_team);
  const int prefix_keys = shared || a.merged ? keys_of(a.prefix_len[0], a.prefix_blocks, a.block_size) : 0;
  Run before{a.prefix_table, a.prefix_blocks, prefix_keys}, own{a.block_tables, 1, 0};
  int part = -1, kv_head = 0, own_from = slices_of(prefix_keys), all_see = 0, first = 0, stop = 0, some = 0;
  if (shared) {
    const int tile = a.by_prefix_tiles.take(u), split = a.by_prefix_splits.take(u);
    kv_head = (int)u;
    if (kv_head < a.kv_heads) {
      part = split;
      first = split * a.prefix_per;
      stop = least(first + a.prefix_per, own_from);
      some = own_from;
      place(tile * kRows + (lane & 31), kv_head);
    }
    own_from = INT_MAX;
  } else {
    // the tiles over the same keys side by side, then the kv heads of a sequence: their rows lie side by side in the
    // cache
    const int tile = a.by_own_tiles.take(u);
    kv_head = a.by_kv_heads.take(u);
    const int split = a.by_own_splits.take(u), b = (int)u;
    if (b < a.batch) {
      own.blocks = a.own_blocks;
      own.table += (long long)b * own.blocks;
      own.keys = keys_of(a.seq_lens[b], own.blocks, a.block_size);
      part = a.prefix_splits + split;
      unsigned i = (unsigned)(tile * kRows + (lane & 31));
      const int g = a.by_group.take(i);
      if ((int)i < a.seq) {
        row.place(a, b, (int)i, kv_head * a.group + g);
        row.limit = own.keys - a.seq + (int)i;
      }
      // the tile's first token sees the least (where the sequence begins in the tile: some token one key), its last the
      // most
      all_see = own.keys - a.seq + (int)a.by_group.of((unsigned)(tile * kRows));
      all_see = all_see < 0 ? 0 : all_see;
      const int last = least((int)a.by_group.of((unsigned)(tile * kRows + kRows - 1)), a.seq - 1);
      const int end = own.keys - a.seq + 1 + last;
      first = split * a.own_per;
      stop = least(first + a.own_per, own_from + slices_of(end < 0 ? 0 : end));
      some = own_from + slices_of(own.keys);
    }
  }
  // a part that nothing reads is not written: a split without keys, unless it is the only one
  if (first >= some && parts > 1) row.at = -1;
  Tile<T, D> t;
  start_tile<T, D>(t, row, lane);
  char* mine = lds + wave * 2 * Dims<D>::slice;
  char* pages = lds + WAVES * 2 * Dims<D>::slice + wave * kWave * 4;
  if (part >= 0)
    attend_slices<T, D>(t, a, before, own, own_from, all_see, first, stop, wave & (team - 1), team,
                        (shared ? a.prefix_tiles : a.own_tiles) == 1 && !a.merged, kv_head, row, mine, pages, lane);
  if (team > 1) __syncthreads();  // finish() reuses the waves' LDS
  else wave_lds_sync();
  finish<T, D, WAVES>(t, a, row, part, parts, team, lds, stats, wave, lane);
}

// A row's parts joined: a wave per row (a workgroup: heads 4 y ... of token x, and of 2^21 z more). Lengths, stats and
// the first parts' sums are asked for at once, before it is known which parts have been written (a split without keys
// writes none).
template <typename T, int D>
__global__ void __launch_bounds__(256) join(Args a) {
  constexpr int E = D <= 64 ? 1 : D <= 128 ? 2 : 4, batch = 8;  // values per lane; parts per trip to memory
  const int lane = lane_id(), token = (int)(blockIdx.z << rw_host::kGridShift | blockIdx.x);
  const int head = (int)blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(wave_id());
  if (head >= a.q_heads || token >= a.batch * a.seq) return;
  const long long at = (long long)token * a.q_heads + head;
  const int parts = a.prefix_splits + a.own_splits;
  const float2* stats = a.stats + at * parts;
  const float* sums = a.sums + at * parts * D + lane * E;
  const bool mine = lane * E < D;
  auto fetch = [&](float (&x)[E], int p) {
    if (mine) {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = sums[(long long)p * D + e];
    }
  };
  float2 stat = make_float2(kNone, 0.0f);
  if (lane < parts) stat = stats[lane];
  float x[batch][E];
#pragma unroll
  for (int i = 0; i < batch; ++i)
    if (i < parts) fetch(x[i], i);
  unsigned b = (unsigned)token;
  const int s = a.by_seq.take(b);
  const int own = keys_of(a.seq_lens[b], a.own_blocks, a.block_size);
  const int prefix = a.prefix_splits || a.merged ? keys_of(a.prefix_len[0], a.prefix_blocks, a.block_size) : 0;
  const int own_slices = slices_of(own) + (a.merged ? slices_of(prefix) : 0);
  auto written = [&](int p) {
    return p < a.prefix_splits ? p * a.prefix_per < slices_of(prefix)
                               : p < parts && (p - a.prefix_splits) * a.own_per < own_slices;
  };
  float o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
  float total = 0.0f;
  auto add = [&](const float (&y)[E], float f) {  // NaN is not zero
    if (f != 0.0f) {
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += y[e] * f;
    }
  };
  if (own - a.seq + s >= 0) {
    float m = written(lane) ? stat.x : kNone;
    for (int p = lane + kWave; p < parts; p += kWave)
      if (written(p)) m = fmaxf(m, stats[p].x);
    m = wave_max(m);
    for (int p0 = 0; p0 < parts; p0 += kWave) {
      float w = 0.0f, l = 0.0f;
      if (written(p0 + lane)) {
        if (p0) stat = stats[p0 + lane];
        w = __builtin_amdgcn_exp2f(stat.x - m);
        l = stat.y * w;
      }
      total += wave_sum(l);
      const int n = least(parts - p0, kWave);
      for (int first = 0; first < n; first += batch) {
        if (p0 + first) {
#pragma unroll
          for (int i = 0; i < batch; ++i)
            if (first + i < n) fetch(x[i], p0 + first + i);
        }
#pragma unroll
        for (int i = 0; i < batch; ++i)
          if (first + i < n) add(x[i], readlane(w, first + i));
      }
    }
  }
  const float inverse = total > 0.0f || total != total ? 1.0f / total : 0.0f;
  if (mine) {
#pragma unroll
    for (int e = 0; e < E; ++e) store_elem<T>(a.out, at * D + lane * E + e, o[e] * inverse);
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------

enum { kTunePrefix = 0, kTuneOwn = 1, kTuneWide = 2, kTuneTeam = 3 };
constexpr long long kMostKeys = 1 << 30;  // of a table
constexpr int kNarrow = 4;                // waves of a workgroup over 32-row tiles
constexpr double kMemory = 5.2e6, kCaches = 5.5e6;  // bytes a us

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

bool sizes_ok(long long batch, long long seq, int q_heads, int kv_heads, int head_dim, long long prefix_blocks,
              long long own_blocks, long long block_size) {
  const bool dim = head_dim == 64 || head_dim == 80 || head_dim == 96 || head_dim == 128 || head_dim == 192 ||
                   head_dim == 256;
  return dim && kv_heads >= 1 && q_heads >= kv_heads && q_heads <= 65536 && q_heads % kv_heads == 0 &&
         block_size >= 1 && block_size <= kMostKeys && prefix_blocks >= 0 && prefix_blocks <= kMostKeys / block_size &&
         own_blocks >= 0 && own_blocks <= kMostKeys / block_size && seq <= INT_MAX / 2 / q_heads &&
         batch <= INT_MAX / 2 / (seq * q_heads);
}

// Slices of a split (whole pairs) and splits, at most 256, of `slices`.
void cut(long long slices, long long splits, int& per, int& n) {
  splits = splits > 256 ? 256 : splits < 1 ? 1 : splits;
  per = (int)((ceil_div(slices, splits) + 1) & ~1LL);
  n = (int)ceil_div(slices, per);
}

// How to cut the prefix and the own keys into splits is a search over a model of what it takes. Its numbers are
// measured: a wave's first slice and each next one, a workgroup's of the shared tiles, the memory's rate, a join's
// launch, parts and bytes. Against the best of some 500 splits, tiles and teams it takes 1.00 to 1.05 times the time on
// batches of 32 to 96 sequences of 4 to 8 kv heads behind 4096 to 20000 keys, and 1.36 and 1.25 on 16 sequences of a
// single kv head behind 16384 and 30000, where 32-row tiles would be the better ones. 64 tokens of 32/8 heads of 128
// behind 8192 keys: 8 splits of the prefix (chosen) 51.8 us, 6 50.4, 4 60.5, 12 53.6; 96 x 4 tokens behind 20000: 4
// (chosen) 148 to 152 us, 3 174, 5 171, 8 162. Splits are equal and a workgroup has one, so the first of these leaves
// 64 of 256 CUs without any and the second 64 without one over the prefix. A short prefix is read before each
// sequence's own keys, in one launch that joins nothing: 104 x 7 tokens of 32 heads of 80 behind 146 keys 12 us, with
// the prefix apart 26.
//
// The host does not know the lengths, so the tables' width stands for them (own keys are taken to fill 0.6 of it).
// Tables much wider than what they hold are cut into splits that are too long for it: 16 contexts of 2048 to 8192 keys
// 65 us, in tables of 16384 keys 89, of 32768 155, of 131072 522.
//
// A way to cut the prefix or the own keys and what it costs: us of one of its workgroups from start to end, their
// number, and the us that the memory needs for what they read.
struct Cost {
  double one, groups, memory, busy;  // busy: the share of the memory's rate that so many waves reach
  int per, splits, team;  // team 0: 256-row tiles
};

// The sizes that costs depend on.
struct Sizes {
  double cus;
  long long prefix, own, rows, all_rows;  // slices; rows of a kv head, of all
  int head_dim, batch, kv_heads, prefix_tiles, own_tiles;  // 32-row tiles
};

double most(double a, double b) { return a > b ? a : b; }
double fewer(double a, double b) { return a < b ? a : b; }

enum class Keys { kPrefix, kOwn, kMerged };

// Teams of `team` waves over 32 rows, each wave one slice after the other.
Cost cost_narrow(const Sizes& z, Keys which, long long splits, int team) {
  const bool shared = which == Keys::kPrefix;
  const long long slices = shared ? z.prefix : which == Keys::kOwn ? z.own : z.prefix + z.own;
  const int tiles = shared ? z.prefix_tiles : z.own_tiles, d = z.head_dim;
  Cost c{};
  c.team = team;
  cut(slices, splits, c.per, c.splits);
  const double chain = (double)ceil_div(c.per, team);
  const double waves = (double)(shared ? 1 : z.batch) * z.kv_heads * tiles * c.splits * team;
  c.groups = waves / kNarrow;
  const double first = d <= 64 ? 4.0 : d <= 128 ? 4.9 : 6.7, slice = d <= 64 ? 0.76 : d <= 128 ? 1.06 : 2.4;
  // sequences are shorter than their tables
  const double some = shared ? 1.0 : 1.0 - 0.25 * z.own / (double)slices;
  c.one = first + slice * some * chain + (team > 1 ? 0.4 : 0.0);
  // the tiles of a workgroup read the same keys together, others again; few waves do not keep the memory busy
  const double again = tiles / fewer(tiles, kNarrow / team), bytes = 4.0 * kKeys * d * z.kv_heads;
  const double prefix = bytes * z.prefix, own = bytes * z.own * 0.6 * z.batch * again;
  c.busy = 1.0;
  if (shared) {
    c.memory = most(prefix / kMemory, prefix * again / kCaches);
  } else {
    const double resident = z.cus * (d <= 128 ? 8 : 4);
    c.busy = (0.8 + 0.2 * fewer(1.0, waves / resident)) * (team == 1 ? 1.0 : team == 2 ? 0.97 : 0.94);
    c.memory = own / kMemory + (which == Keys::kMerged ? prefix * again * z.batch / kCaches : 0.0);
  }
  return c;
}

// 256-row tiles, a CU to a workgroup.
Cost cost_wide(const Sizes& z, long long splits) {
  Cost c{};
  cut(z.prefix, splits, c.per, c.splits);
  c.groups = (double)z.kv_heads * (double)ceil_div(z.rows, z.head_dim <= 128 ? 256 : 128) * c.splits;
  c.one = 5.0 + (0.72 + 0.62 * z.head_dim / 128) * c.per / 2;
  c.memory = 4.0 * kKeys * z.head_dim * z.kv_heads * (double)z.prefix / kMemory;
  return c;
}

// Both, the prefix's workgroups first, and what joins their parts.
double time_of(const Sizes& z, const Cost& prefix, const Cost& own) {
  const bool wide = prefix.splits && prefix.team == 0;
  const double slots = z.cus * (wide || z.head_dim > 128 ? 1 : 2);
  const double groups = wide && z.head_dim <= 128 ? own.groups / 2 : own.groups;
  const double rounds = __builtin_floor(prefix.groups / slots), last = prefix.groups - rounds * slots;
  const double free = slots - last, turns = own.splits ? __builtin_floor(prefix.one / own.one) : 0.0;
  double work = rounds * prefix.one;
  if (last <= 0.0) work += __builtin_ceil(groups / slots) * own.one;
  else if (groups <= free * most(turns, 1.0)) work += most(prefix.one, __builtin_ceil(groups / free) * own.one);
  else work += prefix.one + __builtin_ceil((groups - free * turns) / slots) * own.one;
  const double memory = prefix.memory + own.memory / (wide || own.splits == 0 ? 1.0 : own.busy) + 2.0;
  const double body = most(work, memory) + 0.2 * fewer(work, memory);
  const int parts = prefix.splits + own.splits;
  if (parts == 1) return body;
  const double rows = (double)z.all_rows;
  return body + 3.0 + 0.06 * parts + rows * parts * z.head_dim * 8.0 / kMemory + rows / 8192.0;
}

constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256};

void plan(Args& a, int head_dim) {
  const long long cus = rw_host::device_cus();
  Sizes z{};
  z.cus = (double)cus;
  z.rows = (long long)a.batch * a.seq * a.group;
  z.all_rows = z.rows * a.kv_heads;
  z.prefix = ceil_div((long long)a.prefix_blocks * a.block_size, kKeys);
  z.own = ceil_div((long long)a.own_blocks * a.block_size, kKeys);
  z.head_dim = head_dim, z.batch = a.batch, z.kv_heads = a.kv_heads;
  z.prefix_tiles = (int)ceil_div(z.rows, kRows);
  z.own_tiles = (int)ceil_div((long long)a.seq * a.group, kRows);
  const int splits = rw_host::tune_get(kTunePrefix), own_splits = rw_host::tune_get(kTuneOwn);
  const int wide = rw_host::tune_get(kTuneWide), team = rw_host::tune_get(kTuneTeam);
  Cost prefix{}, own{};
  double best = 0.0;
  const auto keep = [&](Cost& kept, const Cost& c, double time) {
    if (kept.splits == 0 || time < best) kept = c, best = time;
  };
  const auto choose_own = [&](const Cost& beside) {
    own = Cost{};
    for (int n : kSplits)
      for (int t = 1; t <= kNarrow && (n == 1 || 2 * n <= z.own + 1); t *= 2) {
        const Cost c = cost_narrow(z, Keys::kOwn, n, t);
        keep(own, c, time_of(z, beside, c));
      }
  };
  const auto choose_prefix = [&]() {
    prefix = Cost{};
    for (int n : kSplits) {
      if (n > 1 && 2 * n > z.prefix + 1) break;
      for (int t = 1; t <= kNarrow && wide != 2; t *= 2) {
        const Cost c = cost_narrow(z, Keys::kPrefix, n, t);
        keep(prefix, c, time_of(z, c, own));
      }
      if (wide != 1) {
        const Cost c = cost_wide(z, n);
        keep(prefix, c, time_of(z, c, own));
      }
    }
  };
  const auto choose_merged = [&](double apart) {
    Cost merged{};
    const long long slices = z.prefix + z.own;
    for (int n : kSplits)
      for (int t = 1; t <= kNarrow && (n == 1 || 2 * n <= slices + 1); t *= 2) {
        const Cost c = cost_narrow(z, Keys::kMerged, n, t);
        keep(merged, c, time_of(z, Cost{}, c));
      }
    if (best < apart || wide == 3) a.merged = 1, prefix = Cost{}, own = merged;
  };
  if (z.own) choose_own(prefix);
  if (z.prefix) {
    // one given the other in turn, from the own keys' best alone and from their least parts
    Cost kept[2];
    double time = 0.0;
    for (int from = 0; from < (z.own ? 2 : 1); ++from) {
      if (from) own = cost_narrow(z, Keys::kOwn, 1, 2);
      for (int i = 0; i < 2; ++i) {
        choose_prefix();
        if (z.own) choose_own(prefix);
      }
      const double now = time_of(z, prefix, own);
      if (from == 0 || now < time) kept[0] = prefix, kept[1] = own, time = now;
    }
    prefix = kept[0], own = kept[1];
    if (z.own && (wide == 3 || (wide == 0 && splits == 0))) choose_merged(time_of(z, prefix, own));
    if (splits > 0 && !a.merged) cut(z.prefix, splits, prefix.per, prefix.splits);
  }
  if (z.own && own_splits > 0) cut(z.own + (a.merged ? z.prefix : 0), own_splits, own.per, own.splits);
  const bool set = team > 0 && team <= kNarrow && (team & (team - 1)) == 0;
  if (set && prefix.team) prefix.team = team;
  if (set) own.team = team;
  a.wide = prefix.splits && prefix.team == 0;
  a.waves = a.wide && head_dim <= 128 ? 8 : kNarrow;
  a.prefix_tiles = a.wide ? (int)ceil_div(z.rows, a.waves * kRows) : z.prefix_tiles;
  a.own_tiles = z.own_tiles;
  a.prefix_per = prefix.per, a.prefix_splits = prefix.splits, a.prefix_team = prefix.team;
  a.own_per = own.per, a.own_splits = own.splits, a.own_team = own.team;
}

long long work_bytes(const Args& a, int head_dim) {
  const long long parts = a.prefix_splits + a.own_splits;
  if (parts == 0 || (parts == 1 && a.own_splits)) return 0;
  return (long long)a.batch * a.seq * a.q_heads * parts * (4LL * head_dim + 8);
}

// The sizes and how they are cut. A search takes some microseconds: each thread keeps its last four.
Args sized(long long batch, long long seq, int q_heads, int kv_heads, int head_dim, long long prefix_blocks,
           long long own_blocks, long long block_size) {
  using Key = std::array<long long, 12>;
  thread_local struct {
    Key key;
    Args args;
  } kept[4];
  thread_local unsigned turn = 0;
  const Key key{batch, seq, q_heads, kv_heads, head_dim, prefix_blocks, own_blocks, block_size,
                rw_host::tune_get(kTunePrefix), rw_host::tune_get(kTuneOwn),
                rw_host::tune_get(kTuneWide) + 16LL * rw_host::tune_get(kTuneTeam), rw_host::device_cus()};
  for (const auto& k : kept)
    if (k.key == key) return k.args;
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
  kept[turn % 4].key = key;
  kept[turn++ % 4].args = a;
  return a;
}

// Workgroups over the prefix and over own keys; the waves of a grid's last row of them are numbered within 31 bits.
constexpr long long kMostGroups = (1LL << 28) - (1LL << rw_host::kGridShift);
long long groups_of(const Args& a, long long& shared) {
  const long long parts = (long long)a.kv_heads * a.prefix_splits;
  shared = a.wide ? ceil_div(parts, 8) * 8 * a.prefix_tiles
                  : ceil_div(parts * a.prefix_tiles * a.prefix_team, a.waves);
  return shared +
         ceil_div((long long)a.batch * a.kv_heads * a.own_splits * a.own_tiles * a.own_team, a.waves);
}

template <typename T, int D>
int launch_dim(Args a, hipStream_t stream) {
  long long shared = 0;
  const long long groups = groups_of(a, shared);
  a.prefix_groups = (unsigned)shared;
  const dim3 grid = rw_host::grid_of(groups), threads(a.waves * kWave);
  if (groups) {
    if (a.wide) hipLaunchKernelGGL((attend<T, D, Wide<D>::waves, true>), grid, threads, 0, stream, a);
    else hipLaunchKernelGGL((attend<T, D, kNarrow, false>), grid, threads, 0, stream, a);
  }
  const int err = (int)hipGetLastError();
  if (err || (a.prefix_splits == 0 && a.own_splits == 1)) return err;  // the only part is the result
  dim3 tokens = rw_host::grid_of((long long)a.batch * a.seq);
  tokens.z = tokens.y, tokens.y = (unsigned)ceil_div(a.q_heads, 4);
  hipLaunchKernelGGL((join<T, D>), tokens, dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

bool too_many(const Args& a) {
  long long shared = 0;
  return groups_of(a, shared) > kMostGroups;
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
  const Args a = sized(batch, seq, q_heads, kv_heads, head_dim, prefix_blocks, own_blocks, block_size);
  return too_many(a) ? -1 : work_bytes(a, head_dim);
}

extern "C" int prefix_attention_launch_sized(const void* q, const void* k_cache, const void* v_cache,
                                             const void* prefix_table, const void* prefix_len,
                                             const void* block_tables, const void* seq_lens, void* out, void* work,
                                             long long work_size, const long long* strides, long long batch,
                                             long long seq, long long slots, int q_heads, int kv_heads, int head_dim,
                                             long long prefix_blocks, long long own_blocks, long long block_size,
                                             float scale, int dtype, hipStream_t stream) {
  using rw_host::aligned16;
  if (batch <= 0 || seq <= 0) return rw_host::kOk;
  if (!sizes_ok(batch, seq, q_heads, kv_heads, head_dim, prefix_blocks, own_blocks, block_size) || slots < 0 ||
      slots > INT_MAX || (dtype != 1 && dtype != 2) || !q || !aligned16(q) || !out || !aligned16(out) || !seq_lens ||
      (slots && (!k_cache || !v_cache)) || !aligned16(k_cache) || !aligned16(v_cache) ||
      (prefix_blocks && (!prefix_table || !prefix_len)) || (own_blocks && !block_tables) ||
      !(scale >= 1.0e-30f && scale <= 1.0e30f))
    return rw_host::kInvalid;
  Args a = sized(batch, seq, q_heads, kv_heads, head_dim, prefix_blocks, own_blocks, block_size);
  const long long need = work_bytes(a, head_dim);
  if (too_many(a)) return rw_host::kInvalid;
  if (need && (!work || !aligned16(work) || work_size < need)) return rw_host::kInvalid;
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
  if (batch == 1) a.qb = 0;  // a single one's stride is not used, and may be anything
  if (seq == 1) a.qs = 0;
  if (q_heads == 1) a.qh = 0;
  if (a.qb % 8 || a.qs % 8 || a.qh % 8) return rw_host::kInvalid;
  a.slots = (int)slots;
  a.by_block = divisor(block_size);
  a.by_seq = divisor(seq);
  a.by_group = divisor(a.group);
  a.by_kv_heads = divisor(kv_heads);
  a.by_prefix_tiles = divisor(a.prefix_tiles);
  a.by_prefix_splits = divisor(a.prefix_splits);
  a.by_own_tiles = divisor(a.own_tiles);
  a.by_own_splits = divisor(a.own_splits);
  a.cache_blocks = (int)ceil_div(slots, block_size);
  a.scale = scale * 1.44269504088896341f;
  return dtype == 1 ? launch_type<BF16>(a, head_dim, stream) : launch_type<F16>(a, head_dim, stream);
}

extern "C" int prefix_attention_launch(const void* q, const void* k_cache, const void* v_cache,
                                       const void* prefix_table, const void* prefix_len, const void* block_tables,
                                       const void* seq_lens, void* out, void* work, const long long* strides,
                                       long long batch, long long seq, long long slots, int q_heads, int kv_heads,
                                       int head_dim, long long prefix_blocks, long long own_blocks,
                                       long long block_size, float scale, int dtype, hipStream_t stream) {
  return prefix_attention_launch_sized(q, k_cache, v_cache, prefix_table, prefix_len, block_tables, seq_lens, out, work,
                                       LLONG_MAX, strides, batch, seq, slots, q_heads, kv_heads, head_dim,
                                       prefix_blocks, own_blocks, block_size, scale, dtype, stream);
}

extern "C" int prefix_attention_tune(int slot, int value) { return rw_host::tune_set(slot, value); }
