// Causal attention of whole prompts, packed one behind the other, over their own keys (include/prompt_attention.h has the
// formula).
//
// The rows of a kv head are its prompt's tokens times the query heads that share it, token by token; a workgroup does a
// tile of them over all the keys that its last token sees. So a tile of 256 rows in groups of 4 is 64 tokens, whose own
// keys alone are partly hidden, and K and V are read once for the 4 heads. tiles.hpp has the products and the softmax.
//
// K and V go through a ring of LDS buffers that the workgroup's waves share, 32 rows of its own to a wave, loaded without
// registers three or four groups of slices ahead. In the turn of slice i a wave does three things that do not depend on
// each other, woven together product by product: the scores of slice i + 1, the weights of slice i and the values of slice
// i - 1. There is a barrier to a group.
//
// Tiles are dealt out the longest first, so that short ones fill the end of the launch. The lengths are on the device, so a
// workgroup finds its tile itself.
//
// 16384 tokens of 32/8 heads of 128 in 1.85 to 2.02 ms, 1.09 to 1.19 PFLOP/s with the matrix cores busy 58% of a clock that the
// power holds at 1.75 GHz (cards differ); 8192 of 64 in 309 to 332 us, 0.83 to 0.89 PFLOP/s, where 54 vector instructions
// beside a slice's 8 products bound it.
#include <climits>
#include <type_traits>

#include "divide.hpp"
#include "host.hpp"
#include "matrix.hpp"
#include "tiles.hpp"

#pragma clang fp contract(off)

using namespace rw;

namespace {

struct Args {
  const char *q, *k, *v;
  char* out;
  const int* offsets;
  long long qt, qh, kt, kh, vt, vh;  // strides of a token and a head, in bytes
  int tokens, batch, q_heads, kv_heads, group;
  int slots;                         // of tiles
  Divisor by_heads, by_group;
  float scale;                       // times log2(e)
};

// W waves of 32 rows, G slices to a group.
template <int D, int W, int G> struct Ring {
  static constexpr int groups = 4;
  static constexpr int lead = G == 2 ? 3 : 4;          // how many groups ahead K is loaded; V two
  static constexpr int group = G * Dims<D>::slice;     // bytes of K or of V
  static constexpr int bytes = 2 * groups * group;
};

// A wave's rows: per lane (its column's row) the row's place, token * q_heads + head, or -1; the last key that it sees;
// its query.
struct Row {
  int at, limit;
  const char* q;
};

__device__ __forceinline__ int offset_of(const Args& a, int b) {
  const int n = a.offsets[b];
  return n < 0 ? 0 : n < a.tokens ? n : a.tokens;
}

// A tile: its prompt's first row and number of keys (0: there is none), and the tile's first row among the prompt's; and
// the rows that some prompt has.
struct Place {
  int begin, keys, row, first, last;
};
// Of up to kSorted prompts the tiles in the order of their length: place i of every prompt that has so many, i from the
// most down. With n(i) the tiles at place i and beyond, of all prompts, tile `rank` is at the i with n(i + 1) <= rank <
// n(i), which is looked for among 64 places at a time, a lane to each. (4 x 8192 tokens of 8 heads of 128: 262 us, prompt
// after prompt 290. It takes four instructions a prompt, twice: of 24 prompts of up to 1401 tokens it cost 2 us a tile,
// where prompt after prompt ends as early.)
//
// Of more, prompt after prompt from the last one's end: prompt b's tile slots begin at (rows before it) / (rows of a tile) +
// b, and are at least as many as its tiles.
//
// Offsets are looked at 64 at a time, a lane to each; of fewer prompts that is one trip to memory for all that a workgroup
// wants to know.
constexpr int kSorted = 8;
template <int TILE> __device__ __forceinline__ Place place_of(const Args& a, int rank, int lane) {
  const int slot = a.slots - 1 - rank;
  auto begun = [&](int offset, int b) { return offset * a.group / TILE + b <= slot; };
  if (a.batch < kWave) {
    const int offset = offset_of(a, least(lane, a.batch));
    Place p = {0, 0, 0, __builtin_amdgcn_readlane(offset, 0), __builtin_amdgcn_readlane(offset, a.batch)};
    int b, tile;
    if (a.batch <= kSorted) {
      const int keys = from_lane(offset, least(lane + 1, a.batch)) - offset;
      const int tiles = keys > 0 && lane < a.batch ? (keys * a.group + TILE - 1) / TILE : 0;
      int low = 0, span = (int)wave_max((float)tiles), next = 0;  // (fewer than 2^23 tiles: exact)
      do {
        span = (span + kWave - 2) / (kWave - 1);  // n(low + 63 span) <= rank
        const int at = low + lane * span;
        int n = 0;
        for (int i = 0; i < a.batch; ++i) {
          const int more = __builtin_amdgcn_readlane(tiles, i) - at;
          n += more > 0 ? more : 0;
        }
        const int count = __popcll(__ballot(n > rank));
        if (count == 0) return p;
        low += (count - 1) * span;
        next = __builtin_amdgcn_readlane(n, least(count, kWave - 1));
      } while (span > 1);
      uint64_t mask = __ballot(tiles > low);
      for (int skip = rank - next; skip; --skip) mask &= mask - 1;
      b = __builtin_ctzll(mask), tile = low;
    } else {
      b = __popcll(__ballot(lane < a.batch && begun(offset, lane))) - 1;
      if (b < 0) return p;
      tile = slot - (__builtin_amdgcn_readlane(offset, b) * a.group / TILE + b);
    }
    p.begin = __builtin_amdgcn_readlane(offset, b);
    p.keys = __builtin_amdgcn_readlane(offset, b + 1) - p.begin;
    p.row = tile * TILE;
    return p;
  }
  int first = 0, n = a.batch, offset, count;
  Place p = {0, 0, 0, offset_of(a, 0), offset_of(a, a.batch)};
  for (;;) {  // 63 places, and the last one's end beside them
    const int step = (n + kWave - 2) / (kWave - 1), b = first + lane * step;
    offset = offset_of(a, least(b, a.batch));
    count = __popcll(__ballot(b < a.batch && lane * step < n && begun(offset, b)));
    if (count == 0) return p;
    if (step == 1) break;
    first += (count - 1) * step;
    n = step;
  }
  first += count - 1;
  p.begin = __builtin_amdgcn_readlane(offset, count - 1);
  p.keys = __builtin_amdgcn_readlane(offset, count) - p.begin;
  p.row = (slot - (p.begin * a.group / TILE + first)) * TILE;
  return p;
}

// The reference point of a row's weights is its first slice's largest score, and moves only when a slice's weights have
// come to sum up to more than this in a lane: finding each slice's largest is 14 of the 69 vector instructions beside the
// products, and the weights wait for it. A reference far below the largest costs nothing: weights are floating point, the
// sums have room for 2^12 times as many (fp16 weights, which start 2^7 up, end at 2^16). Two bf16 numbers of 2^12 and more
// are as exact as two below 1.
template <typename T> constexpr float kMostSum = 0x1p12f;
template <> constexpr float kMostSum<F16> = 0x1p15f;

// The weights of scores 2 e and 2 e + 1, rounded to 16 bits, and `sum` with them (tiles.hpp has what the rounding costs). In
// two numbers, a high and a low part, outputs have their own rounding's error alone (bf16 0.0016 from the formula in 64 bits
// and not 0.0018 to 0.0021), and the products and the splitting take 35% more time: 16384 tokens of 32/8 heads of 128 2690 us
// for 2000, 8192 of 64 461 for 332, 24 prompts of up to 1401 173 for 128, heads of 256 60 to 100% more.
template <typename T>
__device__ __forceinline__ float weigh_two(const f32x16& s, float scale, float m, int e, u32x4* p, float sum) {
  uint32_t two = pack2<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * e], scale, -m)),
                          __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * e + 1], scale, -m)));
  settle(two);
  sum = add_pair<T>(two, sum);
  settle(sum);  // and not all of them behind each other in the end
  p[e / 4][e % 4] = two;
  return sum;
}
// Moves the rows' reference points up to a slice's largest scores. Returns what the values' sums are to be multiplied by.
template <typename T, int D>
__device__ __forceinline__ float move_point(Tile<T, D>& t, const f32x16& s, float scale) {
  const float m = fmaxf(t.m, max_of_halves(largest(s)) * scale - kBias<T>), f = __builtin_amdgcn_exp2f(t.m - m);
  t.m = m;
  t.l *= f;
  return f;
}

// What the places of row r's chunks of K are XORed with: 16 rows' same chunk lie in different banks, of which there are two
// rows of 64 values to a turn.
template <int D> __device__ __forceinline__ int k_turn(int r) { return Dims<D>::chunks == 8 ? r >> 1 : r; }

template <typename T, int D, int W, int G>
__device__ __forceinline__ void attend_tile(Tile<T, D>& t, const Args& a, const char* kb, const char* vb, int keys,
                                            int slices, int all_see, const Row& row, char* lds, int wave, int lane) {
  using R = Ring<D, W, G>;
  constexpr int slice = Dims<D>::slice, group = R::group, C = Dims<D>::chunks, rows = kWave / C, lead = R::lead;
  constexpr int group_keys = G * kKeys, ring = R::groups;
  constexpr int loads = group_keys / rows / W;  // of a wave, of K's group; row r of the group is at r * row in LDS
  static_assert(loads * rows * W == group_keys, "");
  static_assert(W * kRows * Dims<D>::row <= R::bytes, "the results fit the ring");
  const int n = (slices + G - 1) / G;           // groups
  char* kt = lds;
  char* vt = lds + ring * group;
  // this lane's rows of its loads and its place in them
  const int r0 = wave * rows + lane / C, place = lane & (C - 1);
  uint32_t k_chunk[loads], v_chunk[loads];
  bool k_mine[loads], v_mine[loads];
#pragma unroll
  for (int x = 0; x < loads; ++x) {
    const int r = r0 + x * W * rows;
    k_chunk[x] = 16u * ((place ^ k_turn<D>(r)) & (C - 1)), v_chunk[x] = 16u * ((place ^ (2 * r)) & (C - 1));
    k_mine[x] = Dims<D>::used == C || k_chunk[x] < 2 * D;
    v_mine[x] = Dims<D>::used == C || v_chunk[x] < 2 * D;
  }
  // Group i's rows; a key behind the prompt's last is read as the last, and hidden like all that a row does not see.
  auto load = [&](const char* base, long long stride, const uint32_t (&chunk)[loads], const bool (&mine)[loads], int i,
                  char* to) {
    const int first = least(i * group_keys, keys - 1), left = keys - 1 - first;
    const char* from = base + (long long)first * stride;
    const uint32_t most = (uint32_t)(left < group_keys ? left : group_keys) * (uint32_t)stride;
#pragma unroll
    for (int x = 0; x < loads; ++x) {
      const uint32_t at = (uint32_t)(r0 + x * W * rows) * (uint32_t)stride;
      load_to_lds_at(from, (at < most ? at : most) + chunk[x], to + (wave + W * x) * kWave * 16, mine[x]);
    }
  };
  auto load_k = [&](int i, int where) { load(kb, a.kt, k_chunk, k_mine, i, kt + where * group); };
  auto load_v = [&](int i, int where) { load(vb, a.vt, v_chunk, v_mine, i, vt + where * group); };
  // what the first turn reads, and behind it what the next does
#pragma unroll
  for (int i = 0; i + 1 < lead; ++i) load_k(i, i);
  load_v(0, 0);
  {
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
  constexpr int S = Dims<D>::steps, V = 2 * Dims<D>::blocks, parts_of = S > V ? S : V, ahead = parts_of / 2;
  u32x4 kf[S], vf[V], p[2];
  f32x16 even, odd;  // the scores of slice i at its turn
  // this lane's places in the first slices; V's of 8 rows on are as many bytes on, but of more than 16 chunks to a row
  constexpr int eight = 8 * Dims<D>::row;
  lds_ptr kl[S], vl[V / 2], vl8[C > 16 ? V / 2 : 1];
#pragma unroll
  for (int c = 0; c < S; ++c) kl[c] = own(in_lds(kt) + (lane & 31) * Dims<D>::row +
                                                   (((2 * c + (lane >> 5)) ^ k_turn<D>(lane & 31)) & (C - 1)) * 16);
#pragma unroll
  for (int d = 0; d < V / 2; ++d) {
    vl[d] = own(values_at<D>(vt, 0, d, lane));
    if (C > 16) vl8[d % (C > 16 ? V / 2 : 1)] = own(values_at<D>(vt, 8, d, lane));
  }
  auto value = [&](int d, int at) {
    const lds_ptr first = vl[d] + at;
    return read_values(first, C > 16 ? vl8[d % (C > 16 ? V / 2 : 1)] + at : first + eight);
  };
  wait_loads();
  meet();
  load_k(lead - 1, lead - 1);
  load_v(1, 1);
#pragma unroll
  for (int c = 0; c < S; ++c) kf[c] = lds_vector(kl[c]);
  scores<T, D>(even, t, kf);
#pragma unroll
  for (int c = 0; c < ahead && c < S; ++c) kf[c] = lds_vector(kl[c] + slice);
  if (G == 1) {  // the first turn loads over the first slice
    wait_lds();
    meet();
  }

  // what row sees of slice i
  auto hide_from = [&](f32x16& s, int i) {
    const int limit = row.limit - i * kKeys - 4 * (lane >> 5);
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (8 * (e / 4) + e % 4 > limit) s[e] = -INFINITY;
  };
  if (kKeys - 1 > all_see) hide_from(even, 0);
  move_point<T, D>(t, even, a.scale);

  // The turn of slice i, in place X = i % (G ring) of its ring; in that of a group's first, the loads behind its barrier.
  // The next slice's scores go beside this one's: the two take turns, so that none are moved.
  auto turn = [&](int i, auto where, auto begun) {
    constexpr int X = decltype(where)::value, E = G * ring, here = X / G;
    f32x16 &s = X % 2 ? odd : even, &x = X % 2 ? even : odd;
    constexpr int k_place = (here + lead) % ring, v_place = (here + 2) % ring;
    constexpr int k1 = (X + 1) % E * slice, k2 = (X + 2) % E * slice;  // K's slices i + 1, i + 2
    constexpr int v0 = (X + E - 1) % E * slice, v1 = X * slice;         // V's slices i - 1, i
    if (i * kKeys + kKeys - 1 > all_see) hide_from(s, i);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0.0f;
    float sum = 0.0f;
    u32x4 q[2];
#pragma unroll
    for (int c = 0; c < parts_of; ++c) {
      if (c < S) x = product32<T>(kf[c], t.q[c], x);
      if (decltype(begun)::value && c < V)
        t.o[c % (V / 2)] = product32<T>(vf[c], p[c / (V / 2)], t.o[c % (V / 2)]);
      const int m = (c + ahead) % parts_of;
      if (m < S) kf[m] = lds_vector(kl[m] + (c + ahead < parts_of ? k1 : k2));
      if (m < V && (decltype(begun)::value || c + ahead >= parts_of))
        vf[m] = value(m % (V / 2), (c + ahead < parts_of ? v0 : v1) + 2 * eight * (m / (V / 2)));
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c == e * parts_of / 8) sum = weigh_two<T>(s, a.scale, t.m, e, q, sum);
      if (X % G == 0) {
        if (c == 0) load_v(i / G + 2, v_place);
        if (c == parts_of - 1) load_k(i / G + lead, k_place);
      }
      keep_order();
    }
    if (__ballot(sum > kMostSum<T>)) {  // a score far above the reference point: the slice is weighed again from its own
      const float f = move_point<T, D>(t, s, a.scale);
      sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = weigh_two<T>(s, a.scale, t.m, e, q, sum);
      rescale<T, D>(t, f);
    }
    t.l += sum;
    p[0] = q[0], p[1] = q[1];
  };
  auto group_turn = [&](int i, auto where, auto begun) {
    constexpr int here = decltype(where)::value;
    if (decltype(begun)::value) {
      wait_loads<2 * loads>();
      meet();
    }
    turn(G * i, std::integral_constant<int, G * here>{}, begun);
    if constexpr (G == 2) turn(2 * i + 1, std::integral_constant<int, 2 * here + 1>{}, std::true_type{});
  };
  group_turn(0, std::integral_constant<int, 0>{}, std::false_type{});
  for (int i = 1; i < n;) {
    group_turn(i++, std::integral_constant<int, 1>{}, std::true_type{});
    if (i < n) group_turn(i++, std::integral_constant<int, 2>{}, std::true_type{});
    if (i < n) group_turn(i++, std::integral_constant<int, 3>{}, std::true_type{});
    if (i < n) group_turn(i++, std::integral_constant<int, 0>{}, std::true_type{});
  }
#pragma unroll
  for (int c = 0; c < V; ++c) {
    const int d = c % (V / 2);
    const u32x4 v = value(d, (G * n - 1) % (G * ring) * slice + 2 * eight * (c / (V / 2)));
    t.o[d] = product32<T>(v, p[c / (V / 2)], t.o[d]);
  }
  wait_loads();  // none may arrive after the workgroup has gone
}

// A hidden key's weight is 0, but 0 times a NaN or an infinity is NaN: where a wave's sums are not all finite and a key
// that some of its rows do not see holds one, these rows are done again, a key's lane and then a value's lane at a time.
template <typename T, int D>
__device__ __forceinline__ void mend(const Args& a, const char* kb, const char* vb, int keys, int first, int end,
                                     const Row& row, int lane) {
  wait_loads();  // the results that are written again have been written
  int bad = -1;  // the last key with such a value
  for (int j = first + lane; j < least(end, keys); j += kWave) {
    bool found = false;
    for (int c = 0; c < D / 8; ++c) {
      float f[8];
      unpack<T>(load16<false>(vb + j * a.vt, c), f);
#pragma unroll
      for (int e = 0; e < 8; ++e) found = found || !(fabsf(f[e]) < INFINITY);
    }
    if (found) bad = j;
  }
  for (int d = 1; d < kWave; d *= 2) {
    const int other = from_lane(bad, lane ^ d);
    bad = other > bad ? other : bad;
  }
  for (int r = 0; r < kRows; ++r) {
    const int at = from_lane(row.at, r), limit = from_lane(row.limit, r);
    if (at < 0 || limit >= bad) continue;
    const uint64_t address = (uint64_t)row.q;
    const char* q = reinterpret_cast<const char*>(
        (uint64_t)(uint32_t)from_lane((int)(address >> 32), r) << 32 | (uint32_t)from_lane((int)(uint32_t)address, r));
    constexpr int E = (D + kWave - 1) / kWave;
    float o[E], m = kNone, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
    for (int j0 = 0; j0 <= limit; j0 += kWave) {
      float s = -INFINITY;
      if (j0 + lane <= limit) {
        s = 0.0f;
        for (int c = 0; c < D / 8; ++c) {
          float x[8], y[8];
          unpack<T>(load16<false>(q, c), x);
          unpack<T>(load16<false>(kb + (j0 + lane) * a.kt, c), y);
#pragma unroll
          for (int e = 0; e < 8; ++e) s = __builtin_fmaf(x[e], y[e], s);
        }
        s *= a.scale;
      }
      const float top = fmaxf(m, wave_max(s)), f = __builtin_amdgcn_exp2f(m - top), w = __builtin_amdgcn_exp2f(s - top);
      m = top;
      l = l * f + wave_sum(w);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] *= f;
      for (int j = 0; j < least(kWave, limit + 1 - j0); ++j) {
        const float by = readlane(w, j);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e * kWave + lane < D)
            o[e] = __builtin_fmaf(by, load_elem<T>(vb + (j0 + j) * a.vt, e * kWave + lane), o[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e * kWave + lane < D) store_elem<T>(a.out, (long long)at * D + e * kWave + lane, o[e] / l);
  }
}

template <typename T, int D, int W, int G>
__global__ void __launch_bounds__(W* kWave, D <= 128 ? 2 : 1) attend(Args a) {
  constexpr int tile_rows = W * kRows;
  __shared__ __align__(16) char lds[Ring<D, W, G>::bytes];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  unsigned u = (unsigned)rw_host::workgroup();
  const unsigned group = u;
  const int head = a.by_heads.take(u), rank = (int)u;
  if (rank >= a.slots) return;
  const Place place = place_of<tile_rows>(a, rank, lane);
  {  // rows of no prompt are zeros: each workgroup has a share of them
    const int end = place.last > place.first ? place.last : place.first, idle = place.first + a.tokens - end;
    if (idle) {
      const int vectors = a.q_heads * (D / 8);
      for (int i = (int)group; i < idle; i += a.slots * a.kv_heads) {
        const long long token = i < place.first ? i : i + (end - place.first);
        for (int c = (int)threadIdx.x; c < vectors; c += W * kWave)
          store16<false>(a.out + token * a.q_heads * (2 * D), c, (u32x4){0u, 0u, 0u, 0u});
      }
    }
  }
  const int begin = place.begin, keys = place.keys, first_row = place.row;
  if (keys <= 0 || (unsigned)first_row >= (unsigned)(keys * a.group)) return;  // (below 0: of offsets that decrease)
  // the tile's last token, and how far it sees
  const int last = least((int)a.by_group.of((unsigned)(first_row + tile_rows - 1)), keys - 1);
  const int slices = last / kKeys + 1;
  unsigned token = (unsigned)(first_row + wave * kRows + (lane & 31));
  const int g = a.by_group.take(token);
  Row row = {-1, -1, nullptr};
  if ((int)token < keys) {
    row.at = (begin + (int)token) * a.q_heads + head * a.group + g;
    row.limit = (int)token;
    row.q = a.q + (long long)(begin + (int)token) * a.qt + (long long)(head * a.group + g) * a.qh;
  }
  const int all_see = (int)a.by_group.of((unsigned)(first_row + wave * kRows));  // the wave's first token
  const char* kb = a.k + (long long)begin * a.kt + (long long)head * a.kh;
  const char* vb = a.v + (long long)begin * a.vt + (long long)head * a.vh;
  Tile<T, D> t;
  attend_tile<T, D, W, G>(t, a, kb, vb, keys, slices, all_see, row, lds, wave, lane);
  // The results go through LDS, so that whole rows are stored: 8 bytes of 32 rows to an instruction took 4400 cycles.
  wait_lds();
  meet();
  const float inverse = 1.0f / sum_of_halves(t.l);
  const int r = lane & 31, h = lane >> 5;
  char* mine = lds + wave * kRows * Dims<D>::row;
  bool wild = false;
#pragma unroll
  for (int d = 0; d < Dims<D>::blocks; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = sums_at<D>(d, e, h);
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = t.o[d][4 * e + i] * inverse;
        wild = wild || (c < D && !(fabsf(x[i]) < INFINITY));
      }
      *reinterpret_cast<u32x2*>(mine + r * Dims<D>::row + ((c / 8) ^ (k_turn<D>(r) & 7)) * 16 + 2 * (c % 8)) =
          (u32x2){pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
    }
  wave_lds_sync();
#pragma unroll
  for (int first = 0; first < kRows * Dims<D>::used; first += kWave) {
    const int i = first + lane, to = i / Dims<D>::used, c = i % Dims<D>::used;
    const long long at = from_lane(row.at, to);
    const u32x4 x = *reinterpret_cast<const u32x4*>(mine + to * Dims<D>::row + (c ^ (k_turn<D>(to) & 7)) * 16);
    if (at >= 0) store16<false>(a.out + at * (2 * D), c, x);
  }
  wild = wild && row.at >= 0;
  if (__ballot(wild)) mend<T, D>(a, kb, vb, keys, all_see + 1, (slices + G - 1) / G * G * kKeys, row, lane);
}

// ---- host side ------------------------------------------------------------------------------------------------------

enum { kTuneWaves = 0 };

template <typename T, int D, int W, int G>
int launch_form(Args a, hipStream_t stream) {
  a.slots = (int)((long long)a.tokens * a.group / (W * kRows)) + a.batch + (a.batch == 0);
  const dim3 grid = rw_host::grid_of((long long)a.slots * a.kv_heads), threads(W * kWave);
  hipLaunchKernelGGL((attend<T, D, W, G>), grid, threads, 0, stream, a);
  return (int)hipGetLastError();
}
// 8 waves to a workgroup read K and V half as often as 4 and are one to a CU, so nothing is done while one begins or ends:
// they pay where prompts are long and tiles many. 1 x 16384 tokens of 32/8 heads of 128: 8 waves 1881 us, 4 1993; 1 x 8192
// 502, 534; 1 x 4096 146, 147; 24 of up to 1401 256, 244; 4 x 8192 of 8/8 267, 266; 1 x 8192 of 8/1 (256 tiles of 256 rows)
// 197, 179. Heads of 64, whose LDS allows 3 workgroups of 4 waves to a CU: 16384 tokens 1162, 1164, 24 of up to 1401 150, 120.
template <typename T, int D>
int launch_dim(const Args& a, hipStream_t stream) {
  if constexpr (D > 64 && D <= 128) {
    const long long tiles = (long long)a.tokens * a.group / 256 * a.kv_heads;
    const bool wide = tiles >= 3LL * rw_host::device_cus() && a.tokens >= 4096LL * a.batch;
    const int waves = rw_host::tune_get(kTuneWaves);
    if (waves ? waves == 8 : wide) return launch_form<T, D, 8, 2>(a, stream);
  }
  return launch_form<T, D, 4, 1>(a, stream);
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

extern "C" int prompt_attention_launch(const void* q, const void* k, const void* v, const void* cu_seqlens, void* out,
                                       const long long* strides, long long tokens, long long batch, int q_heads,
                                       int kv_heads, int head_dim, float scale, int dtype, hipStream_t stream) {
  using rw_host::aligned16;
  if (tokens <= 0) return rw_host::kOk;
  const bool dim = head_dim == 64 || head_dim == 80 || head_dim == 96 || head_dim == 128 || head_dim == 192 ||
                   head_dim == 256;
  if (!dim || kv_heads < 1 || q_heads < kv_heads || q_heads > 65536 || q_heads % kv_heads || batch < 0 ||
      tokens > INT_MAX / 2 / q_heads || batch > INT_MAX / 4 / kv_heads || (dtype != 1 && dtype != 2) || !q || !k || !v ||
      !out || !cu_seqlens || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) ||
      !(scale >= 1.0e-30f && scale <= 1.0e30f))
    return rw_host::kInvalid;
  const int heads[3] = {q_heads, kv_heads, kv_heads};
  long long s[6];
  for (int i = 0; i < 3; ++i) {
    // the stride of a single token or head decides nothing
    s[2 * i] = tokens == 1 ? 0 : strides ? strides[2 * i] : (long long)heads[i] * head_dim;
    s[2 * i + 1] = heads[i] == 1 ? 0 : strides ? strides[2 * i + 1] : head_dim;
    if (s[2 * i] % 8 || s[2 * i + 1] % 8) return rw_host::kInvalid;
    if (i && (s[2 * i] < 0 || s[2 * i] > 1 << 23)) return rw_host::kInvalid;  // 64 rows' offsets in 32 bits
  }
  Args a{};
  a.q = static_cast<const char*>(q), a.k = static_cast<const char*>(k), a.v = static_cast<const char*>(v);
  a.out = static_cast<char*>(out);
  a.offsets = static_cast<const int*>(cu_seqlens);
  a.qt = 2 * s[0], a.qh = 2 * s[1], a.kt = 2 * s[2], a.kh = 2 * s[3], a.vt = 2 * s[4], a.vh = 2 * s[5];
  a.tokens = (int)tokens, a.batch = (int)batch;
  a.q_heads = q_heads, a.kv_heads = kv_heads, a.group = q_heads / kv_heads;
  a.by_heads = divisor(kv_heads), a.by_group = divisor(a.group);
  a.scale = scale * 1.44269504088896341f;
  return dtype == 1 ? launch_type<BF16>(a, head_dim, stream) : launch_type<F16>(a, head_dim, stream);
}

extern "C" int prompt_attention_tune(int slot, int value) { return rw_host::tune_set(slot, value); }
