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
// Tiles are dealt out from the prompts' ends, the longest first, so that short ones fill the end of the launch. The
// lengths are on the device: tile slots of prompt b begin at (rows before it) / (rows of a tile) + b, which is at least as
// many as it has tiles, and a workgroup finds its prompt by looking at 64 offsets at a time.
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

// The prompt whose tile slots `slot` is among, -1 where it is before the first's.
template <int TILE> __device__ __forceinline__ int prompt_of(const Args& a, int slot, int lane) {
  int first = 0, n = a.batch;
  do {
    const int step = (n + kWave - 1) / kWave, b = first + lane * step;
    const bool begun = b < a.batch && lane * step < n && offset_of(a, b) * a.group / TILE + b <= slot;
    const int count = __popcll(__ballot(begun));
    if (count == 0) return -1;
    first += (count - 1) * step;
    n = step;
  } while (n > 1);
  return first;
}

template <typename T, int D, int W, int G>
__device__ __forceinline__ void attend_tile(Tile<T, D>& t, const Args& a, const char* kb, const char* vb, int keys,
                                            int slices, int all_see, const Row& row, char* lds, int wave, int lane) {
  using R = Ring<D, W, G>;
  constexpr int slice = Dims<D>::slice, group = R::group, C = Dims<D>::chunks, rows = kWave / C, lead = R::lead;
  constexpr int group_keys = G * kKeys, ring = R::groups;
  constexpr int loads = group_keys / rows / W;  // of a wave, of K's group; row r of the group is at r * row in LDS
  static_assert(loads * rows * W == group_keys, "");
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
    k_chunk[x] = 16u * ((place ^ r) & (C - 1)), v_chunk[x] = 16u * ((place ^ (2 * r)) & (C - 1));
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
#pragma unroll
  for (int i = 0; i < lead; ++i) {
    load_k(i, i);
    if (i < 2) load_v(i, i);
  }
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

  // The turn of slice i, in place X = i % (G ring) of its ring; in that of a group's first, the loads behind its barrier.
  auto turn = [&](int i, auto where, auto begun) {
    constexpr int X = decltype(where)::value, E = G * ring, here = X / G;
    constexpr int k_place = (here + lead) % ring, v_place = (here + 2) % ring;
    constexpr int k1 = (X + 1) % E * slice, k2 = (X + 2) % E * slice;  // K's slices i + 1, i + 2
    constexpr int v0 = (X + E - 1) % E * slice, v1 = X * slice;         // V's slices i - 1, i
    if (i * kKeys + kKeys - 1 > all_see) {
      const int limit = row.limit - i * kKeys - 4 * (lane >> 5);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (8 * (e / 4) + e % 4 > limit) s[e] = -INFINITY;
    }
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
      const int m = (c + ahead) % parts_of;
      if (m < S) kf[m] = lds_vector(kl[m] + (c + ahead < parts_of ? k1 : k2));
      if (m < V && (decltype(begun)::value || c + ahead >= parts_of))
        vf[m] = value(m % (V / 2), (c + ahead < parts_of ? v0 : v1) + 2 * eight * (m / (V / 2)));
      if (c == 0) top = largest(s);
      if (c == 1) f = refer<T, D>(t, top, a.scale);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c == 2 + e * (parts_of - 2) / 8) weigh<T, D>(t, s, a.scale, e, q);
      if (X % G == 0) {
        if (c == 0) load_v(i / G + 2, v_place);
        if (c == parts_of - 1) load_k(i / G + lead, k_place);
      }
      keep_order();
    }
    s = x;
    p[0] = q[0], p[1] = q[1];
    rescale<T, D>(t, f);
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
  const int head = a.by_heads.take(u), slot = a.slots - 1 - (int)u;
  if (slot < 0) return;
  {  // rows of no prompt are zeros: each workgroup has a share of them
    const int before = a.batch ? offset_of(a, 0) : 0, end = a.batch ? offset_of(a, a.batch) : 0;
    const int idle = before + a.tokens - (end > before ? end : before);
    if (idle) {
      const int vectors = a.q_heads * (D / 8);
      for (int i = (int)group; i < idle; i += a.slots * a.kv_heads) {
        const long long token = i < before ? i : i + (end > before ? end - before : 0);
        for (int c = (int)threadIdx.x; c < vectors; c += W * kWave)
          store16<false>(a.out + token * a.q_heads * (2 * D), c, (u32x4){0u, 0u, 0u, 0u});
      }
    }
  }
  if (a.batch == 0) return;
  const int b = __builtin_amdgcn_readfirstlane(prompt_of<tile_rows>(a, slot, lane));
  if (b < 0) return;
  const int begin = __builtin_amdgcn_readfirstlane(offset_of(a, b));
  const int keys = __builtin_amdgcn_readfirstlane(offset_of(a, b + 1)) - begin;
  const int first_row = (slot - (begin * a.group / tile_rows + b)) * tile_rows;
  if (keys <= 0 || first_row >= keys * a.group) return;
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
  const float l = sum_of_halves(t.l), inverse = 1.0f / l;
  const int h = lane >> 5;
  bool wild = false;
  if (row.at >= 0) {
#pragma unroll
    for (int d = 0; d < Dims<D>::blocks; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = sums_at<D>(d, e, h);
        if (c >= D) continue;
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = t.o[d][4 * e + i] * inverse;
          wild = wild || !(fabsf(x[i]) < INFINITY);
        }
        *reinterpret_cast<u32x2*>(a.out + 2 * ((long long)row.at * D + c)) =
            (u32x2){pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
      }
  }
  if (__ballot(wild)) mend<T, D>(a, kb, vb, keys, all_see + 1, (slices + G - 1) / G * G * kKeys, row, lane);
}

// ---- host side ------------------------------------------------------------------------------------------------------

enum { kTuneWaves = 0 };

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

template <typename T, int D, int W, int G>
int launch_form(Args a, hipStream_t stream) {
  a.slots = (int)((long long)a.tokens * a.group / (W * kRows)) + a.batch + (a.batch == 0);
  const dim3 grid = rw_host::grid_of((long long)a.slots * a.kv_heads), threads(W * kWave);
  hipLaunchKernelGGL((attend<T, D, W, G>), grid, threads, 0, stream, a);
  return (int)hipGetLastError();
}
template <typename T, int D>
int launch_dim(const Args& a, hipStream_t stream) {
  const int waves = rw_host::tune_get(kTuneWaves);
  if constexpr (D <= 128) {
    if (waves == 4) return launch_form<T, D, 4, 1>(a, stream);
    return launch_form<T, D, 8, 2>(a, stream);
  } else {
    return launch_form<T, D, 4, 1>(a, stream);
  }
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
