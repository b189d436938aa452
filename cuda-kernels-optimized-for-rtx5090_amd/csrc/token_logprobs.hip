// The log probability of a given token in each row of logits, the row's entropy, and its likeliest alternatives
// (include/token_logprobs.h has the formulas).
//
// One pass over the logits, which bounds it. A lane keeps its largest element m, the sum S of e^d over its elements and
// the sum W of e^d d log2(e), with d = x - m (exact where it matters, so a token that is sure has log probability 0):
//   log p(x) = d - ln S,   entropy = ln S - W ln 2 / S   (both terms of the entropy are positive).
// An element costs some eleven instructions (widening, maximum, difference, product, exponential, two sums), which at 16
// bits an element is most of what the vector units can issue at the memory's rate; 16 or 32 of them are summed in fp32,
// these sums in fp64. Beside the largest, whose e^d is 1, fp32 has lost what is left of a row whose token is sure; so
// a wave whose S is hardly more goes over the elements around its largest again and sums them in fp64.
//
// The alternatives are kept by a wave as a sorted list, a 64-bit key to a lane: the value's order above the inverted
// index, so that of equal values the first comes first. A lane compares only its vectors' maxima, which the sums want
// anyway, with the list's last value; a vector that is above goes to a buffer in LDS whole, and 64 of them are taken
// apart, sorted and merged together. Some k (1 + ln(trips)) vectors of a wave come that far. While there is no list, the
// limit is one that k of the lanes' maxima reach, looked for whenever the trips have doubled (4096 rows, 5 alternatives:
// 191 us, with the first trip's limit alone 197).
//
// A workgroup reads a row, or where there are few rows a part of one; a second launch joins the parts.
//
// 4096 rows of 128256 bf16 in 167 us without alternatives (6.3 TB/s), 182 to 194 with 5, 210 with 20, 275 with 64; 64 rows with
// 20 in 19.2 us (14.5 and the join's 4.6); 700 rows of 49999 fp32 in 25.6 us, 5.5 TB/s.
#include <climits>

#include "host.hpp"
#include "matrix.hpp"

#pragma clang fp contract(off)

using namespace rw;

namespace {

constexpr int kWaves = 4, kUnroll = 4, kMostTop = 64, kMostParts = 64;
constexpr int kBuffer = 2 * kWave;  // vectors, keys: fewer than a wave's, and a wave's more
constexpr double kLog2E = 1.44269504088896340736, kLn2 = 0.693147180559945309417;

struct Args {
  const void* x;
  const long long* tokens;
  float *logprobs, *entropy, *top_logprobs;
  long long* top_indices;
  double* stats;     // [rows][parts][3]
  uint64_t* keys;    // [rows][parts][top]
  long long stride;  // of rows, in elements
  long long rows;
  int n, top, parts, part;  // elements of a part, a multiple of 8
};

// A lane's, a part's or a row's sums.
struct Sums {
  double m, s, w;
};
// What the sums are when their elements' largest becomes `d` (0 or less) further from the reference. A lane's, once or
// more as it goes over a row, with an exponential in fp32: it counts as an element's does.
template <typename R> __device__ __forceinline__ void shift(double& s, double& w, R d) {
  const R t = d * (R)kLog2E;
  R f;
  if constexpr (sizeof(R) == 4) f = __builtin_amdgcn_exp2f(t);
  else f = exp2(t);
  w = f == (R)0 ? 0.0 : (w + s * (double)t) * (double)f;
  s = s * (double)f;
}
__device__ __forceinline__ uint64_t from_lane(uint64_t u, int lane) {
  const uint32_t lo = (uint32_t)rw::from_lane((int)(uint32_t)u, lane), hi = (uint32_t)rw::from_lane((int)(u >> 32), lane);
  return (uint64_t)hi << 32 | lo;
}
// Over the wave's lanes, in a fixed order: each is moved to the largest once, and then they are added. (m is an element, or
// minus infinity where there is none.)
__device__ __forceinline__ Sums wave_sums(float m, double s, double w) {
  const float most = wave_max(m);
  if (s != 0.0) shift(s, w, (double)m - (double)most);
  return {(double)most, wave_sum(s), wave_sum(w)};
}

// A value's place in the order, and back; an element's key (0: none).
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return __builtin_bit_cast(float, order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) { return (uint64_t)order_of(x) << 32 | ~index; }

template <int D> __device__ __forceinline__ uint32_t across_lanes(uint32_t v) { return across<D>(v); }
template <int D> __device__ __forceinline__ uint64_t across_lanes(uint64_t v) {
  return (uint64_t)across<D>((uint32_t)(v >> 32)) << 32 | across<D>((uint32_t)v);
}
// One step of a network: lanes l and l ^ D keep the lesser (l & D clear: `up`, the greater) and the other of theirs.
template <int D, typename K> __device__ __forceinline__ K step(K v, int lane, bool up) {
  const K other = across_lanes<D>(v);
  return ((lane & D) == 0) == up == (v > other) ? v : other;
}
template <int D, typename K> __device__ __forceinline__ K steps(K v, int lane, bool up) {
  v = step<D>(v, lane, up);
  if constexpr (D > 1) v = steps<D / 2>(v, lane, up);
  return v;
}
// The wave's keys sorted, the least in lane 0.
template <int SIZE = 2, typename K> __device__ __forceinline__ K sorted(K v, int lane) {
  v = steps<SIZE / 2>(v, lane, SIZE < kWave && (lane & SIZE) != 0);
  if constexpr (SIZE < kWave) v = sorted<2 * SIZE>(v, lane);
  return v;
}
// The 64 largest of a list (the largest in lane 0) and of keys sorted the other way round, as a list.
__device__ __forceinline__ uint64_t merged(uint64_t list, uint64_t keys, int lane) {
  return steps<kWave / 2>(list > keys ? list : keys, lane, true);
}

// The largest; NaN where one is (maximum, not fmax: it needs no copies of what may be a signaling NaN, and three numbers
// take one instruction).
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }
template <int V> __device__ __forceinline__ float most_of(const float* f) {
  float m = f[0];
#pragma unroll
  for (int e = 1; e < V; ++e) m = larger(m, f[e]);
  return m;
}

// A value that k of the wave's lanes reach, by halving what is between the least and the largest: one vector comparison to
// a step. Eight leave a 256th of it; sorting the wave would be exact and cost some 120 instructions.
__device__ __forceinline__ float least_of(float v, int k) {
  const uint32_t order = order_of(v);
  uint32_t lo = __builtin_amdgcn_readfirstlane(order_of(-wave_max(-v)));  // k lanes reach it
  uint32_t hi = __builtin_amdgcn_readfirstlane(order_of(wave_max(v)));
#pragma unroll 1
  for (int i = 0; i < 8 && lo < hi; ++i) {
    const uint32_t middle = hi - (hi - lo) / 2;
    if (__popcll(__ballot(order >= middle)) >= k) lo = middle;
    else hi = middle - 1;
  }
  return value_of(lo);
}

// The bits of minus infinity where a row has no element.
template <typename T> constexpr uint32_t kNothing = 0xff800000u;
template <> constexpr uint32_t kNothing<BF16> = 0xff80ff80u;
template <> constexpr uint32_t kNothing<F16> = 0xfc00fc00u;

// Elements at ... + V - 1 of a row's end, those from `end` on as nothing.
template <typename T>
__device__ __forceinline__ u32x4 some_of(const char* row, int at, int end) {
  u32x4 r = {kNothing<T>, kNothing<T>, kNothing<T>, kNothing<T>};
  if (at + T::V <= end) {
    r = load16_at<true>(row, (uint32_t)at * (uint32_t)T::bytes);
  } else if (at < end) {
#pragma unroll
    for (int e = 0; e < T::V; ++e) {
      if (at + e >= end) continue;
      if constexpr (T::bytes == 4) {
        r[e] = reinterpret_cast<const uint32_t*>(row)[at + e];
      } else {
        const uint32_t u = reinterpret_cast<const uint16_t*>(row)[at + e];
        r[e / 2] = e % 2 ? (r[e / 2] & 0xffffu) | u << 16 : (r[e / 2] & 0xffff0000u) | u;
      }
    }
  }
  return r;
}

// A wave's list of the largest elements that it has met.
struct List {
  uint64_t key;     // lane i: the i-th largest
  uint64_t last;    // the k-th, 0 where there are fewer
  int vectors;      // in the buffer
};
struct Buffer {
  u32x4 vector[kBuffer];
  uint64_t key[kBuffer];
  int at[kBuffer];
};

__device__ __forceinline__ int rank_in(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// The buffer's vectors taken apart and their elements above the list's last merged with it.
template <typename T>
__device__ __forceinline__ void empty_buffer(List& list, Buffer& b, int k, int n, int lane) {
  wave_lds_sync();
  int keys = 0;
  for (int first = 0; first < list.vectors; first += kWave) {
    const bool mine = first + lane < list.vectors;
    float f[T::V];
    unpack<T>(b.vector[first + lane], f);
    const int at = b.at[first + lane];
#pragma unroll
    for (int e = 0; e < T::V; ++e) {
      const uint64_t key = key_of(f[e], (uint32_t)(at + e));
      const bool wanted = mine && at + e < n && key > list.last;
      const uint64_t mask = __ballot(wanted);
      if (mask == 0) continue;
      if (wanted) b.key[keys + rank_in(mask)] = key;
      keys += __popcll(mask);
      wave_lds_sync();
      const bool end = e == T::V - 1 && first + kWave >= list.vectors;
      if (keys < kWave && !end) continue;
      list.key = merged(list.key, sorted(lane < keys ? b.key[lane] : 0, lane), lane);
      list.last = from_lane(list.key, k - 1);
      const uint64_t more = b.key[kWave + lane];
      wave_lds_sync();
      keys = keys > kWave ? keys - kWave : 0;
      if (lane < keys) b.key[lane] = more;
      wave_lds_sync();
    }
  }
  if (keys) {
    list.key = merged(list.key, sorted(lane < keys ? b.key[lane] : 0, lane), lane);
    list.last = from_lane(list.key, k - 1);
    wave_lds_sync();
  }
  list.vectors = 0;
}

// A row's token and its logit (0 of a token outside the row).
struct Asked {
  long long token;
  float logit;
};
template <typename T> __device__ __forceinline__ Asked asked(const Args& a, long long row) {
  const long long token = a.tokens[row], at = token >= 0 && token < a.n ? token : 0;
  return {token, load_elem<T>(static_cast<const char*>(a.x) + T::bytes * (row * a.stride), at)};
}
// A row's results from its sums and its list.
__device__ __forceinline__ void conclude(const Args& a, long long row, const Asked& of, const Sums& sums, uint64_t key,
                                         int lane) {
  const bool any = sums.s > 0.0 && sums.s < INFINITY;  // else a NaN, a positive infinity, or nothing above a negative one
  const double total = log(sums.s), none = __builtin_nan("");
  const auto log_of = [&](float x) { return (double)x - sums.m - total; };
  if (lane == 0) {
    const double p = any && of.token < a.n ? log_of(of.logit) : none;
    a.logprobs[row] = of.token < 0 ? 0.0f : (float)p;
    a.entropy[row] = (float)(any ? total - sums.w / sums.s * kLn2 : none);
  }
  if (lane < a.top) {
    a.top_logprobs[row * a.top + lane] = (float)(any ? log_of(value_of((uint32_t)(key >> 32))) : none);
    a.top_indices[row * a.top + lane] = any ? (long long)~(uint32_t)key : -1;
  }
}

// What a lane's fp32 sum of e^d over its elements of the trip at `from`, against their largest m, lost.
template <typename T>
__device__ __forceinline__ double lost(const char* row, int from, int end, float m, int lane) {
  u32x4 raw[kUnroll];
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) raw[j] = some_of<T>(row, from + (j * kWave + lane) * T::V, end);
  float sum = 0.0f;
  double exact = 0.0;
#pragma unroll
  for (int j = 0; j < kUnroll; ++j) {
    float f[T::V];
    unpack<T>(raw[j], f);
#pragma unroll
    for (int e = 0; e < T::V; ++e) {
      const float p = __builtin_amdgcn_exp2f((f[e] - m) * (float)kLog2E);
      sum += p;
      exact += (double)p;
    }
  }
  return exact - (double)sum;
}
// Where a wave's sum is below this the trip of its largest is gone over again: above, 2^-20 that 32 elements lose are 2^-16 of
// what is left.
constexpr double kSure = 1.0 + 0x1p-4;

template <typename T, bool TOP>
__global__ void __launch_bounds__(kWaves* kWave) score(Args a) {
  constexpr int V = T::V, U = kUnroll, trip = U * kWave * V;
  __shared__ Buffer buffers[TOP ? kWaves : 1];
  __shared__ Sums all[kWaves];
  __shared__ uint64_t lists[TOP ? kWaves * kWave : 1];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  const long long group = rw_host::workgroup();
  long long row = group;
  int part = 0;
  if (a.parts > 1) row = (unsigned)group / (unsigned)a.parts, part = (int)((unsigned)group % (unsigned)a.parts);
  if (row >= a.rows) return;
  const char* x = static_cast<const char*>(a.x) + T::bytes * (row * a.stride);
  const int begin = part * a.part, end = a.n - begin < a.part ? a.n : begin + a.part;
  Buffer& buffer = buffers[TOP ? wave : 0];
  List list = {0, 0, 0};
  float m = -INFINITY;
  double s = 0.0, w = 0.0;
  int met = 0;              // the trip in which the lane met m
  float limit = -INFINITY;  // of the list: vectors above it are wanted
  bool also = true;         // and those that reach it
  int trips = 0, next = 1;  // this many behind; the limit is looked for at
  for (int from = begin + wave * trip; from < end; from += kWaves * trip) {
    u32x4 raw[U];
    if (from + trip <= end) {
#pragma unroll
      for (int j = 0; j < U; ++j)
        raw[j] = load16_at<true>(x, (uint32_t)(from + (j * kWave + lane) * V) * (uint32_t)T::bytes);
    } else {
#pragma unroll
      for (int j = 0; j < U; ++j) raw[j] = some_of<T>(x, from + (j * kWave + lane) * V, end);
    }
    float most[U], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float f[V];
      unpack<T>(raw[j], f);
      most[j] = most_of<V>(f);
      top = larger(top, most[j]);
    }
    if (__ballot(!(top <= m))) {
      if (!(top <= m)) {
        if (s != 0.0) shift(s, w, m - top);
        m = top;
        met = from;
      }
    }
    const float at = m > -INFINITY ? m : 0.0f;
    float trip_s = 0.0f, trip_w = 0.0f;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float f[V];
      unpack<T>(raw[j], f);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float t = (f[e] - at) * (float)kLog2E, p = __builtin_amdgcn_exp2f(t);
        trip_s += p;
        trip_w = __builtin_fmaf(p, fmaxf(t, -1000.0f), trip_w);  // 0 of what is hidden, not 0 times infinity
      }
    }
    s += (double)trip_s;
    w += (double)trip_w;
    if constexpr (TOP) {
      if (also && ++trips == next) {
        next *= 2;
        const float least = least_of(m, a.top);
        if (least > limit) limit = least, also = true;
      }
      if (__ballot(top > limit || (also && top >= limit)) == 0) continue;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int v = from + (j * kWave + lane) * V;
        const bool wanted = (most[j] > limit || (also && most[j] >= limit)) && v < end;
        const uint64_t mask = __ballot(wanted);
        if (mask == 0) continue;
        if (wanted) {
          const int to = list.vectors + rank_in(mask);
          buffer.vector[to] = raw[j];
          buffer.at[to] = v;
        }
        list.vectors += __popcll(mask);
        if (list.vectors < kWave) continue;
        empty_buffer<T>(list, buffer, a.top, end, lane);
        // what is still to come has larger indices, so it has to be above the last to displace it (as +0 is above -0)
        const uint32_t order = (uint32_t)(list.last >> 32);
        const float last = value_of(order);
        if (list.last && last >= limit) limit = last, also = order == order_of(-0.0f);
      }
    }
  }
  if constexpr (TOP) {
    if (list.vectors) empty_buffer<T>(list, buffer, a.top, end, lane);
    lists[wave * kWave + lane] = list.key;
  }
  Sums mine = wave_sums(m, s, w);
  if (__builtin_amdgcn_readfirstlane(mine.s > 0.0 && mine.s < kSure)) {
    double more = 0.0;
    if (m == (float)mine.m) more = lost<T>(x, met, end, m, lane);
    mine.s += wave_sum(more);
  }
  if (lane == 0) all[wave] = mine;
  __syncthreads();
  if (wave) return;
  const Sums& of = all[lane < kWaves ? lane : 0];
  const Sums sums = wave_sums(lane < kWaves ? (float)of.m : -INFINITY, lane < kWaves ? of.s : 0.0, lane < kWaves ? of.w : 0.0);
  uint64_t key = list.key;
  if constexpr (TOP)
    for (int i = 1; i < kWaves; ++i) key = merged(key, lists[i * kWave + kWave - 1 - lane], lane);
  if (a.parts == 1) {
    conclude(a, row, asked<T>(a, row), sums, key, lane);
  } else {
    const long long at = row * a.parts + part;
    if (lane == 0) a.stats[3 * at] = sums.m, a.stats[3 * at + 1] = sums.s, a.stats[3 * at + 2] = sums.w;
    if (lane < a.top) a.keys[at * a.top + lane] = key;
  }
}

// A wave joins a row's parts.
template <typename T>
__global__ void __launch_bounds__(kWave) join(Args a) {
  const long long row = rw_host::workgroup();
  const int lane = lane_id();
  if (row >= a.rows) return;
  const Asked of = asked<T>(a, row);
  Sums mine = {-INFINITY, 0.0, 0.0};
  if (lane < a.parts) {
    const double* p = a.stats + 3 * (row * a.parts + lane);
    mine = {p[0], p[1], p[2]};
  }
  const uint64_t* keys = a.keys + row * a.parts * a.top;
  uint64_t key = lane < a.top ? keys[lane] : 0;
  constexpr int batch = 8;  // parts to a trip to memory
  const int at = kWave - 1 - lane;
  for (int p = 1; a.top && p < a.parts; p += batch) {
    uint64_t next[batch];
#pragma unroll
    for (int i = 0; i < batch; ++i) next[i] = at < a.top && p + i < a.parts ? keys[(p + i) * a.top + at] : 0;
#pragma unroll
    for (int i = 0; i < batch; ++i)
      if (p + i < a.parts) key = merged(key, next[i], lane);
  }
  conclude(a, row, of, wave_sums((float)mine.m, mine.s, mine.w), key, lane);
}

// ---- host side ------------------------------------------------------------------------------------------------------

enum { kTuneParts = 0 };

bool sizes_ok(long long rows, long long vocabulary, int top, int dtype) {
  return rows <= 1LL << 31 && vocabulary >= 1 && vocabulary <= 1 << 28 && top >= 0 && top <= kMostTop &&
         top <= vocabulary && dtype >= 0 && dtype <= 2;
}

void cut(long long rows, long long vocabulary, int dtype, int& parts, int& part) {
  const long long trip = (long long)kUnroll * kWave * (dtype == 0 ? 4 : 8) * kWaves;
  long long n = rw_host::tune_get(kTuneParts);
  if (n <= 0) {
    // two workgroups to a CU, of two trips of each wave at least: 64 rows of 128256 bf16 19.3 us in 8 parts, 23 in 4, 40 in
    // one; 700 of 49999 fp32 25.6 in one, 28.6 in 2
    n = (2LL * rw_host::device_cus() + rows - 1) / rows;
    const long long most = (vocabulary + 2 * trip - 1) / (2 * trip);
    if (n > most) n = most;
  }
  n = n < 1 ? 1 : n > kMostParts ? kMostParts : n;
  part = (int)(((vocabulary + n - 1) / n + 7) / 8 * 8);
  parts = (int)((vocabulary + part - 1) / part);
  if (rows * parts > INT_MAX) parts = 1, part = (int)((vocabulary + 7) / 8 * 8);  // a workgroup's number in 32 bits
}

template <typename T>
int launch_type(const Args& a, hipStream_t stream) {
  const dim3 grid = rw_host::grid_of(a.rows * a.parts), threads(kWaves * kWave);
  if (a.top) hipLaunchKernelGGL((score<T, true>), grid, threads, 0, stream, a);
  else hipLaunchKernelGGL((score<T, false>), grid, threads, 0, stream, a);
  const int err = (int)hipGetLastError();
  if (err || a.parts == 1) return err;
  hipLaunchKernelGGL((join<T>), rw_host::grid_of(a.rows), dim3(kWave), 0, stream, a);
  return (int)hipGetLastError();
}

}  // namespace

extern "C" long long token_logprobs_work(long long rows, long long vocabulary, int top, int dtype) {
  if (rows <= 0) return 0;
  if (!sizes_ok(rows, vocabulary, top, dtype)) return -1;
  int parts, part;
  cut(rows, vocabulary, dtype, parts, part);
  return parts == 1 ? 0 : rows * parts * (3LL + top) * 8;
}

extern "C" int token_logprobs_launch(const void* logits, const void* tokens, float* logprobs, float* entropy,
                                     float* top_logprobs, void* top_indices, void* work, long long work_bytes,
                                     long long row_stride, long long rows, long long vocabulary, int top, int dtype,
                                     hipStream_t stream) {
  if (rows <= 0) return rw_host::kOk;
  const uintptr_t size = dtype == 0 ? 4 : 2;
  if (!sizes_ok(rows, vocabulary, top, dtype) || !logits || reinterpret_cast<uintptr_t>(logits) % size || !tokens ||
      !logprobs || !entropy || (top && (!top_logprobs || !top_indices)))
    return rw_host::kInvalid;
  Args a{};
  cut(rows, vocabulary, dtype, a.parts, a.part);
  const long long bytes = a.parts == 1 ? 0 : rows * a.parts * (3LL + top) * 8;
  if (bytes && (!work || reinterpret_cast<uintptr_t>(work) % 8 || work_bytes < bytes)) return rw_host::kInvalid;
  a.x = logits;
  a.tokens = static_cast<const long long*>(tokens);
  a.logprobs = logprobs, a.entropy = entropy, a.top_logprobs = top_logprobs;
  a.top_indices = static_cast<long long*>(top_indices);
  a.stats = static_cast<double*>(work);
  a.keys = reinterpret_cast<uint64_t*>(a.stats + 3 * rows * a.parts);
  a.stride = row_stride;
  a.rows = rows;
  a.n = (int)vocabulary;
  a.top = top;
  return dtype == 0 ? launch_type<F32>(a, stream) : dtype == 1 ? launch_type<BF16>(a, stream)
                                                               : launch_type<F16>(a, stream);
}

extern "C" int token_logprobs_tune(int slot, int value) { return rw_host::tune_set(slot, value); }
