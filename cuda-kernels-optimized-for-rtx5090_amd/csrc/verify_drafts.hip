// Verification of drafted tokens against a target model's probabilities, and the draw behind the kept ones
// (include/verify_drafts.h has the rule). Of the drafts + 1 rows of a sequence only the drafted entries and ONE row
// (with the draft's beside it where a draft was refused) matter, so the kernel finds the row first and reads only that.
//
// Every wave decides the row for itself (a draft per lane, a ballot), which saves a launch or a barrier for a few
// hundred bytes read again. A row is split into at most 1024 segments of a whole number of 16-byte vectors per wave;
// a wave adds up its segments in fp64 (the weights are differences of close values, and the draw's threshold has to
// fall on the same side of a running sum whatever the split: sums of 2^18 fp32 terms in fp32 would move it by many
// entries). Where a row has several workgroups, the one that arrives last finds the segment of the threshold from the
// segments' sums (the others' handed over by agent-scope stores, a wait for them, an arrival count and agent-scope
// loads), else the only one does; it reads that segment once more for the entry. The sums' order is fixed by the sizes,
// so results do not depend on the split or on timing.
//
// Between memory and its chain: the drafted entries, the row, the arrival and the segment's second read are a trip to
// memory each, 5.8 us for one row of 50000. 64 sequences over 128256 in fp32, some with the draft's row, are 59 MB (9.5
// us at a copy's rate) and take 15.2 us.
#include <climits>

#include "host.hpp"
#include "rowwise.hpp"

#pragma clang fp contract(off)

using namespace rw;

namespace {

constexpr int kSegments = 1024;
constexpr int kPieces = 4;  // 16-byte vectors per lane of a shortest segment

struct Args {
  const void* target;
  const void* draft;
  const long long* tokens;
  const int* lens;
  const float* uniforms;
  long long* out;
  long long* accepted;
  uint64_t* work;  // doubles' bits
  unsigned* counters;
  long long tb, ts, db, ds;  // element strides: batch and row
  int drafts, vocabulary, blocks;
  unsigned groups;       // workgroups: rows times `blocks`
  int segments, pieces;  // pieces: 16-byte vectors per lane of a segment
};

// A row's weights: target entries, less the draft's (DRAFT, where q is there) or without one token (where it is not
// -1).
struct Row {
  const char* p;
  const char* q;
  int without;
};

// The weights of one 16-byte vector's entries from `first` on, loaded and then formed, so that loads can run ahead.
template <typename T, bool DRAFT>
struct Entries {
  u32x4 p, q;
  __device__ __forceinline__ void load(const Row& r, int first, int n) {
    if (first + T::V <= n) {
      p = load16_at<false>(r.p, (uint32_t)first * T::bytes);
      if (DRAFT && r.q) q = load16_at<false>(r.q, (uint32_t)first * T::bytes);
    } else {
      float x[T::V], y[T::V];
#pragma unroll
      for (int e = 0; e < T::V; ++e) {
        x[e] = first + e < n ? load_elem<T>(r.p, first + e) : 0.0f;
        y[e] = DRAFT && r.q && first + e < n ? load_elem<T>(r.q, first + e) : 0.0f;
      }
      p = pack<T>(x);  // exact: they are the format's own values
      q = pack<T>(y);
    }
  }
  // (the larger of NaN and 0 is 0)
  __device__ __forceinline__ void weights(const Row& r, int first, double* w) const {
    float x[T::V], y[T::V];
    unpack<T>(p, x);
    if (DRAFT && r.q) {
      unpack<T>(q, y);
#pragma unroll
      for (int e = 0; e < T::V; ++e) w[e] = __builtin_fmax((double)x[e] - (double)y[e], 0.0);
    } else {
#pragma unroll
      for (int e = 0; e < T::V; ++e) w[e] = (double)fmaxf(x[e], 0.0f);
    }
    if (!DRAFT && (unsigned)(r.without - first) < (unsigned)T::V) {
#pragma unroll
      for (int e = 0; e < T::V; ++e)
        if (first + e == r.without) w[e] = 0.0;
    }
  }
};

// The sum of the lanes up to and including this one: within rows of 16 lanes by DPP shifts, then the rows before.
__device__ __forceinline__ double running_sum(double v, int lane) {
  v += dpp<0x111>(v);
  v += dpp<0x112>(v);
  v += dpp<0x114>(v);
  v += dpp<0x118>(v);
  const double a = readlane(v, 15), b = a + readlane(v, 31), c = b + readlane(v, 47);
  const int row = lane >> 4;
  return v + (row == 0 ? 0.0 : row == 1 ? a : row == 2 ? b : c);
}

// A segment's sum, in every lane.
template <typename T, bool DRAFT>
__device__ __forceinline__ double segment_sum(const Row& r, const Args& a, int segment, int lane) {
  const int piece = kWave * T::V;
  const long long first = (long long)segment * a.pieces * piece;
  double sum = 0.0;
  for (int i = 0; i < a.pieces; i += kPieces) {
    Entries<T, DRAFT> x[kPieces];
    int at[kPieces];
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const long long begin = first + (long long)(i + k) * piece + lane * T::V;
      at[k] = begin < a.vocabulary ? (int)begin : a.vocabulary;
      x[k].load(r, at[k], a.vocabulary);
    }
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      double w[T::V];
      x[k].weights(r, at[k], w);
#pragma unroll
      for (int e = 0; e < T::V; ++e) sum += w[e];
    }
  }
  return wave_sum(sum);
}

// The entry of the segment where the running sum, from `before`, first is above `level`; the segment's last positive
// entry where rounding leaves it below. A lane holds kPieces vectors in a row here, so that the entries are in order.
template <typename T, bool DRAFT>
__device__ __forceinline__ long long entry(const Row& r, const Args& a, int segment, double before, double level,
                                           int lane) {
  constexpr int N = kPieces * T::V;
  const long long first = (long long)segment * a.pieces * kWave * T::V;
  long long last = -1;
  for (int i = 0; i < a.pieces; i += kPieces) {
    const long long begin = first + ((long long)i * kWave + (long long)lane * kPieces) * T::V;
    Entries<T, DRAFT> x[kPieces];
    double w[N], sum = 0.0;
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const long long at = begin + k * T::V;
      x[k].load(r, at < a.vocabulary ? (int)at : a.vocabulary, a.vocabulary);
    }
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const long long at = begin + k * T::V;
      x[k].weights(r, at < a.vocabulary ? (int)at : a.vocabulary, w + k * T::V);
    }
    int positive = -1, found = -1;
#pragma unroll
    for (int e = 0; e < N; ++e) sum += w[e];
    const double through = running_sum(sum, lane);
    double run = before + (through - sum);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      run += w[e];
      const bool there = w[e] > 0.0;
      positive = there ? e : positive;
      found = found < 0 && there && run > level ? e : found;
    }
    const uint64_t hit = __ballot(found >= 0), any = __ballot(positive >= 0);
    const int l = hit ? __builtin_ctzll(hit) : any ? 63 - __builtin_clzll(any) : 0;
    const long long at = first + ((long long)i * kWave + (long long)l * kPieces) * T::V;
    if (hit) return at + __builtin_amdgcn_readlane(found, l);
    if (any) last = at + __builtin_amdgcn_readlane(positive, l);
    before += readlane(through, kWave - 1);
  }
  return last;
}

// From the segments' sums: the total, and the segment where the running sum first is above u * total with the sum
// before it. A level that rounding leaves above all running sums gives the last positive segment and no bound.
__device__ __forceinline__ double find_segment(const double* sums, int n, double u, int lane, int& segment,
                                               double& before, double& level) {
  const int each = (n + kWave - 1) / kWave, first = lane * each;
  double sum = 0.0;
  for (int i = 0; i < each; ++i) sum += first + i < n ? sums[first + i] : 0.0;
  const double through = running_sum(sum, lane);
  const double total = readlane(through, kWave - 1);
  level = u * total;
  double run = through - sum, at = 0.0;
  int found = -1, positive = -1;
  for (int i = 0; i < each; ++i) {
    const double s = first + i < n ? sums[first + i] : 0.0;
    if (s > 0.0) positive = first + i;
    if (found < 0 && s > 0.0 && run + s > level) found = first + i, at = run;
    run += s;
  }
  const uint64_t hit = __ballot(found >= 0), any = __ballot(positive >= 0);
  segment = -1;
  before = 0.0;
  if (hit) {
    const int l = __builtin_ctzll(hit);
    segment = __builtin_amdgcn_readlane(found, l);
    before = readlane(at, l);
  } else if (any) {
    segment = __builtin_amdgcn_readlane(positive, 63 - __builtin_clzll(any));
    level = INFINITY;
  }
  return total;
}

template <typename T, bool DRAFT, int WAVES>
__global__ void __launch_bounds__(WAVES* kWave) verify_rows(Args a) {
  __shared__ double sums[kSegments];
  __shared__ unsigned arrived;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
  const unsigned group = (unsigned)rw_host::workgroup();  // of at most 2^30, rounded up to a row of the grid
  if (blockIdx.y && group >= a.groups) return;            // (a grid of one row has no others)
  const long long b = group / (unsigned)a.blocks;
  const int block = (int)(group - b * a.blocks);
  const long long* tokens = a.tokens + b * a.drafts;
  const float* uniforms = a.uniforms + b * (a.drafts + 1);
  const char* target = static_cast<const char*>(a.target) + b * a.tb * T::bytes;
  const char* draft = static_cast<const char*>(a.draft) + (DRAFT ? b * a.db * T::bytes : 0);

  // tokens, uniforms and the count of drafts at once, then the drafted entries at once
  int n = a.lens ? a.lens[b] : a.drafts;
  n = n < 0 ? 0 : n < a.drafts ? n : a.drafts;
  int j = n;
  for (int i0 = 0; i0 < a.drafts && j == n; i0 += kWave) {
    const int i = i0 + lane;
    bool refused = false;
    if (i < a.drafts) {
      const long long x = tokens[i];
      const double u = (double)uniforms[i];
      double p = 0.0, q = 1.0;
      if (x >= 0 && x < a.vocabulary) {
        p = load_elem<T>(target + i * a.ts * T::bytes, x);
        if (DRAFT) q = load_elem<T>(draft + i * a.ds * T::bytes, x);
      }
      refused = i < n && !(u * q < p);
    }
    const uint64_t mask = __ballot(refused);
    if (mask) j = i0 + __builtin_ctzll(mask);
  }
  bool rest = j < n;  // the draw is from what the draft left
  Row row{target + j * a.ts * T::bytes, nullptr, -1};
  if (rest) {
    if (DRAFT) {
      row.q = draft + j * a.ds * T::bytes;
    } else {
      const long long x = tokens[j];
      row.without = x >= 0 && x < a.vocabulary ? (int)x : -1;
    }
  }

  const bool split = a.blocks > 1;
  uint64_t* work = split ? a.work + b * a.segments : nullptr;
  for (int s = block * WAVES + wave; s < a.segments; s += a.blocks * WAVES) {
    const double v = segment_sum<T, DRAFT>(row, a, s, lane);
    if (lane == 0) {
      if (split) {
        const uint64_t bits = __builtin_bit_cast(uint64_t, v);
        __hip_atomic_store(work + s, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      } else {
        sums[s] = v;
      }
    }
  }
  if (split) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the sums are at agent scope before the arrival counts
    __syncthreads();
    if (threadIdx.x == 0)
      arrived = __hip_atomic_fetch_add(a.counters + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived != (unsigned)a.blocks - 1) return;
    if (threadIdx.x == 0) __hip_atomic_store(a.counters + b, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int s = threadIdx.x; s < a.segments; s += WAVES * kWave) {
      const uint64_t bits = __hip_atomic_load(work + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      sums[s] = __builtin_bit_cast(double, bits);
    }
  }
  __syncthreads();

  const double u = uniforms[a.drafts];
  int segment;
  double before, level;
  const double total = find_segment(sums, a.segments, u, lane, segment, before, level);
  if (rest && !(total > 0.0)) {  // the draft left nothing: the target's own probabilities, by this workgroup alone
    row.q = nullptr;
    row.without = -1;
    __syncthreads();  // every wave has read the sums
    for (int s = wave; s < a.segments; s += WAVES) {
      const double v = segment_sum<T, DRAFT>(row, a, s, lane);
      if (lane == 0) sums[s] = v;
    }
    __syncthreads();
    find_segment(sums, a.segments, u, lane, segment, before, level);
  }
  if (wave != 0) return;
  const long long drawn = segment >= 0 ? entry<T, DRAFT>(row, a, segment, before, level, lane) : -1;
  long long* out = a.out + b * (a.drafts + 1);
  for (int i = lane; i <= a.drafts; i += kWave) out[i] = i < j ? tokens[i] : i == j ? drawn : -1;
  if (lane == 0) a.accepted[b] = j;
}

// ---- host side ------------------------------------------------------------------------------------------------------

constexpr int kFew = 4, kMany = 16;  // waves of a workgroup: of several to a row, of the only one

bool sizes_ok(long long batch, long long vocabulary, int dtype) {
  return batch <= (1 << 22) && vocabulary >= 1 && vocabulary <= (1 << 28) && (dtype == 0 || dtype == 1);
}

// A segment's 16-byte vectors per lane: as few as leave at most kSegments segments.
int pieces_of(long long vocabulary, int dtype) {
  const long long piece = kWave * (dtype == 0 ? F32::V : BF16::V);
  int pieces = kPieces;
  while ((vocabulary + pieces * piece - 1) / (pieces * piece) > kSegments) pieces *= 2;
  return pieces;
}

int segments_of(long long vocabulary, int dtype) {
  const long long length = (long long)pieces_of(vocabulary, dtype) * kWave * (dtype == 0 ? F32::V : BF16::V);
  return (int)((vocabulary + length - 1) / length);
}

template <typename T, bool DRAFT>
int launch_rows(const Args& a, bool many, hipStream_t stream) {
  const dim3 grid = rw_host::grid_of(a.groups), threads((many ? kMany : kFew) * kWave);
  if (many) hipLaunchKernelGGL((verify_rows<T, DRAFT, kMany>), grid, threads, 0, stream, a);
  else hipLaunchKernelGGL((verify_rows<T, DRAFT, kFew>), grid, threads, 0, stream, a);
  return (int)hipGetLastError();
}

}  // namespace

// About 2048 waves, eight of a CU: many rows by a workgroup of 16 waves each, which hands nothing over, few by several
// workgroups of four. One row of 50000: thirteen of 4 5.8 us, one of 16 7.7. At 64, 102, 103, 128 and 200 rows of one
// draft, one workgroup of 16 against the best of two to eight of 4 (us; the border is between 102 and 103):
//   fp32 128256, refused  17.6 15.9   27.8 21.7   27.8 22.2   30.5 28.0   39.7 41.7
//   fp32 128256, kept     14.7 12.5   14.9 14.4   15.0 14.4   15.8 15.9   20.9 22.4
//   bf16 128256, refused  15.9 13.5   15.9 15.0   16.5 15.4   16.9 16.5   22.2 23.2
//   bf16 128256, kept     12.9 10.6   13.0 11.4   13.0 11.5   14.0 12.4   14.3 15.5
//   fp32 50000, refused    9.8 10.5   11.0 12.3   11.1 12.3   12.3 13.9   16.4 17.6
//   bf16 50000, kept       9.6  9.0    9.6  9.6    8.7  9.4    9.8 10.3   10.3 11.5
// So long rows just above the border lose up to a quarter, short ones below it up to an eighth.
extern "C" long long verify_plan(long long batch, long long vocabulary, int dtype) {
  if (!sizes_ok(batch, vocabulary, dtype)) return -1;
  if (batch < 1) return 1;
  const long long most = (segments_of(vocabulary, dtype) + kFew - 1) / kFew;
  const long long want = 8LL * rw_host::device_cus() / batch / kFew;
  return want <= kMany / kFew ? 1 : want < most ? want : most;
}

// (the segments of a longer vocabulary may be fewer, since longer; the answer grows with the vocabulary all the same,
// so that a buffer for the largest sizes serves smaller ones)
extern "C" long long verify_work(long long batch, long long vocabulary, int dtype) {
  if (!sizes_ok(batch, vocabulary, dtype)) return -1;
  const long long shortest = (long long)kPieces * kWave * (dtype == 0 ? F32::V : BF16::V);
  const long long most = (vocabulary + shortest - 1) / shortest;
  return batch < 1 ? 0 : batch * (most < kSegments ? most : kSegments);
}

extern "C" int verify_launch(const void* target, const void* draft, const void* tokens, const void* lens,
                             const float* uniforms, void* out_tokens, void* accepted, void* work, void* counters,
                             const long long* strides, long long batch, int drafts, long long vocabulary, int dtype,
                             int blocks, hipStream_t stream) {
  if (batch <= 0) return rw_host::kOk;
  if (!sizes_ok(batch, vocabulary, dtype) || drafts < 0 || drafts > 65535 || blocks < 1 || blocks > 256 || !target ||
      (drafts && !tokens) || !uniforms || !out_tokens || !accepted || (blocks > 1 && (!work || !counters)))
    return rw_host::kInvalid;
  Args a{target, draft, (const long long*)tokens, (const int*)lens, uniforms, (long long*)out_tokens,
         (long long*)accepted, (uint64_t*)work, (unsigned*)counters};
  a.ts = a.ds = vocabulary;
  a.tb = (drafts + 1) * vocabulary;
  a.db = drafts * vocabulary;
  if (strides) a.tb = strides[0], a.ts = strides[1], a.db = strides[2], a.ds = strides[3];
  a.drafts = drafts;
  a.vocabulary = (int)vocabulary;
  a.blocks = blocks;
  a.groups = (unsigned)(batch * blocks);
  a.pieces = pieces_of(vocabulary, dtype);
  a.segments = segments_of(vocabulary, dtype);
  const bool many = blocks == 1 && a.segments > kFew;
  if (dtype == 0)
    return draft ? launch_rows<F32, true>(a, many, stream) : launch_rows<F32, false>(a, many, stream);
  return draft ? launch_rows<BF16, true>(a, many, stream) : launch_rows<BF16, false>(a, many, stream);
}
