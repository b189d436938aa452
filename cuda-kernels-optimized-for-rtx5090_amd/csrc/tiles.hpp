// Tiles of attention on the 32x32x16 products, for kernels whose keys come by slices of 32 through LDS.
//
// The products are transposed, so that a lane keeps one row throughout: S^T = K Q^T has a key per matrix row and a
// query per column, its result puts 16 keys of one query into a lane, and these are, packed in pairs, the B operand of
// O^T = V^T P^T without a move between lanes (the order of the 16 keys of a product is free, and V's transposing LDS
// read takes them in the same order). So maximum, sum and rescaling are a lane's own, but for one exchange of the two
// halves of the wave. Softmax in base 2 with the scale folded into the exponent; the reference point moves only when a
// row's maximum has grown by 2^8 (no result depends on it but for rounding, and the sum of values is rescaled only
// then).
#pragma once

#include "matrix.hpp"

#pragma clang fp contract(off)

namespace rw {

constexpr int kRows = 32;   // query rows of a wave: the columns of a product
constexpr int kKeys = 32;   // keys of a slice: the rows of a product
constexpr float kGrow = 8.0f;

// 2^kBias is the weight of a row's reference point: fp16 weights start 2^7 up, so that those down to 2^-21 of the
// largest stay normal numbers; at most 2^(7 + 8).
template <typename T> constexpr float kBias = 0.0f;
template <> constexpr float kBias<F16> = 7.0f;

template <int D> struct Dims {
  static constexpr int chunks = D <= 64 ? 8 : D <= 128 ? 16 : 32;  // 16-byte places of a row in LDS
  static constexpr int used = D / 8;                               // of these hold the row
  static constexpr int row = chunks * 16;
  static constexpr int slice = kKeys * row;                        // bytes of a slice of K or V
  static constexpr int steps = D / 16;                             // products of a slice's scores
  static constexpr int blocks = (D + 31) / 32;                     // 32-wide blocks of the values
};

// 32 rows of a wave.
template <typename T, int D>
struct Tile {
  u32x4 q[Dims<D>::steps];
  f32x16 o[Dims<D>::blocks];
  float m, l;  // reference point; sum of weights over this lane's half of the keys
};
constexpr float kNone = -3.0e38f;  // the reference point of a row that has met no key

// Where chunk c of row r of a slice lies: XORed with the row, so that the lanes of a read (8 rows' same chunk for K, 4
// rows' same pair of chunks for V) meet different banks.
template <int D> __device__ __forceinline__ int k_place(int r, int c) {
  return r * Dims<D>::row + ((c ^ r) & (Dims<D>::chunks - 1)) * 16;
}
template <int D> __device__ __forceinline__ int v_place(int r, int c) {
  return r * Dims<D>::row + ((c ^ (2 * r)) & (Dims<D>::chunks - 1)) * 16;
}

// Where a lane reads step c of a slice's keys, the scores' left operand.
template <int D>
__device__ __forceinline__ lds_ptr keys_at(char* k, int c, int lane) {
  return in_lds(k) + k_place<D>(lane & 31, 2 * c + (lane >> 5));
}

// The scores of a slice of 32 keys, 16 of them in each lane.
template <typename T, int D>
__device__ __forceinline__ void scores(f32x16& s, const Tile<T, D>& t, const u32x4* kf) {
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
  for (int c = 0; c < Dims<D>::steps; ++c) s = product32<T>(kf[c], t.q[c], s);
}

// The largest of a lane's 16 scores.
__device__ __forceinline__ float largest(const f32x16& s) {
  float top = s[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
  return top;
}
// Moves the row's reference point where its largest score asks for it. Returns what its sum of values so far is to be
// multiplied by.
template <typename T, int D>
__device__ __forceinline__ float refer(Tile<T, D>& t, float top, float scale) {
  top = max_of_halves(top) * scale - kBias<T>;
  const float m = top > t.m + kGrow ? top : t.m, f = __builtin_amdgcn_exp2f(t.m - m);
  t.m = m;
  t.l *= f;
  return f;
}
// The weights of scores 2 i and 2 i + 1, rounded to 16 bits: the matrix core's operands are both of V's type, and fp32
// weights would take two products, a high and a low half. They are summed as rounded, so that the weights that multiply
// the values add up to what divides them. Against the formula in 64 bits the output is then off by 0.0023 in bf16 and
// 0.00029 in fp16 (relative, over 64 tokens behind 8192 keys and 33 x 5 behind 4999), where its own rounding alone is
// 0.0017 and 0.00021. Maxima, sums and the sums of values are fp32.
template <typename T, int D>
__device__ __forceinline__ void weigh(Tile<T, D>& t, const f32x16& s, float scale, int i, u32x4* p) {
  uint32_t two = pack2<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i], scale, -t.m)),
                          __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + 1], scale, -t.m)));
  settle(two);
  t.l = add_pair<T>(two, t.l);
  p[i / 4][i % 4] = two;
}

template <typename T, int D>
__device__ __forceinline__ void rescale(Tile<T, D>& t, float f) {
  if (__ballot(f != 1.0f) == 0) return;
#pragma unroll
  for (int d = 0; d < Dims<D>::blocks; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) t.o[d][i] *= f;
}

// Which values the 16 rows n (0 or 1) of block d of the sums are: for 128 values and more the two are half the row
// apart, so that the 32 lanes of a read meet all banks (with neighbours they met half of them twice).
template <int D> __device__ __forceinline__ int value_of(int d, int n) {
  return D % 128 == 0 ? 16 * d + D / 2 * n : 32 * d + 16 * n;
}

// Where a lane reads block d of a slice's values from row `first` on: of the keys 16 j ..., first 16 j and 16 j + 8.
template <int D>
__device__ __forceinline__ lds_ptr values_at(char* v, int first, int d, int lane) {
  const int i16 = lane & 15, n = (lane >> 4) & 1;
  return in_lds(v) + v_place<D>(first + 4 * (lane >> 5) + (i16 >> 2), value_of<D>(d, n) / 8 + ((i16 & 3) >> 1)) +
         8 * (lane & 1);
}
// Transposed, from both, the left operand of the weighted sums.
__device__ __forceinline__ u32x4 read_values(lds_ptr lo, lds_ptr hi) {
  const u32x2 a = lds_column(lo), b = lds_column(hi);
  return (u32x4){a.x, a.y, b.x, b.y};
}

// Where lane (r, h)'s four sums i of block d start among the values.
template <int D> __device__ __forceinline__ int sums_at(int d, int i, int h) {
  return value_of<D>(d, i / 2) + 8 * (i % 2) + 4 * h;
}

}  // namespace rw
