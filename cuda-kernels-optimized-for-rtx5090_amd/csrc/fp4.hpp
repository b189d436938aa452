// Keys and values in 4 bits: e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, the first of the
// two in the low half, and a power of two to every 32 of them, 2^(byte - 127), 255 for a group that stands for NaN. These
// are the forms that gfx950 converts itself (v_cvt_scalef32_pk_*).
#pragma once

#include "matrix.hpp"

namespace rw {

constexpr int kShared = 32;                 // elements that share a scale
constexpr uint32_t kNanScale = 255;

// The largest scale that is written: 6 times it is finite in the type.
template <typename T> constexpr int kMostScale = 252;
template <> constexpr int kMostScale<F16> = 140;

// The scale of a group from the largest of its elements' magnitudes, as the bits of an fp32 number: the least power of
// two that leaves it below 7, which 6 is within half a step of (so no element is further from its code than half a step
// of the coarsest). What is too large for the type's largest scale is cut to 6 times it; an infinity or a NaN makes the
// group NaN.
__device__ __forceinline__ int scale_of(uint32_t most, int limit) {
  if (most >= 0x7f800000u) return (int)kNanScale;
  const int e = (int)((most + 0x200000u) >> 23) - 2;
  return e < 1 ? 1 : e > limit ? limit : e;
}
__device__ __forceinline__ float power_of(uint32_t scale) { return __builtin_bit_cast(float, scale << 23); }
// Scales above the largest that is written read as NaN, so that what is read in bf16 is finite or NaN (fp16, whose largest
// written scale is lower, overflows to infinity where a cache was written in bf16).
__device__ __forceinline__ uint32_t scale_in(uint32_t byte) { return byte > 252u ? kNanScale : byte; }

// The two elements of byte BYTE of `codes`, packed; the codes of a packed pair put into byte BYTE of `old` (the nearest,
// ties to the even code, the largest for what is beyond). Both exact against the definition over all codes and all
// 2^16 patterns of both types, and v_cvt_scalef32_pk_*'s scale of NaN gives NaN.
template <int BYTE> struct Fp4 {
  static __device__ __forceinline__ uint32_t to_bf16(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, BYTE));
  }
  static __device__ __forceinline__ uint32_t to_f16(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, BYTE));
  }
  static __device__ __forceinline__ uint32_t of_bf16(uint32_t old, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2, pair), scale, BYTE);
  }
  static __device__ __forceinline__ uint32_t of_f16(uint32_t old, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(f16x2, pair), scale, BYTE);
  }
};
// The 8 elements of 4 bytes of codes, and back.
template <typename T> __device__ __forceinline__ u32x4 widen4(uint32_t codes, float scale);
template <> __device__ __forceinline__ u32x4 widen4<BF16>(uint32_t codes, float scale) {
  return (u32x4){Fp4<0>::to_bf16(codes, scale), Fp4<1>::to_bf16(codes, scale), Fp4<2>::to_bf16(codes, scale),
                 Fp4<3>::to_bf16(codes, scale)};
}
template <> __device__ __forceinline__ u32x4 widen4<F16>(uint32_t codes, float scale) {
  return (u32x4){Fp4<0>::to_f16(codes, scale), Fp4<1>::to_f16(codes, scale), Fp4<2>::to_f16(codes, scale),
                 Fp4<3>::to_f16(codes, scale)};
}
template <typename T> __device__ __forceinline__ uint32_t narrow4(const u32x4& x, float scale);
template <> __device__ __forceinline__ uint32_t narrow4<BF16>(const u32x4& x, float scale) {
  const uint32_t a = Fp4<1>::of_bf16(Fp4<0>::of_bf16(0u, x[0], scale), x[1], scale);
  return Fp4<3>::of_bf16(Fp4<2>::of_bf16(a, x[2], scale), x[3], scale);
}
template <> __device__ __forceinline__ uint32_t narrow4<F16>(const u32x4& x, float scale) {
  const uint32_t a = Fp4<1>::of_f16(Fp4<0>::of_f16(0u, x[0], scale), x[1], scale);
  return Fp4<3>::of_f16(Fp4<2>::of_f16(a, x[2], scale), x[3], scale);
}

}  // namespace rw
