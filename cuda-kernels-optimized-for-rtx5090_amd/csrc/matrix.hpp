// Matrix cores, transposing LDS reads and loads that go from memory to LDS without registers, for gfx950.
//
// Layouts of the 32x32x16 product, lane l with r = l % 32 and h = l / 32: A's row r and B's column r, both at the 8
// contraction indices 8 h ...; the result's column r at the rows 8 (i / 4) + 4 h + i % 4, i = 0..15.
#pragma once

#include "rowwise.hpp"

namespace rw {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

template <typename T>
__device__ __forceinline__ f32x16 product32(const u32x4& a, const u32x4& b, const f32x16& c);
template <>
__device__ __forceinline__ f32x16 product32<BF16>(const u32x4& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}
template <>
__device__ __forceinline__ f32x16 product32<F16>(const u32x4& a, const u32x4& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Within 16 lanes, lane i gives the address of 4 elements: row i / 4 of a 4 x 16 block, columns 4 (i % 4) ...; it gets
// column i of the block, its 4 rows.
__device__ __forceinline__ u32x2 lds_column(const char* at) {
  typedef __attribute__((address_space(3))) s16x4* ptr;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(uintptr_t)at));
}

// 16 bytes from a lane's own address to LDS at `at` + 16 * lane (`at` the same in the wave's lanes). Asynchronous:
// counted with the vector memory loads, which wait_loads() waits for.
__device__ __forceinline__ void load_to_lds(const void* from, char* at) {
  typedef const __attribute__((address_space(1))) void* gptr;
  typedef __attribute__((address_space(3))) void* lptr;
  __builtin_amdgcn_global_load_lds((gptr)(uintptr_t)from, (lptr)(uintptr_t)at, 16, 0, 0);
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// This wave's LDS reads are in registers.
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// v of lane `from` (any lane of the wave).
__device__ __forceinline__ int from_lane(int v, int from) { return __builtin_amdgcn_ds_bpermute(4 * from, v); }

// The value of lane l ^ 32.
__device__ __forceinline__ float other_half(float v, int lane) {
  return __builtin_bit_cast(float, from_lane(__builtin_bit_cast(int, v), lane ^ 32));
}

// sum + the two elements of a packed pair.
template <typename T>
__device__ __forceinline__ float add_pair(uint32_t pair, float sum);
template <>
__device__ __forceinline__ float add_pair<BF16>(uint32_t pair, float sum) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum,
                                         false);
}
template <>
__device__ __forceinline__ float add_pair<F16>(uint32_t pair, float sum) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), __builtin_bit_cast(f16x2, 0x3c003c00u), sum, false);
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<BF16>(float a, float b) { return pack_bf16x2(a, b); }
template <> __device__ __forceinline__ uint32_t pack2<F16>(float a, float b) { return pack_f16x2(a, b); }

}  // namespace rw
