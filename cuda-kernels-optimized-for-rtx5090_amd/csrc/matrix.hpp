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

// Layouts of the 16x16x32 product, lane l with r = l % 16 and h = l / 16: A's row r and B's column r, both at the 8
// contraction indices 8 h ...; the result's column r at the rows 4 h + i, i = 0..3.
__device__ __forceinline__ f32x4 product16(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}

// An address in LDS. own(): one that is computed here and kept, so that constants are added to it in the instructions
// that use it (left to itself the compiler adds them first, with an instruction or a register for each).
typedef __attribute__((address_space(3))) char* lds_ptr;
__device__ __forceinline__ lds_ptr in_lds(char* p) { return (lds_ptr)p; }
__device__ __forceinline__ lds_ptr own(lds_ptr p) {
  asm volatile("" : "+v"(p));
  return p;
}
__device__ __forceinline__ u32x4 lds_vector(lds_ptr at) {
  return *(const __attribute__((address_space(3))) u32x4*)at;
}
// Within 16 lanes, lane i gives the address of 4 elements: row i / 4 of a 4 x 16 block, columns 4 (i % 4) ...; it gets
// column i of the block, its 4 rows.
__device__ __forceinline__ u32x2 lds_column(lds_ptr at) {
  typedef __attribute__((address_space(3))) s16x4* ptr;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)at));
}
// Computed here, and not where it is used.
__device__ __forceinline__ void settle(uint32_t& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void settle(float& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void settle(int& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void settle(const char*& p) { asm volatile("" : "+v"(p)); }

// 16 bytes from an active lane's own address to LDS at `at` + 16 * lane (`at` the same in the wave's lanes; some lane
// is active, so that the wave counts one load). Asynchronous: counted with the vector memory loads, which wait_loads()
// waits for, and nothing else does: the compiler's builtin for it makes every later LDS read wait for all of them, also
// the reads of another buffer. (The instruction has no register output; a wave counts it in order with its other loads,
// so the compiler's own waits stay sufficient.)
__device__ __forceinline__ void load_to_lds(const void* from, char* at, bool active) {
  const uint32_t to = __builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)at);
  if (active) asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}
// The same from `offset` bytes behind an address that all of the wave's lanes have.
__device__ __forceinline__ void load_to_lds_at(const char* base, uint32_t offset, char* at, bool active) {
  const uint32_t to = __builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)at);
  if (active)
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory");
}
// The same for what is read once: it does not displace what the caches hold for others.
__device__ __forceinline__ void stream_to_lds(const void* from, char* at, bool active) {
  const uint32_t to = __builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)at);
  if (active) asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(to), "v"(from) : "memory");
}
// The same of 4 bytes, to `at` + 4 * lane.
__device__ __forceinline__ void load_word_to_lds(const void* from, char* at) {
  const uint32_t to = __builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)at);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(from) : "memory");
}
// All but this wave's `newer` last loads have arrived.
template <int newer = 0>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(newer) : "memory");
}
// This wave's LDS reads are in registers.
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// LDS accesses stay on their side of this place: a wave's are executed in order, so that is all that what one lane writes
// and another reads asks for.
__device__ __forceinline__ void order_lds() { asm volatile("" ::: "memory"); }
// Nothing is moved across this place by the compiler's scheduler.
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0); }
// The workgroup's barrier alone, without a wait for loads that are under way; nothing is moved across it.
__device__ __forceinline__ void meet() {
  keep_order();
  asm volatile("s_barrier" ::: "memory");
  keep_order();
}

// v of lane `from` (any lane of the wave).
__device__ __forceinline__ int from_lane(int v, int from) { return __builtin_amdgcn_ds_bpermute(4 * from, v); }

// v of lane l ^ D, D a power of two, without a trip to LDS.
template <int D> __device__ __forceinline__ uint32_t across(uint32_t v) {
  if constexpr (D == 16 || D == 32) {
    const bool upper = (threadIdx.x & D) != 0;
    if constexpr (D == 16) {
      const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
      return upper ? (uint32_t)r[0] : (uint32_t)r[1];
    } else {
      const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
      return upper ? (uint32_t)r[0] : (uint32_t)r[1];
    }
  } else {
    // within 16 lanes: l ^ 4 is l ^ 7 of l ^ 3, l ^ 8 half a turn of the row
    float f = __builtin_bit_cast(float, v);
    if constexpr (D == 1) f = dpp<kDppXor1>(f);
    if constexpr (D == 2) f = dpp<kDppXor2>(f);
    if constexpr (D == 4) f = dpp<kDppHalfMirror>(dpp<0x1B>(f));
    if constexpr (D == 8) f = dpp<0x128>(f);
    return __builtin_bit_cast(uint32_t, f);
  }
}

// The larger and the sum of a lane's and lane l ^ 32's values.
__device__ __forceinline__ float max_of_halves(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float sum_of_halves(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// The largest and the sum of the values of lanes l, l ^ 16, l ^ 32 and l ^ 48.
__device__ __forceinline__ float max_of_quarters(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return max_of_halves(fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])));
}
__device__ __forceinline__ float sum_of_quarters(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return sum_of_halves(__builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]));
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
