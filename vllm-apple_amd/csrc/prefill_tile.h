// What the MFMA prefill kernels share: LDS layout of a K/V tile, cross-lane and
// LDS helpers, direct-to-LDS loads.
#pragma once

#include "common.h"

namespace vaa {

typedef short i16x4 __attribute__((ext_vector_type(4)));

// Chunk swizzle: physical chunk = logical chunk ^ swz(row).  For 8 or 16
// chunks per row the XOR takes all 8 values over 8 consecutive rows (K reads
// conflict-free) and distinct pairs over 4 aligned rows (V^T reads
// conflict-free); for 4 or 12 chunks it stays inside aligned groups of 4.
template <int D>
__device__ __forceinline__ int swz(int row) {
  if constexpr (D == 64 || D == 128) return ((row & 3) << 1) | ((row >> 2) & 1);
  else return (row >> 1) & 3;
}

// K tiles at D = 128: the chunk XOR takes all 16 values over 16 consecutive
// rows, so a ds_read_b128 of one logical chunk down 16 rows hits 16 distinct
// chunk slots (measured 201 against 121 B/clk per CU with the 8-value XOR).
// V keeps swz, which the transposed reads need.
template <int D>
__device__ __forceinline__ int swzk(int row) {
  if constexpr (D == 128) return row & 15;
  else return swz<D>(row);
}

__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, kWave));
  return v;
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, kWave));
  return v;
}

// max / sum of x over lanes l and l ^ 32.  v_permlane32_swap exchanges the
// upper half of its first operand with the lower half of its second, so with
// x in both, one result holds x's lower half twice and the other its upper
// half twice: a VALU exchange with no LDS round trip.  The sum adds the same
// two values in both halves, so both hold the identical result.
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x),
                                                  false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x),
                                                  false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <typename T>
__device__ __forceinline__ typename Elem<T>::x4 lds_tr4(const f16* p) {
  const i16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) i16x4*)(p));
  return __builtin_bit_cast(typename Elem<T>::x4, r);
}

// s_waitcnt vmcnt(0) lgkmcnt(0) (gfx9 encoding: vmcnt bits 3:0 and 15:14,
// expcnt 6:4 left at its maximum, lgkmcnt 11:8): every direct load and LDS
// access of this wave has landed.
__device__ __forceinline__ void wait_all() { __builtin_amdgcn_s_waitcnt(0x0070); }
// A wave-uniform 32-bit read through the scalar unit (s_load_dword, via the
// constant address space: the block table is not written during the
// kernel).  lgkmcnt counts it, so waiting for it does not wait for the vector
// loads in flight, which complete in order.
__device__ __forceinline__ int32_t scalar_load_i32(const int32_t* p) {
  return *((const __attribute__((address_space(4))) int32_t*)(reinterpret_cast<uintptr_t>(p)));
}

// Workgroup barrier for LDS traffic only: s_waitcnt lgkmcnt(0) (vmcnt and
// expcnt at their maxima), so outstanding global loads stay in flight.
__device__ __forceinline__ void lds_bar() {
  __builtin_amdgcn_s_waitcnt(0xC07F);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}


// One 16-byte direct load per lane into LDS at lds + 16 * lane, issued as
// inline asm so that the compiler does not track it: a tracked LDS DMA makes
// it wait for every outstanding LDS read (lgkmcnt(0)) before any operand use,
// which defeats the read-ahead.  The explicit wait_all() + barrier at each
// tile boundary orders the DMA against the reads.
__device__ __forceinline__ void dma16(const void* g, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(g), "s"(lds)
               : "memory", "m0");
}
// The same from a wave-uniform base address (an SGPR pair) plus each lane's
// 32-bit byte offset: no per-lane 64-bit address arithmetic.
__device__ __forceinline__ void dma16s(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(base), "s"(lds)
               : "memory", "m0");
}

}  // namespace vaa
