// Rows of the quantised KV cache: e4m3 codes (OCP, largest value 448) with one
// exponent byte b per row; code c stands for c * 2^(b - 127).  b = 0 stands for
// 2^-127 and b = 255, which no written row has, for 2^128.
#pragma once

#include "common.h"

namespace vaa {

// The scale operand of v_cvt_scalef32_*: its exponent field alone counts.
__device__ __forceinline__ float scale_of(uint32_t b) { return __uint_as_float(b << 23); }

// Two codes of a 32-bit word (the lower or the upper pair), times the scale,
// rounded to nearest even.
template <typename T, bool kHigh>
__device__ __forceinline__ uint32_t deq2(uint32_t w, float scale);
template <>
__device__ __forceinline__ uint32_t deq2<f16, false>(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
}
template <>
__device__ __forceinline__ uint32_t deq2<f16, true>(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true));
}
template <>
__device__ __forceinline__ uint32_t deq2<bf16, false>(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
}
template <>
__device__ __forceinline__ uint32_t deq2<bf16, true>(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true));
}

// Eight codes (two words) as eight 16-bit values.
template <typename T>
__device__ __forceinline__ u32x4 deq8(uint32_t w0, uint32_t w1, float scale) {
  return u32x4{deq2<T, false>(w0, scale), deq2<T, true>(w0, scale), deq2<T, false>(w1, scale),
               deq2<T, true>(w1, scale)};
}

}  // namespace vaa
