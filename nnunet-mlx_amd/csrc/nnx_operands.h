// 16 x 16 x 32 matrix products of 16-bit operands, and float32 as operands of them.
#pragma once

#include "nnx_elements.h"

namespace nnx {

// What is held in 8 bits or packed in 4: below kLeastTop, 2^-60, a largest magnitude counts as zero; scales are of kMostTop
// at most, so that scale times largest code is finite.
constexpr float kLeastTop = 0x1p-60f, kMostTop = 3.4028233e38f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <class T>
using Frag = T __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma(Frag<f16> a, Frag<f16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(Frag<bf16> a, Frag<bf16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// What a type is multiplied in: 16-bit types as they are, float32 in three bfloat16 operands that add up to it.
template <class T>
struct Operand {
  using E = T;
  static constexpr int kTerms = 1;
};
template <>
struct Operand<float> {
  using E = bf16;
  static constexpr int kTerms = 3;
};

// Eight values as three operands: cut, not rounded, the next bits eight at a time.  Of infinity nothing is left (NaN
// without INFINITE, where it does not occur or has to be one).
template <bool INFINITE>
__device__ __forceinline__ void cut_in_three(float (&left)[8], Frag<bf16> (&q)[3]) {
#pragma unroll
  for (int term = 0; term < 3; ++term) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = __builtin_amdgcn_perm(__float_as_uint(left[2 * i + 1]), __float_as_uint(left[2 * i]), 0x07060302);
    __builtin_memcpy(&q[term], &r, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float rest = left[i] - __uint_as_float(__float_as_uint(left[i]) & 0xffff0000u);
      left[i] = INFINITE && term == 0 && fabsf(left[i]) == INFINITY ? 0.f : rest;
    }
  }
}

}  // namespace nnx
