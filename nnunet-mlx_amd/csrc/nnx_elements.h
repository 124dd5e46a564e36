// Element types of the token operators (NNX_TYPE_*) and their conversions to float32.
#pragma once

#include "nnx_internal.h"

namespace nnx {

using f16 = _Float16;
using bf16 = __bf16;

// Runs fn(T{}) with the element type of an NNX_TYPE_* code.
template <class F>
void with_type(int type, F&& fn) {
  if (type == NNX_TYPE_F32) {
    fn(float{});
  } else if (type == NNX_TYPE_F16) {
    fn(f16{});
  } else {
    fn(bf16{});
  }
}

inline bool known_type(int type) { return type >= NNX_TYPE_F32 && type <= NNX_TYPE_BF16; }
inline int type_bytes(int type) { return type == NNX_TYPE_F32 ? 4 : 2; }

template <class T>
__device__ __forceinline__ float to_float(T v) {
  return (float)v;
}

// One rounding, to nearest even.
template <class T>
__device__ __forceinline__ T from_float(float v) {
  return (T)v;
}

}  // namespace nnx
