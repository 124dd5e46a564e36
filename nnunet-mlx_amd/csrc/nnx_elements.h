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

// N elements of any alignment (gfx950 takes wide global accesses at every address), one wide
// access each way.
template <class T, int N>
struct Vec {
  T v[N];
};

template <int N, class T>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
  Vec<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}

template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& r) {
  __builtin_memcpy(p, &r, sizeof(r));
}

// Stands between what lanes of a wave write to LDS and what other lanes of it read there, and before they
// write there again.  LDS serves a wave's accesses in order, so this costs no instruction: it holds the
// compiler to that order.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
}

// Value of another lane of the same 16 (CTRL: a DPP control word) without a trip through LDS.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

constexpr int kDppSwap1 = 0xb1, kDppSwap2 = 0x4e;  // quad_perm: lane ^ 1, lane ^ 2
constexpr int kDppHalfMirror = 0x141, kDppMirror = 0x140;

// op over the 16 or 64 lanes that share a row; every lane gets the result.  Mirrors stand for
// lane ^ 4 and lane ^ 8 once groups of 4 and 8 agree.
template <int LANES, class F>
__device__ __forceinline__ float lanes_reduce(float v, F op) {
  static_assert(LANES == 16 || LANES == 64, "");
  v = op(v, dpp<kDppSwap1>(v));
  v = op(v, dpp<kDppSwap2>(v));
  v = op(v, dpp<kDppHalfMirror>(v));
  v = op(v, dpp<kDppMirror>(v));
  if (LANES == 64) {
    v = op(v, __shfl_xor(v, 16));
    v = op(v, __shfl_xor(v, 32));
  }
  return v;
}

}  // namespace nnx
