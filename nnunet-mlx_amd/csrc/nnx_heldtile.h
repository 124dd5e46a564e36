// Attention over held tokens on matrix instructions; included by one source a type.
#pragma once

#include <type_traits>

#include "nnx_held.h"

namespace nnx {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <class T>
using Frag = T __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma(Frag<f16> a, Frag<f16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(Frag<bf16> a, Frag<bf16> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Eight codes as E, exactly.
template <class E>
__device__ __forceinline__ Frag<E> codes_to(uint32_t lo, uint32_t hi) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int w = (int)(i ? hi : lo);
    const float f0 = (float)(int8_t)w, f1 = (float)(int8_t)(w >> 8), f2 = (float)(int8_t)(w >> 16), f3 = (float)(w >> 24);
    if constexpr (std::is_same<E, bf16>::value) {
      r[2 * i] = __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302);
      r[2 * i + 1] = __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x07060302);
    } else {
      r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(f0, f1));
      r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(f2, f3));
    }
  }
  Frag<E> f;
  __builtin_memcpy(&f, &r, 16);
  return f;
}

// The four lanes that hold a row (l, l ^ 16, l ^ 32, l ^ 48) agree.
template <class F>
__device__ __forceinline__ float rows_reduce(float v, F op) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// What a query's element is multiplied in: float16 as it is, the others in bfloat16 operands that add up to it.
template <class T>
struct Query {
  using E = bf16;
  static constexpr int kTerms = std::is_same<T, float>::value ? 3 : 1;
};
template <>
struct Query<f16> {
  using E = f16;
  static constexpr int kTerms = 1;
};
// A weight times its value's scale goes into the second product as two bfloat16 operands (16 bits), of float32 three.
template <class T>
constexpr int kWeightTerms = std::is_same<T, float>::value ? 3 : 2;

// A wave's rows: 16 to a matrix instruction's columns, R of those.  Lane l = 16 g + n has row n; of 64
// slots the logits of 16 t + 4 g + i (t, i < 4), which are the second product's operand as they
// stand, and of the result channels 16 c + 4 g + i.
template <class T, int DP, int R>
struct Rows {
  static constexpr int KF = DP / 32, CT = DP / 16, QT = Query<T>::kTerms;
  Frag<typename Query<T>::E> q[R][QT][KF];
  f32x4 o[R][CT];
  float m[R], l[R];  // l of the lane's slots only
  int count[R];      // slots that the row sees, but for the mask
};

// 64 slots' codes as a wave holds them.
template <int DP>
struct Codes {
  static constexpr int K16 = DP / 64, K8 = DP % 64 / 32;
  u32x4 k[4][K16 ? K16 : 1];
  u32x2 k8[4];
  f32x4 ks[4];
};
template <int DP>
struct Values {
  u32x4 v[DP / 16];
  f32x4 vs[4];
};

// First dimension of the eight that fragment s takes in lane group g: 16 bytes a lane in whole 64s, 8 in what is left.
template <int DP>
__device__ __forceinline__ int dims_at(int s, int g) {
  return s < DP / 64 * 2 ? s / 2 * 64 + 16 * g + s % 2 * 8 : DP / 64 * 64 + 8 * g;
}

template <class T, int DP, int R>
__global__ __launch_bounds__(256) void held_kernel(HeldAttention h) {
  using Q = Query<T>;
  using E = typename Q::E;
  using Row = Rows<T, DP, R>;
  constexpr int KF = Row::KF, CT = Row::CT, WT = kWeightTerms<T>;
  __shared__ __attribute__((aligned(16))) f32x4 exchange[2][R * CT][64];
  __shared__ float exchange_ml[2][2 * R][64];
  const HeldArgs& a = h.a;
  const int lane = threadIdx.x % 64, n16 = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  // units of one key head and part next to each other, on one XCD: they read the same slots
  const int unit = xcd_remap(blockIdx.x, gridDim.x);
  const int tile = unit % h.tiles, rest = unit / h.tiles, split = rest % h.splits, bg = rest / h.splits;
  const int b = bg / a.kv_heads, kh = bg - b * a.kv_heads;
  const int64_t item = bg;

  const int held = min(max(a.lengths ? a.lengths[b] : a.keys, 0), a.keys);
  const int64_t at0 = a.start0 + (a.start ? a.start[b] : 0) + 1;
  const int row0 = tile * 16 * R;
  auto sees = [&](int row) {
    return a.causal ? (int)min(max(at0 + row / h.group, (int64_t)0), (int64_t)held) : held;
  };
  const int least = sees(row0), most = sees(min(row0 + 16 * R, h.rows) - 1);

  Row w;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = row0 + 16 * r + n16;
    const bool live = row < h.rows;
    const int t = live ? row / h.group : 0, hd = live ? row - t * h.group : 0;
    const T* q = (const T*)h.q + b * a.s[0][0] + t * a.s[0][1] + (int64_t)(kh * h.group + hd) * a.s[0][2];
#pragma unroll
    for (int s = 0; s < KF; ++s) {
      const int d = dims_at<DP>(s, g);
      Vec<T, 8> x{};
      if (live && d < a.dim) x = load_vec<8>(q + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float left = to_float(x.v[e]) * h.query;
#pragma unroll
        for (int term = 0; term < Q::kTerms; ++term) {
          const E part = from_float<E>(left);
          w.q[r][term][s][e] = part;
          left -= to_float(part);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) w.o[r][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    w.m[r] = -INFINITY, w.l[r] = 0.f;
    w.count[r] = live ? sees(row) : 0;
  }

  const int all = (most + 63) / 64;
  const int j0 = (int)((int64_t)all * split / h.splits), j1 = (int)((int64_t)all * (split + 1) / h.splits);
  const int8_t* kc = h.k_codes + item * a.slots * a.dim;
  const int8_t* vc = h.v_codes + item * a.slots * a.dim;
  const float* ks = h.k_scales + item * a.slots;
  const float* vs = h.v_scales + item * a.slots;
  const uint8_t* mask = a.mask ? a.mask + b * a.ms : nullptr;
  auto load_keys = [&](Codes<DP>& c, int j) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int8_t* row = kc + ((int64_t)j * 64 + 16 * t + n16) * a.dim;
#pragma unroll
      for (int s = 0; s < Codes<DP>::K16; ++s) {
        const int d = 64 * s + 16 * g;  // past the end: any codes, the query is zero there
        c.k[t][s] = *(const u32x4*)__builtin_assume_aligned(row + (d < a.dim ? d : 0), 16);
      }
      if constexpr (Codes<DP>::K8) {
        const int d = DP / 64 * 64 + 8 * g;
        c.k8[t] = *(const u32x2*)__builtin_assume_aligned(row + (d < a.dim ? d : 0), 8);
      }
      c.ks[t] = *(const f32x4*)__builtin_assume_aligned(ks + (int64_t)j * 64 + 16 * t + 4 * g, 16);
    }
  };
  auto load_values = [&](Values<DP>& c, int j) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int channels = min(16 * ct, a.dim - 16);
      c.v[ct] = *(const u32x4*)__builtin_assume_aligned(vc + (int64_t)j * 64 * a.dim + (channels + n16) * 64 + 16 * g, 16);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
      c.vs[t] = *(const f32x4*)__builtin_assume_aligned(vs + (int64_t)j * 64 + 16 * t + 4 * g, 16);
  };

  Codes<DP> keys;
  Values<DP> values;
  int j = j0 + wave;
  if (j < j1) {
    load_keys(keys, j);
    load_values(values, j);
  }
  for (; j < j1; j += 4) {
    // which of the 64 slots are seen, but for each row's own end
    uint64_t seen = ~0ull;
    if (mask) seen = __ballot(64 * j + lane < a.keys && mask[min(64 * j + lane, a.keys - 1)]);
    const bool whole = seen == ~0ull && 64 * (j + 1) <= least;
    f32x4 x[R][4];  // logits in units of log 2
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      keys.ks[t] *= h.c2;
#pragma unroll
      for (int r = 0; r < R; ++r) x[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KF; ++s) {
        Frag<E> k;
        if (s < Codes<DP>::K16 * 2) {
          k = codes_to<E>(keys.k[t][s / 2][s % 2 * 2], keys.k[t][s / 2][s % 2 * 2 + 1]);
        } else {
          k = codes_to<E>(keys.k8[t][0], keys.k8[t][1]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int term = 0; term < Q::kTerms; ++term) x[r][t] = mfma(k, w.q[r][term][s], x[r][t]);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) x[r][t] *= keys.ks[t];
    }
    if (j + 4 < j1) load_keys(keys, j + 4);
#pragma unroll
    for (int t = 0; t < 4; ++t) values.vs[t] *= h.unit;
    Frag<bf16> p[R][WT][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int end = whole ? 64 : w.count[r] - 64 * j;
      auto hidden = [&](int t, int i) {
        const int slot = 16 * t + 4 * g + i;
        return !((seen >> slot) & 1) || slot >= end;
      };
      if (!whole) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[r][t][i] = hidden(t, i) ? -INFINITY : x[r][t][i];
      }
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, x[r][t][i]);
      top = fmaxf(w.m[r], rows_reduce(top, [](float u, float v) { return fmaxf(u, v); }));
      if (__any(top > w.m[r])) {
        const float back = w.m[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w.m[r] - top);
        w.l[r] *= back;
#pragma unroll
        for (int c = 0; c < CT; ++c) w.o[r][c] *= back;
        w.m[r] = top;
      }
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(x[r][t][i] - base);
          sum += e;
          float left = e * values.vs[t][i];
          if (!whole) left = hidden(t, i) ? 0.f : left;
#pragma unroll
          for (int term = 0; term < WT; ++term) {
            const bf16 part = from_float<bf16>(left);
            p[r][term][t / 2][t % 2 * 4 + i] = part;
            left -= to_float(part);
          }
        }
      w.l[r] += sum;
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const Frag<bf16> v = codes_to<bf16>(values.v[c][2 * u], values.v[c][2 * u + 1]);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int term = 0; term < WT; ++term) w.o[r][c] = mfma(v, p[r][term][u], w.o[r][c]);
      }
    if (j + 4 < j1) load_values(values, j + 4);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) w.l[r] = rows_reduce(w.l[r], [](float u, float v) { return u + v; });

  // waves 2 and 3 into 0 and 1, then 1 into 0; lanes hold the same places
#pragma unroll
  for (int step = 2; step >= 1; step /= 2) {
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        exchange_ml[wave - step][2 * r][lane] = w.m[r];
        exchange_ml[wave - step][2 * r + 1][lane] = w.l[r];
#pragma unroll
        for (int c = 0; c < CT; ++c) exchange[wave - step][r * CT + c][lane] = w.o[r][c];
      }
    }
    __syncthreads();
    if (wave < step) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float m = exchange_ml[wave][2 * r][lane], top = fmaxf(m, w.m[r]);
        const float mine = w.m[r] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(w.m[r] - top);
        const float theirs = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top);
        w.l[r] = w.l[r] * mine + exchange_ml[wave][2 * r + 1][lane] * theirs;
#pragma unroll
        for (int c = 0; c < CT; ++c) w.o[r][c] = w.o[r][c] * mine + exchange[wave][r * CT + c][lane] * theirs;
        w.m[r] = top;
      }
    }
    __syncthreads();
  }
  if (wave) return;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = row0 + 16 * r + n16;
    if (row >= h.rows) continue;
    if (h.splits == 1) {
      const int t = row / h.group, hd = row - t * h.group;
      T* out = (T*)h.out + b * a.s[1][0] + t * a.s[1][1] + (int64_t)(kh * h.group + hd) * a.s[1][2];
      const float whole = w.l[r] == 0.f && w.m[r] == -INFINITY ? 0.f : 1.f / w.l[r];  // nothing seen: zeros
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        if (16 * c >= a.dim) break;
        Vec<T, 4> y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.v[i] = from_float<T>(w.o[r][c][i] * whole * h.back);
        store_vec(out + 16 * c + 4 * g, y);
      }
    } else {
      const int64_t at = ((int64_t)bg * h.splits + split) * h.rows + row;
#pragma unroll
      for (int c = 0; c < CT; ++c)
        if (16 * c < a.dim) *(f32x4*)__builtin_assume_aligned(h.part + at * a.dim + 16 * c + 4 * g, 16) = w.o[r][c];
      if (g == 0) h.meta[at] = make_float2(w.m[r], w.l[r]);
    }
  }
}

template <class T, int DP, int R>
void held_launch(const HeldAttention& h, const HeldPlan& p, hipStream_t st) {
  held_kernel<T, DP, R><<<(unsigned)(p.units * p.splits), 256, 0, st>>>(h);
  launch_check("held_attention");
}

template <class T>
void held_units(const HeldAttention& h, const HeldPlan& p, hipStream_t st) {
  using std::integral_constant;
  auto rows = [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    if (p.r == 1) return held_launch<T, DP, 1>(h, p, st);
    held_launch<T, DP, 2>(h, p, st);
  };
  if (h.a.dim <= 32) return rows(integral_constant<int, 32>{});
  if (h.a.dim <= 64) return rows(integral_constant<int, 64>{});
  if (h.a.dim <= 96) return rows(integral_constant<int, 96>{});
  rows(integral_constant<int, 128>{});
}

}  // namespace
}  // namespace nnx
