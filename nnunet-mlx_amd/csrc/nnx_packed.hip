// Products with 4-bit weights under group scales, and their packing.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "nnx_operands.h"

namespace nnx {

namespace {

struct PackedArgs {
  int inputs, outputs, group, blocks, act;
  int64_t rows, xs, ys;
};

PackedArgs make_args(const nnx_packed_config& c) {
  return {c.inputs, c.outputs, c.group, (int)ceil_div(c.inputs, 128), c.gate_activation, c.rows, c.x_stride, c.y_stride};
}

// Byte of a weight's code, input i of output o; an odd input's code is its upper half.
__device__ __forceinline__ int64_t code_at(const PackedArgs& a, int o, int i) {
  const int p = i % 128;
  return ((int64_t)(o / 16) * a.blocks + i / 128) * 1024 + (p % 32 / 8 * 16 + o % 16) * 16 + p / 32 * 4 + p % 8 / 2;
}
__device__ __forceinline__ int64_t scale_at(const PackedArgs& a, int o, int group) {
  return ((int64_t)(o / 16) * a.blocks * (128 / a.group) + group) * 16 + o % 16;
}

__device__ __forceinline__ float level(int code) {
  const int e = code & 7;
  const float v = e < 4 ? 0.5f * e : e < 6 ? e - 2.f : 2.f * e - 8.f;
  return code & 8 ? -v : v;
}

// A thread a group.
template <class T>
__global__ __launch_bounds__(256) void pack_kernel(PackedArgs a, const T* w, uint8_t* codes, float* scales) {
  const int groups = a.blocks * (128 / a.group);
  const int64_t all = (int64_t)((a.outputs + 15) / 16 * 16) * groups;
  for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < all; n += (int64_t)gridDim.x * 256) {
    const int o = (int)(n / groups), g = (int)(n - (int64_t)o * groups);
    const int i0 = g * a.group, i1 = o < a.outputs ? min(i0 + a.group, a.inputs) : i0;
    const T* row = w + o * a.xs;
    float top = 0.f;
    bool odd = false;
    for (int i = i0; i < i1; ++i) {
      const float e = fabsf(to_float(row[i]));
      top = fmaxf(top, e);
      odd |= !(e < INFINITY);
    }
    const bool zero = odd || top < kLeastTop;
    const float up = zero ? 0.f : 6.f / top;
    auto code_of = [&](int i) {
      if (zero || i >= i1) return 0;
      const float x = to_float(row[i]), s = fabsf(x) * up;
      const int e = (s > 0.25f) + (s >= 0.75f) + (s > 1.25f) + (s >= 1.75f) + (s > 2.5f) + (s >= 3.5f) + (s > 5.f);
      return e | (e && x < 0.f ? 8 : 0);
    };
    for (int i = i0; i < i0 + a.group; i += 2) codes[code_at(a, o, i)] = (uint8_t)(code_of(i) | code_of(i + 1) << 4);
    scales[scale_at(a, o, g)] = odd ? NAN : zero ? 0.f : fminf(top, kMostTop) / 6.f;
  }
}

template <class T>
__global__ __launch_bounds__(256) void unpack_kernel(PackedArgs a, const uint8_t* codes, const float* scales, T* w) {
  const int64_t all = (int64_t)a.outputs * a.inputs;
  for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < all; n += (int64_t)gridDim.x * 256) {
    const int o = (int)(n / a.inputs), i = (int)(n - (int64_t)o * a.inputs);
    const int code = codes[code_at(a, o, i)] >> (i % 2 * 4) & 15;
    float v = level(code) * scales[scale_at(a, o, i / a.group)];
    asm("" : "+v"(v));  // one instruction with the conversion would round a float16 from the exact product
    w[o * a.xs + i] = from_float<T>(v);
  }
}

__device__ __forceinline__ float open_gate(float g, int act) {
  if (act == NNX_GATE_NONE) return g;
  const float s = 1.f / (1.f + expf(-g));
  return act == NNX_GATE_SIGMOID ? s : g * s;
}

template <class T>
__device__ __forceinline__ void split(const Vec<T, 8>& x, Frag<typename Operand<T>::E> (&q)[Operand<T>::kTerms]) {
  if constexpr (sizeof(T) == 2) {
    __builtin_memcpy(&q[0], &x, 16);
  } else {
    float left[8];
    __builtin_memcpy(left, &x, 32);
    cut_in_three<true>(left, q);
  }
}

// Products are formed 2^-10 times as large, by what a code stands for: 128 of them add up to no more than the largest of x.
// (Of x below 2^-110 last places fall below float32's least value on the way.)
constexpr float kDown = 0x1p-10f, kUp = 0x1p10f;

// Eight codes as E, exactly.
template <class E>
__device__ __forceinline__ Frag<E> decode(uint32_t w) {
  u32x4 r;
  if constexpr (std::is_same<E, bf16>::value) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, kDown, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, kDown, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, kDown, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, kDown, 3));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, kDown, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, kDown, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, kDown, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, kDown, 3));
  }
  Frag<E> f;
  __builtin_memcpy(&f, &r, 16);
  return f;
}

struct LinearArgs {
  PackedArgs a;
  const void* x;
  const uint8_t* codes[2];
  const float* scales[2];
  const float* bias;
  void* y;
};

// Four neighbouring outputs of a row from o on: bias, gate, one rounding.
template <class T, int MATRICES>
__device__ __forceinline__ void finish(const LinearArgs& h, int64_t row, int o, f32x4 u, f32x4 gate) {
  const PackedArgs& a = h.a;
  T* y = (T*)h.y + row * a.ys + o;
  Vec<T, 4> v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float z = u[i] * kUp;
    if (h.bias) z += h.bias[min(o + i, a.outputs - 1)];
    if constexpr (MATRICES == 2) z *= open_gate(gate[i] * kUp, a.act);
    v.v[i] = from_float<T>(z);
  }
  if (o + 4 <= a.outputs) {
    store_vec(y, v);
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (o + i < a.outputs) y[i] = v.v[i];
  }
}

// Eight elements of a row from `at` on, zeros past its end.
template <class T>
__device__ __forceinline__ Vec<T, 8> load_row(const T* row, int at, int end) {
  if (at + 8 <= end) return load_vec<8>(row + at);
  Vec<T, 8> x{};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (at + e < end) x.v[e] = row[at + e];
  return x;
}

// A workgroup 16 outputs of 16 R rows, its eight waves blocks of 128 inputs in turn, without a word to each other
// until their sums are added up.  Weights are the matrix instruction's rows, x its columns: a lane's 16 bytes of
// codes are its operands of four instructions, and its results four neighbouring outputs of one row, which a
// group's scales multiply as they stand.  Bound by memory: one row by two matrices of 16384 x 4096 in 13.5 us (71 MB,
// 5.3 TB/s, part of it from the last-level cache), by one of them in 9.7, as long as the call from Python takes.  More than
// 16 rows are read in pieces of 256 bytes and more and turned in LDS (64 rows by 4096 x 4096 11.4 us; straight into the
// operands, 64 bytes of 16 rows an access, 18 us); 128 rows take 19 us, bound by the L2, from which every workgroup reads
// its rows (268 MB).
constexpr int kFewWaves = 8;

template <class T, int G32, int MATRICES, int R>
__global__ __launch_bounds__(64 * kFewWaves) void linear_kernel(LinearArgs h, int row_tiles, int64_t units) {
  using E = typename Operand<T>::E;
  constexpr int TERMS = Operand<T>::kTerms, S = 4 / G32;
  __shared__ __attribute__((aligned(16))) f32x4 sums[4][MATRICES * R][64];
  extern __shared__ __attribute__((aligned(16))) char lds[];  // x of R > 1: 16 R rows of 128 elements a wave
  const PackedArgs& a = h.a;
  const int lane = threadIdx.x % 64, n16 = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int tile = (int)(u / row_tiles);
    const int64_t row0 = (u - (int64_t)tile * row_tiles) * 16 * R;
    const T* x[R];
    bool live[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      live[r] = row0 + 16 * r + n16 < a.rows;
      x[r] = (const T*)h.x + (live[r] ? row0 + 16 * r + n16 : 0) * a.xs;
    }
    f32x4 sum[MATRICES][R];
#pragma unroll
    for (int m = 0; m < MATRICES; ++m)
#pragma unroll
      for (int r = 0; r < R; ++r) sum[m][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 c[MATRICES];
    f32x4 sc[MATRICES][S];
    const auto load_weights = [&](int kb) {
      const int64_t block = (int64_t)tile * a.blocks + kb;
#pragma unroll
      for (int m = 0; m < MATRICES; ++m) {
        c[m] = *(const u32x4*)__builtin_assume_aligned(h.codes[m] + block * 1024 + lane * 16, 16);
#pragma unroll
        for (int s = 0; s < S; ++s)
          sc[m][s] = *(const f32x4*)__builtin_assume_aligned(h.scales[m] + (block * S + s) * 16 + 4 * g, 16);
      }
    };
    const auto multiply = [&](auto&& elements) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        Frag<E> q[G32][R][TERMS];
#pragma unroll
        for (int j = 0; j < G32; ++j)
#pragma unroll
          for (int r = 0; r < R; ++r) split(elements(r, s * G32 + j), q[j][r]);
#pragma unroll
        for (int m = 0; m < MATRICES; ++m) {
          f32x4 part[R];
#pragma unroll
          for (int r = 0; r < R; ++r) part[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < G32; ++j) {
            const Frag<E> w = decode<E>(c[m][s * G32 + j]);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int term = 0; term < TERMS; ++term) part[r] = mfma(w, q[j][r][term], part[r]);
          }
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[m][r][i] = fmaf(part[r][i], sc[m][s][i], sum[m][r][i]);
        }
      }
    };
    // whole blocks first: a load under a condition would be waited for at once
    const int whole = a.inputs / 128;
    int kb = wave;
    if constexpr (R == 1) {
      for (; kb < whole; kb += kFewWaves) {
        load_weights(kb);
        Vec<T, 8> xv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) xv[j] = load_vec<8>(x[0] + kb * 128 + 32 * j + 8 * g);
        multiply([&](int, int j) { return xv[j]; });
      }
    } else if (kb < whole) {
      // rows in pieces of 256 bytes and more, turned to the operands' 16 rows of 8 elements through the wave's own LDS:
      // chunk k of row r at place 16 r + (k ^ r % 16)
      Vec<T, 8>* staged = (Vec<T, 8>*)__builtin_assume_aligned(lds, 16) + wave * 16 * R * 16;
      const T* rows[4 * R];
#pragma unroll
      for (int n = 0; n < 4 * R; ++n)
        rows[n] = (const T*)h.x + min(row0 + 4 * n + g, a.rows - 1) * a.xs + n16 * 8;
      Vec<T, 8> xv[4 * R];
      const auto load_x = [&](int kb) {
#pragma unroll
        for (int n = 0; n < 4 * R; ++n) xv[n] = load_vec<8>(rows[n] + kb * 128);
      };
      load_x(kb);
      for (; kb < whole; kb += kFewWaves) {
        load_weights(kb);
        wave_sync();
#pragma unroll
        for (int n = 0; n < 4 * R; ++n) {
          const int r = 4 * n + g;
          staged[r * 16 + (n16 ^ (r % 16))] = xv[n];
        }
        wave_sync();
        load_x(min(kb + kFewWaves, whole - 1));
        multiply([&](int r, int j) { return staged[(16 * r + n16) * 16 + ((4 * j + g) ^ n16)]; });
      }
    }
    if (kb < a.blocks) {
      load_weights(kb);
      Vec<T, 8> xv[R][4];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < 4; ++j) xv[r][j] = load_row(x[r], kb * 128 + 32 * j + 8 * g, a.inputs);
      multiply([&](int r, int j) { return xv[r][j]; });
    }
    // waves 4 to 7 into 0 to 3, then a wave a tile of rows
#pragma unroll
    for (int w0 = 4; w0 >= 0; w0 -= 4) {
      if (wave >= w0 && wave < w0 + 4) {
#pragma unroll
        for (int m = 0; m < MATRICES; ++m)
#pragma unroll
          for (int r = 0; r < R; ++r) sums[wave - w0][m * R + r][lane] = sum[m][r];
      }
      __syncthreads();
      if (w0 == 0) break;
      if (wave < 4) {
#pragma unroll
        for (int m = 0; m < MATRICES; ++m)
#pragma unroll
          for (int r = 0; r < R; ++r) sum[m][r] += sums[wave][m * R + r][lane];
      }
      __syncthreads();
    }
    const int64_t row = row0 + 16 * wave + n16;
    if (wave < R && row < a.rows) {
      f32x4 v[MATRICES];
#pragma unroll
      for (int m = 0; m < MATRICES; ++m) {
        v[m] = sums[0][m * R + wave][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) v[m] += sums[w][m * R + wave][lane];
      }
      finish<T, MATRICES>(h, row, tile * 16 + 4 * g, v[0], v[MATRICES - 1]);
    }
    __syncthreads();  // sums are read before the next unit's
  }
}

// A workgroup 64 outputs of 64 rows, a wave 32 of 32.  A block of 128 inputs of x goes through LDS, split into operands
// once; its weights are the waves' own, as above.  Chunk c (8 inputs) of row r lies at place c * 64 + (r ^ c), so that
// neither the rows' chunks on their way in nor the chunks' rows on their way out meet in a bank.  What bounds it is the
// way of a block from memory, so two are on theirs while one is multiplied: 4096 rows by 320 x 1280 in float16 14 us
// (with 32 rows a workgroup, and four workgroups a CU, 13.8), 512 rows by 4096 x 4096 32 us, 530 TFLOP/s (39).
template <class T, int G32, int MATRICES>
__global__ __launch_bounds__(256, 2) void linear_many_kernel(LinearArgs h, int row_tiles, int64_t units) {
  using E = typename Operand<T>::E;
  constexpr int TERMS = Operand<T>::kTerms, BUFFERS = TERMS == 1 ? 2 : 1, S = 4 / G32;
  __shared__ __attribute__((aligned(16))) Frag<E> staged[BUFFERS * TERMS * 1024];  // [buffer][operand][place]
  const PackedArgs& a = h.a;
  const int lane = threadIdx.x % 64, n16 = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int wr = wave % 2, wo = wave / 2;
  const int last_tile = (a.outputs - 1) / 16, whole = a.inputs / 128;
  const int chunk = threadIdx.x % 16, first = threadIdx.x / 16;  // of x, of rows first + 16 n
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int tile0 = (int)(u / row_tiles) * 4 + wo * 2;
    const int64_t row0 = (u - u / row_tiles * row_tiles) * 64;
    Vec<T, 8> x[2][4];
    u32x4 c[2][MATRICES][2];
    f32x4 sc[2][MATRICES][2][S];
    f32x4 sum[MATRICES][2][2];
#pragma unroll
    for (int m = 0; m < MATRICES; ++m)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r) sum[m][t][r] = f32x4{0.f, 0.f, 0.f, 0.f};
    const T* rows[4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
      rows[n] = (const T*)h.x + min(row0 + first + 16 * n, a.rows - 1) * a.xs + chunk * 8;
    const auto load_x = [&](int which, int kb) {
#pragma unroll
      for (int n = 0; n < 4; ++n) x[which][n] = load_vec<8>(rows[n] + kb * 128);
    };
    const auto load_weights = [&](int which, int kb) {
#pragma unroll
      for (int m = 0; m < MATRICES; ++m)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int64_t block = (int64_t)min(tile0 + t, last_tile) * a.blocks + kb;
          c[which][m][t] = *(const u32x4*)__builtin_assume_aligned(h.codes[m] + block * 1024 + lane * 16, 16);
#pragma unroll
          for (int s = 0; s < S; ++s)
            sc[which][m][t][s] = *(const f32x4*)__builtin_assume_aligned(h.scales[m] + (block * S + s) * 16 + 4 * g, 16);
        }
    };
    const auto stage = [&](int which, int buffer) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        Frag<E> q[TERMS];
        split(x[which][n], q);
        const int at = chunk * 64 + ((first + 16 * n) ^ chunk);
#pragma unroll
        for (int term = 0; term < TERMS; ++term) staged[(buffer * TERMS + term) * 1024 + at] = q[term];
      }
    };
    const auto multiply = [&](int which, int buffer) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        f32x4 part[MATRICES][2][2];
#pragma unroll
        for (int m = 0; m < MATRICES; ++m)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) part[m][t][r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = s * G32; j < (s + 1) * G32; ++j) {
          Frag<E> q[2][TERMS];
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int term = 0; term < TERMS; ++term)
              q[r][term] = staged[(buffer * TERMS + term) * 1024 + (4 * j + g) * 64 + ((wr * 32 + r * 16 + n16) ^ (4 * j + g))];
#pragma unroll
          for (int m = 0; m < MATRICES; ++m)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const Frag<E> w = decode<E>(c[which][m][t][j]);
#pragma unroll
              for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int term = 0; term < TERMS; ++term) part[m][t][r] = mfma(w, q[r][term], part[m][t][r]);
            }
        }
#pragma unroll
        for (int m = 0; m < MATRICES; ++m)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                sum[m][t][r][i] = fmaf(part[m][t][r][i], sc[which][m][t][s][i], sum[m][t][r][i]);
      }
    };
    __syncthreads();  // the unit before has been read
    // Whole blocks first: a load under a condition would be waited for at once.
    if (whole > 0) {
      const int second = min(1, whole - 1);
      load_x(0, 0);
      load_weights(0, 0);
      load_x(1, second);
      load_weights(1, second);
      stage(0, 0);
      __syncthreads();
    }
    const auto round = [&](int which, int kb) {
      const int next = min(kb + 2, whole - 1);  // past the last the last again
      load_x(which, next);
      multiply(which, BUFFERS == 2 ? which : 0);
      load_weights(which, next);
      if (BUFFERS == 1) __syncthreads();
      stage(1 - which, BUFFERS == 2 ? 1 - which : 0);
      __syncthreads();
    };
    int kb = 0;
    for (; kb + 2 <= whole; kb += 2) {
      round(0, kb);
      round(1, kb + 1);
    }
    if (kb < whole) round(0, kb);
    if (whole < a.blocks) {
      load_weights(0, whole);
#pragma unroll
      for (int n = 0; n < 4; ++n) x[0][n] = load_row(rows[n] - chunk * 8, whole * 128 + chunk * 8, a.inputs);
      stage(0, 0);
      __syncthreads();
      multiply(0, 0);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int64_t row = row0 + wr * 32 + r * 16 + n16;
        if (row >= a.rows) continue;
        finish<T, MATRICES>(h, row, (tile0 + t) * 16 + 4 * g, sum[0][t][r], sum[MATRICES - 1][t][r]);
      }
  }
}

// Pieces of 64 rows by 64 outputs, half as many as CUs: with more of them waves that take a piece each are faster, with
// fewer or as many waves that share the inputs of smaller pieces (us, shared and a piece each, bfloat16): 128 pieces of
// 4096 inputs 18.8 and 23.7; 160 of 1280 inputs 13.3 and 10.7, 165 of 960 with a gate 22.0 and 13.8, 256 of 4096 inputs
// 35.3 and 24.3.  Float32 alike: 96 pieces of 1280 inputs 17.6 and 20.7, 128 of 4096 52.2 and 54.7; 160 of 1280 28.4 and 21.0,
// 256 of 4096 146 and 55.5.
constexpr int kManyUnits = 128;

template <class T, int G32, int MATRICES>
void linear_launch(const LinearArgs& h, hipStream_t st) {
  using std::integral_constant;
  const int tiles = (int)ceil_div(h.a.outputs, 16);
  auto few = [&](auto r) {
    constexpr int R = decltype(r)::value;
    const int row_tiles = (int)ceil_div(h.a.rows, 16 * R);
    const int64_t units = (int64_t)tiles * row_tiles;
    linear_kernel<T, G32, MATRICES, R>
        <<<(unsigned)std::min<int64_t>(units, 1 << 20), 64 * kFewWaves,
            R > 1 ? kFewWaves * 16 * R * 128 * sizeof(T) : 0, st>>>(h, row_tiles, units);
  };
  const int row_tiles = (int)ceil_div(h.a.rows, 64);
  const int64_t units = ceil_div(tiles, 4) * row_tiles;
  if (h.a.rows <= 16) return few(integral_constant<int, 1>{});
  if (h.a.rows <= 32) return few(integral_constant<int, 2>{});
  if (units <= kManyUnits) return few(integral_constant<int, sizeof(T) == 2 ? 4 : 2>{});
  linear_many_kernel<T, G32, MATRICES><<<(unsigned)std::min<int64_t>(units, 1 << 20), 256, 0, st>>>(h, row_tiles, units);
}

void check_config(const nnx_packed_config& c, const char* name) {
  const std::string n(name);
  require(known_type(c.type), n + ": unknown type");
  require(c.inputs >= 1 && c.inputs <= 1 << 20 && c.outputs >= 1 && c.outputs <= 1 << 20,
          n + ": 1 to 2^20 inputs and outputs");
  require(c.group == 32 || c.group == 64 || c.group == 128, n + ": group must be 32, 64 or 128");
}

void check_packed(const void* codes, const void* scales, const char* name) {
  require(codes && scales, std::string(name) + ": null pointer");
  require((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) % 16 == 0,
          std::string(name) + ": codes and scales must be 16-byte aligned");
}

}  // namespace

void pack_weight(const nnx_packed_config& c, const void* w, uint8_t* codes, float* scales, hipStream_t st) {
  check_config(c, "pack weight");
  require(w, "pack weight: null pointer");
  check_packed(codes, scales, "pack weight");
  const PackedArgs a = make_args(c);
  const int64_t groups = ceil_div(c.outputs, 16) * 16 * a.blocks * (128 / c.group);
  ProfScope prof("pack_weight", 0.0, (double)c.outputs * c.inputs * (type_bytes(c.type) + 0.5), st);
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    pack_kernel<T><<<(unsigned)std::min<int64_t>(ceil_div(groups, 256), 1 << 20), 256, 0, st>>>(a, (const T*)w, codes, scales);
  });
  launch_check("pack_weight");
}

void unpack_weight(const nnx_packed_config& c, const uint8_t* codes, const float* scales, void* w, hipStream_t st) {
  check_config(c, "unpack weight");
  require(w, "unpack weight: null pointer");
  check_packed(codes, scales, "unpack weight");
  const PackedArgs a = make_args(c);
  const int64_t n = (int64_t)c.outputs * c.inputs;
  ProfScope prof("unpack_weight", 0.0, (double)n * (type_bytes(c.type) + 0.5), st);
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    unpack_kernel<T><<<(unsigned)std::min<int64_t>(ceil_div(n, 256), 1 << 20), 256, 0, st>>>(a, codes, scales, (T*)w);
  });
  launch_check("unpack_weight");
}

void packed_linear(const nnx_packed_config& c, const void* x, const uint8_t* codes, const float* scales,
                   const float* bias, const uint8_t* gate_codes, const float* gate_scales, void* y,
                   hipStream_t st) {
  check_config(c, "packed linear");
  require(c.rows >= 1 && c.rows < (int64_t)1 << 31, "packed linear: 1 to 2^31 - 1 rows");
  require(c.gate_activation >= NNX_GATE_NONE && c.gate_activation <= NNX_GATE_SILU,
          "packed linear: unknown gate activation");
  require(x && y && !gate_codes == !gate_scales, "packed linear: null pointer");
  check_packed(codes, scales, "packed linear");
  if (gate_codes) check_packed(gate_codes, gate_scales, "packed linear");
  const PackedArgs a = make_args(c);
  const double n = (double)c.inputs * c.outputs * (gate_codes ? 2 : 1);
  ProfScope prof("packed_linear", 2.0 * n * c.rows,
                 n * (0.5 + 4.0 / c.group) + (double)c.rows * (c.inputs + c.outputs) * type_bytes(c.type), st);
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    LinearArgs h{a, x, {codes, gate_codes}, {scales, gate_scales}, bias, y};
    auto groups = [&](auto m) {
      constexpr int M = decltype(m)::value;
      if (c.group == 32) return linear_launch<T, 1, M>(h, st);
      if (c.group == 64) return linear_launch<T, 2, M>(h, st);
      linear_launch<T, 4, M>(h, st);
    };
    if (gate_codes) return groups(std::integral_constant<int, 2>{});
    groups(std::integral_constant<int, 1>{});
  });
  launch_check("packed_linear");
}

}  // namespace nnx
