// Row operators over tokens: rotary positions, and the norms around a block with its gate,
// scale and residual sum.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "nnx_elements.h"

namespace nnx {

// ---- rotary positions ------------------------------------------------------------------
//
// (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t), t = 2 pi position * frequency.
// The frequency is a whole number of 2^-64 turns, so position * step mod 2^64 is the exact
// fraction of a turn whatever the position (a float32 product is 0.1 rad off at position 2^20).

namespace {

struct RotaryArgs {
  const void* x[2];
  void* y[2];
  int heads[2];
  int64_t xs[2][3], ys[2][3];
  const int32_t* pos;
  const int64_t* steps;
  const int32_t* pair_axes;
  int64_t ps[2];
  int batch, tokens, dim, half, axes, interleaved;
  float amp, amp_sin;
};

// sin and cos of a signed number of 2^-32 turns.  The nearest quarter turn is split off in whole
// numbers; the rest is z eighths of a turn, |z| <= 1, where the Taylor series of sin(pi z / 4) and
// cos(pi z / 4) end below 2e-9.
__device__ __forceinline__ void sincos_turns(int32_t turns, float& s, float& c) {
  const int quarter = (int)((uint32_t)turns + 0x20000000u) >> 30;
  const float z = (float)(int32_t)((uint32_t)turns - ((uint32_t)quarter << 30)) * 1.862645149230957e-09f;  // 2^-29
  const float zz = z * z;
  const float ps = z * fmaf(zz, fmaf(zz, fmaf(zz, fmaf(zz, 3.1336162e-07f, -3.6576204e-05f),
                                             2.4903946e-03f), -8.0745512e-02f), 7.8539816e-01f);
  const float pc = fmaf(zz, fmaf(zz, fmaf(zz, fmaf(zz, fmaf(zz, -2.4611370e-08f, 3.5908605e-06f),
                                                   -3.2599189e-04f), 1.5854344e-02f), -3.0842514e-01f), 1.f);
  const float a = quarter & 1 ? pc : ps, b = quarter & 1 ? ps : pc;
  s = quarter & 2 ? -a : a;
  c = (quarter + 1) & 2 ? -b : b;
}

// Bound by memory: 2 x 65536 tokens of 20 heads of 128 float16, 96 of them rotated, move 1.34 GB in 258 us,
// 5.2 TB/s (a large copy reaches 4.8).  A wave turns heads of one token, each lane W neighbouring
// elements of a head, so that its accesses are whole rows of memory whatever the rotated part;
// lanes / head = dim / W.  A lane forms its elements' sines once and keeps them for all its heads.
// When the pairs lie half the rotated part apart, the partners come from the lane that holds them.
// HB heads' loads are in flight at a time.  (Threads that load both elements of their pairs, half a
// row apart, as below, took 543 us.)
template <class T, int W, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_wave_kernel(RotaryArgs a, int lanes, int steps_per,
                                                          int groups, int64_t waves) {
  constexpr int HB = 4, BYTES = W * sizeof(T), WORDS = BYTES < 4 ? 1 : BYTES / 4;
  const int lane = threadIdx.x % 64, at_once = 64 / lanes;
  const int sub = lane / lanes, u = lane - sub * lanes, e = u * W;
  const int all = a.heads[0] + a.heads[1];
  const bool turned = e < 2 * a.half, upper = e >= a.half;
  const int first = INTERLEAVED ? e / 2 : (upper ? e - a.half : e);
  const int partner = turned ? lane + (upper ? -a.half / W : a.half / W) : lane;
  for (int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; i < waves; i += (int64_t)gridDim.x * 4) {
    const int64_t bt = i / groups;
    const int h0 = (int)(i - bt * groups) * steps_per * at_once + sub;
    const int b = (int)(bt / a.tokens), t = (int)(bt - (int64_t)b * a.tokens);
    float sn[W], cs[W];
    if (turned) {
      const int32_t* pos = a.pos + b * a.ps[0] + t * a.ps[1];
#pragma unroll
      for (int p = 0; p < (INTERLEAVED ? W / 2 : W); ++p) {
        const int axis = min(max(a.pair_axes[first + p], 0), a.axes - 1);
        const uint64_t phase = (uint64_t)(int64_t)pos[axis] * (uint64_t)a.steps[first + p];
        float s, c;
        sincos_turns((int32_t)(phase >> 32), s, c);
        s *= a.amp_sin;
        c *= a.amp;
        if constexpr (INTERLEAVED) {
          sn[2 * p] = -s, sn[2 * p + 1] = s;
          cs[2 * p] = c, cs[2 * p + 1] = c;
        } else {
          sn[p] = upper ? s : -s;
          cs[p] = c;
        }
      }
    }
    const T* x[2] = {(const T*)a.x[0] + b * a.xs[0][0] + t * a.xs[0][1] + e,
                     (const T*)a.x[1] + b * a.xs[1][0] + t * a.xs[1][1] + e};
    T* y[2] = {(T*)a.y[0] + b * a.ys[0][0] + t * a.ys[0][1] + e,
               (T*)a.y[1] + b * a.ys[1][0] + t * a.ys[1][1] + e};
    for (int k0 = 0; k0 < steps_per; k0 += HB) {
      Vec<T, W> v[HB];
      bool in[HB];
      T* to[HB];
#pragma unroll
      for (int k = 0; k < HB; ++k) {
        const int h = h0 + (k0 + k) * at_once;
        in[k] = k0 + k < steps_per && sub < at_once && h < all;
        const bool second = h >= a.heads[0];
        const int hh = second ? h - a.heads[0] : h;
        to[k] = second ? y[1] + hh * a.ys[1][2] : y[0] + hh * a.ys[0][2];
        if (in[k]) v[k] = load_vec<W>(second ? x[1] + hh * a.xs[1][2] : x[0] + hh * a.xs[0][2]);
      }
#pragma unroll
      for (int k = 0; k < HB; ++k) {
        Vec<T, W> w;
        if constexpr (!INTERLEAVED) {
          uint32_t mine[WORDS] = {}, theirs[WORDS];
          __builtin_memcpy(mine, &v[k], BYTES);
#pragma unroll
          for (int j = 0; j < WORDS; ++j)
            theirs[j] = (uint32_t)__builtin_amdgcn_ds_bpermute(partner * 4, (int)mine[j]);
          __builtin_memcpy(&w, theirs, BYTES);
        }
        if (!in[k]) continue;
        if (turned) {
          Vec<T, W> o;
#pragma unroll
          for (int p = 0; p < W; ++p) {
            const float other = to_float(INTERLEAVED ? v[k].v[p ^ 1] : w.v[p]);
            o.v[p] = from_float<T>(fmaf(to_float(v[k].v[p]), cs[p], other * sn[p]));
          }
          v[k] = o;
        }
        store_vec(to[k], v[k]);
      }
    }
  }
}

template <class T, int W>
void rotary_wave_launch(const RotaryArgs& a, hipStream_t st) {
  const int lanes = a.dim / W, at_once = 64 / lanes;
  const int steps = (int)ceil_div(a.heads[0] + a.heads[1], at_once);
  // Heads a wave: as many as leave each SIMD 2 waves, so that few sines are formed twice (all 20 heads of
  // 128: 4096 tokens 13.6 us against 24.8 with 4 heads a wave, 65536 tokens 140 against 336).
  const int64_t rows = (int64_t)a.batch * a.tokens;
  int per = 1;
  while (per < steps && rows * ceil_div(steps, 2 * per) >= 2048) per *= 2;
  per = std::min(per, steps);
  const int groups = (int)ceil_div(steps, per);
  const int64_t waves = rows * groups;
  const int grid = (int)std::min<int64_t>(ceil_div(waves, 4), 1 << 23);
  if (a.interleaved) {
    if constexpr (W > 1) rotary_wave_kernel<T, W, true><<<grid, 256, 0, st>>>(a, lanes, per, groups, waves);
  } else {
    rotary_wave_kernel<T, W, false><<<grid, 256, 0, st>>>(a, lanes, per, groups, waves);
  }
}

// Heads that a wave does not hold (dim / W above 64: wide heads, or pairs that W must divide and are
// odd).  A thread holds the sines of W neighbouring elements' pairs of one token (of W / 2 pairs
// when they are interleaved) and turns them in `per` heads, HB heads' loads in flight at a time;
// the elements past the pairs are copied by further threads.  Bound by memory where accesses are wide (32768
// tokens of 2 heads of 1024 float32, 1000 rotated: 537 MB in 154 us, 3.5 TB/s), by the number of accesses
// where an odd count of pairs leaves one element each (8 heads of 80 bfloat16, 22 rotated: 84 MB in 70 us,
// 1.2 TB/s; all 80 rotated, in the kernel above, 38 us).
template <class T, int W, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a, int units, int rotated, int per,
                                                     int groups, int64_t threads) {
  constexpr int HB = 4, PAIRS = INTERLEAVED ? W / 2 : W;
  const int all = a.heads[0] + a.heads[1];
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < threads; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / units;
    const int u = (int)(i - r * units);
    const int64_t bt = r / groups;
    const int h0 = (int)(r - bt * groups) * per, h1 = min(h0 + per, all);
    const int b = (int)(bt / a.tokens), t = (int)(bt - (int64_t)b * a.tokens);
    const int64_t xo[2] = {b * a.xs[0][0] + t * a.xs[0][1], b * a.xs[1][0] + t * a.xs[1][1]};
    const int64_t yo[2] = {b * a.ys[0][0] + t * a.ys[0][1], b * a.ys[1][0] + t * a.ys[1][1]};
    auto from = [&](int h) {
      return h < a.heads[0] ? (const T*)a.x[0] + xo[0] + h * a.xs[0][2]
                            : (const T*)a.x[1] + xo[1] + (h - a.heads[0]) * a.xs[1][2];
    };
    auto to = [&](int h) {
      return h < a.heads[0] ? (T*)a.y[0] + yo[0] + h * a.ys[0][2]
                            : (T*)a.y[1] + yo[1] + (h - a.heads[0]) * a.ys[1][2];
    };
    if (u >= rotated) {  // past the pairs
      const int e = 2 * a.half + (u - rotated) * W;
      if (e + W > a.dim) {
        for (int h = h0; h < h1; ++h)
          for (int d = e; d < a.dim; ++d) to(h)[d] = from(h)[d];
        continue;
      }
      for (int h = h0; h < h1; h += HB) {
        Vec<T, W> v[HB];
#pragma unroll
        for (int k = 0; k < HB; ++k)
          if (h + k < h1) v[k] = load_vec<W>(from(h + k) + e);
#pragma unroll
        for (int k = 0; k < HB; ++k)
          if (h + k < h1) store_vec(to(h + k) + e, v[k]);
      }
      continue;
    }
    const int first = INTERLEAVED ? u * (W / 2) : u * W;
    float sn[PAIRS], cs[PAIRS];
    const int32_t* pos = a.pos + b * a.ps[0] + t * a.ps[1];
#pragma unroll
    for (int p = 0; p < PAIRS; ++p) {
      const int axis = min(max(a.pair_axes[first + p], 0), a.axes - 1);
      const uint64_t phase = (uint64_t)(int64_t)pos[axis] * (uint64_t)a.steps[first + p];
      sincos_turns((int32_t)(phase >> 32), sn[p], cs[p]);
      sn[p] *= a.amp_sin;
      cs[p] *= a.amp;
    }
    const int e0 = u * W, e1 = e0 + a.half;
    for (int h = h0; h < h1; h += HB) {
      Vec<T, W> v[HB], w[INTERLEAVED ? 1 : HB];
#pragma unroll
      for (int k = 0; k < HB; ++k) {
        if (h + k < h1) {
          v[k] = load_vec<W>(from(h + k) + e0);
          if constexpr (!INTERLEAVED) w[k] = load_vec<W>(from(h + k) + e1);
        }
      }
#pragma unroll
      for (int k = 0; k < HB; ++k) {
        if (h + k >= h1) continue;
        if constexpr (INTERLEAVED) {
#pragma unroll
          for (int p = 0; p < PAIRS; ++p) {
            const float x0 = to_float(v[k].v[2 * p]), x1 = to_float(v[k].v[2 * p + 1]);
            v[k].v[2 * p] = from_float<T>(fmaf(x0, cs[p], -(x1 * sn[p])));
            v[k].v[2 * p + 1] = from_float<T>(fmaf(x1, cs[p], x0 * sn[p]));
          }
          store_vec(to(h + k) + e0, v[k]);
        } else {
#pragma unroll
          for (int p = 0; p < PAIRS; ++p) {
            const float x0 = to_float(v[k].v[p]), x1 = to_float(w[k].v[p]);
            v[k].v[p] = from_float<T>(fmaf(x0, cs[p], -(x1 * sn[p])));
            w[k].v[p] = from_float<T>(fmaf(x1, cs[p], x0 * sn[p]));
          }
          store_vec(to(h + k) + e0, v[k]);
          store_vec(to(h + k) + e1, w[k]);
        }
      }
    }
  }
}

template <class T, int W>
void rotary_launch(const RotaryArgs& a, hipStream_t st) {
  const bool in_place = a.x[0] == a.y[0] && a.x[1] == a.y[1];
  const int rotated = a.interleaved ? 2 * a.half / W : a.half / W;
  const int units = rotated + (in_place ? 0 : (int)ceil_div(a.dim - 2 * a.half, W));
  const int all = a.heads[0] + a.heads[1];
  // Heads a thread: as many as leave every CU 1024 threads, so that few sines are formed twice.
  const int64_t rows = (int64_t)a.batch * a.tokens * units;
  int per = 1;
  while (per < all && per < 32 && rows * ceil_div(all, 2 * per) >= 262144) per *= 2;
  const int groups = (int)ceil_div(all, per);
  const int64_t threads = rows * groups;
  const int grid = (int)std::min<int64_t>(ceil_div(threads, 256), 1 << 23);
  if (a.interleaved) {
    if constexpr (W > 1) {
      rotary_kernel<T, W, true><<<grid, 256, 0, st>>>(a, units, rotated, per, groups, threads);
    }
  } else {
    rotary_kernel<T, W, false><<<grid, 256, 0, st>>>(a, units, rotated, per, groups, threads);
  }
}

}  // namespace

void rotary(const nnx_rotary_config& c, const void* x1, const void* x2, const int32_t* positions,
            const int64_t* steps, const int32_t* pair_axes, void* y1, void* y2, hipStream_t st) {
  require(known_type(c.type), "rotary: unknown type");
  require(c.batch >= 1 && c.tokens >= 1, "rotary: batch and tokens must be positive");
  require(c.heads[0] >= 0 && c.heads[1] >= 0 && c.heads[0] <= 65536 && c.heads[1] <= 65536 &&
              c.heads[0] + c.heads[1] >= 1,
          "rotary: 0 to 65536 heads a tensor, at least one in all");
  require(c.head_dim >= 2 && c.head_dim <= 1024, "rotary: head_dim must be 2..1024");
  require(c.rotary_dim >= 2 && c.rotary_dim % 2 == 0 && c.rotary_dim <= c.head_dim,
          "rotary: rotary_dim must be even and 2..head_dim");
  require(c.axes >= 1 && c.axes <= 8, "rotary: 1 to 8 position axes");
  require(std::isfinite(c.amplitude), "rotary: the amplitude must be finite");
  require((c.heads[0] == 0 || (x1 && y1)) && (c.heads[1] == 0 || (x2 && y2)) && positions && steps &&
              pair_axes,
          "rotary: null pointer");
  const double elems = (double)c.batch * c.tokens * (c.heads[0] + c.heads[1]) * c.head_dim;
  require(elems < 9e18, "rotary: too many elements");
  RotaryArgs a;
  a.x[0] = x1, a.x[1] = x2, a.y[0] = y1, a.y[1] = y2;
  for (int i = 0; i < 2; ++i) {
    a.heads[i] = c.heads[i];
    for (int j = 0; j < 3; ++j) {
      a.xs[i][j] = c.x_strides[3 * i + j];
      a.ys[i][j] = c.y_strides[3 * i + j];
    }
  }
  a.pos = positions, a.steps = steps, a.pair_axes = pair_axes;
  a.ps[0] = c.position_strides[0], a.ps[1] = c.position_strides[1];
  a.batch = c.batch, a.tokens = c.tokens, a.dim = c.head_dim, a.half = c.rotary_dim / 2;
  a.axes = c.axes, a.interleaved = c.interleaved != 0;
  a.amp = c.amplitude, a.amp_sin = c.inverse ? -c.amplitude : c.amplitude;
  ProfScope prof("rotary", 3.0 * elems, 2.0 * elems * type_bytes(c.type), st);
  // The widest access (up to 16 bytes) that divides the rotated elements (their half).
  int w = 16 / type_bytes(c.type);
  while ((a.interleaved ? c.rotary_dim : a.half) % w) w /= 2;
  int wave_w = w;  // and that divides the head, for a wave to hold it
  while (c.head_dim % wave_w) wave_w /= 2;
  const bool wave = c.head_dim / wave_w <= 64 && (wave_w > 1 || !a.interleaved);
  if (wave) w = wave_w;
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) {
      if (w == 8) return wave ? rotary_wave_launch<T, 8>(a, st) : rotary_launch<T, 8>(a, st);
    }
    if (w == 4) return wave ? rotary_wave_launch<T, 4>(a, st) : rotary_launch<T, 4>(a, st);
    if (w == 2) return wave ? rotary_wave_launch<T, 2>(a, st) : rotary_launch<T, 2>(a, st);
    wave ? rotary_wave_launch<T, 1>(a, st) : rotary_launch<T, 1>(a, st);
  });
  launch_check("rotary");
}

// ---- norms, gate and residual ----------------------------------------------------------

namespace {

struct NormArgs {
  const void *x, *residual, *gate;
  const float *scale, *post_w, *post_b, *pre_w, *pre_b;
  void *out, *y;
  int64_t rows, xs, rs, gs, os, ys;
  int channels, post, act;
  float residual_scale, eps;
};

template <int G>
__device__ __forceinline__ float row_sum(float v, float* lds) {
  const auto add = [](float a, float b) { return a + b; };
  if constexpr (G <= 64) {
    return lanes_reduce<G>(v, add);
  } else {
    v = lanes_reduce<64>(v, add);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < G / 64; ++w) s += lds[w];
    return s;
  }
}

__device__ __forceinline__ float open_gate(float g, int act) {
  if (act == NNX_GATE_NONE) return g;
  const float s = 1.f / (1.f + expf(-g));
  return act == NNX_GATE_SIGMOID ? s : g * s;
}

// Bound by memory: 262144 rows of 320, bf16 with a float32 residual and both norms, move 1.0 GB in 193 us,
// 5.2 TB/s (a large copy reaches 4.8).  G threads a row, each K runs of W channels; the row stays in
// registers from its one read to its one write, and both norms take their moments there (mean first,
// then squares about it).  A run
// that passes the row's end is moved back to end with it: its first `skip` channels are another
// thread's, written twice with the same values and left out of the sums; runs wholly past the
// end skip all W and write nothing.  Needs channels >= W.
template <class T, class R, int G, int K>
__global__ __launch_bounds__(G > 256 ? G : 256) void residual_norm_kernel(NormArgs a, int rms) {
  constexpr int W = 16 / sizeof(T), ROWS = G > 256 ? 1 : 256 / G;
  __shared__ float lds[G > 64 ? G / 64 : 1];
  const int lane = threadIdx.x % G;
  const float inv = 1.f / (float)a.channels;
  int at[K], skip[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * G + lane) * W;
    at[k] = min(c, a.channels - W);
    skip[k] = min(c - at[k], W);
  }
  for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < a.rows; row0 += (int64_t)gridDim.x * ROWS) {
    const int64_t row = row0 + threadIdx.x / G;
    if (G <= 64 && row >= a.rows) break;  // whole rows leave; a workgroup's row is uniform
    const T* x = (const T*)a.x + row * a.xs;
    const R* res = (const R*)a.residual + row * a.rs;
    const T* gate = (const T*)a.gate + row * a.gs;
    float u[K][W];
    Vec<R, W> r[K];
    Vec<T, W> g[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const Vec<T, W> v = load_vec<W>(x + at[k]);
#pragma unroll
      for (int i = 0; i < W; ++i) u[k][i] = to_float(v.v[i]);
    }
    if (a.residual) {
#pragma unroll
      for (int k = 0; k < K; ++k) r[k] = load_vec<W>(res + at[k]);
    }
    if (a.gate) {
#pragma unroll
      for (int k = 0; k < K; ++k) g[k] = load_vec<W>(gate + at[k]);
    }
    auto sum = [&](auto term) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < W; ++i) s += i >= skip[k] ? term(u[k][i]) : 0.f;
      return row_sum<G>(s, lds) * inv;
    };
    auto normalise = [&](const float* weight, const float* bias) {
      if (!rms) {
        const float mean = sum([](float v) { return v; });
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < W; ++i) u[k][i] -= mean;
      }
      const float rstd = 1.f / sqrtf(sum([](float v) { return v * v; }) + a.eps);
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < W; ++i) u[k][i] *= rstd;
        if (weight) {
          const Vec<float, W> w = load_vec<W>(weight + at[k]);
#pragma unroll
          for (int i = 0; i < W; ++i) u[k][i] *= w.v[i];
        }
        if (bias) {
          const Vec<float, W> w = load_vec<W>(bias + at[k]);
#pragma unroll
          for (int i = 0; i < W; ++i) u[k][i] += w.v[i];
        }
      }
    };
    if (a.post) normalise(a.post_w, a.post_b);
    // a row written in place: every thread has read before any writes
    if (G > 64) __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (a.gate) {
#pragma unroll
        for (int i = 0; i < W; ++i) u[k][i] *= open_gate(to_float(g[k].v[i]), a.act);
      }
      if (a.scale) {
        const Vec<float, W> w = load_vec<W>(a.scale + at[k]);
#pragma unroll
        for (int i = 0; i < W; ++i) u[k][i] *= w.v[i];
      }
      if (a.residual) {
#pragma unroll
        for (int i = 0; i < W; ++i) u[k][i] = fmaf(a.residual_scale, to_float(r[k].v[i]), u[k][i]);
      }
      if (a.out && skip[k] < W) {
        Vec<R, W> o;
#pragma unroll
        for (int i = 0; i < W; ++i) o.v[i] = from_float<R>(u[k][i]);
        store_vec((R*)a.out + row * a.os + at[k], o);
      }
    }
    if (!a.y) continue;
    normalise(a.pre_w, a.pre_b);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (skip[k] >= W) continue;
      Vec<T, W> o;
#pragma unroll
      for (int i = 0; i < W; ++i) o.v[i] = from_float<T>(u[k][i]);
      store_vec((T*)a.y + row * a.ys + at[k], o);
    }
  }
}

// Rows of fewer channels than a wide access holds: a thread a row.
template <class T, class R>
__global__ __launch_bounds__(256) void residual_norm_narrow_kernel(NormArgs a, int rms) {
  constexpr int W = 16 / sizeof(T);
  const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows) return;
  float u[W];
  auto normalise = [&](const float* weight, const float* bias) {
    float mean = 0.f, s = 0.f;
    if (!rms) {
      for (int c = 0; c < W; ++c) mean += c < a.channels ? u[c] : 0.f;
      mean /= (float)a.channels;
    }
    for (int c = 0; c < W; ++c) {
      u[c] = c < a.channels ? u[c] - mean : 0.f;
      s = fmaf(u[c], u[c], s);
    }
    const float rstd = 1.f / sqrtf(s / (float)a.channels + a.eps);
    for (int c = 0; c < W; ++c) {
      if (c >= a.channels) continue;
      u[c] *= rstd;
      if (weight) u[c] *= weight[c];
      if (bias) u[c] += bias[c];
    }
  };
  for (int c = 0; c < W; ++c) u[c] = c < a.channels ? to_float(((const T*)a.x)[row * a.xs + c]) : 0.f;
  if (a.post) normalise(a.post_w, a.post_b);
  for (int c = 0; c < W; ++c) {
    if (c >= a.channels) continue;
    if (a.gate) u[c] *= open_gate(to_float(((const T*)a.gate)[row * a.gs + c]), a.act);
    if (a.scale) u[c] *= a.scale[c];
    if (a.residual)
      u[c] = fmaf(a.residual_scale, to_float(((const R*)a.residual)[row * a.rs + c]), u[c]);
    if (a.out) ((R*)a.out)[row * a.os + c] = from_float<R>(u[c]);
  }
  if (!a.y) return;
  normalise(a.pre_w, a.pre_b);
  for (int c = 0; c < W; ++c)
    if (c < a.channels) ((T*)a.y)[row * a.ys + c] = from_float<T>(u[c]);
}

// The fewest lanes that hold a row in at most 24 channels a thread, the fewest runs a thread that do.
// 16 lanes put four rows in a wave and keep its sums within 16 lanes, but leave few rows too few waves
// to hide their loads.  16 lanes against 64, in us (one norm; both):
//   bf16, bf16 residual, 256 channels   4096 rows 3.9 and 4.2   8192 4.9 and 6.2    262144 99, 104 and 128, 175
//                        320            4.7 and 4.4             6.0 and 6.7         120, 139 and 137, 184
//                        384            4.8 and 4.5             6.3 and 6.6         146, 153 and 150, 194
//   bf16, float32        256            4.4 and 4.5             6.1 and 6.9         142, 154 and 158, 196
//                        320            5.2 and 4.8             7.6 and 7.9         190, 198 and 186, 210
//                        384            5.5 and 5.1             8.4 and 8.7         223, 230 and 216, 237
//   float32              256            5.2 and 5.2             7.2 and 7.9         193, 194 and 199, 229
//                        320            6.3 and 5.6             9.5 and 9.5         282, 268 and 241, 274
//                        384            6.7 and 6.0             10.5 and 10.5       327, 304 and 278, 298
// so from 8192 rows on, up to 384 channels, of float32 up to 256; fewer channels gain more (136: 262144
// rows 63 and 116).
constexpr int64_t kManyRows = 8192;

template <class T, class R>
void residual_norm_launch(const NormArgs& a, int rms, hipStream_t st) {
  constexpr int W = 16 / sizeof(T), S = 8 / W;
  using std::integral_constant;
  if (a.channels < W) {
    residual_norm_narrow_kernel<T, R><<<(unsigned)ceil_div(a.rows, 256), 256, 0, st>>>(a, rms);
    return;
  }
  auto go = [&](auto g, auto k) {
    constexpr int G = decltype(g)::value, K = decltype(k)::value * S;
    constexpr int ROWS = G > 256 ? 1 : 256 / G;
    const int grid = (int)std::min<int64_t>(ceil_div(a.rows, ROWS), 1 << 20);
    residual_norm_kernel<T, R, G, K><<<grid, G > 256 ? G : 256, 0, st>>>(a, rms);
  };
  const integral_constant<int, 1> one;
  const integral_constant<int, 2> two;
  const integral_constant<int, 3> three;
  auto lanes = [&](auto g) {
    const int need = (int)ceil_div(a.channels, decltype(g)::value * 8);
    if (need <= 1) return go(g, one);
    if (need <= 2) return go(g, two);
    go(g, three);
  };
  constexpr int kMost = sizeof(T) == 4 ? 256 : 16 * 24;
  if (a.channels <= 128 || (a.channels <= kMost && a.rows >= kManyRows)) return lanes(integral_constant<int, 16>{});
  if (a.channels <= 64 * 24) return lanes(integral_constant<int, 64>{});
  if (a.channels <= 256 * 24) return lanes(integral_constant<int, 256>{});
  go(integral_constant<int, 1024>{}, two);
}

}  // namespace

void residual_norm(const nnx_residual_norm_config& c, const void* x, const void* residual,
                   const void* gate, const float* scale, const float* post_weight,
                   const float* post_bias, const float* pre_weight, const float* pre_bias,
                   void* residual_out, void* y, hipStream_t st) {
  require(known_type(c.type), "residual norm: unknown type");
  require(c.residual_type == c.type || c.residual_type == NNX_TYPE_F32,
          "residual norm: the residual is of the branch's type or float32");
  require(c.rows >= 1 && c.rows < (int64_t)1 << 31, "residual norm: 1 to 2^31 - 1 rows");
  require(c.channels >= 1 && c.channels <= 16384, "residual norm: channels must be 1..16384");
  require(c.kind == NNX_TOKEN_NORM_LAYER || c.kind == NNX_TOKEN_NORM_RMS,
          "residual norm: unknown norm");
  require(c.gate_activation >= NNX_GATE_NONE && c.gate_activation <= NNX_GATE_SILU,
          "residual norm: unknown gate activation");
  require(c.eps >= 0.f && std::isfinite(c.eps) && std::isfinite(c.residual_scale),
          "residual norm: eps must be finite and not negative, the residual scale finite");
  require(x && (residual_out || y), "residual norm: null pointer");
  const NormArgs a{x,           residual,   gate,          scale,           post_weight,
                   post_bias,   pre_weight, pre_bias,      residual_out,    y,
                   c.rows,      c.x_stride, c.residual_stride, c.gate_stride, c.residual_out_stride,
                   c.y_stride,  c.channels, c.post != 0,   c.gate_activation, c.residual_scale,
                   c.eps};
  const double n = (double)c.rows * c.channels;
  ProfScope prof("residual_norm", 10.0 * n,
                 n * (type_bytes(c.type) * (1.0 + !!gate + !!y) +
                      type_bytes(c.residual_type) * (1.0 * !!residual + !!residual_out)),
                 st);
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    const int rms = c.kind == NNX_TOKEN_NORM_RMS;
    if (c.residual_type == c.type) {
      residual_norm_launch<T, T>(a, rms, st);
    } else {
      residual_norm_launch<T, float>(a, rms, st);
    }
  });
  launch_check("residual_norm");
}

}  // namespace nnx
