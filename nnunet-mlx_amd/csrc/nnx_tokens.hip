// Row operators over tokens: rotary positions, and the norms around a block with its gate,
// scale and residual sum.
#include <cmath>

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

template <class T>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  const int units = a.half + (a.dim - 2 * a.half);  // pairs, then copied elements
  const int all = a.heads[0] + a.heads[1];
  const int64_t n = (int64_t)a.batch * a.tokens * all * units;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int u = (int)(i % units);
    int64_t r = i / units;
    int h = (int)(r % all);
    r /= all;
    const int t = (int)(r % a.tokens), b = (int)(r / a.tokens);
    const int which = h >= a.heads[0];
    if (which) h -= a.heads[0];
    const T* x = (const T*)a.x[which] + b * a.xs[which][0] + t * a.xs[which][1] + h * a.xs[which][2];
    T* y = (T*)a.y[which] + b * a.ys[which][0] + t * a.ys[which][1] + h * a.ys[which][2];
    if (u >= a.half) {
      y[a.half + u] = x[a.half + u];
      continue;
    }
    const int axis = min(max(a.pair_axes[u], 0), a.axes - 1);
    const int64_t p = a.pos[b * a.ps[0] + t * a.ps[1] + axis];
    const uint64_t phase = (uint64_t)p * (uint64_t)a.steps[u];
    float s, c;
    sincospif((float)(int32_t)(phase >> 32) * 4.656612873077393e-10f, &s, &c);
    c *= a.amp;
    s *= a.amp_sin;
    const int i0 = a.interleaved ? 2 * u : u, i1 = a.interleaved ? 2 * u + 1 : u + a.half;
    const float v0 = to_float(x[i0]), v1 = to_float(x[i1]);
    y[i0] = from_float<T>(fmaf(v0, c, -(v1 * s)));
    y[i1] = from_float<T>(fmaf(v1, c, v0 * s));
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
  const int64_t units = (int64_t)c.batch * c.tokens * (c.heads[0] + c.heads[1]) * (c.head_dim - a.half);
  const int grid = (int)std::min<int64_t>(ceil_div(units, 256), 1 << 20);
  ProfScope prof("rotary", 3.0 * elems, 2.0 * elems * type_bytes(c.type), st);
  with_type(c.type, [&](auto t) { rotary_kernel<decltype(t)><<<grid, 256, 0, st>>>(a); });
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

__device__ float block_sum(float v, float* lds) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

// A workgroup a row; every pass forms its values again from global memory.
template <class T, class R, bool RMS>
__global__ __launch_bounds__(256) void residual_norm_kernel(NormArgs a) {
  __shared__ float lds[4];
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.xs;
  const float inv = 1.f / (float)a.channels;
  auto stats = [&](auto value, float& mean, float& rstd) {
    float s = 0.f;
    mean = 0.f;
    if (!RMS) {
      for (int c = threadIdx.x; c < a.channels; c += 256) s += value(c);
      mean = block_sum(s, lds) * inv;
    }
    s = 0.f;
    for (int c = threadIdx.x; c < a.channels; c += 256) {
      const float d = value(c) - mean;
      s = fmaf(d, d, s);
    }
    rstd = rsqrtf(block_sum(s, lds) * inv + a.eps);
  };
  auto branch = [&](int c) { return to_float(x[c]); };
  float mean = 0.f, rstd = 1.f;
  if (a.post) stats(branch, mean, rstd);
  auto total = [&](int c) {
    float u = branch(c);
    if (a.post) {
      u = (u - mean) * rstd * (a.post_w ? a.post_w[c] : 1.f);
      if (a.post_b) u += a.post_b[c];
    }
    if (a.gate) {
      float g = to_float(((const T*)a.gate)[row * a.gs + c]);
      if (a.act != NNX_GATE_NONE) {
        const float s = 1.f / (1.f + expf(-g));
        g = a.act == NNX_GATE_SIGMOID ? s : g * s;
      }
      u *= g;
    }
    if (a.scale) u *= a.scale[c];
    if (a.residual) u = fmaf(a.residual_scale, to_float(((const R*)a.residual)[row * a.rs + c]), u);
    return u;
  };
  float mean2 = 0.f, rstd2 = 1.f;
  if (a.y) stats(total, mean2, rstd2);
  for (int c = threadIdx.x; c < a.channels; c += 256) {
    const float r = total(c);
    if (a.y) {
      float v = (r - mean2) * rstd2 * (a.pre_w ? a.pre_w[c] : 1.f);
      if (a.pre_b) v += a.pre_b[c];
      ((T*)a.y)[row * a.ys + c] = from_float<T>(v);
    }
    if (a.out) ((R*)a.out)[row * a.os + c] = from_float<R>(r);
  }
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
    auto run = [&](auto r) {
      using R = decltype(r);
      if (c.kind == NNX_TOKEN_NORM_RMS) {
        residual_norm_kernel<T, R, true><<<(unsigned)c.rows, 256, 0, st>>>(a);
      } else {
        residual_norm_kernel<T, R, false><<<(unsigned)c.rows, 256, 0, st>>>(a);
      }
    };
    if (c.residual_type == c.type) {
      run(T{});
    } else {
      run(float{});
    }
  });
  launch_check("residual_norm");
}

}  // namespace nnx
