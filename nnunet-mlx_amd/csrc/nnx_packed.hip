// Products with 4-bit weights under group scales, and their packing.
#include <algorithm>
#include <cmath>

#include "nnx_elements.h"

namespace nnx {

namespace {

constexpr float kTiny = 8.673617379884035e-19f;  // 2^-60
constexpr float kMost = 3.4028233e38f;           // 6 * (kMost / 6) is finite

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
  const int groups = a.blocks * (128 / a.group), padded = (a.outputs + 15) / 16 * 16;
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= (int64_t)padded * groups) return;
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
  const bool zero = odd || top < kTiny;
  const float up = zero ? 0.f : 6.f / top;
  auto code_of = [&](int i) {
    if (zero || i >= i1) return 0;
    const float x = to_float(row[i]), s = fabsf(x) * up;
    const int e = (s > 0.25f) + (s >= 0.75f) + (s > 1.25f) + (s >= 1.75f) + (s > 2.5f) + (s >= 3.5f) + (s > 5.f);
    return e | (e && x < 0.f ? 8 : 0);
  };
  for (int i = i0; i < i0 + a.group; i += 2) codes[code_at(a, o, i)] = (uint8_t)(code_of(i) | code_of(i + 1) << 4);
  scales[scale_at(a, o, g)] = odd ? NAN : zero ? 0.f : fminf(top, kMost) / 6.f;
}

template <class T>
__global__ __launch_bounds__(256) void unpack_kernel(PackedArgs a, const uint8_t* codes, const float* scales, T* w) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= (int64_t)a.outputs * a.inputs) return;
  const int o = (int)(n / a.inputs), i = (int)(n - (int64_t)o * a.inputs);
  const int code = codes[code_at(a, o, i)] >> (i % 2 * 4) & 15;
  float v = level(code) * scales[scale_at(a, o, i / a.group)];
  asm("" : "+v"(v));  // one instruction with the conversion would round a float16 from the exact product
  w[o * a.xs + i] = from_float<T>(v);
}

__device__ __forceinline__ float open_gate(float g, int act) {
  if (act == NNX_GATE_NONE) return g;
  const float s = 1.f / (1.f + expf(-g));
  return act == NNX_GATE_SIGMOID ? s : g * s;
}

// A wave an output and row, a group at a time.
template <class T>
__global__ __launch_bounds__(64) void linear_kernel(PackedArgs a, const T* x, const uint8_t* codes, const float* scales,
                                                    const float* bias, const uint8_t* gate_codes,
                                                    const float* gate_scales, T* y) {
  const int o = blockIdx.x;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    auto product = [&](const uint8_t* codes, const float* scales) {
      float sum = 0.f;
      for (int g = 0; g * a.group < a.inputs; ++g) {
        float part = 0.f;
        for (int i = g * a.group + threadIdx.x; i < min((g + 1) * a.group, a.inputs); i += 64)
          part = fmaf(to_float(x[row * a.xs + i]), level(codes[code_at(a, o, i)] >> (i % 2 * 4) & 15), part);
        sum = fmaf(part, scales[scale_at(a, o, g)], sum);
      }
      return lanes_reduce<64>(sum, [](float p, float r) { return p + r; });
    };
    float u = product(codes, scales);
    if (bias) u += bias[o];
    if (gate_codes) u *= open_gate(product(gate_codes, gate_scales), a.act);
    if (threadIdx.x == 0) y[row * a.ys + o] = from_float<T>(u);
  }
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
    pack_kernel<T><<<(unsigned)ceil_div(groups, 256), 256, 0, st>>>(a, (const T*)w, codes, scales);
  });
  launch_check("pack_weight");
}

void unpack_weight(const nnx_packed_config& c, const uint8_t* codes, const float* scales, void* w, hipStream_t st) {
  check_config(c, "unpack weight");
  require(w, "unpack weight: null pointer");
  check_packed(codes, scales, "unpack weight");
  const PackedArgs a = make_args(c);
  const int64_t n = (int64_t)c.outputs * c.inputs;
  require(n < (int64_t)1 << 38, "unpack weight: fewer than 2^38 weights");
  ProfScope prof("unpack_weight", 0.0, (double)n * (type_bytes(c.type) + 0.5), st);
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    unpack_kernel<T><<<(unsigned)ceil_div(n, 256), 256, 0, st>>>(a, codes, scales, (T*)w);
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
    const dim3 grid((unsigned)c.outputs, (unsigned)std::min<int64_t>(c.rows, 65535));
    linear_kernel<T><<<grid, 64, 0, st>>>(a, (const T*)x, codes, scales, bias, gate_codes, gate_scales, (T*)y);
  });
  launch_check("packed_linear");
}

}  // namespace nnx
