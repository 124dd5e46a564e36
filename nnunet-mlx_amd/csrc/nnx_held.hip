// Keys and values held in 8 bits: quantised as they are written, read back, and the attention that
// reads them as they are.
#include <algorithm>
#include <cmath>

#include "nnx_elements.h"

namespace nnx {

namespace {

constexpr float kTiny = 8.673617379884035e-19f;  // 2^-60
constexpr float kMost = 3.4028233e38f;           // 127 * (kMost / 127) is finite

struct HeldArgs {
  int batch, tokens, slots, keys, heads, kv_heads, dim, causal;
  float scale;
  int64_t start0;
  int64_t s[2][3], ms;
  const int32_t *start, *lengths;
  const uint8_t* mask;
};

HeldArgs make_args(const nnx_held_config& c, const int32_t* start, const int32_t* lengths, const uint8_t* mask) {
  HeldArgs a;
  a.batch = c.batch, a.tokens = c.tokens, a.slots = c.slots, a.keys = c.keys;
  a.heads = c.heads, a.kv_heads = c.kv_heads, a.dim = c.head_dim, a.causal = c.causal != 0;
  a.scale = c.scale, a.start0 = c.start, a.ms = c.mask_stride;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 3; ++j) a.s[i][j] = c.strides[i][j];
  a.start = start, a.lengths = lengths, a.mask = mask;
  return a;
}

// Place of a value's code among those of its item and key head.
__device__ __forceinline__ int64_t value_at(int slot, int d, int dim) {
  const int s = slot % 64;
  return ((int64_t)(slot / 64) * dim + d) * 64 + s / 4 % 4 * 16 + s / 16 * 4 + s % 4;
}

template <class T>
__global__ __launch_bounds__(256) void hold_kernel(HeldArgs a, const T* k, const T* v, int8_t* k_codes,
                                                   float* k_scales, int8_t* v_codes, float* v_scales) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t rows = (int64_t)a.batch * a.tokens * a.kv_heads;
  if (i >= 2 * rows) return;
  const int which = i >= rows;
  const int64_t r = which ? i - rows : i, bt = r / a.kv_heads;
  const int g = (int)(r - bt * a.kv_heads), b = (int)(bt / a.tokens), t = (int)(bt - (int64_t)b * a.tokens);
  const int64_t slot = a.start0 + (a.start ? a.start[b] : 0) + t;
  if (slot < 0 || slot >= a.slots || (a.lengths && t >= a.lengths[b])) return;
  const T* x = (which ? v : k) + b * a.s[which][0] + t * a.s[which][1] + g * a.s[which][2];
  float top = 0.f;
  bool odd = false;
  for (int d = 0; d < a.dim; ++d) {
    const float e = fabsf(to_float(x[d]));
    top = fmaxf(top, e);
    odd |= !(e < INFINITY);
  }
  const bool zero = odd || top < kTiny;
  const float up = zero ? 0.f : 127.f / top;
  const int64_t item = (int64_t)b * a.kv_heads + g;
  int8_t* codes = (which ? v_codes : k_codes) + item * a.slots * a.dim;
  for (int d = 0; d < a.dim; ++d) {
    const int8_t code = zero ? 0 : (int8_t)(int)rintf(to_float(x[d]) * up);
    codes[which ? value_at((int)slot, d, a.dim) : slot * a.dim + d] = code;
  }
  (which ? v_scales : k_scales)[item * a.slots + slot] = odd ? NAN : zero ? 0.f : fminf(top, kMost) / 127.f;
}

// code * scale in float32.  Kept apart from its conversion: the two as one instruction round a float16 from
// the exact product.
__device__ __forceinline__ float stands_for(float code, float scale) {
  float v = code * scale;
  asm("" : "+v"(v));
  return v;
}

template <class T>
__global__ __launch_bounds__(256) void read_kernel(HeldArgs a, const int8_t* k_codes, const float* k_scales,
                                                   const int8_t* v_codes, const float* v_scales, T* k, T* v) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t all = (int64_t)a.batch * a.tokens * a.kv_heads * a.dim;
  if (i >= 2 * all) return;
  const int which = i >= all;
  const int64_t e = which ? i - all : i, r = e / a.dim, bt = r / a.kv_heads;
  const int d = (int)(e - r * a.dim), g = (int)(r - bt * a.kv_heads);
  const int b = (int)(bt / a.tokens), t = (int)(bt - (int64_t)b * a.tokens), slot = (int)a.start0 + t;
  const int64_t item = (int64_t)b * a.kv_heads + g;
  const int8_t* codes = (which ? v_codes : k_codes) + item * a.slots * a.dim;
  const float code = (float)codes[which ? value_at(slot, d, a.dim) : (int64_t)slot * a.dim + d];
  T* y = (which ? v : k) + b * a.s[which][0] + t * a.s[which][1] + g * a.s[which][2];
  y[d] = from_float<T>(stands_for(code, (which ? v_scales : k_scales)[item * a.slots + slot]));
}

// A workgroup a query and head: 256 slots at a time, their logits a thread each, then a thread a channel.
template <class T>
__global__ __launch_bounds__(256) void attend_kernel(HeldArgs a, float down, const T* q, const int8_t* k_codes,
                                                     const float* k_scales, const int8_t* v_codes,
                                                     const float* v_scales, T* out) {
  __shared__ float qs[128], ws[256], red[4];
  const int h = blockIdx.x % a.heads;
  const int64_t bt = blockIdx.x / a.heads;
  const int b = (int)(bt / a.tokens), t = (int)(bt - (int64_t)b * a.tokens);
  const int64_t item = (int64_t)b * a.kv_heads + h / (a.heads / a.kv_heads);
  const T* row = q + b * a.s[0][0] + t * a.s[0][1] + h * a.s[0][2];
  if (threadIdx.x < a.dim) qs[threadIdx.x] = to_float(row[threadIdx.x]) * 0x1p-14f;  // products with codes stay finite
  int64_t n = a.lengths ? min(a.lengths[b], a.keys) : a.keys;
  if (a.causal) n = min(n, a.start0 + (a.start ? a.start[b] : 0) + t + 1);
  const float c2 = a.scale * (1.4426950408889634f * 0x1p14f), unit = exp2f(-down);
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int s0 = 0; s0 < n; s0 += 256) {
    __syncthreads();
    const int slot = s0 + threadIdx.x;
    const bool seen = slot < n && (!a.mask || a.mask[b * a.ms + slot]);
    float x = -INFINITY;
    if (seen) {
      const int8_t* key = k_codes + (item * a.slots + slot) * a.dim;
      float dot = 0.f;
      for (int d = 0; d < a.dim; ++d) dot = fmaf(qs[d], (float)key[d], dot);
      x = dot * k_scales[item * a.slots + slot] * c2;
    }
    const float most = lanes_reduce<64>(x, [](float p, float r) { return fmaxf(p, r); });
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = most;
    __syncthreads();
    const float next = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float top = next == -INFINITY ? 0.f : next;
    const float back = m == -INFINITY ? 0.f : exp2f(m - next);
    m = next;
    ws[threadIdx.x] = seen ? exp2f(x - top) : -1.f;
    __syncthreads();
    float ls = 0.f, os = 0.f;  // of 256 slots: sums of sums lose less
    for (int j = 0; j < 256 && s0 + j < n; ++j) {
      const float w = ws[j];
      if (w < 0.f) continue;  // not seen
      ls += w;
      if (threadIdx.x < a.dim)
        os = fmaf(w * (v_scales[item * a.slots + s0 + j] * unit),
                 (float)v_codes[item * a.slots * a.dim + value_at(s0 + j, threadIdx.x, a.dim)], os);
    }
    l = fmaf(l, back, ls), o = fmaf(o, back, os);
  }
  if (threadIdx.x < a.dim)
    (out + b * a.s[1][0] + t * a.s[1][1] + h * a.s[1][2])[threadIdx.x] = from_float<T>(l == 0.f ? 0.f : o / l / unit);
}

void check_config(const nnx_held_config& c, const char* name, bool attention) {
  const std::string n(name);
  require(known_type(c.type), n + ": unknown type");
  require(c.batch >= 1 && c.batch <= 65535 && c.tokens >= 1, n + ": 1 to 65535 items of at least one token");
  require(c.slots >= 64 && c.slots % 64 == 0, n + ": slots must be a positive multiple of 64");
  require(c.kv_heads >= 1 && c.kv_heads <= 65536, n + ": 1 to 65536 key heads");
  require(c.head_dim >= 16 && c.head_dim <= 128 && c.head_dim % 16 == 0,
          n + ": head_dim must be a multiple of 16, 16..128");
  require((double)c.batch * c.slots * c.kv_heads * c.head_dim < 9e18, n + ": too many elements");
  require(c.start >= 0 && c.start < (int64_t)1 << 40, n + ": start must be 0..2^40 - 1");
  if (!attention) return;
  require(c.keys >= 1 && c.keys <= c.slots, n + ": keys must be 1 to the slots");
  require(c.heads >= 1 && c.heads <= 65536 && c.heads % c.kv_heads == 0,
          n + ": heads must be a multiple of the key heads, up to 65536");
  require((double)c.batch * c.tokens * c.heads < 2147483648.0, n + ": fewer than 2^31 queries times heads");
  require(std::isfinite(c.scale), n + ": the scale must be finite");
}

void check_held(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                const char* name) {
  require(k_codes && k_scales && v_codes && v_scales, std::string(name) + ": null pointer");
  require((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(k_scales) |
           reinterpret_cast<uintptr_t>(v_codes) | reinterpret_cast<uintptr_t>(v_scales)) % 16 == 0,
          std::string(name) + ": codes and scales must be 16-byte aligned");
}

}  // namespace

void hold_tokens(const nnx_held_config& c, const void* k, const void* v, const int32_t* start,
                 const int32_t* lengths, int8_t* k_codes, float* k_scales, int8_t* v_codes,
                 float* v_scales, hipStream_t st) {
  check_config(c, "hold tokens", false);
  const double rows = 2.0 * c.batch * c.tokens * c.kv_heads;
  require(rows < 2147483648.0, "hold tokens: fewer than 2^30 tokens times key heads");
  require(k && v, "hold tokens: null pointer");
  check_held(k_codes, k_scales, v_codes, v_scales, "hold tokens");
  const HeldArgs a = make_args(c, start, lengths, nullptr);
  ProfScope prof("hold_tokens", 4.0 * rows * c.head_dim, rows * (c.head_dim * (type_bytes(c.type) + 1.0) + 4.0), st);
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    hold_kernel<T><<<(unsigned)ceil_div((int64_t)rows, 256), 256, 0, st>>>(
        a, (const T*)k, (const T*)v, k_codes, k_scales, v_codes, v_scales);
  });
  launch_check("hold_tokens");
}

void read_held(const nnx_held_config& c, const int8_t* k_codes, const float* k_scales,
               const int8_t* v_codes, const float* v_scales, void* k, void* v, hipStream_t st) {
  check_config(c, "read held", false);
  const double rows = 2.0 * c.batch * c.tokens * c.kv_heads;
  require(rows < 2147483648.0, "read held: fewer than 2^30 tokens times key heads");
  require(c.start + c.tokens <= c.slots, "read held: slots start to start + tokens - 1 must be there");
  require(k && v, "read held: null pointer");
  check_held(k_codes, k_scales, v_codes, v_scales, "read held");
  const HeldArgs a = make_args(c, nullptr, nullptr, nullptr);
  ProfScope prof("read_held", rows * c.head_dim, rows * (c.head_dim * (type_bytes(c.type) + 1.0) + 4.0), st);
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    read_kernel<T><<<(unsigned)ceil_div((int64_t)rows * c.head_dim, 256), 256, 0, st>>>(
        a, k_codes, k_scales, v_codes, v_scales, (T*)k, (T*)v);
  });
  launch_check("read_held");
}

size_t held_attention_workspace(const nnx_held_config& c) {
  try {
    check_config(c, "held attention", true);
    return 0;
  } catch (...) {  // nothing may leave a C entry
    return 0;
  }
}

void held_attention(const nnx_held_config& c, const void* q, const int8_t* k_codes,
                    const float* k_scales, const int8_t* v_codes, const float* v_scales,
                    const int32_t* start, const int32_t* lengths, const uint8_t* mask, void* out,
                    void* ws, size_t ws_bytes, hipStream_t st) {
  check_config(c, "held attention", true);
  require(q && out, "held attention: null pointer");
  check_held(k_codes, k_scales, v_codes, v_scales, "held attention");
  const HeldArgs a = make_args(c, start, lengths, mask);
  const double rows = (double)c.batch * c.tokens * c.heads;
  ProfScope prof("held_attention", 4.0 * rows * c.keys * c.head_dim,
                 2.0 * rows * c.head_dim * type_bytes(c.type) +
                     2.0 * c.batch * c.kv_heads * c.keys * (c.head_dim + 4.0),
                 st);
  const float down = ceilf(log2f((float)c.keys));
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    attend_kernel<T><<<(unsigned)(int64_t)rows, 256, 0, st>>>(a, down, (const T*)q, k_codes, k_scales, v_codes,
                                                             v_scales, (T*)out);
  });
  launch_check("held_attention");
}

}  // namespace nnx
