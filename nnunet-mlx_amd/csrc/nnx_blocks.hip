// Attention over blocks of keys that a cheap score selects for each query: block summaries,
// selection and the attention itself.
#include <algorithm>
#include <cmath>

#include "nnx_elements.h"

namespace nnx {
namespace {

constexpr int kMaxBlocks = 32768;
constexpr int kMaxKeep = 256;
constexpr float kTiny = 8.673617379884035e-19f;  // 2^-60

struct BlockArgs {
  int batch, queries, keys, heads, kv_heads, group, dim, block, blocks, keep, first, local, causal;
  int64_t start0;
  float scale;
  int64_t qs[3], ks[3], vs[3], os[3], ms;
  const int32_t *start, *lengths;
  const uint8_t* mask;
};

void check_config(const nnx_block_config& c, const char* what, bool queries) {
  const std::string w = std::string(what) + ": ";
  require(known_type(c.type), w + "unknown type");
  require(c.batch >= 1 && c.batch <= 65535 && c.keys >= 1, w + "1 to 65535 items with keys");
  require(c.kv_heads >= 1 && c.kv_heads <= 65535, w + "1 to 65535 key heads");
  require(c.head_dim >= 8 && c.head_dim <= 128 && c.head_dim % 8 == 0,
          w + "head_dim must be a multiple of 8, 8..128");
  require(c.block == 16 || c.block == 32 || c.block == 64 || c.block == 128,
          w + "block must be 16, 32, 64 or 128");
  require(ceil_div(c.keys, c.block) <= kMaxBlocks, w + "at most 32768 blocks");
  if (queries) {
    require(c.queries >= 1, w + "no queries");
    require(c.heads >= 1 && c.heads % c.kv_heads == 0, w + "heads must be a multiple of the key heads");
    require(c.keep >= 1 && c.keep <= kMaxKeep, w + "keep must be 1..256");
    require((double)c.batch * c.queries * c.kv_heads * c.keep < 2147483648.0 &&
                (double)c.batch * c.queries * c.heads < 2147483648.0,
            w + "at most 2^31 - 1 kept blocks and query rows");
    require(std::isfinite(c.scale), w + "the scale must be finite");
    require(c.start >= 0 && c.start < (int64_t)1 << 40, w + "start must be 0..2^40");
    require(c.first >= 0 && c.local >= 0, w + "first and local must not be negative");
  }
}

BlockArgs make_args(const nnx_block_config& c, const int32_t* start, const int32_t* lengths,
                    const uint8_t* mask) {
  BlockArgs a;
  a.batch = c.batch, a.queries = c.queries, a.keys = c.keys, a.heads = c.heads;
  a.kv_heads = c.kv_heads, a.group = c.heads / c.kv_heads, a.dim = c.head_dim, a.block = c.block;
  a.blocks = (int)ceil_div(c.keys, c.block), a.keep = c.keep, a.first = c.first, a.local = c.local;
  a.causal = c.causal != 0, a.start0 = c.start, a.scale = c.scale, a.ms = c.mask_stride;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = c.q_strides[i], a.ks[i] = c.k_strides[i], a.vs[i] = c.v_strides[i];
    a.os[i] = c.out_strides[i];
  }
  a.start = start, a.lengths = lengths, a.mask = mask;
  return a;
}

__device__ __forceinline__ int item_length(const BlockArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.keys) : a.keys;
}

__device__ __forceinline__ int64_t item_start(const BlockArgs& a, int b) {
  return a.start0 + (a.start ? a.start[b] : 0);
}

__device__ __forceinline__ float finite_or_zero(float v) { return fabsf(v) < INFINITY ? v : 0.f; }

// A workgroup of 128 threads a block of keys, a thread a channel.
template <class T>
__global__ __launch_bounds__(128) void summarize_kernel(BlockArgs a, const T* k, int first,
                                                        int8_t* codes, float* scales) {
  __shared__ float top_lds[2];
  __shared__ int most_lds[2];
  const int j = first + blockIdx.x, g = blockIdx.y, b = blockIdx.z, d = threadIdx.x;
  const int lo = j * a.block, hi = min(lo + a.block, item_length(a, b));
  const T* kb = k + b * a.ks[0] + g * a.ks[2];
  const bool has = d < a.dim;
  int count = 0;
  float top = 0.f;
  for (int i = lo; i < hi; ++i) {
    if (a.mask && !a.mask[b * a.ms + i]) continue;
    ++count;
    if (has) top = fmaxf(top, fabsf(finite_or_zero(to_float(kb[i * a.ks[1] + d]))));
  }
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (d % 64 == 0) top_lds[d / 64] = top;
  __syncthreads();
  top = fmaxf(top_lds[0], top_lds[1]);
  int sum = 0;
  if (has && top >= kTiny) {
    const float up = __fdiv_rn(32767.f, top);
    for (int i = lo; i < hi; ++i) {
      if (a.mask && !a.mask[b * a.ms + i]) continue;
      sum += (int)rintf(finite_or_zero(to_float(kb[i * a.ks[1] + d])) * up);
    }
  }
  int most = abs(sum);
  for (int o = 32; o; o >>= 1) most = max(most, __shfl_xor(most, o));
  if (d % 64 == 0) most_lds[d / 64] = most;
  __syncthreads();
  most = max(most_lds[0], most_lds[1]);
  const int64_t at = ((int64_t)b * a.kv_heads + g) * a.blocks + j;
  if (has) {
    const float down = most ? __fdiv_rn(127.f, (float)most) : 0.f;
    codes[at * a.dim + d] = (int8_t)(int)rintf((float)sum * down);
  }
  if (d == 0) {
    scales[at] = count == 0 ? -1.f
                 : most == 0 ? 0.f
                             : __fdiv_rn(top, 4161409.f * (float)count) * (float)most;
  }
}

// A workgroup a query and key head: all scores in LDS, then `keep` times the best.
template <class T>
__global__ __launch_bounds__(256) void select_kernel(BlockArgs a, const T* q, const int8_t* codes,
                                                     const float* scales, int32_t* ids) {
  extern __shared__ float score[];  // blocks
  __shared__ int8_t qc[128];
  __shared__ float qtop;
  __shared__ float best_v[4];
  __shared__ int best_i[4];
  const int t = blockIdx.x, g = blockIdx.y, b = blockIdx.z;
  const int64_t at = (item_start(a, b) + t) / a.block;
  const int64_t unit = (int64_t)b * a.kv_heads + g;
  int32_t* row = ids + (((int64_t)b * a.queries + t) * a.kv_heads + g) * a.keep;
  for (int j = threadIdx.x; j < a.blocks; j += 256) score[j] = -INFINITY;
  for (int h = 0; h < a.group; ++h) {
    const T* qr = q + b * a.qs[0] + t * a.qs[1] + (g * a.group + h) * a.qs[2];
    __syncthreads();
    if (threadIdx.x < 64) {
      const int d = threadIdx.x;
      const float v0 = d < a.dim ? finite_or_zero(to_float(qr[d])) : 0.f;
      const float v1 = d + 64 < a.dim ? finite_or_zero(to_float(qr[d + 64])) : 0.f;
      float top = fmaxf(fabsf(v0), fabsf(v1));
      for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
      const float up = top < kTiny ? 0.f : __fdiv_rn(127.f, top);
      qc[d] = (int8_t)(int)rintf(v0 * up);
      qc[d + 64] = (int8_t)(int)rintf(v1 * up);
      if (d == 0) qtop = top < kTiny ? 1.f : top;
    }
    __syncthreads();
    for (int j = threadIdx.x; j < a.blocks; j += 256) {
      const int8_t* cb = codes + (unit * a.blocks + j) * a.dim;
      int dot = 0;
      for (int d = 0; d < a.dim; ++d) dot += (int)cb[d] * (int)qc[d];
      const float sc = scales[unit * a.blocks + j];
      float s = ((float)dot * qtop) * sc;
      if (j < a.first || (j <= at && j > at - a.local)) s = INFINITY;
      if (sc < 0.f || (a.causal && j > at)) s = -INFINITY;
      score[j] = fmaxf(score[j], s);
    }
  }
  __syncthreads();
  int found = 0;
  for (; found < a.keep; ++found) {
    float v = -INFINITY;
    int at_i = a.blocks;
    for (int j = threadIdx.x; j < a.blocks; j += 256) {
      if (score[j] > v) v = score[j], at_i = j;
    }
    for (int o = 32; o; o >>= 1) {
      const float ov = __shfl_xor(v, o);
      const int oi = __shfl_xor(at_i, o);
      if (ov > v || (ov == v && oi < at_i)) v = ov, at_i = oi;
    }
    __syncthreads();
    if (threadIdx.x % 64 == 0) best_v[threadIdx.x / 64] = v, best_i[threadIdx.x / 64] = at_i;
    __syncthreads();
    for (int w = 0; w < 4; ++w) {
      if (best_v[w] > v || (best_v[w] == v && best_i[w] < at_i)) v = best_v[w], at_i = best_i[w];
    }
    if (v == -INFINITY) break;
    // ascending: the kept ones stay marked and are written in order below
    if (threadIdx.x == 0) score[at_i] = NAN;
    __syncthreads();
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    for (int j = 0; j < a.blocks && n < found; ++j) {
      if (score[j] != score[j]) row[n++] = j;
    }
    for (; n < a.keep; ++n) row[n] = -1;
  }
}

// A wave a query row: running maximum and sum over 64 keys at a time, a lane a key.
template <class T>
__global__ __launch_bounds__(64) void attention_kernel(BlockArgs a, const T* q, const T* k,
                                                       const T* v, const int32_t* ids, T* out) {
  __shared__ float qv[128];
  const int lane = threadIdx.x;
  const int h = blockIdx.y, b = blockIdx.z, g = h / a.group;
  const int t = blockIdx.x;
  const T* qr = q + b * a.qs[0] + t * a.qs[1] + h * a.qs[2];
  for (int d = lane; d < a.dim; d += 64) qv[d] = to_float(qr[d]);
  __syncthreads();
  const int length = item_length(a, b);
  const int64_t pos = item_start(a, b) + t;
  const int32_t* row = ids + (((int64_t)b * a.queries + t) * a.kv_heads + g) * a.keep;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int s = 0; s < a.keep; ++s) {
    const int j = row[s];
    if (j < 0 || j >= a.blocks) continue;
    for (int base = j * a.block; base < min((j + 1) * a.block, length); base += 64) {
      const int i = base + lane;
      bool see = i < min((j + 1) * a.block, length) && (!a.causal || i <= pos);
      if (see && a.mask) see = a.mask[b * a.ms + i] != 0;
      float x = -INFINITY;
      if (see) {
        const T* kr = k + b * a.ks[0] + i * a.ks[1] + g * a.ks[2];
        float dot = 0.f;
        for (int d = 0; d < a.dim; ++d) dot = fmaf(qv[d], to_float(kr[d]), dot);
        x = dot * a.scale;
      }
      float top = x;
      for (int w = 32; w; w >>= 1) top = fmaxf(top, __shfl_xor(top, w));
      const float mn = fmaxf(m, top);
      if (mn == -INFINITY) continue;
      const float p = see ? expf(x - mn) : 0.f;
      float sum = p;
      for (int w = 32; w; w >>= 1) sum += __shfl_xor(sum, w);
      const float old = expf(m - mn);
      l = l * old + sum;
      o0 *= old, o1 *= old;
      m = mn;
      for (int w = 0; w < 64; ++w) {
        const float pw = __shfl(p, w);
        if (pw == 0.f) continue;  // unseen values are never read
        const T* vr = v + b * a.vs[0] + (int64_t)(base + w) * a.vs[1] + g * a.vs[2];
        if (lane < a.dim) o0 = fmaf(pw, to_float(vr[lane]), o0);
        if (lane + 64 < a.dim) o1 = fmaf(pw, to_float(vr[lane + 64]), o1);
      }
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  T* orow = out + b * a.os[0] + t * a.os[1] + h * a.os[2];
  if (lane < a.dim) orow[lane] = from_float<T>(o0 * inv);
  if (lane + 64 < a.dim) orow[lane + 64] = from_float<T>(o1 * inv);
}

}  // namespace

void block_summarize(const nnx_block_config& c, const void* k, const int32_t* lengths,
                     const uint8_t* mask, int first_block, int blocks, int8_t* codes,
                     float* scales, hipStream_t st) {
  check_config(c, "block summaries", false);
  const BlockArgs a = make_args(c, nullptr, lengths, mask);
  require(first_block >= 0 && blocks >= 0 && blocks <= a.blocks && first_block <= a.blocks - blocks,
          "block summaries: the asked blocks are not blocks of the keys");
  require(k && codes && scales, "block summaries: null pointer");
  if (blocks == 0) return;
  const double n = (double)c.batch * blocks * c.block * c.kv_heads * c.head_dim;
  ProfScope prof("block_summarize", 3.0 * n, n * type_bytes(c.type), st);
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    summarize_kernel<T><<<dim3(blocks, c.kv_heads, c.batch), 128, 0, st>>>(a, (const T*)k, first_block,
                                                                           codes, scales);
  });
  launch_check("block_summarize");
}

void block_select(const nnx_block_config& c, const void* q, const int8_t* codes,
                  const float* scales, const int32_t* start, int32_t* ids, hipStream_t st) {
  check_config(c, "block selection", true);
  require(q && codes && scales && ids, "block selection: null pointer");
  const BlockArgs a = make_args(c, start, nullptr, nullptr);
  const double rows = (double)c.batch * c.queries * c.heads;
  ProfScope prof("block_select", 2.0 * rows * a.blocks * c.head_dim,
                 rows * c.head_dim * type_bytes(c.type), st);
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    select_kernel<T><<<dim3(c.queries, c.kv_heads, c.batch), 256, a.blocks * sizeof(float), st>>>(
        a, (const T*)q, codes, scales, ids);
  });
  launch_check("block_select");
}

size_t block_attention_workspace(const nnx_block_config& c) {
  try {
    check_config(c, "block attention", true);
  } catch (const Error&) {
    return 0;
  }
  return 16;
}

void block_attention(const nnx_block_config& c, const void* q, const void* k, const void* v,
                     const int32_t* ids, const int32_t* start, const int32_t* lengths,
                     const uint8_t* mask, void* out, void* ws, size_t ws_bytes, hipStream_t st) {
  check_config(c, "block attention", true);
  require(q && k && v && ids && out && ws, "block attention: null pointer");
  require(ws_bytes >= block_attention_workspace(c), "block attention: workspace too small");
  const BlockArgs a = make_args(c, start, lengths, mask);
  const double pairs = (double)c.batch * c.queries * c.heads * c.keep * c.block;
  ProfScope prof("block_attention", 4.0 * pairs * c.head_dim, 0.0, st);
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    attention_kernel<T><<<dim3(c.queries, c.heads, c.batch), 64, 0, st>>>(
        a, (const T*)q, (const T*)k, (const T*)v, ids, (T*)out);
  });
  launch_check("block_attention");
}

}  // namespace nnx
