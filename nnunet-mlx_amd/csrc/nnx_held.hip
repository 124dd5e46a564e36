// Keys and values held in 8 bits: quantised as they are written, read back, and the attention that
// reads them as they are.
#include <algorithm>
#include <cmath>

#include "nnx_held.h"
#include "nnx_operands.h"

namespace nnx {

namespace {

constexpr int kMostSplits = 512, kUnits = 256;  // a workgroup a CU

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

// Bound by memory: 32768 tokens of 5 heads of 64 in bfloat16 are written in 18 us (42 MB in, 22 out) and read back in
// 13 (5.1 TB/s; a large copy reaches 5.2), both in 29 back to back.  A workgroup a tile of 64 slots of one key head's keys or values, a thread 8
// channels of four slots in a row: rows come in and go out whole (a thread a row: 692 us for both).  Four slots of a
// value channel are one word of its 64 places (slot 16 t + 4 g + i at 16 g + 4 t + i), so value tiles change between
// rows of channels and rows of places by words, through LDS.
constexpr int kPlaceWords = 17;  // from channel to channel there: 16 and a turn of the banks

struct Unit {
  int which, b, g, tile;
};

__device__ __forceinline__ Unit unit_of(const HeldArgs& a, int64_t u, int tiles) {
  Unit r;
  const int64_t rest = u / tiles;
  r.tile = (int)(u - rest * tiles);
  r.which = (int)(rest % 2);
  r.g = (int)(rest / 2 % a.kv_heads);
  r.b = (int)(rest / 2 / a.kv_heads);
  return r;
}

// rint(v) in two's complement, |v| <= 127, in the lowest byte: beside 1.5 * 2^23 a float's last place is 1.
__device__ __forceinline__ uint32_t code_of(float v) { return __float_as_uint(v + 12582912.f); }
__device__ __forceinline__ uint32_t lowest_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400), __builtin_amdgcn_perm(b, a, 0x0c0c0400), 0x05040100);
}

inline int tile_threads(int dim) { return (16 * (dim / 8) + 63) / 64 * 64; }

template <class T>
__global__ __launch_bounds__(256, 4) void hold_kernel(HeldArgs a, const T* k, const T* v, int8_t* k_codes,
                                                   float* k_scales, int8_t* v_codes, float* v_scales, int tiles,
                                                   int64_t units) {
  __shared__ float tops[64 * kPlaceWords];
  __shared__ float ups[64];
  __shared__ uint32_t placed[128 * kPlaceWords];
  const int chunks = a.dim / 8, quad = threadIdx.x / chunks, c = threadIdx.x - quad * chunks;
  const bool works = quad < 16;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const Unit w = unit_of(a, u, tiles);
    const int64_t start = a.start0 + (a.start ? a.start[w.b] : 0);
    const int64_t slot0 = ((start >> 6) + w.tile) * 64;  // of the tile; may lie outside the slots
    const int given = a.lengths ? min(max(a.lengths[w.b], 0), a.tokens) : a.tokens;
    // tokens of the tile: rows r0 to r1, row r token slot0 - start + r
    const int r0 = (int)max((int64_t)0, start - slot0);
    const int r1 = slot0 < 0 || slot0 >= a.slots ? 0 : (int)max((int64_t)0, min((int64_t)64, start + given - slot0));
    if (r0 >= r1) continue;
    const T* x = (w.which ? v : k) + w.b * a.s[w.which][0] + w.g * a.s[w.which][2] + c * 8;
    const int64_t ts = a.s[w.which][1], t0 = slot0 - start;
    const int64_t item = (int64_t)w.b * a.kv_heads + w.g;
    Vec<T, 8> rows[4];
    if (works) {
#pragma unroll
      for (int i = 0; i < 4; ++i)  // of rows that are none: a neighbour's
        rows[i] = load_vec<8>(x + (t0 + min(max(quad * 4 + i, r0), r1 - 1)) * ts);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float m = fabsf(to_float(rows[i].v[e]));
          top = m < INFINITY ? fmaxf(top, m) : INFINITY;  // stays there
        }
        tops[(quad * 4 + i) * kPlaceWords + c] = top;
      }
    }
    __syncthreads();
    for (int r = threadIdx.x; r < 64; r += blockDim.x) {
      float top = 0.f;
      for (int n = 0; n < chunks; ++n) top = fmaxf(top, tops[r * kPlaceWords + n]);
      const bool odd = !(top < INFINITY), zero = odd || top < kLeastTop;
      ups[r] = zero ? 0.f : 127.f / top;  // codes of 0 where it is 0
      if (r >= r0 && r < r1)
        (w.which ? v_scales : k_scales)[item * a.slots + slot0 + r] = odd ? NAN : zero ? 0.f : fminf(top, kMostTop) / 127.f;
    }
    __syncthreads();
    int8_t* codes = (w.which ? v_codes : k_codes) + (item * a.slots + slot0) * a.dim;
    if (works) {
      uint32_t code[4][8];  // in the lowest byte
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float up = ups[quad * 4 + i];
#pragma unroll
        for (int e = 0; e < 8; ++e) code[i][e] = up == 0.f ? 0 : code_of(to_float(rows[i].v[e]) * up);
      }
      if (w.which) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          placed[(c * 8 + e) * kPlaceWords + quad % 4 * 4 + quad / 4] = lowest_bytes(code[0][e], code[1][e], code[2][e], code[3][e]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = quad * 4 + i;
          const Vec<uint32_t, 2> y{lowest_bytes(code[i][0], code[i][1], code[i][2], code[i][3]),
                                   lowest_bytes(code[i][4], code[i][5], code[i][6], code[i][7])};
          if (r >= r0 && r < r1) store_vec((uint32_t*)(codes + r * a.dim + c * 8), y);
        }
      }
    }
    if (!w.which) continue;  // the next unit's first barrier is before what this one reads last is written
    __syncthreads();
    const bool whole = r0 == 0 && r1 == 64;
    for (int n = threadIdx.x; n < a.dim * 4; n += blockDim.x) {
      const int d = n / 4, g = n % 4;
      Vec<uint32_t, 4> y;
#pragma unroll
      for (int t = 0; t < 4; ++t) y.v[t] = placed[d * kPlaceWords + g * 4 + t];
      int8_t* to = codes + d * 64 + g * 16;
      if (whole) {
        store_vec((uint32_t*)to, y);
        continue;
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // others' bytes stay as they are
          const int slot = 16 * t + 4 * g + i;
          if (slot >= r0 && slot < r1) to[t * 4 + i] = (int8_t)(y.v[t] >> (8 * i));
        }
    }
  }
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
                                                   const int8_t* v_codes, const float* v_scales, T* k, T* v, int tiles,
                                                   int64_t units) {
  __shared__ uint32_t placed[128 * kPlaceWords];
  const int chunks = a.dim / 8, quad = threadIdx.x / chunks, c = threadIdx.x - quad * chunks;
  const bool works = quad < 16;
  const int first = (int)a.start0, end = first + a.tokens;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const Unit w = unit_of(a, u, tiles);
    const int slot0 = (first / 64 + w.tile) * 64;
    if (slot0 >= end) continue;
    const int r0 = max(0, first - slot0), r1 = min(64, end - slot0);
    const int64_t item = (int64_t)w.b * a.kv_heads + w.g;
    const int8_t* codes = (w.which ? v_codes : k_codes) + (item * a.slots + slot0) * a.dim;
    const float* scales = (w.which ? v_scales : k_scales) + item * a.slots + slot0;
    T* y = (w.which ? v : k) + w.b * a.s[w.which][0] + w.g * a.s[w.which][2] + c * 8;
    const int64_t ts = a.s[w.which][1];
    const Vec<float, 4> scale = load_vec<4>(scales + min(quad, 15) * 4);
    Vec<int8_t, 8> x[4] = {};
    if (w.which) {
      __syncthreads();  // the unit before has been read
      for (int n = threadIdx.x; n < a.dim * 4; n += blockDim.x) {
        const Vec<uint32_t, 4> word = load_vec<4>((const uint32_t*)(codes + n * 16));
#pragma unroll
        for (int t = 0; t < 4; ++t) placed[n / 4 * kPlaceWords + n % 4 * 4 + t] = word.v[t];
      }
      __syncthreads();
      if (works) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const Vec<int8_t, 4> word =
              __builtin_bit_cast(Vec<int8_t, 4>, placed[(c * 8 + e) * kPlaceWords + quad % 4 * 4 + quad / 4]);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i].v[e] = word.v[i];
        }
      }
    } else if (works) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = load_vec<8>(codes + (quad * 4 + i) * a.dim + c * 8);
    }
    if (!works) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = quad * 4 + i;
      if (r < r0 || r >= r1) continue;
      Vec<T, 8> o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o.v[e] = from_float<T>(stands_for((float)x[i].v[e], scale.v[i]));
      store_vec(y + (int64_t)(slot0 + r - first) * ts, o);
    }
  }
}

// The parts' results of rows, weighted by their sums relative to the largest reference and added up in order:
// a workgroup a row, its threads four channels of every 1024 / dim-th part.
template <class T>
__global__ __launch_bounds__(256) void join_kernel(HeldAttention h) {
  __shared__ float weights[kMostSplits], reds[8];
  __shared__ __attribute__((aligned(16))) float4 sums[256];
  const int quads = h.a.dim / 4, lanes = 256 / quads;
  const int64_t bg = blockIdx.x / h.rows;
  const int mine = (int)(blockIdx.x - bg * h.rows);
  const int b = (int)(bg / h.a.kv_heads), kh = (int)(bg - (int64_t)b * h.a.kv_heads);
  const int64_t first = (int64_t)blockIdx.x * h.splits;
  float top = -INFINITY, l = 0.f;
  for (int s = threadIdx.x; s < h.splits; s += 256) top = fmaxf(top, h.meta[first + s].x);
  top = lanes_reduce<64>(top, [](float u, float v) { return fmaxf(u, v); });
  if (threadIdx.x % 64 == 0) reds[threadIdx.x / 64] = top;
  __syncthreads();
  top = fmaxf(fmaxf(reds[0], reds[1]), fmaxf(reds[2], reds[3]));
  for (int s = threadIdx.x; s < h.splits; s += 256) {
    const float2 m = h.meta[first + s];
    // nothing seen: a sum of 0, or of NaN logits
    const float w = m.x == -INFINITY ? m.y : m.y * __builtin_amdgcn_exp2f(m.x - top);
    weights[s] = w;
    l += w;
  }
  l = lanes_reduce<64>(l, [](float u, float v) { return u + v; });
  if (threadIdx.x % 64 == 0) reds[4 + threadIdx.x / 64] = l;
  __syncthreads();
  l = (reds[4] + reds[5]) + (reds[6] + reds[7]);
  const float share = l == 0.f ? 0.f : 1.f / l;
  const int part = threadIdx.x / quads, d = (threadIdx.x - part * quads) * 4;
  float4 o{0.f, 0.f, 0.f, 0.f};
  if (part < lanes) {
#pragma unroll 4
    for (int s = part; s < h.splits; s += lanes) {
      const float w = weights[s] * share;
      const float4 v = *(const float4*)__builtin_assume_aligned(h.part + (first + s) * h.a.dim + d, 16);
      o.x = fmaf(v.x, w, o.x), o.y = fmaf(v.y, w, o.y), o.z = fmaf(v.z, w, o.z), o.w = fmaf(v.w, w, o.w);
    }
  }
  sums[threadIdx.x] = o;
  __syncthreads();
  if (part != 0) return;
  for (int i = 1; i < lanes; ++i) {
    const float4 v = sums[i * quads + threadIdx.x];
    o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
  }
  const int t = mine / h.group, hd = mine - t * h.group;
  T* out = (T*)h.out + b * h.a.s[1][0] + t * h.a.s[1][1] + (int64_t)(kh * h.group + hd) * h.a.s[1][2] + d;
  store_vec(out, Vec<T, 4>{from_float<T>(o.x), from_float<T>(o.y), from_float<T>(o.z), from_float<T>(o.w)});
}

// The same for few parts of many rows: a thread four channels of a row.
constexpr int kFewSplits = 8;
template <class T>
__global__ __launch_bounds__(256) void join_few_kernel(HeldAttention h, int rows) {
  const int quads = h.a.dim / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / quads;
  if (row >= rows) return;
  const int d = (int)(i - row * quads) * 4;
  const int64_t bg = row / h.rows, first = row * h.splits;
  const int mine = (int)(row - bg * h.rows), b = (int)(bg / h.a.kv_heads), kh = (int)(bg - (int64_t)b * h.a.kv_heads);
  float2 m[kFewSplits];
  float4 v[kFewSplits];
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {  // past the last the last again, which then counts 0
    const int64_t at = first + min(s, h.splits - 1);
    m[s] = h.meta[at];
    v[s] = *(const float4*)__builtin_assume_aligned(h.part + at * h.a.dim + d, 16);
  }
  float top = -INFINITY, l = 0.f, w[kFewSplits];
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) top = fmaxf(top, m[s].x);
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    w[s] = m[s].x == -INFINITY ? m[s].y : m[s].y * __builtin_amdgcn_exp2f(m[s].x - top);
    if (s >= h.splits) w[s] = 0.f;
    l += w[s];
  }
  const float share = l == 0.f ? 0.f : 1.f / l;
  float4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    if (s >= h.splits) break;
    const float by = w[s] * share;
    o.x = fmaf(v[s].x, by, o.x), o.y = fmaf(v[s].y, by, o.y), o.z = fmaf(v[s].z, by, o.z), o.w = fmaf(v[s].w, by, o.w);
  }
  const int t = mine / h.group, hd = mine - t * h.group;
  T* out = (T*)h.out + b * h.a.s[1][0] + t * h.a.s[1][1] + (int64_t)(kh * h.group + hd) * h.a.s[1][2] + d;
  store_vec(out, Vec<T, 4>{from_float<T>(o.x), from_float<T>(o.y), from_float<T>(o.z), from_float<T>(o.w)});
}

// Logits are in units of log 2.
float in_octaves(float scale) { return scale * 1.4426950408889634f; }

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
  require(std::isfinite(in_octaves(c.scale)), n + ": the scale must be finite, and so must it be times log2 e");
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
  const int tiles = (int)ceil_div((int64_t)c.tokens + (start || c.start % 64 ? 63 : 0), 64);  // that tokens may lie in
  const int64_t units = 2ll * c.batch * c.kv_heads * tiles;
  ProfScope prof("hold_tokens", 4.0 * rows * c.head_dim, rows * (c.head_dim * (type_bytes(c.type) + 1.0) + 4.0), st);
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    hold_kernel<T><<<(unsigned)std::min<int64_t>(units, 1 << 20), tile_threads(c.head_dim), 0, st>>>(
        a, (const T*)k, (const T*)v, k_codes, k_scales, v_codes, v_scales, tiles, units);
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
  const int tiles = (int)ceil_div(c.start % 64 + c.tokens, 64);
  const int64_t units = 2ll * c.batch * c.kv_heads * tiles;
  ProfScope prof("read_held", rows * c.head_dim, rows * (c.head_dim * (type_bytes(c.type) + 1.0) + 4.0), st);
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    read_kernel<T><<<(unsigned)std::min<int64_t>(units, 1 << 20), tile_threads(c.head_dim), 0, st>>>(
        a, k_codes, k_scales, v_codes, v_scales, (T*)k, (T*)v, tiles, units);
  });
  launch_check("read_held");
}

namespace {

HeldPlan make_plan(const nnx_held_config& c) {
  HeldPlan p;
  p.group = c.heads / c.kv_heads;
  p.rows = c.tokens * p.group;
  p.r = held_rows(c.type, c.head_dim, p.rows);
  p.tiles = (int)ceil_div(p.rows, 16 * p.r);
  p.units = (int64_t)c.batch * c.kv_heads * p.tiles;
  p.splits = 1;
  if (p.units < kUnits) {
    // Few units: parts of at least 4 tiles of 64 slots, a wave each, up to two workgroups a CU.  (One query of 32 heads
    // over 131072 slots 38.6 us, with four workgroups a CU 47.5.)  Not where one workgroup is done before another
    // launch would begin: one query of 5 heads of 64 over 2048 slots takes 13.8 us in one launch and 15.4 in two, over
    // 3000 18.7 and 15.3 (heads of 128: 1536 16.8 and 15.7, 2048 19.9 and 15.8).
    if ((int64_t)c.keys * c.head_dim > 2048 * 64)
      p.splits = (int)std::max<int64_t>(1, std::min(kMostSplits / p.units, ceil_div(c.keys, 256)));
  } else {
    // Many: parts that even out what the CUs get, in tiles a wave and with what a workgroup (6) and the join (8) cost.
    // 640 units over 32768 slots: 550, 468, 505 and 487 us in 1 to 4 parts; 1280 units over 4096: 135 in 1, 155 in 2.
    int64_t least = INT64_MAX;
    for (int s = 1; s <= 4; ++s) {
      const int64_t cost = ceil_div(p.units * s, kUnits) * (ceil_div(c.keys, 256 * s) + 6) + (s > 1 ? 8 : 0);
      if (cost < least) least = cost, p.splits = s;
    }
  }
  require(p.units * p.splits < 1 << 24, "held attention: fewer than 2^24 items times key heads times tiles of rows");
  p.meta = p.bytes = 0;
  if (p.splits > 1) {
    const size_t rows = (size_t)c.batch * c.kv_heads * p.splits * p.rows;
    p.meta = rows * c.head_dim * 4;
    p.bytes = p.meta + rows * 8;
  }
  return p;
}

}  // namespace

size_t held_attention_workspace(const nnx_held_config& c) {
  try {
    check_config(c, "held attention", true);
    return make_plan(c).bytes;
  } catch (...) {  // nothing may leave a C entry
    return 0;
  }
}

void held_attention(const nnx_held_config& c, const void* q, const int8_t* k_codes,
                    const float* k_scales, const int8_t* v_codes, const float* v_scales,
                    const int32_t* start, const int32_t* lengths, const uint8_t* mask, void* out,
                    void* ws, size_t ws_bytes, hipStream_t st) {
  check_config(c, "held attention", true);
  const HeldPlan p = make_plan(c);
  require(q && out, "held attention: null pointer");
  check_held(k_codes, k_scales, v_codes, v_scales, "held attention");
  require(p.bytes == 0 || (ws && ws_bytes >= p.bytes && reinterpret_cast<uintptr_t>(ws) % 16 == 0),
          "held attention: the workspace is too small or not 16-byte aligned");
  // Of factors up to 2^26 the keys' scales are multiplied by 64 at most, which none of them overflows by, and the queries
  // by the rest, 2^20 at most: their products with codes are finite below 2^122 and so are logits up to the type's
  // end.  A float16 query is taken as it is and its keys' scales by the whole factor, as by what larger ones leave.
  const float factor = in_octaves(c.scale);
  const float query = c.type == NNX_TYPE_F16 || factor == 0.f
                          ? 1.f : std::exp2(std::min(20.f, std::max(-16.f, std::ceil(std::log2(std::fabs(factor) / 64.f)))));
  HeldAttention h{make_args(c, start, lengths, mask), q, k_codes, v_codes, k_scales, v_scales, out, (float*)ws,
                  (float2*)((char*)ws + p.meta), p.group, p.rows, p.tiles, p.splits,
                  query, factor / query};
  const double rows = (double)c.batch * c.tokens * c.heads;
  ProfScope prof("held_attention", 4.0 * rows * c.keys * c.head_dim,
                 2.0 * rows * c.head_dim * type_bytes(c.type) +
                     2.0 * c.batch * c.kv_heads * c.keys * (c.head_dim + 4.0),
                 st);
  if (c.type == NNX_TYPE_F32) {
    held_units_f32(h, p, st);
  } else if (c.type == NNX_TYPE_F16) {
    held_units_f16(h, p, st);
  } else {
    held_units_bf16(h, p, st);
  }
  if (p.splits == 1) return;
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    if (p.splits <= kFewSplits) {
      const int64_t threads = (int64_t)rows * (c.head_dim / 4);
      join_few_kernel<T><<<(unsigned)ceil_div(threads, 256), 256, 0, st>>>(h, (int)rows);
    } else {
      join_kernel<T><<<(unsigned)(int64_t)rows, 256, 0, st>>>(h);
    }
  });
  launch_check("held_join");
}

}  // namespace nnx
