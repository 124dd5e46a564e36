// Shared by the kernels of attention over selected blocks: arguments, the chunk of work that one
// pass of launches covers, and per-item lengths and positions.
#pragma once

#include "nnx_elements.h"

namespace nnx {

// n / d for 0 <= n < 2^31 by one product: m = ceil(2^(31 + l) / d) with 2^l >= d errs by less than
// d / 2^(31 + l) a unit, less than 1 / d over n.
struct FastDiv {
  uint32_t m;
  int l;
  explicit FastDiv(uint32_t d = 1) : l(0) {
    while ((1ull << l) < d) ++l;
    m = (uint32_t)(((1ull << (31 + l)) + d - 1) / d);
  }
  __device__ __forceinline__ int operator()(int n) const {
    return (int)(__umulhi((uint32_t)n << 1, m) >> l);
  }
};

struct BlockArgs {
  int batch, queries, keys, heads, kv_heads, group, dim, block, blocks, keep, first, local, causal;
  int64_t start0;
  float scale;
  int64_t qs[3], ks[3], vs[3], os[3], ms;
  const int32_t *start, *lengths;
  const uint8_t* mask;
};

__device__ __forceinline__ int item_length(const BlockArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.keys) : a.keys;
}

__device__ __forceinline__ int64_t item_start(const BlockArgs& a, int b) {
  return a.start0 + (a.start ? a.start[b] : 0);
}

// The queries of each key head of each item are cut into `splits` spans of `nt`; span v = (item *
// kv_heads + key head) * splits + split.  A launch covers spans [span0, span0 + spans).  Row =
// (span, query of the span, head of the group), counted from span0; every row has `keep`
// partials, one a kept block: `dim` values (Partial<T>), sums over the block's keys with weights 2^(x - m),
// and (m, l), l the sum of the weights.  A negative l: the block holds values that are not finite, which
// count as 0 in the partial.
struct ChunkArgs {
  BlockArgs a;
  const void *q, *k, *v;
  const int32_t* ids;
  void* part;
  float2* meta;
  int span0, spans, splits, nt;
  FastDiv by_keep, by_group, by_nt;
  // by block: pairs (query, slot) of a span that keep it, list[start[u]...], in tiles of kTileRows
  // rows (pairs * group heads), tiles[u] of them before block u = (span - span0) * blocks + block
  const int32_t *list, *start, *tiles;
};

// What the values of a partial result are held in.  bfloat16's are float16 times a power of two that
// puts the row's largest below 2^15: 11 bits for every channel down to 2^-29 of it, where the result
// keeps 8, so an error of 2^-12 of a channel's own partials; the power's exponent is kept in the last 8
// bits of l, which leaves l 16.  float16's result keeps 11 bits itself, and its partials are float32.
template <class T>
struct PartialOf {
  using type = float;
};
template <>
struct PartialOf<bf16> {
  using type = f16;
};
template <class T>
using Partial = typename PartialOf<T>::type;

constexpr uint32_t kExponentBits = 255, kExponentZero = 128;

inline int partial_bytes(int type) { return type == NNX_TYPE_BF16 ? 2 : 4; }

struct Span {
  int b, g, t0, queries;
};

__device__ __forceinline__ Span span_of(const ChunkArgs& c, int v) {
  const int unit = v / c.splits, b = unit / c.a.kv_heads, t0 = (v - unit * c.splits) * c.nt;
  return {b, unit - b * c.a.kv_heads, t0, min(c.nt, c.a.queries - t0)};
}

constexpr int kTileRows = 128;

// Buffer accesses take 32-bit offsets, and past the buffer's end load 0 and store nothing; the check is of
// the lane's offset, so all of it goes there and the scalar offset is 0.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, size_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)(uint32_t)bytes, 0x00027000);
}

// Attention of a launch's rows to each of their kept blocks, a partial result each.  `by_block`:
// rows gathered by the block that they keep (list, start, tiles; at most `grid` tiles), else a
// workgroup for each of `grid` kept blocks of queries.
void block_partials_f32(const ChunkArgs& c, bool by_block, int grid, hipStream_t st);
void block_partials_f16(const ChunkArgs& c, bool by_block, int grid, hipStream_t st);
void block_partials_bf16(const ChunkArgs& c, bool by_block, int grid, hipStream_t st);

}  // namespace nnx
