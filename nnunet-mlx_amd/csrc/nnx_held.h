// Shared by the kernels over held tokens.
#pragma once

#include "nnx_elements.h"

namespace nnx {

struct HeldArgs {
  int batch, tokens, slots, keys, heads, kv_heads, dim, causal;
  float scale;
  int64_t start0;
  int64_t s[2][3], ms;
  const int32_t *start, *lengths;
  const uint8_t* mask;
};

// Attention by units: (item, key head, tile of 16 * r rows, part of the slots that its rows see), rows counting
// (query, head of the key head's group).  A unit of several parts leaves its sums for the join.
struct HeldPlan {
  int group, rows, r, tiles, splits;
  int64_t units;  // batch * kv_heads * tiles
  size_t meta, bytes;  // the workspace: results, then (reference logit, sum of weights), by key head, row and part
};

struct HeldAttention {
  HeldArgs a;
  const void* q;
  const int8_t *k_codes, *v_codes;
  const float *k_scales, *v_scales;
  void* out;
  float* part;
  float2* meta;
  int group, rows, tiles, splits;
  float query, c2;   // factors of the queries, a power of two, and of the keys' scales: scale * log2 e together
};

// 16 rows a wave or 32: two share what a code's conversion costs, where a wave's registers hold them beside two
// waves a SIMD.
constexpr bool held_pairs(bool f32, int dim) { return !f32 && dim <= 96; }
inline int held_rows(int type, int dim, int rows) { return rows > 16 && held_pairs(type == NNX_TYPE_F32, dim) ? 2 : 1; }

void held_units_f32(const HeldAttention& h, const HeldPlan& p, hipStream_t st);
void held_units_f16(const HeldAttention& h, const HeldPlan& p, hipStream_t st);
void held_units_bf16(const HeldAttention& h, const HeldPlan& p, hipStream_t st);

}  // namespace nnx
