// Attention of query rows to one block of keys, the partial results of attention over selected
// blocks; included by one source a type.
#pragma once

#include <algorithm>
#include <type_traits>

#include "nnx_blocks.h"

namespace nnx {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// One of the two lane halves' values in both: {lower half's, upper half's}.
__device__ __forceinline__ float2 both_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <class T>
using Frag = T __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x16 mfma(Frag<f16> a, Frag<f16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(Frag<bf16> a, Frag<bf16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(float a, float b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

// Tile geometry.  Rows of keys and values lie in LDS in 16-byte chunks, chunk c of row r at place
// c ^ turn(r), so that 16 lanes that read the same chunk of 16 rows meet all banks.
template <class T, int DP, int BK>
struct Tile {
  static constexpr int CH = 16 / sizeof(T);        // elements of a chunk
  static constexpr int CHUNKS = DP / CH;           // chunks of a row
  static constexpr int ROWS = BK < 32 ? 32 : BK;   // rows of keys that the products read
  static constexpr int KT = ROWS / 32;             // 32-key tiles
  static constexpr int REGS = BK < 32 ? 8 : 16;    // scores of a 32-key tile that a lane uses
  static constexpr int ROW_BYTES = DP * sizeof(T);
  static constexpr int PER = ROW_BYTES >= 256 ? 1 : 256 / ROW_BYTES;  // rows in 256 bytes
  static constexpr int TURNS = CHUNKS & -CHUNKS;   // a power of two that divides CHUNKS
  // keys, values, what their scores are replaced by, and for each wave 32 rows of 128 bytes on their way out
  static constexpr int OUT = 32 * 128;
  static constexpr size_t LDS = (size_t)2 * ROWS * ROW_BYTES + ROWS * sizeof(float) + 16 + 4 * OUT;
  static __device__ __forceinline__ int at(int row, int chunk) {
    const int turn = (row / PER) & (TURNS - 1);
    return row * DP + (chunk ^ turn) * CH;
  }
};

struct Staged {
  bool full;  // every key is valid
  bool odd;   // some value is not finite
};

// The block's keys and values into LDS, zeros for those that are not valid and for values that are not
// finite (a weight of 0 would not keep them out of a product; the join takes them from the rows that see
// them), and the scores of keys that are not valid: -inf, 0 for the others.
template <class T, int DP, int BK>
__device__ __forceinline__ Staged stage_block(const ChunkArgs& c, int b, int g, int j, T* lk, T* lv,
                                            float* bias, bool negate) {
  using G = Tile<T, DP, BK>;
  const int length = item_length(c.a, b), first = j * BK;
  const T* k = (const T*)c.k + b * c.a.ks[0] + g * c.a.ks[2];
  const T* v = (const T*)c.v + b * c.a.vs[0] + g * c.a.vs[2];
  const uint8_t* mask = c.a.mask ? c.a.mask + b * c.a.ms : nullptr;
  constexpr int N = BK * G::CHUNKS, EACH = (N + 255) / 256;
  Vec<T, G::CH> kr[EACH], vr[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int n = threadIdx.x + i * 256, row = n / G::CHUNKS, d = (n % G::CHUNKS) * G::CH;
    const int64_t key = first + row;
    kr[i] = vr[i] = Vec<T, G::CH>{};
    if (n < N && d < c.a.dim && key < length && (!mask || mask[key])) {
      kr[i] = load_vec<G::CH>(k + key * c.a.ks[1] + d);
      vr[i] = load_vec<G::CH>(v + key * c.a.vs[1] + d);
    }
  }
  bool odd = false;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int n = threadIdx.x + i * 256;
    bool here = false;
#pragma unroll
    for (int e = 0; e < G::CH; ++e) here |= !(fabsf(to_float(vr[i].v[e])) < INFINITY);
    if (here) {
#pragma unroll
      for (int e = 0; e < G::CH; ++e)
        vr[i].v[e] = fabsf(to_float(vr[i].v[e])) < INFINITY ? vr[i].v[e] : from_float<T>(0.f);
    }
    odd |= here;
    if (negate) {
#pragma unroll
      for (int e = 0; e < G::CH; ++e) kr[i].v[e] = -kr[i].v[e];
    }
    if (n < N) {
      const int at = G::at(n / G::CHUNKS, n % G::CHUNKS);
      *(Vec<T, G::CH>*)__builtin_assume_aligned(lk + at, 16) = kr[i];
      *(Vec<T, G::CH>*)__builtin_assume_aligned(lv + at, 16) = vr[i];
    }
  }
  bool missing = false;
  if (threadIdx.x < BK) {
    const int key = first + threadIdx.x;
    missing = !(key < length && (!mask || mask[key]));
    bias[threadIdx.x] = missing ? -INFINITY : 0.f;
  }
  int* seen = (int*)(bias + G::ROWS);  // of each wave
  const int mine = (__any(odd) ? 1 : 0) | (__any(missing) ? 2 : 0);
  if (threadIdx.x % 64 == 0) seen[threadIdx.x / 64] = mine;
  __syncthreads();
  const int any = __builtin_amdgcn_readfirstlane(seen[0] | seen[1] | seen[2] | seen[3]);
  return {!(any & 2), (any & 1) != 0};
}

// Stores into the partials go through buffer instructions: 32-bit offsets, and one past the buffer's
// end stores nothing, so that a tile's dead rows need no branch (a branch around a store leaves its
// count of outstanding accesses open, and the next tile's queries would be waited for with it).
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr uint32_t kNowhere = 0xffffff00u;

// Chunks of 16 bytes, one row's in two lanes (8 of them make 128 bytes of a row), leave as whole
// rows: through LDS, 8 lanes a row.
struct RowWriter {
  char* lds;  // of the wave
  __amdgpu_buffer_rsrc_t part;
  uint32_t row;  // offset of the lane's row, kNowhere for none
  uint32_t bytes;  // of a row
  __device__ __forceinline__ void put(int chunk, u32x4 v) const {
    const int col = threadIdx.x % 32;
    *(u32x4*)__builtin_assume_aligned(lds + col * 128 + ((chunk ^ (col & 7)) * 16), 16) = v;
  }
  __device__ __forceinline__ void flush(int pass) const {
    const int lane = threadIdx.x % 64, chunk = lane % 8;
    const uint32_t at = pass * 128 + chunk * 16;
    wave_sync();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + lane / 8;
      const u32x4 v = *(const u32x4*)__builtin_assume_aligned(lds + r * 128 + ((chunk ^ (r & 7)) * 16), 16);
      const uint32_t to = __shfl(row, r);
      __builtin_amdgcn_raw_buffer_store_b128(v, part, at < bytes && to != kNowhere ? to + at : kNowhere, 0, 0);
    }
    wave_sync();
  }
};

// The partial softmax of rows over one block: m = max x up to a constant, l = sum 2^(x - m), O = sum
// 2^(x - m) v (x the scores in units of log 2; weights, sums and O
// in float32).  In 16-bit types a weight is two operands of the second product, its rounded value and the
// rest: 16 bits of it for bfloat16, 22 for float16, so that the result's own rounding is the only one that
// shows (1.3 times the error with one operand; 329 us of partials against 314 for 32768 queries of 32 blocks).
// 32 query rows, a lane pair (l, l + 32) each: S^T = K Q^T leaves a row's scores in its two
// lanes' registers, so the softmax needs one exchange between halves, and its weights are
// already the second operand of O^T = V^T P^T (the order of keys is that of the registers; values
// are read transposed to match).
template <class T, int DP>
struct QueryRow {
  static constexpr int CH = 16 / sizeof(T), N = DP / (2 * CH);
  u32x4 v[N];  // a half's chunks: 2 s + half
};

// Chunks past the row's end are filled from inside it; the keys are 0 there.
template <class T, int DP>
__device__ __forceinline__ void load_query(QueryRow<T, DP>& row, const T* q, int dim) {
  using Q = QueryRow<T, DP>;
  const int half = threadIdx.x % 64 / 32;
#pragma unroll
  for (int s = 0; s < Q::N; ++s)
    __builtin_memcpy(&row.v[s], q + min((2 * s + half) * Q::CH, dim - Q::CH), 16);
}

template <class T, int DP, int BK, class F, class G0>
__device__ __forceinline__ void attend_rows(const ChunkArgs& c, const T* lk, const T* lv,
                                            const float* bias, char* out_lds,
                                            __amdgpu_buffer_rsrc_t part, __amdgpu_buffer_rsrc_t metas,
                                            QueryRow<T, DP>& q, int last, float c2, Staged block,
                                            uint32_t partial, F&& after_scores, G0&& before_stores) {
  using G = Tile<T, DP, BK>;
  const int lane = threadIdx.x % 64, col = lane % 32, half = lane / 32;
  f32x16 acc[G::KT] = {};
  if constexpr (sizeof(T) == 2) {
    Frag<T> qf[DP / 16];
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) __builtin_memcpy(&qf[s], &q.v[s], 16);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int kt = 0; kt < G::KT; ++kt)
        acc[kt] = mfma(*(const Frag<T>*)(lk + G::at(kt * 32 + col, 2 * s + half)), qf[s], acc[kt]);
  } else {
    // 32 channels at a time: a sum of 128 in one chain errs by twice as much
#pragma unroll
    for (int kt = 0; kt < G::KT; ++kt)
#pragma unroll
      for (int s0 = 0; s0 < DP / 8; s0 += 4) {
        f32x16 part = {};
#pragma unroll
        for (int s = s0; s < s0 + 4; ++s) {
          Vec<float, 4> qf;
          __builtin_memcpy(&qf, &q.v[s], 16);
          const float4 kf = *(const float4*)(lk + G::at(kt * 32 + col, 2 * s + half));
          part = mfma(kf.x, qf.v[0], part);
          part = mfma(kf.y, qf.v[1], part);
          part = mfma(kf.z, qf.v[2], part);
          part = mfma(kf.w, qf.v[3], part);
        }
        acc[kt] = s0 ? acc[kt] + part : part;
      }
  }
  after_scores();
  if (!block.full) {
#pragma unroll
    for (int kt = 0; kt < G::KT; ++kt)
#pragma unroll
      for (int r = 0; r < G::REGS; r += 4) {
        // chosen, not added: a query that is not finite has NaN for the zeros of such keys
        const float4 z = *(const float4*)&bias[kt * 32 + 2 * r + 4 * half];
        acc[kt][r] = z.x < 0.f ? z.x : acc[kt][r];
        acc[kt][r + 1] = z.y < 0.f ? z.y : acc[kt][r + 1];
        acc[kt][r + 2] = z.z < 0.f ? z.z : acc[kt][r + 2];
        acc[kt][r + 3] = z.w < 0.f ? z.w : acc[kt][r + 3];
      }
  }
  if (__any(last < BK - 1)) {  // the query's own block, or one behind it
    const int seen = last - 4 * half;
#pragma unroll
    for (int kt = 0; kt < G::KT; ++kt)
#pragma unroll
      for (int r = 0; r < G::REGS; ++r)
        if (kt * 32 + 8 * (r / 4) + r % 4 > seen) acc[kt][r] = -INFINITY;
  }
  float m = -INFINITY;
#pragma unroll
  for (int kt = 0; kt < G::KT; ++kt)
#pragma unroll
    for (int r = 0; r < G::REGS; ++r) m = fmaxf(m, acc[kt][r]);
  const float2 mh = both_halves(m);
  m = fmaxf(mh.x, mh.y);
  // Weights of at most 2^-kDown, so that the block's values add up to no more than the largest of them
  // (float16's do not reach float32's end).  Nothing seen: all weights 2^-inf.
  constexpr float kDown = std::is_same<T, f16>::value ? 0 : BK == 16 ? 4 : BK == 32 ? 5 : BK == 64 ? 6 : 7;
  const float top = m == -INFINITY ? 0.f : m * c2 + kDown;
  float l = 0.f;
#pragma unroll
  for (int kt = 0; kt < G::KT; ++kt)
#pragma unroll
    for (int r = 0; r < G::REGS; ++r) {
      acc[kt][r] = __builtin_amdgcn_exp2f(fmaf(acc[kt][r], c2, -top));
      l += acc[kt][r];
    }
  const float2 lh = both_halves(l);
  l = lh.x + lh.y;
  f32x16 o[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < BK / 16; ++i) {
      // each weight as two operands, its rounded value and what that leaves
      Frag<T> p, rest;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float w = acc[i / 2][8 * (i % 2) + r];
        p[r] = from_float<T>(w);
        rest[r] = from_float<T>(w - to_float(p[r]));
      }
      const int row = 16 * i + 4 * half + lane % 16 / 4;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const int d = dt * 32 + lane / 16 % 2 * 16 + lane % 4 * 4;
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4* lds_ptr;
        union {
          s16x4 h[2];
          Frag<T> f;
        } vt;
        vt.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lv + G::at(row, d / 8) + d % 8));
        vt.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lv + G::at(row + 8, d / 8) + d % 8));
        o[dt] = mfma(vt.f, p, o[dt]);
        o[dt] = mfma(vt.f, rest, o[dt]);
      }
    }
  } else {
#pragma unroll
    for (int kt = 0; kt < G::KT; ++kt)
#pragma unroll
      for (int r = 0; r < G::REGS; ++r) {
        const int row = kt * 32 + 8 * (r / 4) + 4 * half + r % 4;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) {
          const int d = dt * 32 + col;
          o[dt] = mfma(lv[G::at(row, d / 4) + d % 4], acc[kt][r], o[dt]);
        }
      }
  }
  // Registers 4i .. 4i + 3 of o[dt] are channels 32 dt + 8 i + 4 half + 0..3 of the lane's row.
  before_stores();
  float2 meta = make_float2(l == 0.f ? -INFINITY : top, l);  // 0: nothing seen; NaN stays
  if constexpr (sizeof(Partial<T>) == 2) {
    // The power of two: of the largest magnitude, at least 2^-96, so that both factors are normal.  NaN, of
    // the weights, hides from the largest and stays NaN.
    float big = 0.f;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; r += 2) big = fmaxf(fmaxf(big, fabsf(o[dt][r])), fabsf(o[dt][r + 1]));
    const float2 bh = both_halves(big);
    const int exponent = max(__builtin_amdgcn_frexp_expf(fmaxf(bh.x, bh.y)), -96) - 15;
    const float down = __uint_as_float((uint32_t)(127 - exponent) << 23);
    meta.y = __uint_as_float(((__float_as_uint(l) + (kExponentBits + 1) / 2) & ~kExponentBits) |
                             (uint32_t)(exponent + (int)kExponentZero));
    const uint32_t bytes = c.a.dim * 2;
    const RowWriter writer{out_lds, part, partial == kNowhere ? kNowhere : partial * bytes, bytes};
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const Vec<f16, 2> pair{(f16)(o[dt][8 * i + 2 * r] * down), (f16)(o[dt][8 * i + 2 * r + 1] * down)};
          __builtin_memcpy(&w[r], &pair, 4);
        }
        // channels 8 apart, 4 a half, become 8 neighbours a half
        const auto r0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
        const auto r1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
        writer.put(4 * (dt % 2) + 2 * i + half, u32x4{r0[0], r1[0], r0[1], r1[1]});
      }
      if (dt % 2 || dt + 1 == DP / 32) writer.flush(dt / 2);
    }
  } else {
    const uint32_t bytes = c.a.dim * 4;
    const RowWriter writer{out_lds, part, partial == kNowhere ? kNowhere : partial * bytes, bytes};
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32x4 w;
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = __float_as_uint(o[dt][4 * i + r]);
        writer.put(2 * i + half, w);
      }
      writer.flush(dt);
    }
  }
  if (block.odd) meta.y = -meta.y;  // the join looks
  const u32x2 words{__float_as_uint(meta.x), __float_as_uint(meta.y)};
  __builtin_amdgcn_raw_buffer_store_b64(words, metas, half || partial == kNowhere ? kNowhere : partial * 8, 0, 0);
}

// The last u in [0, n) with tiles[u] <= tile, by all lanes at once.
__device__ __forceinline__ int find_tile(const int32_t* tiles, int n, int tile) {
  const int lane = threadIdx.x % 64;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 63) / 64, at = lane * step;
    const int below = __popcll(__ballot(at < n && tiles[lo + min(at, n - 1)] <= tile));
    const int to = (below - 1) * step;
    lo += to;
    n = min(step, n - to);
  }
  return lo;
}

// How many of a block's keys a query at `at` sees, less one: below 0 none, BK - 1 all.
__device__ __forceinline__ int last_seen(const BlockArgs& a, int64_t at, int first_key) {
  return a.causal ? (int)min(max(at - first_key, (int64_t)-1), (int64_t)1 << 20) : 1 << 20;
}

// Bound by the partials' stores: 1.05 million pairs with blocks of 64 keys of 64 bfloat16 channels, a
// fifth of 32768 queries by 5 heads by 32 blocks, take 61 to 69 us: 26 GFLOP with both operands of the
// weights, and 134 MB of partials with 8 MB of sums, which leave in pieces of 128 and 8 bytes at 2.1 TB/s.
// The products would take 21 us at a large product's rate, the queries' 134 MB are read from the L2.  Two
// tiles of queries in registers, keys and values held in registers, sums by products of ones, and four
// waves a SIMD were all measured, with one operand of the weights, and made nothing faster (297 to 365 us
// for the five launches against 300).  Registers for two waves a
// SIMD where that leaves nothing in memory (accumulators then stay where vector instructions reach
// them); larger tiles take one.
template <class T, int DP, int BK>
constexpr int kWaves = (sizeof(T) == 2 ? DP * BK < 128 * 128 : DP + BK <= 128) ? 2 : 1;

template <class T, int DP, int BK, bool BY_BLOCK>
__global__ __launch_bounds__(256, (kWaves<T, DP, BK>)) void block_partials_kernel(ChunkArgs c) {
  using G = Tile<T, DP, BK>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* lk = (T*)lds;
  T* lv = lk + G::ROWS * DP;
  float* bias = (float*)(lv + G::ROWS * DP);
  char* out_lds = (char*)(bias + G::ROWS) + 16 + threadIdx.x / 64 * G::OUT;
  const BlockArgs& a = c.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), col = threadIdx.x % 32;
  // the scale's sign goes to the keys, so that the largest weight belongs to the largest product; a
  // factor of 0 stays above it, which keeps -inf times it -inf
  const float c2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-35f);
  const bool negate = a.scale < 0.f;
  const size_t partials_all = (size_t)c.spans * c.nt * a.group * a.keep;
  const auto part = buffer_of(c.part, partials_all * a.dim * sizeof(Partial<T>));
  const auto metas = buffer_of(c.meta, partials_all * 8);
  if constexpr (BY_BLOCK) {
    const int all = c.spans * a.blocks, tile0 = c.tiles[0];
    const int64_t total = c.tiles[all] - tile0;
    const int t_hi = tile0 + (int)((blockIdx.x + 1) * total / gridDim.x);
    int tile = tile0 + (int)(blockIdx.x * total / gridDim.x), held = -1;
    while (tile < t_hi) {
      held = held < 0 ? find_tile(c.tiles, all, tile)
                      : held + 1 + find_tile(c.tiles + held + 1, all - held - 1, tile);
      held = __builtin_amdgcn_readfirstlane(held);
      const int span = held / a.blocks, j = held - span * a.blocks;
      const Span s = span_of(c, c.span0 + span);
      const int first_tile = c.tiles[held], to = min(c.tiles[held + 1], t_hi);
      const int32_t* list = c.list + c.start[held];
      const int rows = (c.start[held + 1] - c.start[held]) * a.group;
      const int64_t start = item_start(a, s.b) + s.t0;
      const T* queries = (const T*)c.q + s.b * a.qs[0] + s.t0 * a.qs[1] + (int64_t)s.g * a.group * a.qs[2];
      const uint32_t first = (uint32_t)span * c.nt;
      // a row of the tile: its list entry a tile ahead, its query a tile ahead of its products
      struct Row {
        int entry, h;
        bool live;
      };
      const auto locate = [&](int at) {
        const int row = (at - first_tile) * kTileRows + wave * 32 + col;
        Row r;
        r.live = at < to && row < rows;
        const int pair = r.live ? c.by_group(row) : 0;
        r.h = r.live ? row - pair * a.group : 0;
        r.entry = list[pair];
        return r;
      };
      const auto fetch = [&](const Row& r, QueryRow<T, DP>& q) {
        load_query<T, DP>(q, queries + c.by_keep(r.entry) * a.qs[1] + r.h * a.qs[2], a.dim);
      };
      Row row = locate(tile), next = locate(tile + 1);
      __syncthreads();  // the block before has been read
      const Staged block = stage_block<T, DP, BK>(c, s.b, s.g, j, lk, lv, bias, negate);
      QueryRow<T, DP> q;
      fetch(row, q);
      for (; tile < to; ++tile) {
        Row after = locate(tile + 2);
        const int t = c.by_keep(row.entry), slot = row.entry - t * a.keep;
        const uint32_t partial = ((first + t) * a.keep + slot) * a.group + row.h;
        // The next tile's queries take the registers of this one's after its scores, and are waited for
        // before its stores: accesses end in order, and a wait behind the stores would be one for
        // them too.
        attend_rows<T, DP, BK>(
            c, lk, lv, bias, out_lds, part, metas, q, last_seen(a, start + t, j * BK), c2, block,
            row.live ? partial : kNowhere, [&] { fetch(next, q); },
            [&] {
#pragma unroll
              for (u32x4& v : q.v) asm volatile("" : "+v"(v));
              asm volatile("" : "+v"(after.entry));
            });
        row = next;
        next = after;
      }
    }
  } else {
    const int item = blockIdx.x, vt = c.by_keep(item), slot = item - vt * a.keep;
    const int span = c.by_nt(vt), t = vt - span * c.nt;
    const Span s = span_of(c, c.span0 + span);
    if (t >= s.queries) return;
    const int j = c.ids[(((int64_t)s.b * a.queries + s.t0 + t) * a.kv_heads + s.g) * a.keep + slot];
    if (j < 0 || j >= a.blocks) return;
    const Staged block = stage_block<T, DP, BK>(c, s.b, s.g, j, lk, lv, bias, negate);
    const int last = last_seen(a, item_start(a, s.b) + s.t0 + t, j * BK);
    for (int h0 = wave * 32; h0 < a.group; h0 += 128) {
      const bool live = h0 + col < a.group;
      const int h = live ? h0 + col : 0;
      QueryRow<T, DP> q;
      load_query<T, DP>(q, (const T*)c.q + s.b * a.qs[0] + (s.t0 + t) * a.qs[1] +
                               (int64_t)(s.g * a.group + h) * a.qs[2],
                        a.dim);
      const uint32_t partial = item * a.group + h;
      attend_rows<T, DP, BK>(c, lk, lv, bias, out_lds, part, metas, q, last, c2, block,
                             live ? partial : kNowhere, [] {}, [] {});
    }
  }
}

template <class T, int DP, int BK>
void launch_partials(const ChunkArgs& c, bool by_block, int grid, hipStream_t st) {
  constexpr size_t bytes = Tile<T, DP, BK>::LDS;
  if (by_block) {
    // as many workgroups as run at once: they share the tiles evenly, and a block's keys are staged
    // once for a run of its tiles
    static const int per_cu = [] {
      int n = 0;
      hip_check(hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, block_partials_kernel<T, DP, BK, true>, 256, bytes),
                "block attention: occupancy");
      return std::max(1, n);
    }();
    grid = (int)std::min<int64_t>(grid, (int64_t)per_cu * compute_units());
    block_partials_kernel<T, DP, BK, true><<<grid, 256, bytes, st>>>(c);
  } else {
    block_partials_kernel<T, DP, BK, false><<<grid, 256, bytes, st>>>(c);
  }
  launch_check("block_partials");
}

template <class T>
void block_partials(const ChunkArgs& c, bool by_block, int grid, hipStream_t st) {
  using std::integral_constant;
  auto keys = [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    if (c.a.block == 16) return launch_partials<T, DP, 16>(c, by_block, grid, st);
    if (c.a.block == 32) return launch_partials<T, DP, 32>(c, by_block, grid, st);
    if (c.a.block == 64) return launch_partials<T, DP, 64>(c, by_block, grid, st);
    launch_partials<T, DP, 128>(c, by_block, grid, st);
  };
  if (c.a.dim <= 32) return keys(integral_constant<int, 32>{});
  if (c.a.dim <= 64) return keys(integral_constant<int, 64>{});
  if (c.a.dim <= 96) return keys(integral_constant<int, 96>{});
  keys(integral_constant<int, 128>{});
}

}  // namespace
}  // namespace nnx
