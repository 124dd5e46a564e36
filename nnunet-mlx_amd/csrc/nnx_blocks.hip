// Attention over blocks of keys that a cheap score selects for each query: block summaries,
// selection and the attention itself.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "nnx_blocks.h"

namespace nnx {
namespace {

constexpr int kMaxBlocks = 32768;
constexpr int kMaxKeep = 256;
constexpr float kTiny = 8.673617379884035e-19f;  // 2^-60

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
    require(c.heads / c.kv_heads <= 1024, w + "at most 1024 heads may share a key head");
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

__device__ __forceinline__ float finite_or_zero(float v) { return fabsf(v) < INFINITY ? v : 0.f; }

// ---- summaries -------------------------------------------------------------------------

// The mean key of a block as 8-bit codes under one scale: s = sum of the keys in 15 bits of the block's
// largest magnitude, the codes s in 7 bits of its own largest.  Sums of whole numbers have no order, so
// the codes, and the choices made by them, are the same however the keys are dealt to threads.
// Bound by the launch and one read of the keys: 2560 blocks of 64 keys of 64 bfloat16 (21 MB) take
// 11 us, 4 us of it the read at a large copy's rate.  A workgroup a block, dim / 8 threads a key: whole
// rows of memory, and as many loads in flight as a thread has keys (BK / 16); the keys stay in
// registers between the search for the largest magnitude and the sums.
template <class T, int BK>
__global__ __launch_bounds__(256) void summarize_kernel(BlockArgs a, const T* k, int first,
                                                        int8_t* codes, float* scales) {
  constexpr int EACH = BK / 16;  // of 16 threads a key; fewer channels leave fewer keys a thread
  __shared__ float top_lds[4];
  __shared__ int sums[128], most_lds[4], count_lds[4];
  const int j = first + blockIdx.x, g = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int lanes = a.dim / 8, per = 256 / lanes, sub = tid / lanes, d = (tid - sub * lanes) * 8;
  const int lo = j * BK, hi = min(lo + BK, item_length(a, b));
  const T* kb = k + b * a.ks[0] + g * a.ks[2] + d;
  const uint8_t* mask = a.mask ? a.mask + b * a.ms : nullptr;
  if (tid < 128) sums[tid] = 0;
  Vec<T, 8> v[EACH];
  bool in[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int64_t key = lo + sub + i * per;
    in[i] = sub < per && sub + i * per < BK && key < hi && (!mask || mask[key]);
    if (in[i]) v[i] = load_vec<8>(kb + key * a.ks[1]);
  }
  int count = 0;
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (!in[i]) continue;
    count += d == 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(finite_or_zero(to_float(v[i].v[e]))));
  }
  const auto larger = [](float x, float y) { return fmaxf(x, y); };
  top = lanes_reduce<64>(top, larger);
  count = (int)lanes_reduce<64>((float)count, [](float x, float y) { return x + y; });
  if (tid % 64 == 0) top_lds[tid / 64] = top, count_lds[tid / 64] = count;
  __syncthreads();
  top = fmaxf(fmaxf(top_lds[0], top_lds[1]), fmaxf(top_lds[2], top_lds[3]));
  count = count_lds[0] + count_lds[1] + count_lds[2] + count_lds[3];
  if (top >= kTiny && sub < per) {
    const float up = __fdiv_rn(32767.f, top);
    int s[8] = {};
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if (!in[i]) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += (int)rintf(finite_or_zero(to_float(v[i].v[e])) * up);
    }
    // whole numbers: the order of these additions does not show
#pragma unroll
    for (int e = 0; e < 8; ++e) atomicAdd(&sums[d + e], s[e]);
  }
  __syncthreads();
  const int sum = tid < a.dim ? sums[tid] : 0;
  // below 2^24: exact as floats
  const float most4 = lanes_reduce<64>((float)abs(sum), larger);
  if (tid % 64 == 0) most_lds[tid / 64] = (int)most4;
  __syncthreads();
  const int most = max(most_lds[0], most_lds[1]);
  const int64_t at = ((int64_t)b * a.kv_heads + g) * a.blocks + j;
  if (tid < a.dim) {
    const float down = most ? __fdiv_rn(127.f, (float)most) : 0.f;
    codes[at * a.dim + tid] = (int8_t)(int)rintf((float)sum * down);
  }
  if (tid == 0) {
    scales[at] = count == 0 ? -1.f
                 : most == 0 ? 0.f
                             : __fdiv_rn(top, 4161409.f * (float)count) * (float)most;
  }
}

// ---- selection -------------------------------------------------------------------------

typedef int i32x4 __attribute__((ext_vector_type(4)));

// The kept blocks of one row of scores, written by a wave: the forced ones and the highest scores,
// equal ones by the lower index.  A score that is no candidate is NaN, which no comparison takes.
// A cut is searched by halving until exactly as many scores as are wanted lie above it: of the
// values at first, which ends in some 9 steps for scores with gaps, then of their order as whole
// numbers, which ends in 32 at a value whose equals are taken from the lowest index on.  A step is
// a comparison, a count and an addition for each register, and bound by their issue.  (Steps aimed
// by a line through the counts' logarithms were fewer and took longer, 214 us against 185 for 163840
// rows of 512: the scores have more than one hump.)
struct Cut {
  float above;  // kept: scores above it, and the first `ties` that equal it
  int ties;
};

// Needs above(low) >= want > above(high).
template <class Above>
__device__ __forceinline__ Cut refine_cut(float low, float high, int want, Above&& above) {
  for (int step = 0; step < 14; ++step) {
    const float mid = 0.5f * low + 0.5f * high;
    const int count = (int)above(mid);
    if (count == want) return {mid, 0};
    (count < want ? high : low) = mid;
  }
  const auto order = [](float v) {
    const int32_t b = __float_as_int(v + 0.f);
    return b ^ (b >> 31 & 0x7fffffff);
  };
  const auto back = [](int32_t o) { return __int_as_float(o ^ (o >> 31 & 0x7fffffff)); };
  int32_t lo = order(low), hi = order(high);
  while ((int64_t)hi - lo > 1) {
    const int32_t mid = (int32_t)(((int64_t)lo + hi) >> 1);
    ((int)above(back(mid)) < want ? hi : lo) = mid;
  }
  return {back(hi), want - (int)above(back(hi))};
}

constexpr float kMostFloat = 3.4028235e38f;

template <class Above, class Range>
__device__ __forceinline__ Cut find_cut(int want, Above&& above, Range&& range) {
  if (want <= 0) return {kMostFloat, 0};  // but +inf, which forced blocks have in the end
  if (above(-INFINITY) <= want) return {-INFINITY, 0};
  float low, high;
  range(low, high);
  const int over = above(low);
  if (over < want) return {low, want - over};
  return refine_cut(low, high, want, above);
}

__device__ __forceinline__ int lanes_before(uint64_t lanes, int from) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32),
                                        __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, (uint32_t)from));
}

// The row lies in LDS, `chunks` times 64 filled up with NaN; N > 0: N = chunks, held in N registers a
// lane; N = 0: a multiple of 8 chunks, read again for every step.  `spare`: 256 places, for N > 0 the row's own.
template <int N>
__device__ __forceinline__ void select_row(float* score, float* spare, int chunks, int blocks, int keep,
                                           int first, int local, int own, int32_t* out) {
  const int lane = threadIdx.x % 64;
  constexpr uint32_t kForced = 0x7fc00001u;  // a forced block: a NaN of its own while the others are compared
  int forced = 0;
  const auto force = [&](int begin, int end) {  // blocks begin .. end - 1 as far as they are candidates
    for (int j0 = begin / 64 * 64; j0 < end; j0 += 64) {
      const int j = j0 + lane;
      const bool take = j >= begin && j < end && score[j] > -INFINITY && score[j] < INFINITY;
      if (take) score[j] = __uint_as_float(kForced);
      forced += __popcll(__ballot(take));
    }
  };
  if (first) force(0, min(first, blocks));
  if (local) force(max(own + 1 - local, 0), min(own + 1, blocks));
  float v[N ? N : 1];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = score[i * 64 + lane];
  const auto each = [&](auto&& body) {
    if constexpr (N > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) body(i, v[i]);
    } else {
      for (int i = 0; i < chunks; i += 8) {
        float y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = score[(i + k) * 64 + lane];
#pragma unroll
        for (int k = 0; k < 8; ++k) body(i + k, y[k]);
      }
    }
  };
  const auto above = [&](float x) {
    int count = 0;
    each([&](int, float y) { count += __popcll(__ballot(y > x)); });
    return count;
  };
  const auto larger = [](float x, float y) { return fmaxf(x, y); };
  const auto range = [&](float& low, float& high) {
    low = INFINITY, high = -INFINITY;
    each([&](int, float y) { low = y < low ? y : low, high = y > high ? y : high; });
    low = -lanes_reduce<64>(-low, larger);
    high = lanes_reduce<64>(high, larger);
  };
  const auto restore = [&] {  // forced blocks above all others
    const auto shown = [](float y) { return __float_as_uint(y) == kForced ? INFINITY : y; };
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = shown(v[i]);
    for (int i = 0; !N && i < chunks; ++i) score[i * 64 + lane] = shown(score[i * 64 + lane]);
  };
  int done = 0, tied = 0;
  const auto emit = [&](int block, uint64_t equal, bool take, int ties) {
    if (ties) {
      take |= ((equal >> lane) & 1) && lanes_before(equal, tied) < ties;
      tied += __popcll(equal);
    }
    const uint64_t taken = __ballot(take);
    const int to = lanes_before(taken, done);
    if (take && to < keep) out[(uint32_t)to] = block;
    done += __popcll(taken);
  };
  const auto finish = [&] {
    for (int i = min(done, keep) + lane; i < keep; i += 64) out[i] = -1;
  };
  if constexpr (N == 0 || N >= 4) {
    // Once no more than 128 scores are left above the lower end, they and their blocks are packed into two
    // registers (by way of `spare`), where the rest of the search and the writing cost a fraction.  (A first
    // guess from two or four samples a lane saved steps and no time: 153 us against 153.)
    const int want = keep - forced, room = 128 - forced;
    int over = above(-INFINITY);
    if (keep <= 128 && want > 0 && over > want) {
      float low, high;
      range(low, high);
      low -= fabsf(low) * 1e-6f + 1e-30f;  // below all, -inf at worst
      for (int step = 0; step < 14 && over > room; ++step) {
        const float mid = 0.5f * low + 0.5f * high;
        const int count = above(mid);
        if (count < want) {
          high = mid;
        } else {
          low = mid, over = count;
        }
      }
      if (over <= room) {
        if (forced) restore();
        wave_sync();
        int n = 0;
        each([&](int i, float y) {
          const bool take = y > low;
          const uint64_t taken = __ballot(take);
          const int to = lanes_before(taken, n);
          if (take && to < 128) spare[to] = y, spare[128 + to] = __int_as_float(i * 64 + lane);
          n += __popcll(taken);
        });
        wave_sync();
        float w[2];
        int32_t at[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool in = i * 64 + lane < n;
          w[i] = in ? spare[i * 64 + lane] : NAN;
          at[i] = in ? __float_as_int(spare[128 + i * 64 + lane]) : 0;
        }
        const Cut cut = refine_cut(low, high, keep, [&](float x) {
          return __popcll(__ballot(w[0] > x)) + __popcll(__ballot(w[1] > x));
        });
#pragma unroll
        for (int i = 0; i < 2; ++i) emit(at[i], cut.ties ? __ballot(w[i] == cut.above) : 0, w[i] > cut.above, cut.ties);
        return finish();
      }
    }
  }
  const Cut cut = find_cut(keep - forced, above, range);
  if (forced) restore();
  each([&](int i, float y) {
    emit(i * 64 + lane, cut.ties ? __ballot(y == cut.above) : 0, y > cut.above || y == INFINITY, cut.ties);
  });
  finish();
}

// `rows` <= 16 queries of one item and key head: their scores against 16 blocks at a time by 8-bit
// products in whole numbers, kept in LDS; then a wave a query picks.  Heads that share the key
// head are taken kScoreHeads at a time (their codes in LDS) and meet in the largest score.  A
// wave's next AHEAD times 16 blocks are on their way while it scores the ones before.
// Bound by the issue of instructions: 163840 rows against 512 blocks of 64 channels take 150 us, the
// vector and the scalar units busy for 72 % of it (389 and 383 instructions a row), for 84
// million scores of which 5.2 million are kept; the codes of a key head (32 KB) come from the L2, and
// the scores never leave the CU.  8 queries a workgroup leave half of a
// product unused (240 us against 190), 4 or 16 waves a workgroup fill the CU less evenly than 8 (209
// and 269 against 190) unless there are too few workgroups for the CUs; four tiles of codes in flight
// instead of two spill (40 against 33 us for 12 rows against 2048 blocks of 8 heads of 128).
constexpr int kScoreHeads = 8;
// Rows of up to 2048 blocks (32 registers a lane) are scored and picked from by one workgroup, a tile
// of 16 queries each, unless the tiles are few for the chip.  One kernel against scores by parts and
// picking, with 64 channels: 4 tiles of 256 blocks 6.9 us and 8.1, 16 of 512 8.4 and 8.1, 32 of 512 8.2
// and 9.3, 32 of 1024 10.8 and 10.7, 4 of 2048 16.5 and 11.8, 64 of 2048 16.6 and 19.7; with 8 heads
// of 128 channels 4 tiles of 256 10.9 and 12.2, 4 of 2048 30 and 17, 32 of 2048 31 and 24, 64 31 and 34.
// Longer rows always go by parts (8192 blocks: 6 tiles 167 us in one kernel, which has to read its
// scores again for every step, 8 tiles 32 us by parts).
constexpr int kWholeBlocks = 2048, kPartBlocks = 512, kPartTiles = 32;
constexpr int64_t kScoreBudget = (int64_t)128 << 20;

struct Parts {
  int count, blocks;  // of a row; of a part
  int rows, pitch;    // queries of a launch, places of one
  float* scores;      // by item, key head and query
};

// The block of a query's own position: -1 before the first key, at most 2^24 (past the last block).
__device__ __forceinline__ int own_block(const BlockArgs& a, int b, int t) {
  const int64_t at = (item_start(a, b) + t) >> __builtin_ctz(a.block);
  return (int)min(max(at, (int64_t)-1), (int64_t)1 << 24);
}
constexpr int kPart = -1;  // the scores of a part of the blocks only, to global memory

template <class T, int N>
__global__ __launch_bounds__(1024) void select_kernel(BlockArgs a, const T* q, const int8_t* codes,
                                                      const float* scales, int32_t* ids, int rows,
                                                      int pitch, int from, Parts parts) {
  extern __shared__ __attribute__((aligned(16))) float score[];  // rows x pitch
  i32x4* qcode = (i32x4*)(score + rows * pitch);                 // by head, 64 channels, lane
  __shared__ float qtop[kScoreHeads][16];
  const int t0 = from + (N == kPart ? blockIdx.x / parts.count : blockIdx.x) * rows, g = blockIdx.y, b = blockIdx.z;
  const int begin = N == kPart ? blockIdx.x % parts.count * parts.blocks : 0;
  const int stop = N == kPart ? min(begin + parts.blocks, a.blocks) : a.blocks;
  const int lane = threadIdx.x % 64, col = lane % 16, quad = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64;
  const int64_t unit = (int64_t)b * a.kv_heads + g;
  constexpr int AHEAD = N == kPart ? 1 : 2;
  const bool wide = a.dim > 64;
  const int own = a.causal ? own_block(a, b, t0 + col) : 1 << 24;
  const uint32_t unit_bytes = (uint32_t)a.blocks * a.dim;
  const auto cu = buffer_of(codes + unit * unit_bytes, unit_bytes);
  const auto su = buffer_of(scales + unit * a.blocks, a.blocks * 4);
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  struct Blocks {
    i32x2 k[4];
    int scale[4];
  };
  // Past the last block all is 0 and not kept; past the head's end lie the next block's codes, and the
  // queries' codes are 0.  The whole offset is the lane's: the scalar one is left out of the bounds check.
  const uint32_t code_at = (uint32_t)(col * a.dim + quad * 16), scale_at = (uint32_t)(quad * 16);
  const auto load = [&](Blocks& x, int j0) {
    const uint32_t ca = code_at + (uint32_t)(j0 * a.dim), sa = scale_at + (uint32_t)(j0 * 4);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s > 1 && !wide) break;
      x.k[s] = __builtin_bit_cast(
          i32x2, __builtin_amdgcn_raw_buffer_load_b64(cu, ca + s / 2 * 64 + s % 2 * 8, 0, 0));
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) x.scale[r] = (int)__builtin_amdgcn_raw_buffer_load_b32(su, sa + 4 * r, 0, 0);
  };
  if (N > 0) {
    const int full = (a.blocks + 15) / 16 * 16, rest = N * 64 - full;
    for (int i = threadIdx.x; i < rows * rest; i += blockDim.x)
      score[i / rest * pitch + full + i % rest] = NAN;
  }
  for (int h0 = 0; h0 < a.group; h0 += kScoreHeads) {
    const int heads = min(kScoreHeads, a.group - h0);
    Blocks x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(x[i], begin + (wave + i * waves) * 16);
    if (h0) __syncthreads();
    // 16 lanes a query and head, 8 channels each, into the places of the products' second operand
    for (int i = threadIdx.x / 16; i < heads * 16; i += blockDim.x / 16) {
      const int h = i / 16, t = i % 16, d = lane % 16 * 8;
      Vec<T, 8> x{};
      if (t < rows && t0 + t < a.queries && d < a.dim)
        x = load_vec<8>(q + b * a.qs[0] + (int64_t)(t0 + t) * a.qs[1] + (int64_t)(g * a.group + h0 + h) * a.qs[2] + d);
      float v[8], m = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = finite_or_zero(to_float(x.v[e]));
        m = fmaxf(m, fabsf(v[e]));
      }
      m = lanes_reduce<16>(m, [](float p, float r) { return fmaxf(p, r); });
      const float up = m < kTiny ? 0.f : __fdiv_rn(127.f, m);
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e / 4] |= ((uint32_t)(int)rintf(v[e] * up) & 255u) << (8 * (e % 4));
      if (d < 64 || wide) {
        uint32_t* to = (uint32_t*)&qcode[(h * 2 + d / 64) * 64 + d % 64 / 16 * 16 + t] + d % 16 / 4;
        to[0] = w[0], to[1] = w[1];
      }
      if (lane % 16 == 0) qtop[h][t] = m < kTiny ? 1.f : m;
    }
    __syncthreads();
    const auto compute = [&](const Blocks& x, int j0) {
      const i32x4 k0{x.k[0][0], x.k[0][1], x.k[1][0], x.k[1][1]};
      const i32x4 k1{x.k[2][0], x.k[2][1], x.k[3][0], x.k[3][1]};
      float best[4], scale[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) scale[r] = __int_as_float(x.scale[r]);
      for (int h = 0; h < heads; ++h) {
        i32x4 dot = {0, 0, 0, 0};
        dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(k0, qcode[h * 128 + lane], dot, 0, 0, 0);
        if (wide) dot = __builtin_amdgcn_mfma_i32_16x16x64_i8(k1, qcode[h * 128 + 64 + lane], dot, 0, 0, 0);
        const float top = qtop[h][col];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float y = ((float)dot[r] * top) * scale[r];
          best[r] = h && !(y > best[r]) ? best[r] : y;
        }
      }
      // products can overflow; infinities mean something else to what follows
#pragma unroll
      for (int r = 0; r < 4; ++r) best[r] = __builtin_amdgcn_fmed3f(best[r], -kMostFloat, kMostFloat);
      if (col < rows) {
        float4* to = (float4*)&score[col * pitch + j0 - begin + quad * 4];
        if (h0) {
          const float4 z = *to;
          best[0] = fmaxf(best[0], z.x), best[1] = fmaxf(best[1], z.y);
          best[2] = fmaxf(best[2], z.z), best[3] = fmaxf(best[3], z.w);
        }
        if (__any(fminf(fminf(scale[0], scale[1]), fminf(scale[2], scale[3])) < 0.f)) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (scale[r] < 0.f) best[r] = NAN;  // no valid key
        }
        if (a.causal || j0 + 16 > a.blocks) {
          const int end = min(own, a.blocks - 1);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (j0 + quad * 4 + r > end) best[r] = NAN;
        }
        *to = make_float4(best[0], best[1], best[2], best[3]);
      }
    };
    for (int j0 = begin + wave * 16; j0 < stop; j0 += AHEAD * waves * 16) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int j = j0 + i * waves * 16;
        if (j < stop) compute(x[i], j);
        if (N != kPart || j + AHEAD * waves * 16 < stop) load(x[i], j + AHEAD * waves * 16);
      }
    }
  }
  __syncthreads();
  if constexpr (N == kPart) {
    const int each = (stop - begin + 15) / 16 * 4;  // float4 of a row
    const int last = min(rows, from + parts.rows - t0);  // the launch's may be fewer than the queries
    for (int i = threadIdx.x; i < min(last, a.queries - t0) * each; i += blockDim.x) {
      const int r = i / each, j = i % each * 4;
      *(float4*)(parts.scores + (unit * parts.rows + t0 - from + r) * parts.pitch + begin + j) = *(float4*)&score[r * pitch + j];
    }
  } else {
    for (int r = wave; r < rows && t0 + r < a.queries; r += waves)
      select_row<N>(score + r * pitch, score + r * pitch, N, a.blocks, a.keep, a.first, a.local, own_block(a, b, t0 + r),
                    ids + (((int64_t)b * a.queries + t0 + r) * a.kv_heads + g) * a.keep);
  }
}

// Picks from a row of scores in global memory: a workgroup brings it to LDS, a wave searches.  (Rows of
// up to 8192 blocks held in registers took as long.)
__global__ __launch_bounds__(256) void pick_kernel(BlockArgs a, int from, Parts parts, int32_t* ids) {
  extern __shared__ __attribute__((aligned(16))) float score[];  // 64 a chunk and 256 more
  const int t = from + blockIdx.x, g = blockIdx.y, b = blockIdx.z, chunks = (a.blocks + 511) / 512 * 8;
  const float* row = parts.scores + (((int64_t)b * a.kv_heads + g) * parts.rows + blockIdx.x) * parts.pitch;
#pragma unroll 4
  for (int j = threadIdx.x * 4; j < chunks * 64; j += 1024) {
    const float4 v = *(const float4*)&row[min(j, parts.pitch - 4)];
    *(float4*)&score[j] = j < parts.pitch ? v : make_float4(NAN, NAN, NAN, NAN);
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  select_row<0>(score, score + chunks * 64, chunks, a.blocks, a.keep, a.first, a.local, own_block(a, b, t),
                ids + (((int64_t)b * a.queries + t) * a.kv_heads + g) * a.keep);
}

// Rows of many blocks, or few rows: the scores by parts of a row, a workgroup each, to global memory,
// then a wave a row picks.
struct SelectPlan {
  bool split;
  int chunks, rows, pitch;  // of the kernel that forms scores: 64 blocks each, queries of a workgroup, LDS row
  int queries;              // of a launch
  Parts parts;
  size_t bytes;
};

SelectPlan plan_selection(const nnx_block_config& c) {
  SelectPlan p{};
  const int blocks = (int)ceil_div(c.keys, c.block);
  const int64_t units = (int64_t)c.kv_heads * c.batch, tiles = ceil_div(c.queries, 16) * units;
  p.chunks = 1;
  while (p.chunks * 64 < blocks) p.chunks *= 2;
  p.rows = std::min(16, c.queries);
  p.split = blocks > kWholeBlocks || (blocks >= kPartBlocks && tiles <= std::min(kPartTiles, blocks / 32));
  if (!p.split) {
    p.pitch = p.chunks * 64 + 4;  // with the codes at most 16 * 2052 * 4 + 8 * 2048 bytes of LDS, 144 KB
    return p;
  }
  p.parts.pitch = (int)ceil_div(blocks, 16) * 16;
  p.queries = (int)std::min<int64_t>(c.queries, std::max<int64_t>(16, kScoreBudget / (units * p.parts.pitch * 4) / 16 * 16));
  p.parts.rows = p.queries;
  const double want = (double)blocks * ceil_div(p.queries, 16) * units / 256;
  p.parts.blocks = (int)std::min(1024.0, std::max(1.0, std::ceil(want / 64)) * 64);
  p.parts.count = (int)ceil_div(blocks, p.parts.blocks);
  p.pitch = p.parts.blocks + 4;
  p.bytes = (size_t)units * p.queries * p.parts.pitch * 4;
  return p;
}

// ---- the attention ---------------------------------------------------------------------
//
// Rows that keep the same block need the same keys and values, and rows near each other mostly
// keep different ones.  So the pairs (query, kept block) are gathered by block: dense tiles of
// rows against a block that stays in LDS, one partial softmax a pair, and a last pass that joins
// each row's partials.  Few pairs skip the gathering: a workgroup each.
//
// The lists of 5.2 million pairs (163840 rows of 32 blocks) take 50 us: totals cleared 5, counted 17,
// summed 5, placed 25.  The ids are read twice (42 MB) and 21 MB of entries written in runs of a few;
// counting and placing wait for most of their time, for the ids and the additions in LDS and memory.
// (Sums formed by every placing workgroup, for one launch less, took as long: 58 us against 54.)

// Calls body(entry, block) for the pairs of `per` queries of a span (grid: groups, spans), 16 ids a thread on
// their way at a time (4: 56 us against 52 for the lists above).
template <class F>
__device__ __forceinline__ void each_pair(const ChunkArgs& c, int per, F&& body) {
  constexpr int AHEAD = 16;
  const BlockArgs& a = c.a;
  const Span s = span_of(c, c.span0 + blockIdx.y);
  const int t_lo = blockIdx.x * per, t_hi = min(t_lo + per, s.queries);
  const int32_t* ids = c.ids + (((int64_t)s.b * a.queries + s.t0) * a.kv_heads + s.g) * a.keep;
  const int end = t_hi * a.keep;
  for (int e0 = t_lo * a.keep + threadIdx.x; e0 < end; e0 += AHEAD * 256) {
    int j[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int e = min(e0 + i * 256, end - 1), t = c.by_keep(e);
      j[i] = ids[(int64_t)t * a.kv_heads * a.keep + e - t * a.keep];
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (e0 + i * 256 < end && (unsigned)j[i] < (unsigned)a.blocks) body(e0 + i * 256, j[i]);
  }
}

// Counts by block in LDS; each group takes its range of every block's list by one addition to the
// block's total.  The order of groups and pairs in a list is left to chance and shows in no
// result: a row's partial does not depend on its neighbours in a tile.
__global__ __launch_bounds__(256) void count_pairs_kernel(ChunkArgs c, int per, int32_t* total,
                                                          int32_t* base) {
  extern __shared__ int32_t hist[];
  const int blocks = c.a.blocks;
  for (int j = threadIdx.x; j < blocks; j += 256) hist[j] = 0;
  __syncthreads();
  each_pair(c, per, [&](int, int j) { atomicAdd(&hist[j], 1); });
  __syncthreads();
  int32_t* mine = base + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * blocks;
  for (int j = threadIdx.x; j < blocks; j += 256)
    if (hist[j]) mine[j] = atomicAdd(&total[blockIdx.y * blocks + j], hist[j]);
}

// Where each block's list starts, and its tiles: running sums over n totals, by one workgroup.
__global__ __launch_bounds__(1024) void scan_pairs_kernel(const int32_t* total, int n, int group,
                                                          int32_t* start, int32_t* tiles) {
  __shared__ int2 part[16];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  int2 before = make_int2(0, 0);
  for (int at = 0; at < n; at += 4096) {
    int2 mine[4], sum = make_int2(0, 0);
    const int i0 = at + threadIdx.x * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pairs = i0 + i < n ? total[i0 + i] : 0;
      mine[i] = sum;
      sum.x += pairs;
      sum.y += (int)(((int64_t)pairs * group + kTileRows - 1) / kTileRows);
    }
    int2 run = sum;
    for (int o = 1; o < 64; o *= 2) {
      const int x = __shfl_up(run.x, o), y = __shfl_up(run.y, o);
      if (lane >= o) run.x += x, run.y += y;
    }
    __syncthreads();
    if (lane == 63) part[wave] = run;
    __syncthreads();
    int2 offset = before;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) offset.x += part[w].x, offset.y += part[w].y;
      before.x += part[w].x, before.y += part[w].y;
    }
    offset.x += run.x - sum.x, offset.y += run.y - sum.y;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i0 + i < n) start[i0 + i] = offset.x + mine[i].x, tiles[i0 + i] = offset.y + mine[i].y;
  }
  if (threadIdx.x == 0) start[n] = before.x, tiles[n] = before.y;
}

__global__ __launch_bounds__(256) void place_pairs_kernel(ChunkArgs c, int per, const int32_t* base,
                                                          int32_t* list) {
  extern __shared__ int32_t next[];
  const int blocks = c.a.blocks;
  const int32_t* mine = base + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * blocks;
  // base holds nothing for blocks without pairs here, and their place is not asked for
  for (int j = threadIdx.x; j < blocks; j += 256) next[j] = c.start[blockIdx.y * blocks + j] + mine[j];
  __syncthreads();
  each_pair(c, per, [&](int e, int j) { list[atomicAdd(&next[j], 1)] = e; });
}

// Adds what of block j's values is not finite and seen by query t of a span: the sum becomes the infinity or
// NaN that it is by definition, in the channels that hold one.
template <class T>
__device__ __forceinline__ void add_odd_values(const ChunkArgs& c, const T* v, Span s, int t, int j,
                                                         float (&o)[8]) {
  const BlockArgs& a = c.a;
  const uint8_t* mask = a.mask ? a.mask + s.b * a.ms : nullptr;
  const int64_t first = (int64_t)j * a.block, at = item_start(a, s.b) + s.t0 + t;
  int64_t end = min(first + a.block, (int64_t)item_length(a, s.b));
  if (a.causal) end = min(end, at + 1);
  for (int64_t key = first; key < end; ++key) {
    if (mask && !mask[key]) continue;
    const Vec<T, 8> x = load_vec<8>(v + s.b * a.vs[0] + key * a.vs[1] + s.g * a.vs[2]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = to_float(x.v[e]);
      if (!(fabsf(y) < INFINITY)) o[e] += y;
    }
  }
}

// out = sum_s w_s O_s / sum_s w_s l_s with w_s = 2^(m_s - largest), O_s a partial times its power of
// two, in the order of the slots.  A workgroup forms the weights of its rows together, then dim / 8
// lanes a row add up (`share` groups of them a row, each every share-th partial, where rows are few
// or have many).  Bound by its reads: 143 MB of partials in 27 us (5.3 TB/s, mostly from the
// last-level cache), 8 partials in flight a lane.
constexpr int kJoinWeights = 4096;

template <class T>
__global__ __launch_bounds__(256) void join_partials_kernel(ChunkArgs c, T* out, int share, int each) {
  using P = Partial<T>;
  const float2 nothing = make_float2(-INFINITY, __uint_as_float(kExponentZero));
  // by row and slot (m, l); then the shares' sums
  extern __shared__ float2 weight[];
  float(*sums)[9] = (float(*)[9])(weight + each * c.a.keep);
  const BlockArgs& a = c.a;
  const int64_t row0 = (int64_t)blockIdx.x * each, rows = (int64_t)c.spans * c.nt * a.group;
  const int here = (int)min((int64_t)each, rows - row0);
  const auto place = [&](int64_t row, Span& s, int& t, int& h) {
    const int vt = c.by_group((int)row), span = c.by_nt(vt);
    h = (int)row - vt * a.group;
    t = vt - span * c.nt;
    s = span_of(c, c.span0 + span);
  };
  // partials lie by query, slot and head
  const auto partial_of = [&](int64_t row) {
    const int vt = c.by_group((int)row);
    return (int64_t)vt * a.keep * a.group + (int)row - vt * a.group;
  };
  for (int i = threadIdx.x; i < here * a.keep; i += 256) {
    const int r = c.by_keep(i), slot = i - r * a.keep;
    Span s;
    int t, h;
    place(row0 + r, s, t, h);
    int j = -1;
    if (t < s.queries)
      j = c.ids[(((int64_t)s.b * a.queries + s.t0 + t) * a.kv_heads + s.g) * a.keep + slot];
    weight[i] = (unsigned)j < (unsigned)a.blocks ? c.meta[partial_of(row0 + r) + (int64_t)slot * a.group]
                                                 : nothing;
  }
  const int lanes = a.dim / 8, sub = threadIdx.x / lanes, u = threadIdx.x - sub * lanes;
  const int own = sub / share, part0 = sub - own * share;
  const bool live = own < here;
  // Partials of entries that are no block were never written: whatever is there is left out below.
  constexpr int AHEAD = 8;
  const P* part = (const P*)c.part + partial_of(row0 + (live ? own : 0)) * a.dim + 8 * u;
  bool odd = false;  // some partial leaves out values that are not finite
  Vec<P, 8> x[AHEAD];
  const auto fetch = [&](int s0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) x[i] = load_vec<8>(part + (int64_t)min(s0 + i * share, a.keep - 1) * a.group * a.dim);
  };
  fetch(part0);
  __syncthreads();
  float o[8] = {}, l = 0.f;
  if (live) {
    const float2* w = weight + own * a.keep;
    float top = -INFINITY;
#pragma unroll 8
    for (int s = 0; s < a.keep; ++s) top = fmaxf(top, w[s].x);
    if (top == -INFINITY) top = 0.f;
    top += (float)(32 - __clz(a.keep - 1));  // weights that sum to 1 at most keep the sum in the values' range
    for (int s0 = part0; s0 < a.keep; s0 += AHEAD * share) {
      if (s0 != part0) fetch(s0);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int s = s0 + i * share;
        const float2 m = s < a.keep ? w[s] : nothing;
        const float ws = __builtin_amdgcn_exp2f(m.x - top);
        const bool written = !(m.x == -INFINITY);
        float f = ws, sum = fabsf(m.y);
        if constexpr (sizeof(P) == 2) {
          const uint32_t bits = __float_as_uint(sum);
          f *= __uint_as_float(((bits & kExponentBits) + 127 - kExponentZero) << 23);
          sum = __uint_as_float(bits & ~kExponentBits);
        }
        odd |= m.y < 0.f;
        l = fmaf(ws, sum, l);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          o[e] = fmaf(f, written ? to_float(x[i].v[e]) : 0.f, o[e]);
        }
      }
    }
  }
  if (odd) {
    Span s;
    int t, h;
    place(row0 + own, s, t, h);
    for (int slot = part0; slot < a.keep; slot += share) {
      if (!(weight[own * a.keep + slot].y < 0.f)) continue;
      const int j = c.ids[(((int64_t)s.b * a.queries + s.t0 + t) * a.kv_heads + s.g) * a.keep + slot];
      add_odd_values(c, (const T*)c.v + 8 * u, s, t, j, o);
    }
  }
  if (share > 1) {
    for (int i = 0; i < 8; ++i) sums[threadIdx.x][i] = o[i];
    sums[threadIdx.x][8] = l;
    __syncthreads();
    if (!live || part0) return;
    for (int p = 1; p < share; ++p) {
      for (int i = 0; i < 8; ++i) o[i] += sums[threadIdx.x + p * lanes][i];
      l += sums[threadIdx.x + p * lanes][8];
    }
  }
  if (!live) return;
  Span s;
  int t, h;
  place(row0 + own, s, t, h);
  if (t >= s.queries) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  Vec<T, 8> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = from_float<T>(o[i] * inv);
  store_vec(out + s.b * a.os[0] + (s.t0 + t) * a.os[1] + (int64_t)(s.g * a.group + h) * a.os[2] + 8 * u, r);
}

// Where the work is cut and where it lies in the workspace.  Spans and the launches that cover
// some of them are sized for their partials to stay in the 256 MiB last-level cache until they are
// joined (a launch over everything took 1.35 times as long at 5 x 32768 queries of 32 blocks);
// the lists of many launches are formed at once.
constexpr size_t kPartialBudget = (size_t)160 << 20;
constexpr int64_t kListPairs = (int64_t)1 << 27;
// Pairs go one by one up to so many, and so many bytes of keys and values.  One by one against by block
// (lists and partials): 1280 of 16 KiB 13 us and 16 + 15, 5120 28 and 16 + 16, 8192 of 32 KiB 71 and
// 19 + 21; 19200 of 4 KiB 45 and 25 + 30, 40000 of 1 KiB 67 and 25 + 24.
// More than that go by block where there are more of them than blocks that they may keep (of every item
// and key head): the sums over the blocks' totals cost 1 us a thousand, and a block that few pairs keep is
// staged for little.  A whole call, one by one against by block: 32768 pairs over 2097152 blocks of 4 KiB
// 80 us and 1964, over 1048576 79 and 1079; 16384 over 262144 of 32 KiB 262 and 526, over 32768 246 and
// 282; 32768 over 32768 505 and 424, over 8192 454 and 161; 65536 over 4096 858 and 97; of 8 KiB 32768
// over 16384 90 and 131, 65536 over 16384 167 and 145.
constexpr double kDirectPairs = 20000, kDirectBytes = 80e6;

struct AttentionPlan {
  bool by_block;
  int splits, nt, spans;      // spans in all
  int at_once, listed;        // spans of a launch, spans whose lists are formed together
  int per, groups;            // queries of a counting group, groups of a span
  size_t total, base, start, tiles, list, meta, part, bytes;
};

AttentionPlan make_plan(const nnx_block_config& c) {
  AttentionPlan p;
  const int64_t group = c.heads / c.kv_heads, blocks = ceil_div(c.keys, c.block);
  // bytes of the partials of a query and key head: at most 256 * 130 * 4 a head
  const int64_t query = group * c.keep * (8 + (int64_t)c.head_dim * partial_bytes(c.type));
  const int64_t fit = std::max<int64_t>(1, kPartialBudget / query);
  p.nt = (int)ceil_div(c.queries, ceil_div(c.queries, fit));
  p.splits = (int)ceil_div(c.queries, p.nt);
  const int64_t spans = (int64_t)c.batch * c.kv_heads * p.splits;
  require(spans < (int64_t)1 << 31, "block attention: too many queries and key heads");
  p.spans = (int)spans;
  const double pairs = (double)c.batch * c.kv_heads * c.queries * c.keep;
  p.by_block = pairs > (double)c.batch * c.kv_heads * blocks &&
               (pairs > kDirectPairs || pairs * c.block * c.head_dim * 2 * type_bytes(c.type) > kDirectBytes);
  p.at_once = (int)std::max<int64_t>(1, std::min(spans, fit / p.nt));
  // counts and tiles are 32-bit, and spans a grid axis
  const int64_t most = std::min<int64_t>({spans, 65535, ((int64_t)1 << 30) / blocks, kListPairs / ((int64_t)p.nt * c.keep)});
  p.at_once = (int)std::min<int64_t>(p.at_once, std::max<int64_t>(1, std::min<int64_t>(65535, ((int64_t)1 << 30) / blocks)));
  p.at_once = (int)ceil_div(spans, ceil_div(spans, p.at_once));  // launches of one size
  p.listed = p.by_block ? (int)std::max<int64_t>(p.at_once, most) : p.at_once;
  p.per = (int)std::min<int64_t>(p.nt, ceil_div(std::max<int64_t>(4096, 2 * blocks), c.keep));
  p.groups = (int)ceil_div(p.nt, p.per);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t lists = p.by_block ? (size_t)p.listed * blocks : 0;
  const size_t rows = (size_t)p.at_once * p.nt * group * c.keep;
  p.total = take(lists * 4);
  p.base = take(lists * p.groups * 4);
  p.start = take((lists + 1) * 4);
  p.tiles = take((lists + 1) * 4);
  p.list = take(p.by_block ? (size_t)p.listed * p.nt * c.keep * 4 : 0);
  p.meta = take(rows * 8);
  p.part = take(rows * c.head_dim * partial_bytes(c.type));
  p.bytes = at;
  return p;
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
    const dim3 grid(blocks, c.kv_heads, c.batch);
    auto go = [&](auto bk) {
      summarize_kernel<T, decltype(bk)::value><<<grid, 256, 0, st>>>(a, (const T*)k, first_block, codes, scales);
    };
    using std::integral_constant;
    if (c.block == 16) return go(integral_constant<int, 16>{});
    if (c.block == 32) return go(integral_constant<int, 32>{});
    if (c.block == 64) return go(integral_constant<int, 64>{});
    go(integral_constant<int, 128>{});
  });
  launch_check("block_summarize");
}

void block_select(const nnx_block_config& c, const void* q, const int8_t* codes,
                  const float* scales, const int32_t* start, int32_t* ids, void* ws, size_t ws_bytes,
                  hipStream_t st) {
  check_config(c, "block selection", true);
  require(q && codes && scales && ids, "block selection: null pointer");
  require(reinterpret_cast<uintptr_t>(codes) % 8 == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0,
          "block selection: codes must be 8-byte and scales 4-byte aligned");
  const SelectPlan plan = plan_selection(c);
  require(!plan.split || (ws && ws_bytes >= plan.bytes && reinterpret_cast<uintptr_t>(ws) % 16 == 0),
          "block selection: the workspace is too small or not 16-byte aligned");
  const BlockArgs a = make_args(c, start, nullptr, nullptr);
  const double products = (double)c.batch * c.queries * c.heads * c.head_dim;
  ProfScope prof("block_select", 2.0 * products * a.blocks, products * type_bytes(c.type), st);
  using std::integral_constant;
  const size_t codes_bytes = (size_t)std::min(a.group, kScoreHeads) * 2048;
  const size_t shared = plan.rows * plan.pitch * sizeof(float) + codes_bytes;
  if (plan.split) {
    Parts parts = plan.parts;
    parts.scores = (float*)ws;
    for (int from = 0; from < c.queries; from += parts.rows) {
      const int queries = std::min(parts.rows, c.queries - from);
      const dim3 grid((unsigned)ceil_div(queries, plan.rows) * parts.count, c.kv_heads, c.batch);
      with_type(c.type, [&](auto t) {
        using T = decltype(t);
        select_kernel<T, kPart><<<grid, 256, shared, st>>>(a, (const T*)q, codes, scales, ids, plan.rows, plan.pitch,
                                                           from, parts);
      });
      launch_check("block_select");
      pick_kernel<<<dim3(queries, c.kv_heads, c.batch), 256, (ceil_div(a.blocks, 512) * 512 + 256) * sizeof(float), st>>>(
          a, from, parts, ids);
      launch_check("block_select");
    }
    return;
  }
  // As many queries a workgroup as the products take, and waves by how many workgroups a CU has.  16 waves
  // while CUs would idle: of 64 blocks 190 workgroups 6.0 us against 6.5 with 8 waves, 375 8.8 and 7.6; of
  // 400 8.3 and 10.1, 12.2 and 11.6; of 1000 10.6 and 13.3, 17.0 and 16.3; of 2000 14.7 and 19.3, 26.8 and
  // 35.6, where a workgroup's LDS leaves room for one alone.  4 waves for up to 128 blocks where there are
  // workgroups enough: of 64 blocks 5120 workgroups 29.9 against 35.4 with 8, 1024 14.7 and 15.9, 375 8.6
  // and 7.6; of 128 37.7 and 43.7, 19.2 and 18.1; of 256 49.6 and 54.2, 23.5 and 23.0; of 512 74.5 and
  // 66.4, 39.7 and 29.4.
  const dim3 grid((unsigned)ceil_div(c.queries, plan.rows), c.kv_heads, c.batch);
  const double each = (double)grid.x * grid.y * grid.z / compute_units();
  const int threads = each < (plan.chunks > 16 ? 2 : 1) ? 1024 : plan.chunks <= 2 && each >= 2 ? 256 : 512;
  with_type(c.type, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto k) {
      select_kernel<T, decltype(k)::value><<<grid, threads, shared, st>>>(
          a, (const T*)q, codes, scales, ids, plan.rows, plan.pitch, 0, Parts{});
    };
    if (plan.chunks == 1) return go(integral_constant<int, 1>{});
    if (plan.chunks == 2) return go(integral_constant<int, 2>{});
    if (plan.chunks == 4) return go(integral_constant<int, 4>{});
    if (plan.chunks == 8) return go(integral_constant<int, 8>{});
    if (plan.chunks == 16) return go(integral_constant<int, 16>{});
    go(integral_constant<int, 32>{});
  });
  launch_check("block_select");
}

size_t block_select_workspace(const nnx_block_config& c) {
  try {
    check_config(c, "block selection", true);
    return plan_selection(c).bytes;
  } catch (...) {  // nothing may leave a C entry
    return 0;
  }
}

size_t block_attention_workspace(const nnx_block_config& c) {
  try {
    check_config(c, "block attention", true);
    return make_plan(c).bytes;
  } catch (...) {  // nothing may leave a C entry
    return 0;
  }
}

void block_attention(const nnx_block_config& c, const void* q, const void* k, const void* v,
                     const int32_t* ids, const int32_t* start, const int32_t* lengths,
                     const uint8_t* mask, void* out, void* ws, size_t ws_bytes, hipStream_t st) {
  check_config(c, "block attention", true);
  require(q && k && v && ids && out && ws, "block attention: null pointer");
  const AttentionPlan p = make_plan(c);
  require(ws_bytes >= p.bytes && reinterpret_cast<uintptr_t>(ws) % 16 == 0,
          "block attention: the workspace is too small or not 16-byte aligned");
  ChunkArgs k0;
  k0.a = make_args(c, start, lengths, mask);
  const BlockArgs& a = k0.a;
  char* w = (char*)ws;
  auto at = [&](size_t offset) { return (int32_t*)(w + offset); };
  k0.q = q, k0.k = k, k0.v = v, k0.ids = ids;
  k0.part = w + p.part;
  k0.meta = (float2*)(w + p.meta);
  k0.list = at(p.list);
  k0.splits = p.splits, k0.nt = p.nt;
  k0.by_keep = FastDiv(c.keep), k0.by_group = FastDiv(a.group), k0.by_nt = FastDiv(p.nt);
  const double flops = 4.0 * a.group * c.keep * c.block * c.head_dim * p.nt;
  for (int l0 = 0; l0 < p.spans; l0 += p.listed) {
    const int listed = std::min(p.listed, p.spans - l0);
    if (p.by_block) {
      const int lists = listed * a.blocks;
      ChunkArgs m = k0;
      m.span0 = l0, m.spans = listed;
      m.start = at(p.start);
      ProfScope prof("block_lists", 0.0, 12.0 * listed * p.nt * c.keep, st);
      fill_zero(w + p.total, (size_t)lists * 4, st);
      count_pairs_kernel<<<dim3(p.groups, listed), 256, a.blocks * 4, st>>>(m, p.per, at(p.total), at(p.base));
      launch_check("count_pairs");
      scan_pairs_kernel<<<1, 1024, 0, st>>>(at(p.total), lists, a.group, at(p.start), at(p.tiles));
      launch_check("scan_pairs");
      place_pairs_kernel<<<dim3(p.groups, listed), 256, a.blocks * 4, st>>>(m, p.per, at(p.base), at(p.list));
      launch_check("place_pairs");
    }
    for (int s0 = 0; s0 < listed; s0 += p.at_once) {
      ChunkArgs m = k0;
      m.span0 = l0 + s0, m.spans = std::min(p.at_once, listed - s0);
      m.start = at(p.start) + (size_t)s0 * a.blocks;
      m.tiles = at(p.tiles) + (size_t)s0 * a.blocks;
      const int64_t pairs = (int64_t)m.spans * p.nt * c.keep;
      int grid = (int)pairs;
      if (p.by_block) {
        grid = (int)std::min<int64_t>(ceil_div(pairs * a.group, kTileRows) + (int64_t)m.spans * a.blocks, 1 << 30);
      }
      {
        ProfScope prof("block_partials", flops * m.spans, 0.0, st);
        if (c.type == NNX_TYPE_F32) {
          block_partials_f32(m, p.by_block, grid, st);
        } else if (c.type == NNX_TYPE_F16) {
          block_partials_f16(m, p.by_block, grid, st);
        } else {
          block_partials_bf16(m, p.by_block, grid, st);
        }
      }
      const int64_t rows = (int64_t)m.spans * p.nt * a.group;
      const int lanes = a.dim / 8;
      // groups of lanes a row: more while rows are too few for the CUs (65536 threads are one wave a
      // SIMD) or a workgroup's weights too many for its LDS
      int share = 1;
      const auto each = [&] { return 256 / (lanes * share); };
      while (lanes * share * 2 <= 256 &&
             (each() * c.keep > kJoinWeights || (share * 2 <= c.keep && rows * lanes * share < 65536)))
        share *= 2;
      const int here = std::min(each(), kJoinWeights / c.keep);
      ProfScope prof("block_join", 2.0 * rows * c.keep * c.head_dim,
                     (double)rows * c.keep * (8 + c.head_dim * partial_bytes(c.type)), st);
      with_type(c.type, [&](auto z) {
        using T = decltype(z);
        const size_t bytes = (size_t)here * c.keep * 8 + (share > 1 ? 256 * 9 * 4 : 0);
        join_partials_kernel<T><<<(unsigned)ceil_div(rows, here), 256, bytes, st>>>(m, (T*)out, share, here);
      });
      launch_check("block_join");
    }
  }
}

}  // namespace nnx
