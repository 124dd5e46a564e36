// Attention over held tokens on matrix instructions; included by one source a type.
#pragma once

#include <type_traits>

#include "nnx_held.h"
#include "nnx_operands.h"

namespace nnx {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// Eight codes as E, exactly.  float16: a code's byte under 0x64 is 1024 + (code + 128), less 1152 in pairs: 5
// instructions for 4 codes; bfloat16 takes 6, through float32.
template <class E>
__device__ __forceinline__ Frag<E> codes_to(uint32_t lo, uint32_t hi) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w = i ? hi : lo;
    if constexpr (std::is_same<E, bf16>::value) {
      const int v = (int)w;
      const float f0 = (float)(int8_t)v, f1 = (float)(int8_t)(v >> 8), f2 = (float)(int8_t)(v >> 16), f3 = (float)(v >> 24);
      r[2 * i] = __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302);
      r[2 * i + 1] = __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x07060302);
    } else {
      typedef f16 f16x2 __attribute__((ext_vector_type(2)));
      const f16x2 less = {1152.f, 1152.f};
      const uint32_t above = w ^ 0x80808080u;
      const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, above, 0x04010400)) - less;
      const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, above, 0x04030402)) - less;
      r[2 * i] = __builtin_bit_cast(uint32_t, a);
      r[2 * i + 1] = __builtin_bit_cast(uint32_t, b);
    }
  }
  Frag<E> f;
  __builtin_memcpy(&f, &r, 16);
  return f;
}

// The four lanes that hold a row (l, l ^ 16, l ^ 32, l ^ 48) agree.
template <class F>
__device__ __forceinline__ float rows_reduce(float v, F op) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// A weight times its value's scale is three bfloat16 operands of the second product, eight bits each, that add up to
// it exactly and reach as far as float32 does: no slot's value, seen or not, changes how exact another's is.  (Two float16
// operands, 2^-23 of a power of two that all slots share, lose values 2^-24 as large as another slot's.)

// A row's weights are relative to a logit that a tile leaves alone while 16 slots' weights add up to kMostWeight at
// most (the largest is only looked for when they do not).  Scales are multiplied by kDown: 2^32 slots' weights (2 each at
// most, by the sixteen) times values at float32's end stay below it, and of the smallest scale that is held, 2^-67, the last
// operand's bits are above 2^-126.
constexpr float kMostWeight = 32.f;
constexpr float kDown = 0x1p-34f, kUp = 0x1p34f;

// Beyond this a logit's last place is more than the weights' own errors: there logits are rounded before the
// reference is taken off, so that equal ones stay equal (one instruction more a logit).
constexpr float kFar = 0x1p16f;

// A wave's rows: 16 to a matrix instruction's columns, R of those.  Lane l = 16 g + n has row n; of 64
// slots the logits of 16 t + 4 g + i (t, i < 4), which are the second product's operand as they
// stand, and of the result channels 16 c + 4 g + i.
template <class T, int DP, int R>
struct Rows {
  static constexpr int KF = DP / 32, CT = DP / 16, QT = Operand<T>::kTerms;
  Frag<typename Operand<T>::E> q[R][QT][KF];
  f32x4 o[R][CT];
  // the logit that weights are relative to, how much the weights of 16 slots may add up to before it moves (-1:
  // nothing seen yet), and the sum of the weights of the lane's slots
  float ref[R], most[R], l[R];
  int count[R];  // slots that the row sees, but for the mask
};

// 64 slots' codes as a wave holds them.
template <int DP>
struct Codes {
  static constexpr int K16 = DP / 64, K8 = DP % 64 / 32;
  u32x4 k[4][K16 ? K16 : 1];
  u32x2 k8[4];
};

// Units of one key head and part lie next to each other and read the same slots: kTogether of them run on one
// XCD, then the next XCD's turn comes, so that heads of different lengths are spread over all.
constexpr int kTogether = 4;
__device__ __forceinline__ int unit_of_block(int block, int blocks) {
  constexpr int kXcds = 8;
  if (block >= blocks / (kXcds * kTogether) * (kXcds * kTogether)) return block;
  const int xcd = block % kXcds, at = block / kXcds;
  return (at / kTogether * kXcds + xcd) * kTogether + at % kTogether;
}

// First dimension of the eight that fragment s takes in lane group g: 16 bytes a lane in whole 64s, 8 in what is left.
template <int DP>
__device__ __forceinline__ int dims_at(int s, int g) {
  return s < DP / 64 * 2 ? s / 2 * 64 + 16 * g + s % 2 * 8 : DP / 64 * 64 + 8 * g;
}

// softmax(scale q . k) v of 16 R rows over a part of an item's slots: the four waves take tiles of 64 slots in turn, each
// on its own with a running softmax, and join their results in the end; a tile's codes go from memory to the lanes that
// multiply them, the next tile's are on their way meanwhile.
//
// Few rows are bound by memory: one query of 32 heads over 131072 slots of 4 heads of 128, 138 MB, takes 39 us with the
// join (3.6 TB/s), 4 queries of 16 heads, twice 16 rows a key head that read the same slots through the L2, 53 us for 156 MB.
// Many are bound by vector instructions, of which 64 slots by 32 rows of 64 take 645 (conversions of codes 192, weights
// cut into operands 176, logits to weights 128, of them 32 exponentials at a quarter of the rate, the rest addresses, scales
// and sums) beside 64 matrix instructions: 4096 queries of 5 heads over 32768 slots take 468 us with the join, 370 TFLOP/s,
// the vector units busy for 85% and the matrix units for 29% of it.  32 rows a wave share conversions (16 rows: 558).
// With one operand a weight, 372 us then: 64 rows leave one wave a SIMD (785), three waves a SIMD spill (443); operands
// converted once for four waves' rows and passed through LDS, with a barrier a tile, were slower (355 against 349).
template <class T, int DP, int R>
__global__ __launch_bounds__(256, 2) void held_kernel(HeldAttention h) {
  using Q = Operand<T>;
  using E = typename Q::E;
  using Row = Rows<T, DP, R>;
  constexpr int KF = Row::KF, CT = Row::CT;
  __shared__ __attribute__((aligned(16))) f32x4 exchange[2][R * CT][64];
  __shared__ float exchange_ml[2][2 * R][64];
  __shared__ __attribute__((aligned(16))) float slot_scales[4][128];
  const HeldArgs& a = h.a;
  const int lane = threadIdx.x % 64, n16 = lane % 16, g = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int unit = unit_of_block(blockIdx.x, gridDim.x);
  const int rest = unit / h.tiles, split = rest % h.splits, bg = rest / h.splits;
  const int tile = h.tiles - 1 - (unit - rest * h.tiles);  // causal rows: those that see most first
  const int b = bg / a.kv_heads, kh = bg - b * a.kv_heads;
  const int64_t item = bg;

  const int held = min(max(a.lengths ? a.lengths[b] : a.keys, 0), a.keys);
  const int64_t at0 = a.start0 + (a.start ? a.start[b] : 0) + 1;
  const int row0 = tile * 16 * R;
  auto sees = [&](int row) {
    return a.causal ? (int)min(max(at0 + row / h.group, (int64_t)0), (int64_t)held) : held;
  };
  const int least = sees(row0), most = sees(min(row0 + 16 * R, h.rows) - 1);

  Row w;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = row0 + 16 * r + n16;
    const bool live = row < h.rows;
    const int t = live ? row / h.group : 0, hd = live ? row - t * h.group : 0;
    const T* q = (const T*)h.q + b * a.s[0][0] + t * a.s[0][1] + (int64_t)(kh * h.group + hd) * a.s[0][2];
#pragma unroll
    for (int s = 0; s < KF; ++s) {
      const int d = dims_at<DP>(s, g);
      Vec<T, 8> x{};
      if (live && d < a.dim) x = load_vec<8>(q + d);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = to_float(x.v[e]) * h.query;
        // an infinite element makes its row NaN whatever the signs of its products: logits that are all -inf would
        // look like slots that are not seen
        if (!(fabsf(y[e]) < INFINITY)) y[e] = NAN;
      }
      if constexpr (Q::kTerms == 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w.q[r][0][s][e] = from_float<E>(y[e]);
      } else {
        Frag<bf16> parts[3];
        cut_in_three<false>(y, parts);
#pragma unroll
        for (int term = 0; term < 3; ++term) w.q[r][term][s] = parts[term];
      }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) w.o[r][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    w.ref[r] = 0.f, w.most[r] = -1.f, w.l[r] = 0.f;
    w.count[r] = live ? sees(row) : held;  // rows past the last see what there is, like others
  }

  const int all = (most + 63) / 64;
  const int j0 = (int)((int64_t)all * split / h.splits), j1 = (int)((int64_t)all * (split + 1) / h.splits);
  const int8_t* kc = h.k_codes + item * a.slots * a.dim;
  const int8_t* vc = h.v_codes + item * a.slots * a.dim;
  const float* ks = h.k_scales + item * a.slots;
  const float* vs = h.v_scales + item * a.slots;
  const uint8_t* mask = a.mask ? a.mask + b * a.ms : nullptr;
  // Offsets of the lane in a tile of 64 slots, whose start is the wave's own.  Past the end of a row of keys: any
  // codes, the query is zero there; of values: results that are not stored.
  uint32_t key_at[Codes<DP>::K16 + 1];
#pragma unroll
  for (int s = 0; s <= Codes<DP>::K16; ++s) {
    const int d = s < Codes<DP>::K16 ? 64 * s + 16 * g : DP / 64 * 64 + 8 * g;
    key_at[s] = n16 * a.dim + (d < a.dim ? d : 0);
  }
  const uint32_t value_at = n16 * 64 + 16 * g;
  const int last_channels = a.dim / 16 - 1;
  // scales a lane a slot, spread to the lanes that need them through LDS
  float* scales = slot_scales[wave];
  Codes<DP> keys;
  u32x4 values[CT];
  float key_scale, value_scale;
  // without a mask any byte is loaded and none looked at: a load under a condition would be waited for at once
  const uint8_t* marks = mask ? mask : (const uint8_t*)ks;
  const int last_mark = mask ? a.keys - 1 : 0;
  uint8_t mark;
  auto load_keys = [&](int j) {
    const int8_t* at = kc + (int64_t)j * 64 * a.dim;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int s = 0; s < Codes<DP>::K16; ++s)
        keys.k[t][s] = *(const u32x4*)__builtin_assume_aligned(at + 16 * t * a.dim + key_at[s], 16);
      if constexpr (Codes<DP>::K8 != 0)
        keys.k8[t] = *(const u32x2*)__builtin_assume_aligned(at + 16 * t * a.dim + key_at[Codes<DP>::K16], 8);
    }
    key_scale = ks[(int64_t)j * 64 + lane];
    value_scale = vs[(int64_t)j * 64 + lane];
    mark = marks[min(64 * j + lane, last_mark)];
  };
  auto load_values = [&](int j) {
    const int8_t* at = vc + (int64_t)j * 64 * a.dim;
#pragma unroll
    for (int c = 0; c < CT; ++c)
      values[c] = *(const u32x4*)__builtin_assume_aligned(at + min(c, last_channels) * 1024 + value_at, 16);
  };

  bool far = false;     // some row's reference is further from 0 than kFar
  const auto larger = [](float u, float v) { return fmaxf(u, v); };
  int j = j0 + wave;
  if (j < j1) {
    load_keys(j);
    load_values(j);
  }
  for (; j < j1; j += 4) {
    // which of the 64 slots are seen, but for each row's own end
    const bool shown = (!mask || mark) && 64 * j + lane < most;
    const uint64_t seen = __ballot(shown);
    const bool whole = seen == ~0ull && 64 * (j + 1) <= least;
    wave_sync();
    scales[lane] = key_scale * h.c2;
    scales[64 + lane] = value_scale * kDown;
    wave_sync();
    f32x4 x[R][4];  // logits in units of log 2, relative to the row's reference
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      // A matrix instruction's sum loses up to a last place: what the lower operands add is small, and has sums of its own.
      f32x4 rest[R];
#pragma unroll
      for (int r = 0; r < R; ++r) x[r][t] = rest[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KF; ++s) {
        Frag<E> k;
        if (s < Codes<DP>::K16 * 2) {
          k = codes_to<E>(keys.k[t][s / 2][s % 2 * 2], keys.k[t][s / 2][s % 2 * 2 + 1]);
        } else {
          k = codes_to<E>(keys.k8[t][0], keys.k8[t][1]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          x[r][t] = mfma(k, w.q[r][0][s], x[r][t]);
#pragma unroll
          for (int term = 1; term < Q::kTerms; ++term) rest[r] = mfma(k, w.q[r][term][s], rest[r]);
        }
      }
      if constexpr (Q::kTerms > 1) {
#pragma unroll
        for (int r = 0; r < R; ++r) x[r][t] += rest[r];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_keys(min(j + 4, j1 - 1));  // the last again: no branch, which would double the registers
    if (!far) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 by = *(const f32x4*)__builtin_assume_aligned(scales + 16 * t + 4 * g, 16);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[r][t][i] = fmaf(x[r][t][i], by[i], -w.ref[r]);
      }
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 by = *(const f32x4*)__builtin_assume_aligned(scales + 16 * t + 4 * g, 16);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float rounded = x[r][t][i] * by[i] - w.ref[r];
            x[r][t][i] = fabsf(w.ref[r]) > kFar ? rounded : fmaf(x[r][t][i], by[i], -w.ref[r]);
          }
      }
    }
    // of the lane's four slots from 16 t + 4 g on, those that the row sees
    const auto row_sees = [&](int r, int t) {
      const int first = 16 * t + 4 * g, end = min(max(w.count[r] - 64 * j - first, 0), 4);
      return (uint32_t)(seen >> first) & ((1u << end) - 1);
    };
    if (!whole) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t bits = row_sees(r, t);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[r][t][i] = bits & (1u << i) ? x[r][t][i] : -INFINITY;
        }
    }
    f32x4 e[R][4];  // weights, then times their values' scales
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const auto weights = [&] {
        f32x4 sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[r][t][i] = __builtin_amdgcn_exp2f(x[r][t][i]);
            sum[i] += e[r][t][i];
          }
        return (sum[0] + sum[1]) + (sum[2] + sum[3]);
      };
      float sum = weights();
      if (__any(sum > w.most[r])) {
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, x[r][t][i]);
        top = rows_reduce(top, larger);
        // by the row's own weights: what other rows do does not show
        const bool first = w.most[r] < 0.f;
        const bool moves = rows_reduce(sum, larger) > w.most[r] && top > (first ? -INFINITY : 0.f);
        const float next = moves ? w.ref[r] + top : w.ref[r], by = next - w.ref[r];
        const float back = first ? 1.f : __builtin_amdgcn_exp2f(-by);
        w.l[r] *= back;
#pragma unroll
        for (int c = 0; c < CT; ++c) w.o[r][c] *= back;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[r][t][i] -= by;
        w.ref[r] = next;
        far |= __any(fabsf(next) > kFar);
        w.most[r] = moves ? kMostWeight : w.most[r];
        sum = weights();
      }
      w.l[r] += sum;
#pragma unroll
      for (int t = 0; t < 4; ++t) e[r][t] *= *(const f32x4*)__builtin_assume_aligned(scales + 64 + 16 * t + 4 * g, 16);
    }
    if (!whole) {  // a weight of 0 keeps out no value that is not a number
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t bits = row_sees(r, t);
#pragma unroll
          for (int i = 0; i < 4; ++i) e[r][t][i] = bits & (1u << i) ? e[r][t][i] : 0.f;
        }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      Frag<bf16> p[R][3];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = e[r][2 * u][i], y[4 + i] = e[r][2 * u + 1][i];
        cut_in_three<false>(y, p[r]);
      }
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const Frag<bf16> v = codes_to<bf16>(values[c][2 * u], values[c][2 * u + 1]);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int term = 0; term < 3; ++term) w.o[r][c] = mfma(v, p[r][term], w.o[r][c]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_values(min(j + 4, j1 - 1));
  }
  // the row's own result over its slots, with (reference, sum of weights) to join it by
  float m[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    w.l[r] = rows_reduce(w.l[r], [](float u, float v) { return u + v; });
    m[r] = w.most[r] < 0.f ? -INFINITY : w.ref[r];
    const float whole = w.l[r] == 0.f ? 0.f : 1.f / w.l[r];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) w.o[r][c][i] = w.o[r][c][i] * whole * kUp;
  }

  // waves 2 and 3 into 0 and 1, then 1 into 0; lanes hold the same places
#pragma unroll
  for (int step = 2; step >= 1; step /= 2) {
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        exchange_ml[wave - step][2 * r][lane] = m[r];
        exchange_ml[wave - step][2 * r + 1][lane] = w.l[r];
#pragma unroll
        for (int c = 0; c < CT; ++c) exchange[wave - step][r * CT + c][lane] = w.o[r][c];
      }
    }
    __syncthreads();
    if (wave < step) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float m1 = exchange_ml[wave][2 * r][lane], l1 = exchange_ml[wave][2 * r + 1][lane], top = fmaxf(m1, m[r]);
        // nothing seen: a sum of 0, or of NaN logits
        const float mine = m[r] == -INFINITY ? w.l[r] : w.l[r] * __builtin_amdgcn_exp2f(m[r] - top);
        const float theirs = m1 == -INFINITY ? l1 : l1 * __builtin_amdgcn_exp2f(m1 - top);
        const float l = mine + theirs, share = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int c = 0; c < CT; ++c)
          w.o[r][c] = w.o[r][c] * (mine * share) + exchange[wave][r * CT + c][lane] * (theirs * share);
        m[r] = top, w.l[r] = l;
      }
    }
    __syncthreads();
  }
  if (wave) return;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = row0 + 16 * r + n16;
    if (row >= h.rows) continue;
    if (h.splits == 1) {
      const int t = row / h.group, hd = row - t * h.group;
      T* out = (T*)h.out + b * a.s[1][0] + t * a.s[1][1] + (int64_t)(kh * h.group + hd) * a.s[1][2];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        if (16 * c >= a.dim) break;
        Vec<T, 4> y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.v[i] = from_float<T>(w.o[r][c][i]);
        store_vec(out + 16 * c + 4 * g, y);
      }
    } else {
      const int64_t at = ((int64_t)bg * h.rows + row) * h.splits + split;
#pragma unroll
      for (int c = 0; c < CT; ++c)
        if (16 * c < a.dim) *(f32x4*)__builtin_assume_aligned(h.part + at * a.dim + 16 * c + 4 * g, 16) = w.o[r][c];
      if (g == 0) h.meta[at] = make_float2(m[r], w.l[r]);
    }
  }
}

template <class T, int DP, int R>
void held_launch(const HeldAttention& h, const HeldPlan& p, hipStream_t st) {
  held_kernel<T, DP, R><<<(unsigned)(p.units * p.splits), 256, 0, st>>>(h);
  launch_check("held_attention");
}

template <class T>
void held_units(const HeldAttention& h, const HeldPlan& p, hipStream_t st) {
  using std::integral_constant;
  auto rows = [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    if constexpr (held_pairs(std::is_same<T, float>::value, DP)) {
      if (p.r == 2) return held_launch<T, DP, 2>(h, p, st);
    }
    held_launch<T, DP, 1>(h, p, st);
  };
  if (h.a.dim <= 32) return rows(integral_constant<int, 32>{});
  if (h.a.dim <= 64) return rows(integral_constant<int, 64>{});
  if (h.a.dim <= 96) return rows(integral_constant<int, 96>{});
  rows(integral_constant<int, 128>{});
}

}  // namespace
}  // namespace nnx
