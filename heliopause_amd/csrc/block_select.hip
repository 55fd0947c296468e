// block_select.hip -- which blocks of a long context a token's queries attend to.
//
// Bounds.  Of each block of positions and KV head the least and largest element
// of its keys, lo_d and hi_d, rounded outward to bf16.  For any key k of the
// block q . k <= sum_d max(q_d lo_d, q_d hi_d), the block's score for q; a KV
// head's query heads share their blocks, so a block counts with the largest of
// their scores.  Bounds are bytes: 4 D of a block that itself has 2 e D B.
//
// Score.  Products of a query element with a bf16 bound and their sums are 64
// bits: the vector unit runs f64 at its f32 rate, and the order of two blocks
// then does not depend on how the sum was taken (f32 sums put one block in a
// million on the wrong side of its neighbour).  q is split into its positive and
// its negative part, so that a term is two fused products of which one adds 0.
// A score becomes a 64-bit key that sorts the same way.
//
// Pick.  One workgroup per (sequence, KV head), the keys in its registers where
// they fit: the digits of the budget-th largest key, 8 bits at a time below the
// bits that all keys share, by counting in LDS, until 64 or fewer are left, which
// a wave ranks; then the blocks above it, and of those equal to it the first
// ones, in their order.
//
// Not kept: scores by the matrix cores in parts of bf16 (10.5 us for 12.0 on 24
// contexts, 12.8 for 14.4 on two of 262144), with the blocks that their error
// leaves open scored in 64 bits by the pick, which then took 12.4 and 18.9 us for
// 7.2 and 10.8.
#include "hp_mfma.h"
#include "hp_serving.h"
#include "hp_wave.h"

namespace hp {

namespace {

constexpr float kBf16Most = 3.38953138925153547590e38f;
constexpr float kF32Most = 3.40282346638528860e38f;
constexpr float kInf = __builtin_inff();

// x in bf16, the nearest value that is not below it (UP) or not above; NaN (a
// key that is one could score anything) and what is past the type the largest.
template <bool UP>
__device__ __forceinline__ uint16_t outward(float x) {
  x = x != x ? (UP ? kBf16Most : -kBf16Most) : fminf(fmaxf(x, -kBf16Most), kBf16Most);
  const uint32_t bits = __builtin_bit_cast(uint32_t, x);
  const bool away = UP ? x > 0.0f : x < 0.0f;  // (zero is exact)
  return (uint16_t)((bits + (away ? 0xffffu : 0u)) >> 16);
}

// 16 bytes of a row a lane.  The least and largest are f16's in pairs, two rows
// an instruction (v_pk_minimum3_f16), which keep a NaN: f16 keys as they are, e4m3
// as the halves that they are, i8 as the halves 1152 + q, whose order is theirs;
// bf16 as f32.  Few blocks: a workgroup has a (touched block, KV head), all of its
// loads on their way at once, and the waves' parts are joined in LDS.  Many: a wave
// has it.  (One block of 64 rows, 2 heads of 256, f16: 3.5 us, with a wave each 7.2;
// 100000 rows in blocks of 32, e4m3: 57 MB in 12.8 us, with a workgroup each 36.)
template <int CT>
struct Extremes {
  using V = half2v;
  static constexpr int kPer = 16 / elem_bytes(CT), kN = kPer / 2;  // elements of a lane, registers
  static __device__ __forceinline__ V most(bool up) {
    const _Float16 v = (_Float16)(up ? -kInf : kInf);
    return V{v, v};
  }
  static __device__ __forceinline__ void of(const uint4 &w, V (&v)[kN]) {
    const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (CT == kElemF16) {
        v[i] = as_h2(d[i]);
      } else if (CT == kElemI8) {
        v[2 * i % kN] = magic_pair<kSel01>(d[i] ^ 0x80808080u);
        v[(2 * i + 1) % kN] = magic_pair<kSel23>(d[i] ^ 0x80808080u);
      } else {
        v[2 * i % kN] = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d[i], 1.0f, false));
        v[(2 * i + 1) % kN] = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(d[i], 1.0f, true));
      }
    }
  }
  static __device__ __forceinline__ float value(const V (&v)[kN], int j) {
    return (float)v[j / 2][j & 1] - (CT == kElemI8 ? 1152.0f : 0.0f);
  }
};
template <>
struct Extremes<kElemBf16> {
  using V = float;
  static constexpr int kPer = 8, kN = 8;
  static __device__ __forceinline__ V most(bool up) { return up ? -kInf : kInf; }
  static __device__ __forceinline__ void of(const uint4 &w, V (&v)[kN]) {
    const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[2 * i] = bf16_value(d[i] & 0xffffu);
      v[2 * i + 1] = __builtin_bit_cast(float, d[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float value(const V (&v)[kN], int j) { return v[j]; }
};

template <int D, int CT, int WAVES>
__global__ __launch_bounds__(256) void block_bounds_kernel(const BlockBoundsArgs a, int units) {
  using E = Extremes<CT>;
  using V = typename E::V;
  constexpr int kE = elem_bytes(CT), kPer = E::kPer, kN = E::kN, kLanes = D / kPer, kRows = 64 / kLanes * WAVES;
  constexpr int kDeep = WAVES == 1 ? 8 : 4;  // loads of a lane at a time
  __shared__ V sh[WAVES == 1 ? 1 : 2][WAVES][WAVES == 1 ? 1 : kLanes][kN];
  const int tid = threadIdx.x % (64 * WAVES), lane = threadIdx.x & 63, wave = WAVES == 1 ? 0 : threadIdx.x >> 6;
  const int unit = WAVES == 1 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (unit >= units) return;
  const int h = unit % a.c.nkv, slot = unit / a.c.nkv;
  int seq = slot;
  NewInBlock n;
  const int64_t table_keys = (int64_t)a.c.width << a.c.page_shift;
  if (a.offsets) {
    seq = touched_sequence(a.offsets, a.c.sequences, slot, 1 << a.b.shift);
    const int begin = a.offsets[seq];
    n = new_in_block(a.c.lengths[seq], (int64_t)a.offsets[seq + 1] - begin,
                     slot - touched_first(begin, seq, 1 << a.b.shift), a.b.shift, table_keys);
  } else {
    n = new_in_block(a.c.lengths[seq], 1, 0, a.b.shift, table_keys);
  }
  if (n.end <= n.first) return;  // (the same for the unit's waves)
  const int page = page_or_none(a.c.pages[(int64_t)seq * a.c.width + (n.first >> a.c.page_shift)], a.c.page_count);
  if (page < 0) return;
  const int in_page = n.block & ((1 << (a.c.page_shift - a.b.shift)) - 1), live = n.end - (n.block << a.b.shift);
  const int64_t block_at = (((int64_t)page * a.c.nkv + h) << (a.c.page_shift - a.b.shift)) + in_page;
  const uint8_t *rows = static_cast<const uint8_t *>(a.c.keys) +
                        (page * a.c.page_stride + (((int64_t)h << a.c.page_shift) + ((int64_t)in_page << a.b.shift)) * D) * kE;
  const float scale = a.b.key_scales ? a.b.key_scales[block_at] : CT == kElemE4m3 ? a.c.key_scale : 1.0f;
  const int col = lane % kLanes, sub = tid / kLanes;
  V lo[kN], hi[kN];
#pragma unroll
  for (int i = 0; i < kN; i++) lo[i] = E::most(false), hi[i] = E::most(true);
  for (int r0 = 0; r0 < live; r0 += kRows * kDeep) {
    uint4 w[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; i++) {  // (behind the last row: the last one's again)
      const int r = min(r0 + i * kRows + sub, live - 1);
      w[i] = *reinterpret_cast<const uint4 *>(rows + ((int64_t)r * D + col * kPer) * kE);
    }
#pragma unroll
    for (int i = 0; i < kDeep; i += 2) {
      V u[kN], v[kN];
      E::of(w[i], u);
      E::of(w[i + 1], v);
#pragma unroll
      for (int j = 0; j < kN; j++) {
        lo[j] = __builtin_elementwise_minimum(__builtin_elementwise_minimum(lo[j], u[j]), v[j]);
        hi[j] = __builtin_elementwise_maximum(__builtin_elementwise_maximum(hi[j], u[j]), v[j]);
      }
    }
  }
#pragma unroll
  for (int m = kLanes; m < 64; m *= 2) {
#pragma unroll
    for (int j = 0; j < kN; j++) {
      const int x = __builtin_bit_cast(int, lo[j]), y = __builtin_bit_cast(int, hi[j]);
      lo[j] = __builtin_elementwise_minimum(lo[j], __builtin_bit_cast(V, __shfl_xor(x, m)));
      hi[j] = __builtin_elementwise_maximum(hi[j], __builtin_bit_cast(V, __shfl_xor(y, m)));
    }
  }
  if (WAVES > 1) {
    if (lane < kLanes) {
#pragma unroll
      for (int j = 0; j < kN; j++) {
        sh[0][wave][lane % kLanes][j] = lo[j];
        sh[WAVES == 1 ? 0 : 1][wave][lane % kLanes][j] = hi[j];
      }
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; w++)
#pragma unroll
      for (int j = 0; j < kN; j++) {
        lo[j] = __builtin_elementwise_minimum(lo[j], sh[0][w][col][j]);
        hi[j] = __builtin_elementwise_maximum(hi[j], sh[WAVES == 1 ? 0 : 1][w][col][j]);
      }
  }
  if (lane >= kLanes) return;
  uint16_t *out = a.b.key_bounds + block_at * 2 * D + col * kPer;
#pragma unroll
  for (int j = 0; j < kPer; j += 8) {
    uint32_t l[4], u[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      l[i] = outward<false>(E::value(lo, j + 2 * i) * scale) | (uint32_t)outward<false>(E::value(lo, j + 2 * i + 1) * scale) << 16;
      u[i] = outward<true>(E::value(hi, j + 2 * i) * scale) | (uint32_t)outward<true>(E::value(hi, j + 2 * i + 1) * scale) << 16;
    }
    *reinterpret_cast<uint4 *>(out + j) = make_uint4(l[0], l[1], l[2], l[3]);
    *reinterpret_cast<uint4 *>(out + D + j) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

template <int D, int CT>
hipError_t launch_bounds(const BlockBoundsArgs &a, int slots, int num_cus, hipStream_t s) {
  const int units = slots * a.c.nkv;
  if (units <= 4 * num_cus)
    hipLaunchKernelGGL((block_bounds_kernel<D, CT, 4>), dim3(units), dim3(256), 0, s, a, units);
  else
    hipLaunchKernelGGL((block_bounds_kernel<D, CT, 1>), dim3((units + 3) / 4), dim3(256), 0, s, a, units);
  return hipGetLastError();
}

template <int D>
hipError_t launch_bounds_type(const BlockBoundsArgs &a, int slots, int num_cus, hipStream_t s) {
  switch (a.c.type) {
    case kElemF16: return launch_bounds<D, kElemF16>(a, slots, num_cus, s);
    case kElemBf16: return launch_bounds<D, kElemBf16>(a, slots, num_cus, s);
    case kElemE4m3: return launch_bounds<D, kElemE4m3>(a, slots, num_cus, s);
    case kElemI8: return launch_bounds<D, kElemI8>(a, slots, num_cus, s);
    default: return hipErrorInvalidValue;
  }
}

// ---- scores ------------------------------------------------------------------

constexpr int kScoreWaves = 4;

// Keys that sort as the scores do.  0: no block to take; all ones: a block that
// is taken whatever its score.
constexpr uint64_t kAlways = ~0ull;
__device__ __forceinline__ uint64_t key_of(double score) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, score + 0.0);  // (-0 is 0)
  return bits ^ ((int64_t)bits < 0 ? ~0ull : 1ull << 63);
}

__device__ __forceinline__ int table_blocks_of(const BlockSelectArgs &a) {
  return (int)(((int64_t)a.c.width << a.c.page_shift) >> a.b.shift);
}
__device__ __forceinline__ int blocks_of(const BlockSelectArgs &a, int length) {
  return length > 0 ? (int)min(((int64_t)length + (1 << a.b.shift) - 1) >> a.b.shift, (int64_t)table_blocks_of(a)) : 0;
}
// Bounds of block b of a sequence on `page` for KV head h.
__device__ __forceinline__ const uint16_t *bounds_of(const BlockSelectArgs &a, int page, int h, int b, int head_dim) {
  const int in_page = a.c.page_shift - a.b.shift;
  return a.b.key_bounds + ((((int64_t)page * a.c.nkv + h) << in_page) + (b & ((1 << in_page) - 1))) * 2 * head_dim;
}

// Eight elements of a query row from element i on: a NaN is 0, an infinity the
// largest number.
__device__ __forceinline__ void query_part(const BlockSelectArgs &a, int64_t i, float (&v)[8]) {
  if (a.q_type == kElemF32) {
    const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + i);
    const float4 x = p[0], y = p[1];
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
  } else {
    const uint4 x = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + i);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t b = w[j / 2] >> (16 * (j & 1)) & 0xffffu;
      v[j] = a.q_type == kElemF16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)b) : bf16_value(b);
    }
  }
  float odd = 0.0f;  // a NaN where an element is not finite
#pragma unroll
  for (int j = 0; j < 8; j++) odd += v[j] * 0.0f;
  if (odd != 0.0f) {  // (NaN)
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = v[j] != v[j] ? 0.0f : fminf(fmaxf(v[j], -kF32Most), kF32Most);
  }
}

// A permutation of each 16-lane row that has a source for every lane.
template <int CTRL>
__device__ __forceinline__ uint32_t permuted(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ double permuted(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)permuted<CTRL>((uint32_t)(b >> 32)) << 32 | permuted<CTRL>((uint32_t)b));
}
constexpr int kDppRor4 = 0x124, kDppReverse = 0x1B;  // quad_perm [3,2,1,0]

// Of two sums of every lane, x's over the lane and its partner in the lanes whose
// bit of `odd` is clear, y's in the others.
template <int CTRL>
__device__ __forceinline__ double joined(double x, double y, bool odd) {
  const double keep = odd ? y : x, send = odd ? x : y;
  return keep + permuted<CTRL>(send);
}

// Largest of the HEADS sums over the L lanes of a row (8, 16 or 32).  The lanes
// first share the sums out, so that each step has half as many.
template <int L, int HEADS>
__device__ __forceinline__ double largest_sum(const double (&v)[HEADS], int lane) {
  double s;
  if (HEADS == 4) {
    s = joined<kDppXor2>(joined<kDppXor1>(v[0], v[1 % HEADS], lane & 1), joined<kDppXor1>(v[2 % HEADS], v[3 % HEADS], lane & 1), lane & 2);
  } else {
    s = HEADS == 2 ? joined<kDppXor1>(v[0], v[1 % HEADS], lane & 1) : v[0] + permuted<kDppXor1>(v[0]);
    s += permuted<kDppXor2>(s);
  }
  if (L == 8) {
    s += permuted<kDppReverse>(permuted<kDppRowHalfMirror>(s));  // lane ^ 4
  } else {
    s += permuted<kDppRor8>(s);
    s += permuted<kDppRor4>(s);
    if (L == 32) s += __shfl_xor(s, 16);
  }
  if (HEADS >= 2) s = fmax(s, permuted<kDppXor1>(s));
  if (HEADS == 4) s = fmax(s, permuted<kDppXor2>(s));
  return s;
}

// D / 8 lanes have a block's bounds, 8 elements each, and HEADS of the group's
// queries at a time; a workgroup has `per` blocks of a (sequence, KV head).  The
// next block's bounds are on their way while one is worked on, and the table's
// entry of the one after it (four turns ahead: the same or slower).
template <int D, int HEADS>
__global__ __launch_bounds__(64 * kScoreWaves) void block_score_kernel(const BlockSelectArgs a, uint64_t *__restrict__ keys,
                                                                       int per, int chunks) {
  constexpr int kLanes = D / 8, kRows = 64 / kLanes, kStep = kScoreWaves * kRows;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % kLanes, sub = lane / kLanes;
  const int row = blockIdx.x / chunks, seq = row / a.c.nkv, h = row - seq * a.c.nkv;
  const int group = a.nq / a.c.nkv, in_page = a.c.page_shift - a.b.shift;
  const int64_t q0 = seq * a.q_stride + (int64_t)h * group * D + 8 * l;
  const int *table = a.c.pages + (int64_t)seq * a.c.width;
  const int blocks = blocks_of(a, a.c.lengths[seq]);
  const int begin = blockIdx.x % chunks * per + wave * kRows, end = min((int)(blockIdx.x % chunks) * per + per, blocks), last = end - 1;
  if (begin >= end) return;
  for (int g0 = 0; g0 < group; g0 += HEADS) {
    int entry = table[min(begin + sub, last) >> in_page], entry_next = table[min(begin + sub + kStep, last) >> in_page];
    double up[HEADS][8], down[HEADS][8];
#pragma unroll
    for (int g = 0; g < HEADS; g++) {  // (a head beyond the group: the last one's again)
      float q[8];
      query_part(a, q0 + (int64_t)min(g0 + g, group - 1) * D, q);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        up[g][j] = fmaxf(q[j], 0.0f);
        down[g][j] = fminf(q[j], 0.0f);
      }
    }
    const uint16_t *bound = bounds_of(a, max(page_or_none(entry, a.c.page_count), 0), h, min(begin + sub, last), D) + 8 * l;
    uint4 lo = *reinterpret_cast<const uint4 *>(bound), hi = *reinterpret_cast<const uint4 *>(bound + D);
    for (int b0 = begin; b0 < end; b0 += kStep) {
      const int b = b0 + sub;
      const bool absent = page_or_none(entry, a.c.page_count) < 0;
      const uint32_t low[4] = {lo.x, lo.y, lo.z, lo.w}, high[4] = {hi.x, hi.y, hi.z, hi.w};
      bound = bounds_of(a, max(page_or_none(entry_next, a.c.page_count), 0), h, min(b + kStep, last), D) + 8 * l;
      entry = entry_next;
      entry_next = table[min(b + 2 * kStep, last) >> in_page];
      lo = *reinterpret_cast<const uint4 *>(bound);
      hi = *reinterpret_cast<const uint4 *>(bound + D);
      double sum[HEADS];
#pragma unroll
      for (int g = 0; g < HEADS; g++) sum[g] = 0.0;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const double x = (double)bf16_value(low[j / 2] >> (16 * (j & 1)) & 0xffffu);
        const double y = (double)bf16_value(high[j / 2] >> (16 * (j & 1)) & 0xffffu);
#pragma unroll
        for (int g = 0; g < HEADS; g++) sum[g] = fma(up[g][j], y, fma(down[g][j], x, sum[g]));
      }
      const double best = largest_sum<kLanes>(sum, lane);
      if (l != 0 || b >= end) continue;
      uint64_t *key = keys + (int64_t)row * table_blocks_of(a) + b;
      uint64_t k = key_of(best);
      if (g0 > 0) k = max(k, *key);  // (this lane's own of the heads before)
      if (b < a.first_blocks || b >= blocks - a.last_blocks) k = kAlways;
      *key = absent ? 0 : k;
    }
  }
}

// ---- pick --------------------------------------------------------------------

constexpr int kPickKeys = 8;     // of a thread, in registers where these are enough
template <int NT>
constexpr int digit_bits() {  // (so that one digit mostly leaves few enough)
  return NT > 256 ? 11 : 8;
}
constexpr int kPickAtOnce = 64;  // keys that one wave ranks by comparing all with all

__device__ __forceinline__ uint64_t lane_key(uint64_t k, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, lane);
}

// A row's keys in a workgroup's sweeps: in registers (HELD, up to NT * kPickKeys),
// or read in each.
template <int NT, bool HELD>
struct Keys {
  const uint64_t *key;
  int n;
  uint64_t held[HELD ? kPickKeys : 1];
  __device__ __forceinline__ Keys(const uint64_t *k, int count) : key(k), n(count) {
    if (HELD) {
#pragma unroll
      for (int j = 0; j < kPickKeys; j++) held[j % (HELD ? kPickKeys : 1)] = j * NT + (int)threadIdx.x < n ? key[j * NT + threadIdx.x] : 0;
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {  // f(key, place); behind the last: a key of 0
    if (HELD) {
#pragma unroll
      for (int j = 0; j < kPickKeys; j++)
        if (j * NT < n) f(held[j % (HELD ? kPickKeys : 1)], j * NT + (int)threadIdx.x);
    } else {
      for (int i = threadIdx.x; i < n; i += NT) f(key[i], i);
    }
  }
};

// What the sweeps of a workgroup share.
template <int NT>
struct PickShared {
  static constexpr int kWaves = NT / 64;
  static constexpr int kBins = 1 << digit_bits<NT>(), kEach = kBins / NT;  // of a thread
  uint64_t any[kWaves], all[kWaves], key[kPickAtOnce], least;
  int first[kWaves], second[kWaves], bins[kBins], at[kPickAtOnce], counts[kPickKeys * kWaves + 1];
  int digit, need, in, last, found;
};

// The bits that some, and that all, of a wave's lanes have.
template <int CTRL>
__device__ __forceinline__ void join_bits(uint32_t (&any)[2], uint32_t (&all)[2]) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
    any[i] |= permuted<CTRL>(any[i]);
    all[i] &= permuted<CTRL>(all[i]);
  }
}
__device__ __forceinline__ void wave_bits(uint64_t &some, uint64_t &every) {
  uint32_t any[2] = {(uint32_t)some, (uint32_t)(some >> 32)}, all[2] = {(uint32_t)every, (uint32_t)(every >> 32)};
  join_bits<kDppXor1>(any, all);
  join_bits<kDppXor2>(any, all);
  join_bits<kDppRowHalfMirror>(any, all);
  join_bits<kDppRowMirror>(any, all);
  uint32_t o[2], a[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    auto lane = [](uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
    o[i] = lane(any[i], 0) | lane(any[i], 16) | lane(any[i], 32) | lane(any[i], 48);
    a[i] = lane(all[i], 0) & lane(all[i], 16) & lane(all[i], 32) & lane(all[i], 48);
  }
  some = (uint64_t)o[1] << 32 | o[0];
  every = (uint64_t)a[1] << 32 | a[0];
}

// The need-th of the keys other than 0 and kAlways in the order (larger key, lower
// place), of which there are `in` >= need >= 1 and which have the bits `all` and no
// others than `any`: its key and place.  Digits below the bits that all share,
// counted in LDS, until a wave can compare what is left.
template <int NT, bool HELD>
__device__ void nth_key(PickShared<NT> &sh, const Keys<NT, HELD> &keys, uint64_t any, uint64_t all, int in, int need,
                        uint64_t *at_key, int *at_place) {
  constexpr int kWaves = NT / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint64_t differ = any ^ all;
  int shift = differ ? 64 - __builtin_clzll(differ) : 0;  // they agree in the bits from here on
  uint64_t least = shift < 64 ? all >> shift << shift : 0;
  auto among = [&](uint64_t k) { return k != 0 && k != kAlways && (shift == 64 || k >> shift == least >> shift); };
  while (shift > 0 && in > kPickAtOnce) {
    using S = PickShared<NT>;
    const int low = max(shift - digit_bits<NT>(), 0), digits = (1 << (shift - low)) - 1;
    keys.each([&](uint64_t k, int) {
      if (among(k)) atomicAdd(&sh.bins[(int)(k >> low) & digits], 1);
    });
    __syncthreads();
    // from the largest digit down
    int c[S::kEach], sum = 0;
#pragma unroll
    for (int j = 0; j < S::kEach; j++) {
      sum += c[j] = sh.bins[S::kBins - 1 - S::kEach * tid - j];
      sh.bins[S::kBins - 1 - S::kEach * tid - j] = 0;
    }
    const int to = (int)wave_scan((uint32_t)sum);
    if (lane == 63) sh.first[wave] = to;
    __syncthreads();
    int before = to - sum;
#pragma unroll
    for (int w = 0; w < kWaves; w++) before += w < wave ? sh.first[w] : 0;
#pragma unroll
    for (int j = 0; j < S::kEach; j++) {
      if (before < need && need <= before + c[j]) {  // one thread's one digit
        sh.digit = S::kBins - 1 - S::kEach * tid - j;
        sh.need = need - before;
        sh.in = c[j];
      }
      before += c[j];
    }
    __syncthreads();
    least |= (uint64_t)sh.digit << low;
    need = sh.need;
    in = sh.in;
    shift = low;
  }
  if (in <= kPickAtOnce) {  // the rank of each: how many are ahead of it
    keys.each([&](uint64_t k, int i) {
      if (among(k)) {
        const int at = atomicAdd(&sh.found, 1);
        sh.key[at] = k;
        sh.at[at] = i;
      }
    });
    __syncthreads();
    if (wave == 0) {
      const uint64_t k = lane < in ? sh.key[lane] : 0;
      const int i = lane < in ? sh.at[lane] : 0x7fffffff;
      int ahead = 0;
      for (int j = 0; j < in; j++) {
        const uint64_t other = lane_key(k, j);
        ahead += other > k || (other == k && __builtin_amdgcn_readlane(i, j) < i);
      }
      if (lane < in && ahead == need - 1) {
        sh.least = k;
        sh.last = i;
      }
    }
  } else {  // all alike: the place of the need-th
    int seen = 0;
    for (int i0 = 0; i0 < keys.n && seen < need; i0 += NT) {
      const bool is = i0 + tid < keys.n && keys.key[i0 + tid] == least;
      const uint64_t mask = __ballot(is);
      __syncthreads();
      if (lane == 0) sh.first[wave] = __popcll(mask);
      __syncthreads();
      int rank = seen + __popcll(mask & ((1ull << lane) - 1));
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        rank += w < wave ? sh.first[w] : 0;
        seen += sh.first[w];
      }
      if (is && rank == need - 1) {
        sh.least = least;
        sh.last = i0 + tid;
      }
    }
  }
  __syncthreads();
  *at_key = sh.least;
  *at_place = sh.last;
}

// The places that `taken` says, in their order, and -1 behind them.
template <int NT, bool HELD, class Taken>
__device__ void put_places(PickShared<NT> &sh, const Keys<NT, HELD> &keys, Taken taken, int budget, int *__restrict__ out,
                           int *count) {
  constexpr int kWaves = NT / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int total = 0;
  if (HELD) {
    uint64_t masks[kPickKeys];
#pragma unroll
    for (int j = 0; j < kPickKeys; j++) {
      masks[j] = __ballot(j * NT + tid < keys.n && taken(keys.held[j % (HELD ? kPickKeys : 1)], j * NT + tid));
      if (lane == 0) sh.counts[j * kWaves + wave] = __popcll(masks[j]);
    }
    __syncthreads();
    if (wave == 0) {
      constexpr int kAll = kPickKeys * kWaves, kPer = (kAll + 63) / 64;
      int c[kPer], sum = 0;
#pragma unroll
      for (int j = 0; j < kPer; j++) sum += c[j] = lane * kPer + j < kAll ? sh.counts[lane * kPer + j] : 0;
      const int to = (int)wave_scan((uint32_t)sum);
      int before = to - sum;
#pragma unroll
      for (int j = 0; j < kPer; j++) {
        if (lane * kPer + j < kAll) sh.counts[lane * kPer + j] = before;
        before += c[j];
      }
      if (lane == 63) sh.counts[kAll] = to;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPickKeys; j++) {
      const int at = sh.counts[j * kWaves + wave] + __popcll(masks[j] & ((1ull << lane) - 1));
      if ((masks[j] >> lane & 1) != 0 && at < budget) out[at] = j * NT + tid;
    }
    total = sh.counts[kPickKeys * kWaves];
  } else {
    for (int i0 = 0; i0 < keys.n && total < budget; i0 += NT) {
      const bool is = i0 + tid < keys.n && taken(keys.key[i0 + tid], i0 + tid);
      const uint64_t mask = __ballot(is);
      __syncthreads();
      if (lane == 0) sh.first[wave] = __popcll(mask);
      __syncthreads();
      int at = total + __popcll(mask & ((1ull << lane) - 1));
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        at += w < wave ? sh.first[w] : 0;
        total += sh.first[w];
      }
      if (is && at < budget) out[at] = i0 + tid;
    }
  }
  total = min(total, budget);
  for (int i = total + tid; i < budget; i += NT) out[i] = -1;
  if (tid == 0 && count) *count = total;
}

// One (sequence, KV head).
template <int NT, bool HELD>
__device__ void pick(const BlockSelectArgs &a, const uint64_t *key, int n, int *out, int *count) {
  __shared__ PickShared<NT> sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Keys<NT, HELD> keys(key, n);
  // how many there are, and the bits in which the scored ones differ
  int live = 0, always = 0;  // (a wave's)
  uint64_t any = 0, all = ~0ull;
  keys.each([&](uint64_t k, int) {
    live += __popcll(__ballot(k != 0));
    always += __popcll(__ballot(k == kAlways));
    if (k != 0 && k != kAlways) {
      any |= k;
      all &= k;
    }
  });
  wave_bits(any, all);
  if (!HELD) {  // (the lanes of a sweep's end have not seen it)
    live = __builtin_amdgcn_readfirstlane(live);
    always = __builtin_amdgcn_readfirstlane(always);
  }
  if (lane == 0) {
    sh.first[wave] = live;
    sh.second[wave] = always;
    sh.any[wave] = any;
    sh.all[wave] = all;
  }
  for (int i = tid; i < PickShared<NT>::kBins; i += NT) sh.bins[i] = 0;
  if (tid == 0) sh.found = 0;
  __syncthreads();
  live = always = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; w++) {
    live += sh.first[w];
    always += sh.second[w];
    any |= sh.any[w];
    all &= sh.all[w];
  }
  __syncthreads();  // (the places are used again)

  // taken: keys above `least`, and those equal to it up to place `last`
  uint64_t least = live <= a.budget ? 0 : kAlways - 1;
  int last = -1;
  if (live > a.budget && a.budget > always) nth_key(sh, keys, any, all, live - always, a.budget - always, &least, &last);
  put_places(sh, keys, [&](uint64_t k, int i) { return k > least || (k == least && i <= last); }, a.budget, out, count);
}

template <int NT>
__global__ __launch_bounds__(NT) void block_pick_kernel(const BlockSelectArgs a, const uint64_t *__restrict__ keys) {
  const int row = blockIdx.x, n = blocks_of(a, a.c.lengths[row / a.c.nkv]);
  const uint64_t *key = keys + (int64_t)row * table_blocks_of(a);
  int *out = a.selected + (int64_t)row * a.budget, *count = a.counts ? a.counts + row : nullptr;
  if (n <= NT * kPickKeys)
    pick<NT, true>(a, key, n, out, count);
  else
    pick<NT, false>(a, key, n, out, count);
}

template <int D>
void launch_scores(const BlockSelectArgs &a, uint64_t *keys, int grid, int per, int chunks, hipStream_t s) {
  const int group = a.nq / a.c.nkv;
  if (group == 1)
    hipLaunchKernelGGL((block_score_kernel<D, 1>), dim3(grid), dim3(64 * kScoreWaves), 0, s, a, keys, per, chunks);
  else if (group == 2)
    hipLaunchKernelGGL((block_score_kernel<D, 2>), dim3(grid), dim3(64 * kScoreWaves), 0, s, a, keys, per, chunks);
  else
    hipLaunchKernelGGL((block_score_kernel<D, 4>), dim3(grid), dim3(64 * kScoreWaves), 0, s, a, keys, per, chunks);
}

template <int D>
hipError_t launch_select_width(const BlockSelectArgs &a, uint64_t *keys, int num_cus, hipStream_t s) {
  constexpr int kRows = 64 / (D / 8) * kScoreWaves;  // blocks of a workgroup at once
  const int64_t rows = (int64_t)a.c.sequences * a.c.nkv, table_blocks = ((int64_t)a.c.width << a.c.page_shift) >> a.b.shift;
  // four workgroups a CU where there are as many blocks (24 contexts up to 32768
  // in blocks of 64, 8 KV heads of 128, groups of 4: 11.2 us, eight 14, two 15; two
  // of 262144 in blocks of 32, 4 KV heads: 14.1, 16, 13.0; two heads at a time in
  // place of four cost 0.5 to 1 us more, one 6)
  int64_t per = (rows * table_blocks + 4 * num_cus - 1) / (4 * num_cus);
  per = (per + kRows - 1) / kRows * kRows;
  per = per < kRows ? kRows : per > 64 * kRows ? 64 * kRows : per;
  const int64_t chunks = (table_blocks + per - 1) / per;
  launch_scores<D>(a, keys, (int)(rows * chunks), (int)per, (int)chunks, s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (table_blocks <= 256 * kPickKeys)
    hipLaunchKernelGGL(block_pick_kernel<256>, dim3((unsigned)rows), dim3(256), 0, s, a, keys);
  else
    hipLaunchKernelGGL(block_pick_kernel<1024>, dim3((unsigned)rows), dim3(1024), 0, s, a, keys);
  return hipGetLastError();
}

}  // namespace

bool block_bounds_fits(const BlockBoundsArgs &a) {
  const int64_t slots = a.offsets ? touched_blocks(a.tokens, a.c.sequences, 1 << a.b.shift) : a.c.sequences;
  return !((slots * a.c.nkv) >> 31);
}

hipError_t launch_block_bounds(const BlockBoundsArgs &a, int num_cus, hipStream_t s) {
  if (a.tokens < 1 || a.c.nkv < 1 || !a.b.key_bounds || a.b.shift < 4 || a.b.shift > a.c.page_shift || !block_bounds_fits(a))
    return hipErrorInvalidValue;
  const int64_t slots = a.offsets ? touched_blocks(a.tokens, a.c.sequences, 1 << a.b.shift) : a.c.sequences;
  switch (a.c.head_dim) {
    case 64: return launch_bounds_type<64>(a, (int)slots, num_cus, s);
    case 128: return launch_bounds_type<128>(a, (int)slots, num_cus, s);
    case 256: return launch_bounds_type<256>(a, (int)slots, num_cus, s);
    default: return hipErrorInvalidValue;
  }
}

size_t block_select_scratch_bytes(const BlockSelectArgs &a) {
  return (size_t)a.c.sequences * a.c.nkv * (((size_t)a.c.width << a.c.page_shift) >> a.b.shift) * sizeof(uint64_t);
}

bool block_select_fits(const BlockSelectArgs &a) {  // (a workgroup of the scores has eight blocks at least)
  const int64_t table_blocks = ((int64_t)a.c.width << a.c.page_shift) >> a.b.shift;
  return !((int64_t)a.c.sequences * a.c.nkv * (table_blocks / 8 + 1) >> 31);
}

hipError_t launch_block_select(const BlockSelectArgs &a, void *scratch, int num_cus, hipStream_t s) {
  if (a.c.sequences < 1 || a.c.nkv < 1 || a.nq % a.c.nkv != 0 || a.budget < 1 || !a.b.key_bounds || !scratch ||
      a.b.shift < 4 || a.b.shift > a.c.page_shift || !block_select_fits(a))
    return hipErrorInvalidValue;
  uint64_t *keys = static_cast<uint64_t *>(scratch);
  switch (a.c.head_dim) {
    case 64: return launch_select_width<64>(a, keys, num_cus, s);
    case 128: return launch_select_width<128>(a, keys, num_cus, s);
    case 256: return launch_select_width<256>(a, keys, num_cus, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace hp
