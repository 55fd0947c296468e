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
// Pick.  One workgroup per (sequence, KV head): the digits of the budget-th
// largest key, 8 bits at a time below the bits that all keys share, by counting
// in LDS; then the blocks above it, and of those equal to it the first ones, in
// their order.
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

// One wave per (touched block, KV head): 16 bytes of a row a lane.
constexpr int kBoundWaves = 4;

template <int CT>
__device__ __forceinline__ void elements(const uint4 &w, float (&v)[16 / elem_bytes(CT)]) {
  const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 16 / elem_bytes(CT); i++) {
    if (CT == kElemF16)
      v[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(d[i / 2] >> (16 * (i & 1))));
    else if (CT == kElemBf16)
      v[i] = bf16_value(d[i / 2] >> (16 * (i & 1)) & 0xffffu);
    else if (CT == kElemI8)
      v[i] = (float)(int8_t)(d[i / 4] >> (8 * (i & 3)));
    else
      v[i] = (i & 3) == 0   ? __builtin_amdgcn_cvt_f32_fp8(d[i / 4], 0)
             : (i & 3) == 1 ? __builtin_amdgcn_cvt_f32_fp8(d[i / 4], 1)
             : (i & 3) == 2 ? __builtin_amdgcn_cvt_f32_fp8(d[i / 4], 2)
                            : __builtin_amdgcn_cvt_f32_fp8(d[i / 4], 3);
  }
}

template <int D, int CT>
__global__ __launch_bounds__(64 * kBoundWaves) void block_bounds_kernel(const BlockBoundsArgs a, int units) {
  constexpr int kE = elem_bytes(CT), kPer = 16 / kE, kLanes = D / kPer, kRows = 64 / kLanes, kDeep = 8;
  const int lane = threadIdx.x & 63, unit = blockIdx.x * kBoundWaves + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int h = unit % a.c.nkv, slot = unit / a.c.nkv;
  int seq = slot;
  NewInBlock n;
  const int64_t table_keys = (int64_t)a.c.width << a.c.page_shift;
  if (a.offsets) {
    int lo = 0, left = a.c.sequences;  // the largest sequence whose first slot is not behind this one
    while (left > 64) {
      const int step = (left + 63) >> 6, i = lo + min(lane * step, left - 1);
      const bool le = lane * step < left && touched_first(a.offsets[i], i, 1 << a.b.shift) <= slot;
      const int c = max(__popcll(__ballot(le)), 1) - 1;
      lo += c * step;
      left = min(step, left - c * step);
    }
    const int i = lo + min(lane, left - 1);
    const bool le = lane < left && touched_first(a.offsets[i], i, 1 << a.b.shift) <= slot;
    seq = lo + max(__popcll(__ballot(le)), 1) - 1;
    const int begin = a.offsets[seq];
    n = new_in_block(a.c.lengths[seq], (int64_t)a.offsets[seq + 1] - begin,
                     slot - touched_first(begin, seq, 1 << a.b.shift), a.b.shift, table_keys);
  } else {
    n = new_in_block(a.c.lengths[seq], 1, 0, a.b.shift, table_keys);
  }
  if (n.end <= n.first) return;
  const int page = page_or_none(a.c.pages[(int64_t)seq * a.c.width + (n.first >> a.c.page_shift)], a.c.page_count);
  if (page < 0) return;
  const int in_page = n.block & ((1 << (a.c.page_shift - a.b.shift)) - 1), live = n.end - (n.block << a.b.shift);
  const int64_t block_at = (((int64_t)page * a.c.nkv + h) << (a.c.page_shift - a.b.shift)) + in_page;
  const uint8_t *rows = static_cast<const uint8_t *>(a.c.keys) +
                        (page * a.c.page_stride + (((int64_t)h << a.c.page_shift) + ((int64_t)in_page << a.b.shift)) * D) * kE;
  const int col = lane % kLanes, sub = lane / kLanes;
  float lo[kPer], hi[kPer];
#pragma unroll
  for (int i = 0; i < kPer; i++) lo[i] = kInf, hi[i] = -kInf;
  bool odd = false;  // a NaN is among the lane's elements
  for (int r0 = 0; r0 < live; r0 += kRows * kDeep) {
    uint4 w[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; i++) {  // (behind the last row: the last one's again)
      const int r = min(r0 + i * kRows + sub, live - 1);
      w[i] = *reinterpret_cast<const uint4 *>(rows + ((int64_t)r * D + col * kPer) * kE);
    }
#pragma unroll
    for (int i = 0; i < kDeep; i++) {
      float v[kPer];
      elements<CT>(w[i], v);
#pragma unroll
      for (int j = 0; j < kPer; j++) {
        lo[j] = fminf(lo[j], v[j]);
        hi[j] = fmaxf(hi[j], v[j]);
        odd = odd || v[j] != v[j];
      }
    }
  }
  if (__any(odd)) {  // rare: which elements
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      bool is = false;
      for (int r = sub; r < live; r += kRows) {
        float v[kPer];
        elements<CT>(*reinterpret_cast<const uint4 *>(rows + ((int64_t)r * D + col * kPer) * kE), v);
        is = is || v[j] != v[j];
      }
      lo[j] = is ? -kInf : lo[j];
      hi[j] = is ? kInf : hi[j];
    }
  }
  const float scale = a.b.key_scales ? a.b.key_scales[block_at] : CT == kElemE4m3 ? a.c.key_scale : 1.0f;
#pragma unroll
  for (int m = kLanes; m < 64; m *= 2) {
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      lo[j] = fminf(lo[j], __shfl_xor(lo[j], m));
      hi[j] = fmaxf(hi[j], __shfl_xor(hi[j], m));
    }
  }
  if (sub != 0) return;
  uint16_t *out = a.b.key_bounds + block_at * 2 * D + col * kPer;
#pragma unroll
  for (int j = 0; j < kPer; j += 8) {
    uint32_t l[4], u[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      l[i] = outward<false>(lo[j + 2 * i] * scale) | (uint32_t)outward<false>(lo[j + 2 * i + 1] * scale) << 16;
      u[i] = outward<true>(hi[j + 2 * i] * scale) | (uint32_t)outward<true>(hi[j + 2 * i + 1] * scale) << 16;
    }
    *reinterpret_cast<uint4 *>(out + j) = make_uint4(l[0], l[1], l[2], l[3]);
    *reinterpret_cast<uint4 *>(out + D + j) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

template <int D>
hipError_t launch_bounds_type(const BlockBoundsArgs &a, int units, hipStream_t s) {
  const dim3 grid((units + kBoundWaves - 1) / kBoundWaves), threads(64 * kBoundWaves);
  switch (a.c.type) {
    case kElemF16: hipLaunchKernelGGL((block_bounds_kernel<D, kElemF16>), grid, threads, 0, s, a, units); break;
    case kElemBf16: hipLaunchKernelGGL((block_bounds_kernel<D, kElemBf16>), grid, threads, 0, s, a, units); break;
    case kElemE4m3: hipLaunchKernelGGL((block_bounds_kernel<D, kElemE4m3>), grid, threads, 0, s, a, units); break;
    case kElemI8: hipLaunchKernelGGL((block_bounds_kernel<D, kElemI8>), grid, threads, 0, s, a, units); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

// ---- scores ------------------------------------------------------------------

constexpr int kScoreWaves = 4;
constexpr int kHeadsAtOnce = 4;  // whose queries a lane holds: 8 elements, both parts, 64 bits
constexpr uint64_t kAlways = ~0ull;  // a key of a block that is taken whatever its score; 0: none to take

__device__ __forceinline__ uint64_t key_of(double score) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, score + 0.0);  // (-0 is 0)
  return bits ^ ((int64_t)bits < 0 ? ~0ull : 1ull << 63);
}

// Sum over the L lanes of a row (8, 16 or 32).
template <int L>
__device__ __forceinline__ double row_sum(double v) {
  v += dpp_f64<kDppXor1>(v);
  v += dpp_f64<kDppXor2>(v);
  v += dpp_f64<kDppRowHalfMirror>(v);
  if (L >= 16) v += dpp_f64<kDppRowMirror>(v);
  if (L >= 32) v += __shfl_xor(v, 16);
  return v;
}

__device__ __forceinline__ float query_element(const BlockSelectArgs &a, int64_t i) {
  const float v = a.q_type == kElemF32   ? static_cast<const float *>(a.q)[i]
                  : a.q_type == kElemF16 ? (float)static_cast<const _Float16 *>(a.q)[i]
                                         : bf16_value(static_cast<const uint16_t *>(a.q)[i]);
  return v != v ? 0.0f : fminf(fmaxf(v, -kF32Most), kF32Most);
}

// D / 8 lanes have a block's bounds, 8 elements each; a workgroup `per` blocks
// of a (sequence, KV head).
template <int D>
__global__ __launch_bounds__(64 * kScoreWaves) void block_score_kernel(const BlockSelectArgs a, uint64_t *__restrict__ keys,
                                                                       int per, int chunks) {
  constexpr int kLanes = D / 8, kRows = 64 / kLanes;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % kLanes, sub = lane / kLanes;
  const int row = blockIdx.x / chunks, seq = row / a.c.nkv, h = row - seq * a.c.nkv;
  const int table_blocks = (int)(((int64_t)a.c.width << a.c.page_shift) >> a.b.shift);
  const int length = a.c.lengths[seq];
  const int blocks = length > 0 ? min((int)(((int64_t)length + (1 << a.b.shift) - 1) >> a.b.shift), table_blocks) : 0;
  const int begin = blockIdx.x % chunks * per, end = min(begin + per, blocks);
  if (begin >= end) return;
  const int group = a.nq / a.c.nkv, in_page = a.c.page_shift - a.b.shift;
  const int *table = a.c.pages + (int64_t)seq * a.c.width;
  const int64_t q0 = seq * a.q_stride + (int64_t)h * group * D + 8 * l;
  for (int g0 = 0; g0 < group; g0 += kHeadsAtOnce) {
    double up[kHeadsAtOnce][8], down[kHeadsAtOnce][8];
#pragma unroll
    for (int g = 0; g < kHeadsAtOnce; g++)
#pragma unroll
      for (int j = 0; j < 8; j++) {  // (a head beyond the group: the last one's again)
        const float v = query_element(a, q0 + (int64_t)min(g0 + g, group - 1) * D + j);
        up[g][j] = fmaxf(v, 0.0f);
        down[g][j] = fminf(v, 0.0f);
      }
    for (int b0 = begin + wave * kRows; b0 < end; b0 += kScoreWaves * kRows) {
      const int b = min(b0 + sub, end - 1);
      const int page = page_or_none(table[b >> in_page], a.c.page_count);
      const uint16_t *bound = a.b.key_bounds +
                              ((((int64_t)max(page, 0) * a.c.nkv + h) << in_page) + (b & ((1 << in_page) - 1))) * 2 * D + 8 * l;
      const uint4 lo = *reinterpret_cast<const uint4 *>(bound), hi = *reinterpret_cast<const uint4 *>(bound + D);
      const uint32_t low[4] = {lo.x, lo.y, lo.z, lo.w}, high[4] = {hi.x, hi.y, hi.z, hi.w};
      double sum[kHeadsAtOnce];
#pragma unroll
      for (int g = 0; g < kHeadsAtOnce; g++) sum[g] = 0.0;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const double x = (double)bf16_value(low[j / 2] >> (16 * (j & 1)) & 0xffffu);
        const double y = (double)bf16_value(high[j / 2] >> (16 * (j & 1)) & 0xffffu);
#pragma unroll
        for (int g = 0; g < kHeadsAtOnce; g++) sum[g] = fma(up[g][j], y, fma(down[g][j], x, sum[g]));
      }
      double best = row_sum<kLanes>(sum[0]);
#pragma unroll
      for (int g = 1; g < kHeadsAtOnce; g++) best = fmax(best, row_sum<kLanes>(sum[g]));
      if (l != 0 || b0 + sub >= end) continue;
      uint64_t *key = keys + (int64_t)row * table_blocks + b;
      uint64_t k = key_of(best);
      if (g0 > 0) k = max(k, *key);  // (this lane's own of the heads before)
      if (b < a.first_blocks || b >= blocks - a.last_blocks) k = kAlways;
      *key = page < 0 ? 0 : k;
    }
  }
}

// ---- pick --------------------------------------------------------------------

constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / 64;

__device__ __forceinline__ uint64_t wave_or(uint64_t v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v |= __shfl_xor(v, m);
  return v;
}
__device__ __forceinline__ uint64_t wave_and(uint64_t v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v &= __shfl_xor(v, m);
  return v;
}

__global__ __launch_bounds__(kPickThreads) void block_pick_kernel(const BlockSelectArgs a, const uint64_t *__restrict__ keys) {
  __shared__ uint64_t sh_or[kPickWaves], sh_and[kPickWaves];
  __shared__ int sh_live[kPickWaves], sh_always[kPickWaves];
  __shared__ int sh_bins[256];
  __shared__ int sh_digit, sh_need, sh_in;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x, seq = row / a.c.nkv;
  const int table_blocks = (int)(((int64_t)a.c.width << a.c.page_shift) >> a.b.shift);
  const int length = a.c.lengths[seq];
  const int n = length > 0 ? min((int)(((int64_t)length + (1 << a.b.shift) - 1) >> a.b.shift), table_blocks) : 0;
  const uint64_t *key = keys + (int64_t)row * table_blocks;

  // how many there are, and the bits in which the others' keys differ
  uint64_t any = 0, all = ~0ull;
  int live = 0, always = 0;
  for (int i = tid; i < n; i += kPickThreads) {
    const uint64_t k = key[i];
    live += k != 0;
    always += k == kAlways;
    if (k != 0 && k != kAlways) {
      any |= k;
      all &= k;
    }
  }
  any = wave_or(any);
  all = wave_and(all);
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    live += __shfl_xor(live, m);
    always += __shfl_xor(always, m);
  }
  if (lane == 0) {
    sh_or[wave] = any;
    sh_and[wave] = all;
    sh_live[wave] = live;
    sh_always[wave] = always;
  }
  __syncthreads();
  live = always = 0;
  for (int w = 0; w < kPickWaves; w++) {
    any |= sh_or[w];
    all &= sh_and[w];
    live += sh_live[w];
    always += sh_always[w];
  }
  __syncthreads();  // (the counts' places are used again)

  // the threshold: keys above `least | low bits` are taken, and `need` of those
  // whose bits from `shift` on are its own
  int need = a.budget - always, shift = 64;
  uint64_t least = 0;
  const bool whole = live <= a.budget;  // (the same for the workgroup)
  if (!whole && need > 0) {
    const uint64_t differ = any ^ all;
    shift = differ ? 64 - __builtin_clzll(differ) : 0;  // the bits from here on are the same
    least = shift < 64 ? all >> shift << shift : 0;
    int in = live - always;
    while (shift > 0 && in > need) {
      const int low = max(shift - 8, 0), bits = shift - low;
      for (int i = tid; i < 256; i += kPickThreads) sh_bins[i] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kPickThreads) {
        const uint64_t k = key[i];
        if (k != 0 && k != kAlways && (shift == 64 || k >> shift == least >> shift))
          atomicAdd(&sh_bins[(k >> low) & ((1 << bits) - 1)], 1);
      }
      __syncthreads();
      if (wave == 0) {  // from the largest digit down: four a lane
        int c[4], sum = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) sum += c[j] = sh_bins[255 - 4 * lane - j];
        int to = sum;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
          const int o = __shfl_up(to, d);
          to += lane >= d ? o : 0;
        }
        int before = to - sum;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (before < need && need <= before + c[j]) {  // one lane's one digit
            sh_digit = 255 - 4 * lane - j;
            sh_need = need - before;
            sh_in = c[j];
          }
          before += c[j];
        }
      }
      __syncthreads();
      least |= (uint64_t)sh_digit << low;
      need = sh_need;
      in = sh_in;
      shift = low;
      __syncthreads();
    }
    if (in <= need) need = in;
  }

  // in their order
  int *out = a.selected + (int64_t)row * a.budget;
  int taken = 0, equal = 0;  // up to the blocks at hand, by the whole workgroup
  for (int i0 = 0; i0 < n && taken < a.budget; i0 += kPickThreads) {
    const int i = i0 + tid;
    const uint64_t k = i < n ? key[i] : 0;
    const bool other = k != 0 && k != kAlways;
    const bool same = !whole && need > 0 && other && (shift == 64 || k >> shift == least >> shift);
    const bool above = k == kAlways || (whole && k != 0) || (!whole && need > 0 && other && !same && k > least);
    const uint64_t same_mask = __ballot(same);
    if (lane == 0) sh_live[wave] = __popcll(same_mask);
    __syncthreads();
    int rank = equal + __popcll(same_mask & ((1ull << lane) - 1)), sames = 0;
    for (int w = 0; w < kPickWaves; w++) {
      rank += w < wave ? sh_live[w] : 0;
      sames += sh_live[w];
    }
    const bool take = above || (same && rank < need);
    const uint64_t mask = __ballot(take);
    if (lane == 0) sh_always[wave] = __popcll(mask);
    __syncthreads();
    int at = taken + __popcll(mask & ((1ull << lane) - 1)), takes = 0;
    for (int w = 0; w < kPickWaves; w++) {
      at += w < wave ? sh_always[w] : 0;
      takes += sh_always[w];
    }
    if (take && at < a.budget) out[at] = i;
    taken += takes;
    equal += sames;
  }
  taken = min(taken, a.budget);
  for (int i = taken + tid; i < a.budget; i += kPickThreads) out[i] = -1;
  if (tid == 0 && a.counts) a.counts[row] = taken;
}

template <int D>
hipError_t launch_select_width(const BlockSelectArgs &a, uint64_t *keys, int num_cus, hipStream_t s) {
  constexpr int kRows = 64 / (D / 8) * kScoreWaves;  // blocks of a workgroup at once
  const int64_t rows = (int64_t)a.c.sequences * a.c.nkv, table_blocks = ((int64_t)a.c.width << a.c.page_shift) >> a.b.shift;
  // eight workgroups a CU where there are as many blocks
  int64_t per = (rows * table_blocks + 8 * num_cus - 1) / (8 * num_cus);
  per = (per + kRows - 1) / kRows * kRows;
  per = per < kRows ? kRows : per > 32 * kRows ? 32 * kRows : per;
  const int64_t chunks = (table_blocks + per - 1) / per;
  hipLaunchKernelGGL(block_score_kernel<D>, dim3((unsigned)(rows * chunks)), dim3(64 * kScoreWaves), 0, s, a, keys,
                     (int)per, (int)chunks);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(block_pick_kernel, dim3((unsigned)rows), dim3(kPickThreads), 0, s, a, keys);
  return hipGetLastError();
}

}  // namespace

bool block_bounds_fits(const BlockBoundsArgs &a) {
  const int64_t slots = a.offsets ? touched_blocks(a.tokens, a.c.sequences, 1 << a.b.shift) : a.c.sequences;
  return !((slots * a.c.nkv) >> 31);
}

hipError_t launch_block_bounds(const BlockBoundsArgs &a, hipStream_t s) {
  if (a.tokens < 1 || a.c.nkv < 1 || !a.b.key_bounds || a.b.shift < 4 || a.b.shift > a.c.page_shift || !block_bounds_fits(a))
    return hipErrorInvalidValue;
  const int64_t slots = a.offsets ? touched_blocks(a.tokens, a.c.sequences, 1 << a.b.shift) : a.c.sequences;
  const int units = (int)(slots * a.c.nkv);
  switch (a.c.head_dim) {
    case 64: return launch_bounds_type<64>(a, units, s);
    case 128: return launch_bounds_type<128>(a, units, s);
    case 256: return launch_bounds_type<256>(a, units, s);
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
