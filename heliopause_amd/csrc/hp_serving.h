// hp_serving.h -- arguments and launches of the operators that serve several
// sequences at once: the paged key/value cache (paged_append.hip,
// paged_attn.hip), the attention over packed prompts (packed_attn.hip) and the
// penalties, biases and masks of the logits (logit_rules.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "hp_pages.h"

namespace hp {

// HP_ELEM_* of include/hp_hip.h
constexpr int kElemF32 = 0, kElemF16 = 1, kElemBf16 = 2, kElemE4m3 = 3, kElemI8 = 4;
__host__ __device__ constexpr int elem_bytes(int type) {
  return type == kElemF32 ? 4 : type == kElemE4m3 || type == kElemI8 ? 1 : 2;
}

// The pages of a batch: key row (page p, head h, slot i) at element
// p * page_stride + (h * page_size + i) * head_dim.
struct PagedCache {
  void *keys, *values;
  const int *pages, *lengths;  // [sequences][width], [sequences]
  int64_t page_stride;
  int type, head_dim, nkv, page_count, page_shift, sequences, width;
  float key_scale, value_scale;  // e4m3: value = stored * scale
};

struct PagedAppendArgs {
  PagedCache c;
  const float *q, *k, *v;  // v == nullptr: the key projection's rows
  int64_t q_stride, k_stride, v_stride;
  const int *offsets;  // null: token t is sequence t's
  const float *q_norm, *k_norm, *freq_factors;
  void *q_out, *k_out, *v_out;
  int tokens, nq, out_type, norm_values, rope_dims;
  float eps;
  double log2_base;
};
hipError_t launch_paged_append(const PagedAppendArgs &a, int num_cus, hipStream_t s);

struct PagedAttnArgs {
  PagedCache c;
  const void *q;
  void *out;
  int64_t q_stride, out_stride;
  int nq, q_type, out_type, window;
  float scale;
  float *partials;  // paged_attn_scratch_bytes
  // block_attn.hip: a scale of each block and KV head, [page][kv head][block]; the
  // blocks to attend to, [sequence][kv head][budget], and how many
  const float *key_scales, *value_scales;
  const int *selected, *counts;
  int block_shift, budget;
};
// Shares of a launch's keys, which the scratch goes by (the lengths are on the
// device, so neither depends on them).
int paged_attn_groups(const PagedAttnArgs &a, int num_cus);
size_t paged_attn_scratch_bytes(const PagedAttnArgs &a, int groups);
hipError_t launch_paged_attn(const PagedAttnArgs &a, int groups, hipStream_t s);
hipError_t launch_block_attn(const PagedAttnArgs &a, int groups, hipStream_t s);
// Steps of a batch whose sequences fill their tables; the kernel counts them
// in 32 bits.
uint64_t paged_attn_most_steps(const PagedAttnArgs &a);

// What is kept of a cache's blocks of 1 << shift positions: for each page, KV head
// and block of the page a scale of the keys and one of the values, and the bounds
// of the keys (bf16: head_dim least, head_dim largest elements).
struct CacheBlocks {
  float *key_scales, *value_scales;
  uint16_t *key_bounds;
  int shift;
};

// Whether the launch's grid is within what a launch takes.
bool block_append_fits(const PagedAppendArgs &a, const CacheBlocks &b);
hipError_t launch_block_append(const PagedAppendArgs &a, const CacheBlocks &b, int num_cus, hipStream_t s);

struct BlockBoundsArgs {
  PagedCache c;
  CacheBlocks b;
  const int *offsets;  // null: row s is sequence s's
  int tokens;
};
bool block_bounds_fits(const BlockBoundsArgs &a);
hipError_t launch_block_bounds(const BlockBoundsArgs &a, int num_cus, hipStream_t s);

struct BlockSelectArgs {
  PagedCache c;
  CacheBlocks b;
  const void *q;
  int64_t q_stride;
  int *selected, *counts;  // [sequence][kv head][budget], [sequence][kv head]
  int nq, q_type, budget, first_blocks, last_blocks;
};
bool block_select_fits(const BlockSelectArgs &a);
size_t block_select_scratch_bytes(const BlockSelectArgs &a);
hipError_t launch_block_select(const BlockSelectArgs &a, void *scratch, int num_cus, hipStream_t s);

struct PagePlanArgs {
  int *pages;  // [sequences][width]
  const int *lengths, *fresh, *keep_from;  // fresh null: a token for each sequence that has some
  int *lengths_out, *free, *free_count, *offsets, *missing, *sequence_of, *positions;
  int64_t *slots;
  int sequences, width, page_shift, page_count, rows;
};
int page_plan_launches(const PagePlanArgs &a);  // one: no scratch
size_t page_plan_scratch_bytes(const PagePlanArgs &a);
hipError_t launch_page_plan(const PagePlanArgs &a, void *scratch, hipStream_t s);

struct PackedAttnArgs {
  const void *q, *k, *v;
  void *out;
  const int *offsets;  // [sequences + 1]
  int64_t q_stride, k_stride, v_stride, out_stride;
  int sequences, tokens, nq, nkv, head_dim, type, out_type, window;
  float scale;
};
// Whether the launch's grid is within what a launch takes.
bool packed_attn_fits(const PackedAttnArgs &a);
hipError_t launch_packed_attn(const PackedAttnArgs &a, int num_cus, hipStream_t s);

struct LogitRulesArgs {
  const float *logits;
  float *out;
  const int *history, *history_lengths, *prompt_lengths;
  const float *repetition, *frequency, *presence;
  const int *bias_ids, *bias_counts;
  const float *bias_values;
  const uint32_t *allowed;
  int64_t logits_stride, out_stride, history_stride, bias_stride, allowed_stride;
  int rows, n;
  double softcap;  // 0: none
};
hipError_t launch_logit_rules(const LogitRulesArgs &a, hipStream_t s);

// Largest s in 0 .. n such that offsets[1 .. s] <= t, by a whole wave: the
// sequence of packed row t (n: a row behind the last).  64 entries are probed
// at once.  Offsets that fall give some s of the same range.
__device__ __forceinline__ int packed_sequence_of(const int *__restrict__ offsets, int n, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  while (n > 64) {
    const int step = (n + 63) >> 6, at = (lane + 1) * step;
    const bool le = at <= n && offsets[lo + min(at, n)] <= t;
    const int c = __popcll(__ballot(le));
    lo += c * step;
    n = min(step - 1, n - c * step);
  }
  const bool le = lane < n && offsets[lo + 1 + min(lane, max(n - 1, 0))] <= t;
  return lo + __popcll(__ballot(le));
}

// The sequence whose touched blocks (hp_pages.h) have slot `slot`, by a whole
// wave: the largest s in 0 .. n - 1 whose first slot is not behind it.
__device__ __forceinline__ int touched_sequence(const int *__restrict__ offsets, int n, int slot, int block) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  while (n > 64) {
    const int step = (n + 63) >> 6, i = lo + min(lane * step, n - 1);
    const bool le = lane * step < n && touched_first(offsets[i], i, block) <= slot;
    const int c = max(__popcll(__ballot(le)), 1) - 1;
    lo += c * step;
    n = min(step, n - c * step);
  }
  const int i = lo + min(lane, n - 1);
  const bool le = lane < n && touched_first(offsets[i], i, block) <= slot;
  return lo + max(__popcll(__ballot(le)), 1) - 1;
}

// DPP rotation of each 16-lane row by eight: lane c gets lane c ^ 8's value.
constexpr int kDppRor8 = 0x128;

__device__ __forceinline__ uint16_t bf16_bits(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
__device__ __forceinline__ uint16_t f16_bits(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
__device__ __forceinline__ float bf16_value(uint32_t bits16) { return __builtin_bit_cast(float, bits16 << 16); }

// Four consecutive elements, rounded to nearest even where they leave in 16
// bits (a value past the largest f16 becomes an infinity).
__device__ __forceinline__ void store4(void *p, int64_t i, int type, const float (&v)[4]) {
  if (type == kElemF32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
  uint16_t b[4];
#pragma unroll
  for (int j = 0; j < 4; j++) b[j] = type == kElemF16 ? f16_bits(v[j]) : bf16_bits(v[j]);
  *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + i) =
      make_uint2(b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16);
}

}  // namespace hp
