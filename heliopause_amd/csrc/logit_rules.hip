// logit_rules.hip -- what a request changes about the head's logits before
// the top-k: penalties for tokens that were there already, biases, and the
// grammar's mask.  Per row and token:
//   x = logit, or cap * tanh(logit / cap)
//   x = x > 0 ? x / repetition : x * repetition   (token in the history)
//   x = x - frequency * count                     (count: its occurrences in the
//   x = x - presence             (count > 0)       history after the prompt)
//   x = x + bias                  (the last entry of the token in the list)
//   x = -inf                      (the token's mask bit is 0)
// in f32, each step rounded as it stands (no contraction); the cap is the
// top-k's own, in f64.  It belongs here where there is one: behind the rules it
// would make a masked token's -inf a -cap, which is sampled.  (With a top-k of 40
// behind, 128 rows of 151669: 172 us without a cap, 290 with it here, 451 there.)
//
// Logits in and out, 8 bytes a token, are what it moves.  A workgroup takes a
// slice of a row's vocabulary and counts in LDS what of the row's whole
// history falls into the slice, one word a token, with integer atomics, whose
// order changes nothing; so there is one launch, no scratch and no table of
// the vocabulary's size in memory.  Every slice reads the history again (from
// the L2).  The logits are loaded first and wait in registers while the history
// is counted.  Slices of 2048 tokens by 256 threads: 6.1 us for one row of
// 262144 and 37.5 us (4.2 TB/s) for 128 of 151669, against 7.7 and 39.8 in
// slices of 16384, and 6.0 and 47.9 in slices of 1024.  Stores past the caches
// make the launch alone faster (30 us) and with the top-k behind it, which reads
// them, slower (196 -> 200 us), so they stay ordinary.
#include "hp_serving.h"
#include "hp_tanh.h"

namespace hp {

namespace {

constexpr uint32_t kInPrompt = 0x80000000u;  // of a word: the token is in the prompt part

// Four elements at a 4-byte boundary: rows of odd widths start anywhere.
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef int int4u __attribute__((ext_vector_type(4), aligned(4)));

// A slice: a workgroup's threads with kPer groups of four tokens each.
constexpr int kThreads = 256, kPer = 2, kSlice = kThreads * 4 * kPer;

template <bool CAP>
__global__ __launch_bounds__(kThreads) void logit_rules_kernel(const LogitRulesArgs a) {
  __shared__ uint32_t words[kSlice];
  const int tid = threadIdx.x, row = blockIdx.y, base = blockIdx.x * kSlice;
  const float *in = a.logits + row * a.logits_stride + base;
  float *out = a.out + row * a.out_stride + base;
  const int left = min(kSlice, a.n - base);

  float x[kPer][4];
  uint32_t allowed[kPer];
#pragma unroll
  for (int g = 0; g < kPer; g++) {
    const int i = 4 * (g * kThreads + tid);
    if (i + 4 <= left) {
      const float4u v = *reinterpret_cast<const float4u *>(in + i);
#pragma unroll
      for (int j = 0; j < 4; j++) x[g][j] = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) x[g][j] = i + j < left ? in[i + j] : 0.0f;
    }
    allowed[g] = a.allowed && i < left
                     ? a.allowed[row * a.allowed_stride + (base + i) / 32] >> ((base + i) & 31)
                     : 0xfu;
  }

  if (CAP) {
#pragma unroll
    for (int g = 0; g < kPer; g++)
#pragma unroll
      for (int j = 0; j < 4; j++) x[g][j] = softcap_value(x[g][j], a.softcap);
  }

  const int seen = a.history ? max(a.history_lengths[row], 0) : 0;
  const int told = (int)min((int64_t)seen, a.history_stride);
  const int biases = a.bias_ids ? (int)min((int64_t)max(a.bias_counts[row], 0), a.bias_stride) : 0;
  if (told > 0 || biases > 0) {
#pragma unroll
    for (int g = 0; g < kPer; g++)
      *reinterpret_cast<uint4 *>(&words[4 * (g * kThreads + tid)]) = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  if (told > 0) {
    const int *history = a.history + row * a.history_stride;
    const int prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
    auto count = [&](int token, int i) {
      const uint32_t at = (uint32_t)token - (uint32_t)base;
      if (at >= (uint32_t)left) return;  // another slice's, or no token
      if (i < prompt)
        atomicOr(&words[at], kInPrompt);
      else
        atomicAdd(&words[at], 1u);
    };
    if (told < 4) {
      if (tid < told) count(history[tid], tid);
    } else {
      // four at a time, the loads of kDeep fours on their way together; a four
      // that would pass the end is the last four, of which the thread counts
      // its own
      constexpr int kDeep = 4;
      for (int i0 = 4 * tid; i0 < told; i0 += 4 * kThreads * kDeep) {
        int4u t[kDeep];
#pragma unroll
        for (int k = 0; k < kDeep; k++)
          t[k] = *reinterpret_cast<const int4u *>(history + min(i0 + 4 * kThreads * k, told - 4));
#pragma unroll
        for (int k = 0; k < kDeep; k++) {
          const int i = i0 + 4 * kThreads * k, from = min(i, told - 4);
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (from + j >= i) count(t[k][j], from + j);
        }
      }
    }
    __syncthreads();
    const float r = a.repetition ? a.repetition[row] : 1.0f;
    const float f = a.frequency ? a.frequency[row] : 0.0f, p = a.presence ? a.presence[row] : 0.0f;
#pragma unroll
    for (int g = 0; g < kPer; g++) {
      uint4 *at = reinterpret_cast<uint4 *>(&words[4 * (g * kThreads + tid)]);
      const uint4 w4 = *at;
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
      *at = make_uint4(0, 0, 0, 0);  // the biases'
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (w[j] == 0) continue;
        float v = x[g][j];
        v = v > 0.0f ? v / r : v * r;
        const uint32_t n = w[j] & ~kInPrompt;
        v = v - f * (float)n;
        x[g][j] = n ? v - p : v;
      }
    }
  }
  if (biases > 0) {
    const int *ids = a.bias_ids + row * a.bias_stride;
    const float *values = a.bias_values + row * a.bias_stride;
    __syncthreads();  // every word is 0 again
    for (int i = tid; i < biases; i += kThreads) {
      const uint32_t at = (uint32_t)ids[i] - (uint32_t)base;
      if (at < (uint32_t)left) atomicMax(&words[at], (uint32_t)i + 1);
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < kPer; g++) {
      const uint4 w4 = *reinterpret_cast<const uint4 *>(&words[4 * (g * kThreads + tid)]);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (w[j]) x[g][j] = x[g][j] + values[w[j] - 1];
    }
  }
#pragma unroll
  for (int g = 0; g < kPer; g++) {
    const int i = 4 * (g * kThreads + tid);
    float4u v;
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = (allowed[g] >> j & 1) ? x[g][j] : -__builtin_inff();
    if (i + 4 <= left) {
      *reinterpret_cast<float4u *>(out + i) = v;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (i + j < left) out[i + j] = v[j];
    }
  }
}

}  // namespace

hipError_t launch_logit_rules(const LogitRulesArgs &a, hipStream_t s) {
  if (a.rows < 1 || a.rows > 65535 || a.n < 1) return hipErrorInvalidValue;
  const dim3 grid((a.n + kSlice - 1) / kSlice, a.rows);
  if (a.softcap > 0.0)
    hipLaunchKernelGGL(logit_rules_kernel<true>, grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL(logit_rules_kernel<false>, grid, dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace hp
