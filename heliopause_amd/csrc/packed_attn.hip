// packed_attn.hip -- causal attention over whole prompts that lie end to end
// in one batch: row i of a sequence attends its keys j <= i (of the last
// `window`), out = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j - m), in one
// pass over the keys with a running maximum and sum.
//
// The matrix cores bound it (4 D flop a pair and head), with the vector unit
// close behind: every pair costs one exponential, a quarter-rate instruction.
//
// A workgroup is 128 query rows of one head, 32 for each of its four waves,
// and walks the keys in tiles of kKeys through LDS, double buffered: tile t +
// 1 goes from memory straight into LDS while tile t is worked on.  Two
// workgroups share a CU, and one's products run under the other's softmax.
// Per 32 keys a wave forms, on v_mfma_f32_32x32x16,
//   S^T = K Q^T: the keys are the A rows, read as they lie; the query is the
//     B operand, in registers throughout.  Lane (n, h) then has query row n's
//     scores for keys 8 b + 4 h + {0..3}, b = 0..3;
//   O^T += V^T P^T: the lane's own probabilities are the B operand, so they
//     never leave its registers; V^T comes out of LDS through the transposing
//     read (four keys of one element a lane), in the same order of the keys.
// Rows of a tile are XORed by 16-byte chunks so that both reads touch every
// bank once.
//
// The probabilities are rounded to the operands' type for the second product
// and the normaliser adds the rounded ones, so that the weights of a row still
// sum to one; scores, maximum, sums and output stay f32 until the end.  The
// running maximum moves only when a tile passes it by more than 2^8 (p stays
// below 2^8), so most tiles skip the rescaling.
//
// Masked places are not read into the result whatever they hold: scores there
// become -inf, and where a tile has masked keys its values' infinities and
// NaNs are taken out of the product (0 * inf) and added back for the rows
// that do see them.
#include <type_traits>

#include "hp_mfma.h"
#include "hp_serving.h"

namespace hp {

namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kWaveRows = 32, kRows = kPackedRows;
static_assert(kRows == kWaveRows * kWaves, "a block of rows");
constexpr int kXcds = 8;
constexpr int kWaitLoads = 0x0f70;  // s_waitcnt vmcnt(0)
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLazy = 8.0f;
constexpr float kInf = __builtin_inff();

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t *lds_ptr;

template <bool BF>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// Two f32 as a pair of the operand type, and acc + their rounded values.
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (BF) {
    bf16x2 v;
    v[0] = (__bf16)lo;
    v[1] = (__bf16)hi;
    return __builtin_bit_cast(uint32_t, v);
  }
  halfx2 v;
  v[0] = (_Float16)lo;
  v[1] = (_Float16)hi;
  return __builtin_bit_cast(uint32_t, v);
}
template <bool BF>
__device__ __forceinline__ float add2(uint32_t pair, float acc) {
  if (BF)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, 0x3f803f80u), acc,
                                           false);
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(halfx2, pair), __builtin_bit_cast(halfx2, 0x3c003c00u), acc, false);
}

// The other half's value of a query row (lane ^ 32) and this lane's, in an
// order that a symmetric operation does not see.
__device__ __forceinline__ void halves(float v, float *x, float *y) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  *x = __builtin_bit_cast(float, r0);
  *y = __builtin_bit_cast(float, r1);
}

// Bits 15 and 31 where the low and the high half of w are infinities or NaNs
// (exponents all ones: one more in their last place carries); others are free.
template <bool BF>
__device__ __forceinline__ uint32_t nonfinite(uint32_t w) {
  return BF ? (w & 0x7f807f80u) + 0x00800080u : (w & 0x7c007c00u) + 0x04000400u;
}

// The halves of w that are of a kind -- 0: numbers, as they are; 1: +inf, 2:
// -inf, 3: NaN, as ones -- and zeros for the others.
template <bool BF>
__device__ __forceinline__ uint32_t only_kind(uint32_t w, int kind) {
  const uint32_t inf = BF ? 0x7f80u : 0x7c00u, one = BF ? 0x3f80u : 0x3c00u;
  uint32_t x = 0;
#pragma unroll
  for (int b = 0; b < 2; b++) {
    const uint32_t v = w >> (16 * b) & 0xffffu;
    const int is = (v & inf) != inf ? 0 : v == inf ? 1 : v == (inf | 0x8000u) ? 2 : 3;
    x |= (is == kind ? (kind == 0 ? v : one) : 0u) << (16 * b);
  }
  return x;
}

// 16 bytes a lane from base + offset into LDS, at `lds` (the same for the wave)
// and on by lane.  As assembly, so that the compiler does not take reads of
// the tile at hand to need the next one, which it cannot tell apart; the wait
// is the loop's own.  Nothing comes back in a register; m0 (the LDS address,
// one wait state ahead of its use) is as it was afterwards.
__device__ __forceinline__ void load_to_lds(const uint8_t *base, uint32_t offset, uint32_t lds) {
  uint32_t m0;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %3\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(m0)
      : "v"(offset), "s"(base), "s"(lds)
      : "memory");
}

// Chunk (16 bytes) where a tile's row keeps chunk c, for keys and values.  Keys
// are read 16 rows at a time at one chunk, values 4 rows at 4 chunks.
template <int D>
__device__ __forceinline__ int key_swizzle(int row) {
  return D == 64 ? (row >> 1) & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int value_swizzle(int row) {
  return D == 64 ? (row & 2) << 1 : (row & 3) << 2;
}

template <int D>
struct Shape {
  static constexpr int kKeys = D == 256 ? 32 : 64;     // of a tile
  static constexpr int kRowBytes = 2 * D, kChunks = D / 8;
  static constexpr int kTileBytes = kKeys * kRowBytes;  // of K or V
  static constexpr int kLoads = kTileBytes / 1024 / kWaves;  // 16-byte loads a lane, of K or V
  static constexpr int kLoadRows = 1024 / kRowBytes;    // rows of one load of a wave
};

template <int D, bool BF>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void packed_attn_kernel(const PackedAttnArgs a, int slots) {
  using S = Shape<D>;
  constexpr int kKeys = S::kKeys, kSubs = kKeys / 32, kRowBytes = S::kRowBytes;
  __shared__ __align__(1024) uint8_t lds[2][2][S::kTileBytes];  // [buffer][K, V]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, h = lane >> 5;

  // Work: (slot, KV head) units from the last slot down -- a sequence's last
  // rows have the most keys -- dealt round the XCDs, the heads of a unit one
  // after another on one XCD, whose L2 then has the keys that they share.
  const int group = a.nq / a.nkv;
  const int r = blockIdx.x / kXcds;
  const int unit = r / group * kXcds + blockIdx.x % kXcds;
  if (unit >= slots * a.nkv) return;
  const int slot = slots - 1 - unit / a.nkv, kvh = unit % a.nkv, head = kvh * group + r % group;

  int seq;
  {
    int lo = 0, n = a.sequences;  // the largest whose first block is not behind `slot`
    while (n > 64) {
      const int step = (n + 63) >> 6, at = lo + min(lane * step, n - 1);
      const bool le = lane * step < n && packed_first_block(a.offsets[at], at) <= slot;
      const int c = max(__popcll(__ballot(le)), 1) - 1;
      lo += c * step;
      n = min(step, n - c * step);
    }
    const int at = lo + min(lane, n - 1);
    const bool le = lane < n && packed_first_block(a.offsets[at], at) <= slot;
    seq = lo + max(__popcll(__ballot(le)), 1) - 1;
  }
  const int begin = a.offsets[seq], end = min(a.offsets[seq + 1], a.tokens);
  if (begin < 0 || begin >= end) return;
  const int64_t row_at = (slot - packed_first_block(begin, seq)) * kRows;
  const int len = end - begin;
  if (row_at < 0 || row_at >= len) return;
  const int row0 = (int)row_at;                         // the workgroup's first row
  const int wave0 = row0 + kWaveRows * wave;            // the wave's
  const int row = wave0 + n32;                          // the lane's
  const int window = a.window > 0 ? a.window : 0x7fffffff;
  const int first = max(row - min(row, window - 1), 0);  // first key of the lane's row
  const int tile_first = max(row0 - min(row0, window - 1), 0) / kKeys * kKeys;
  const int tile_stop = min(len, row0 + kRows);

  const uint8_t *kp = static_cast<const uint8_t *>(a.k) + ((int64_t)begin * a.k_stride + kvh * D) * 2;
  const uint8_t *vp = static_cast<const uint8_t *>(a.v) + ((int64_t)begin * a.v_stride + kvh * D) * 2;

  // A lane's part of a tile: load i of this wave brings rows kTurn i + kLoadRows
  // wave + lane / kChunks, LDS chunk lane % kChunks.  Rows behind the sequence
  // are its last, and masked.
  constexpr int kTurn = S::kLoadRows * kWaves;
  const int load_row = S::kLoadRows * wave + lane / S::kChunks, load_chunk = lane % S::kChunks;
  const uint32_t k_row = (uint32_t)a.k_stride * 2, v_row = (uint32_t)a.v_stride * 2;
  const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_ptr)&lds[0][0][0] + 1024 * wave;
  // (the rows of one load of all waves repeat the swizzles', but for heads of
  // 256 every second time)
  constexpr int kKinds = kTurn % 16 == 0 ? 1 : 2;
  static_assert(kTurn * kKinds % 16 == 0, "the swizzles' period");
  uint32_t k_at[kKinds], v_at[kKinds];
#pragma unroll
  for (int i = 0; i < kKinds; i++) {
    const int rr = load_row + kTurn * i;
    k_at[i] = load_row * k_row + 16 * (load_chunk ^ key_swizzle<D>(rr));
    v_at[i] = load_row * v_row + 16 * (load_chunk ^ value_swizzle<D>(rr));
  }
  auto load_tile = [&](int key, int buffer) {
    const uint8_t *kb = kp + (int64_t)key * k_row, *vb = vp + (int64_t)key * v_row;
    const int over = key + kKeys - len;  // rows behind the sequence
    if (over <= 0) {                     // the same for the workgroup
#pragma unroll
      for (int i = 0; i < S::kLoads; i++) {
        const uint32_t at = lds_at + (uint32_t)(buffer * 2 * S::kTileBytes + 1024 * kWaves * i);
        load_to_lds(kb + (uint32_t)(kTurn * i) * (uint64_t)k_row, k_at[i % kKinds], at);
        load_to_lds(vb + (uint32_t)(kTurn * i) * (uint64_t)v_row, v_at[i % kKinds], at + S::kTileBytes);
      }
    } else {
#pragma unroll
      for (int i = 0; i < S::kLoads; i++) {
        const uint32_t at = lds_at + (uint32_t)(buffer * 2 * S::kTileBytes + 1024 * kWaves * i);
        const int from = min(load_row + kTurn * i, kKeys - 1 - over) - load_row;
        load_to_lds(kb, k_at[i % kKinds] + from * k_row, at);
        load_to_lds(vb, v_at[i % kKinds] + from * v_row, at + S::kTileBytes);
      }
    }
  };
  load_tile(tile_first, 0);

  u32x4 q[D / 16];
  {
    const int64_t at = (int64_t)(begin + min(row, len - 1)) * a.q_stride + head * D + 8 * h;
#pragma unroll
    for (int i = 0; i < D / 16; i++)
      q[i] = *reinterpret_cast<const u32x4 *>(static_cast<const uint8_t *>(a.q) + (at + 16 * i) * 2);
  }
  const float factor = a.scale * kLog2e;
  f32x16 acc[D / 32];
#pragma unroll
  for (int t = 0; t < D / 32; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) acc[t][i] = 0.0f;
  float m = -kInf, l = 0.0f;

  // One tile in LDS: scores, weights, products with the values.
  auto work = [&](int key, int buffer, auto edge) {
    constexpr bool kMasked = decltype(edge)::value;
    const uint8_t *kt = lds[buffer][0];
    const uint8_t *vt = lds[buffer][1];
    f32x16 s[kSubs];
#pragma unroll
    for (int u = 0; u < kSubs; u++) {
#pragma unroll
      for (int i = 0; i < 16; i++) s[u][i] = 0.0f;
      const int kr = 32 * u + n32;
#pragma unroll
      for (int i = 0; i < D / 16; i++) {
        const u32x4 kf =
            *reinterpret_cast<const u32x4 *>(kt + kr * kRowBytes + 16 * ((2 * i + h) ^ key_swizzle<D>(kr)));
        s[u] = mfma32<BF>(kf, q[i], s[u]);
      }
    }
    if (kMasked) {
      // the lane's key 32 u + 8 (i / 4) + i % 4 of the tile, from its first
      const int to = row - key - 4 * h, from = first - key - 4 * h;
#pragma unroll
      for (int u = 0; u < kSubs; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int j = 32 * u + 8 * (i >> 2) + (i & 3);
          s[u][i] = j > to ? -kInf : s[u][i];
        }
      if (from > -kKeys) {
#pragma unroll
        for (int u = 0; u < kSubs; u++)
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int j = 32 * u + 8 * (i >> 2) + (i & 3);
            s[u][i] = j < from ? -kInf : s[u][i];
          }
      }
    }
    float most = s[0][0];
#pragma unroll
    for (int u = 0; u < kSubs; u++)
#pragma unroll
      for (int i = 0; i < 16; i++) most = fmaxf(most, s[u][i]);
    {
      float x, y;
      halves(most, &x, &y);
      most = fmaxf(x, y) * factor;
    }
    if (__any(most > m + kLazy)) {
      const float m_new = most > m + kLazy ? most : m;
      const float alpha = m_new == m ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int t = 0; t < D / 32; t++) acc[t] *= alpha;
    }
    const float m_use = m == -kInf ? 0.0f : m;  // no key so far: exp2(-inf)
    u32x4 p[2 * kSubs];
#pragma unroll
    for (int u = 0; u < kSubs; u++)
#pragma unroll
      for (int w = 0; w < 8; w++) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][2 * w], factor, -m_use));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][2 * w + 1], factor, -m_use));
        const uint32_t pair = pack2<BF>(p0, p1);
        l = add2<BF>(pair, l);
        p[2 * u + (w >> 2)][w & 3] = pair;
      }
    // V^T fragments: product jj's k index 8 h + i is key 16 jj + 4 h + i (i < 4)
    // and 16 jj + 8 + 4 h + i - 4; a lane of 16 reads 8 bytes of key row
    // (lane % 16) / 4, elements 4 (lane % 4) .. of its 16
    const int vr = 4 * h + ((lane & 15) >> 2);
    const int vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), vb = 8 * (lane & 1);
    auto value_frag = [&](int jj, int t) -> u32x4 {
      u32x4 f;
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const int rr = 16 * jj + 8 * b + vr;
        const uint8_t *at = vt + rr * kRowBytes + 16 * ((4 * t + vc) ^ value_swizzle<D>(rr)) + vb;
        const short4v w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) short4v *)(lds_ptr)at);
        const uint2 w2 = __builtin_bit_cast(uint2, w);
        f[2 * b] = w2.x;
        f[2 * b + 1] = w2.y;
      }
      return f;
    };
    bool odd = false;
#pragma unroll
    for (int jj = 0; jj < 2 * kSubs; jj++) {
      u32x4 f[D / 32];
#pragma unroll
      for (int t = 0; t < D / 32; t++) f[t] = value_frag(jj, t);
      if (kMasked) {  // (a weight of 0 times an infinity would be a NaN)
        uint32_t bad = 0;
#pragma unroll
        for (int t = 0; t < D / 32; t++)
#pragma unroll
          for (int w = 0; w < 4; w++) bad |= nonfinite<BF>(f[t][w]);
        if (__any((bad & 0x80008000u) != 0)) {
          odd = true;
#pragma unroll
          for (int t = 0; t < D / 32; t++)
#pragma unroll
            for (int w = 0; w < 4; w++) f[t][w] = only_kind<BF>(f[t][w], 0);
        }
      }
#pragma unroll
      for (int t = 0; t < D / 32; t++) acc[t] = mfma32<BF>(f[t], p[jj], acc[t]);
    }
    if (kMasked && odd) {
      // what infinities and NaNs come to in the rows that see them: the weights
      // of +inf, of -inf and of NaN, each as a product of its own
#pragma unroll 1
      for (int kind = 1; kind < 4; kind++) {
        const float add = kind == 1 ? kInf : kind == 2 ? -kInf : __builtin_nanf("");
#pragma unroll
        for (int t = 0; t < D / 32; t++) {
          f32x16 weight;
#pragma unroll
          for (int i = 0; i < 16; i++) weight[i] = 0.0f;
#pragma unroll
          for (int jj = 0; jj < 2 * kSubs; jj++) {
            u32x4 f = value_frag(jj, t);
#pragma unroll
            for (int w = 0; w < 4; w++) f[w] = only_kind<BF>(f[w], kind);
            weight = mfma32<BF>(f, p[jj], weight);
          }
#pragma unroll
          for (int i = 0; i < 16; i++) acc[t][i] += weight[i] > 0.0f ? add : 0.0f;
        }
      }
    }
  };
  // This wave's part of tile `key` is in LDS after the wait; after the barrier
  // every wave's is, and the other buffer has no reader left: the tile after
  // goes there.
  auto next_tile = [&](int key, int buffer) {
    __builtin_amdgcn_s_waitcnt(kWaitLoads);
    __syncthreads();
    if (key + kKeys < tile_stop) load_tile(key + kKeys, buffer ^ 1);
  };
  // Tiles of which every row of the workgroup sees every key, in a loop of their
  // own; the others mask.
  const int whole_first = (row0 + kRows - min(row0 + kRows, window) + kKeys - 1) / kKeys * kKeys;
  const int whole_stop = (row0 + 1) / kKeys * kKeys;
  int buffer = 0;
  for (int key = tile_first; key < tile_stop;) {
    if (key >= whole_first && key < whole_stop) {
      for (; key < whole_stop; key += kKeys, buffer ^= 1) {
        next_tile(key, buffer);
        work(key, buffer, std::false_type{});
      }
      continue;
    }
    next_tile(key, buffer);
    // (what the wave's rows see of it, the same for the wave)
    if (key <= wave0 + kWaveRows - 1 && key + kKeys - 1 >= wave0 - min(wave0, window - 1)) work(key, buffer, std::true_type{});
    key += kKeys;
    buffer ^= 1;
  }

  float x, y;
  halves(l, &x, &y);
  l = x + y;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (row >= len) return;
  const int64_t o = (int64_t)(begin + row) * a.out_stride + head * D;
#pragma unroll
  for (int t = 0; t < D / 32; t++)
#pragma unroll
    for (int b = 0; b < 4; b++) {
      const float v[4] = {acc[t][4 * b] * inv, acc[t][4 * b + 1] * inv, acc[t][4 * b + 2] * inv, acc[t][4 * b + 3] * inv};
      store4(a.out, o + 32 * t + 8 * b + 4 * h, a.out_type, v);
    }
}

int64_t slots_of(const PackedAttnArgs &a) { return packed_blocks(a.tokens, a.sequences); }
int64_t grid_of(const PackedAttnArgs &a) {
  return (slots_of(a) * a.nkv + kXcds - 1) / kXcds * kXcds * (a.nq / a.nkv);
}

template <int D>
hipError_t launch(const PackedAttnArgs &a, hipStream_t s) {
  const int64_t slots = slots_of(a), grid = grid_of(a);
  if (a.type == kElemBf16)
    hipLaunchKernelGGL((packed_attn_kernel<D, true>), dim3((unsigned)grid), dim3(kThreads), 0, s, a, (int)slots);
  else
    hipLaunchKernelGGL((packed_attn_kernel<D, false>), dim3((unsigned)grid), dim3(kThreads), 0, s, a, (int)slots);
  return hipGetLastError();
}

}  // namespace

// (a launch has fewer than 2^32 threads in a dimension)
bool packed_attn_fits(const PackedAttnArgs &a) { return grid_of(a) <= 0xffffffffll / kThreads; }

hipError_t launch_packed_attn(const PackedAttnArgs &a, hipStream_t s) {
  if (a.tokens < 1 || a.sequences < 1 || a.nkv < 1 || a.nq % a.nkv != 0 || !packed_attn_fits(a))
    return hipErrorInvalidValue;
  switch (a.head_dim) {
    case 64: return launch<64>(a, s);
    case 128: return launch<128>(a, s);
    case 256: return launch<256>(a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace hp
