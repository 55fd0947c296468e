// packed_attn.hip -- causal attention over whole prompts that lie end to end
// in one batch: row i of a sequence attends its keys j <= i (of the last
// `window`), out = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j - m), in one
// pass over the keys with a running maximum and sum.
//
// The matrix cores bound it (4 D flop a pair and head), with the vector unit
// close behind: every pair costs one exponential, a quarter-rate instruction.
// 16384 rows of 16 heads of 128, bf16: 1.1 TFLOP in 1000 to 1080 us, 1020 to 1100
// TFLOP/s, by the clock that the card's power leaves it (1190 us at 1.53 GHz, the
// matrix cores busy 58 % of the cycles; a large library matrix product reaches
// 1212); 15 prompts of 12345 rows, 32 heads: 111 GFLOP in 150 to 160 us, 690 to
// 740 TFLOP/s (169 us at 1.96 GHz, 35 %), a quarter of their tiles being the
// diagonal's.
//
// A workgroup is 32 query rows for each of its four waves -- 32 rows of four
// heads that share their keys, 64 of two or 128 of one, by what the heads of a
// group divide into -- and walks the keys in tiles of kKeys through LDS, double
// buffered: the next tiles go from memory straight into LDS while one is worked
// on.  The more heads, the fewer tiles of the diagonal, of a window's edge and
// behind a prompt's end its waves wait through (8 prompts of 2000 rows, 32 / 8
// heads of 128: one head 25.1 us, four 22.3; windows of 500 on 8000 rows of half as
// many 58.2 and 56.0).  Query rows come in and, where blocks fill the card, output rows leave
// through LDS, whole rows a load or store and not 16 bytes of each (the same
// prompts to 19.6, the windows to 52.6; 40 rows of heads of 128 6.0 -> 6.3).
// Up to heads of 128 two workgroups share a CU; the scores of the next tile are
// formed ahead of this one's weights, so that a wave's products run under its
// exponentials as well (heads of 256, one wave a SIMD: 192 -> 166 us on six
// prompts of 9000 rows).  Tiles for heads of 256 are 32 keys, whose one
// accumulator would chain sixteen products: even and odd ones go to one each
// (the same prompts 164 -> 152 us; tiles of 64 keys instead 179).
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
// sum to one; scores, maximum, sums and output stay f32 until the end.  One part
// a weight is off by half a step of its type at most, also where outputs leave as
// f32, and the steps of a row's keys average out: 16-bit outputs are 2.2e-4 (f16,
// 77 rows of heads of 256) and 1.9e-3 (bf16, the batches above) of their size from
// those of 64 bits, and would be 2.0e-4 and 1.7e-3 with f32 weights.  A second
// part, which the one-token kernel has under its bytes, is a third product here:
// 151 -> 196 us on the ragged batch, 1000 -> 1408 on the long prompt, 103 -> 132
// on 4000 rows of heads of 256, 48 -> 71 on 6000 of heads of 64.
//
// The running maximum moves only when a tile passes it by more than 2^8 (p stays
// below 2^8), so most tiles skip the rescaling.  f16 weights carry a factor 2^7
// beside, which cancels: they stay below 2^15, and what is lost of a small one in
// f16's subnormal steps is 2^-32 of the running maximum and not 2^-25, which some
// thousands of keys behind a heavy one would add up to what f16 shows.
//
// Masked places are not read into the result whatever they hold: scores there
// become -inf, and where a tile has masked keys its values' infinities and
// NaNs are taken out of the product (0 * inf) and added back for the rows
// that do see them, as a tile without masked keys has them (a NaN where the
// weight is 0).
#include <type_traits>

#include "hp_mfma.h"
#include "hp_serving.h"

namespace hp {

namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kWaveRows = 32;
constexpr int kXcds = 8;
constexpr int kWaitLoads = 0x0f70;  // s_waitcnt vmcnt(0)
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLazy = 8.0f;
constexpr float kBiasF16 = 7.0f;  // f16 weights carry 2^kBiasF16
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

// The same from a lane's own address.
__device__ __forceinline__ void load_to_lds(const uint8_t *at, uint32_t lds) {
  uint32_t m0;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %2\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(m0)
      : "v"(at), "s"(lds)
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

// Heads of D, the keys of a block split over G groups of waves.
template <int D, int G>
struct Shape {
  static constexpr int kGroupWaves = kWaves / G, kRows = kWaveRows * kGroupWaves;  // (query row, head) pairs of a workgroup
  static constexpr int kKeys = D == 256 ? 32 : 64;                                 // of a tile
  static constexpr int kRowBytes = 2 * D, kChunks = D / 8;
  static constexpr int kTileBytes = kKeys * kRowBytes;            // of K or V
  static constexpr int kLoads = kTileBytes / 1024 / kGroupWaves;  // 16-byte loads a lane, of K or V
  static constexpr int kLoadRows = 1024 / kRowBytes;              // rows of one load of a wave
  static constexpr int kQueryBytes = kRows * kRowBytes;           // of a group's query rows
  // (they come through the place of the second V and, where they are more, on)
  static constexpr int kSpare = kQueryBytes > kTileBytes ? kQueryBytes - kTileBytes : 0;
};

template <int D, bool BF, int G>
__global__ __launch_bounds__(kThreads, D * G >= 256 ? 1 : 2) void packed_attn_kernel(const PackedAttnArgs a, int slots,
                                                                                int heads_log2) {
  using S = Shape<D, G>;
  constexpr int kKeys = S::kKeys, kSubs = kKeys / 32, kRowBytes = S::kRowBytes;
  const int head_rows = 1 << (__builtin_ctz(S::kRows) - heads_log2);  // query rows of each of the workgroup's heads
  __shared__ __align__(1024) uint8_t lds_all[G][4 * S::kTileBytes + S::kSpare];  // [group]: buffer 0's K, V, 1's K, V
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n32 = lane & 31, h = lane >> 5;
  const int part = wave / S::kGroupWaves, member = wave % S::kGroupWaves;  // group of waves, place in it
  auto tile_of = [&](int buffer, int value) { return &lds_all[part][(2 * buffer + value) * S::kTileBytes]; };

  // Work: (slot, KV head) units from the last slot down -- a sequence's last
  // rows have the most keys -- dealt round the XCDs, the heads of a unit one
  // after another on one XCD, whose L2 then has the keys that they share.
  const int group = a.nq / a.nkv, bundles = group >> heads_log2;
  const int r = blockIdx.x / kXcds;
  const int unit = r / bundles * kXcds + blockIdx.x % kXcds;
  if (unit >= slots * a.nkv) return;
  const int slot = slots - 1 - unit / a.nkv, kvh = unit % a.nkv;
  const int head = kvh * group + (r % bundles << heads_log2) + member % (1 << heads_log2);  // the wave's

  int seq, begin, end;
  {
    int lo = 0, n = a.sequences;  // the largest whose first block is not behind `slot`
    while (n > 64) {
      const int step = (n + 63) >> 6, at = lo + min(lane * step, n - 1);
      const bool le = lane * step < n && packed_first_block(a.offsets[at], at, head_rows) <= slot;
      const int c = max(__popcll(__ballot(le)), 1) - 1;
      lo += c * step;
      n = min(step, n - c * step);
    }
    const int at = lo + min(lane, n - 1), o0 = a.offsets[at], o1 = a.offsets[at + 1];
    const bool le = lane < n && packed_first_block(o0, at, head_rows) <= slot;
    const int c = max(__popcll(__ballot(le)), 1) - 1;
    seq = lo + c;
    begin = __builtin_amdgcn_readlane(o0, c);
    end = min(__builtin_amdgcn_readlane(o1, c), a.tokens);
  }
  if (begin < 0 || begin >= end) return;
  const int64_t row_at = (slot - packed_first_block(begin, seq, head_rows)) * head_rows;
  const int len = end - begin;
  if (row_at < 0 || row_at >= len) return;
  const int row0 = (int)row_at;                         // the workgroup's first row
  const int wave0 = row0 + kWaveRows * (member >> heads_log2);           // the wave's
  const int row = wave0 + n32;                          // the lane's
  const int window = a.window > 0 ? a.window : 0x7fffffff;
  const int first = max(row - min(row, window - 1), 0);  // first key of the lane's row
  const int tile_first = max(row0 - min(row0, window - 1), 0) / kKeys * kKeys;
  const int tile_stop = min(len, row0 + head_rows);

  const uint8_t *kp = static_cast<const uint8_t *>(a.k) + ((int64_t)begin * a.k_stride + kvh * D) * 2;
  const uint8_t *vp = static_cast<const uint8_t *>(a.v) + ((int64_t)begin * a.v_stride + kvh * D) * 2;

  // A lane's part of a tile: load i of this wave brings rows kTurn i + kLoadRows
  // member + lane / kChunks, LDS chunk lane % kChunks.  Rows behind the sequence
  // are its last, and masked.
  constexpr int kTurn = S::kLoadRows * S::kGroupWaves;
  const int load_row = S::kLoadRows * member + lane / S::kChunks, load_chunk = lane % S::kChunks;
  const uint32_t k_row = (uint32_t)a.k_stride * 2, v_row = (uint32_t)a.v_stride * 2;
  const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_ptr)tile_of(0, 0) + 1024 * member;
  // (the rows of one load of the group repeat the swizzles' after kKinds)
  constexpr int kKinds = kTurn >= 16 ? 1 : 16 / kTurn;
  static_assert(kTurn * kKinds % 16 == 0, "the swizzles' period");
  uint32_t k_at[kKinds], v_at[kKinds];
#pragma unroll
  for (int i = 0; i < kKinds; i++) {
    const int rr = load_row + kTurn * i;
    k_at[i] = load_row * k_row + 16 * (load_chunk ^ key_swizzle<D>(rr));
    v_at[i] = load_row * v_row + 16 * (load_chunk ^ value_swizzle<D>(rr));
  }
  auto load_rows = [&](const uint8_t *rows, uint32_t row_bytes, const uint32_t (&at)[kKinds], int key, uint32_t lds) {
    const uint8_t *base = rows + (int64_t)key * row_bytes;
    const int over = key + kKeys - len;  // rows behind the sequence
    if (over <= 0) {                     // the same for the workgroup
#pragma unroll
      for (int i = 0; i < S::kLoads; i++)
        load_to_lds(base + (uint32_t)(kTurn * i) * (uint64_t)row_bytes, at[i % kKinds], lds + 1024 * S::kGroupWaves * i);
    } else {
#pragma unroll
      for (int i = 0; i < S::kLoads; i++) {
        const int from = min(load_row + kTurn * i, kKeys - 1 - over) - load_row;
        load_to_lds(base, at[i % kKinds] + from * row_bytes, lds + 1024 * S::kGroupWaves * i);
      }
    }
  };
  auto load_keys = [&](int key, int buffer) { load_rows(kp, k_row, k_at, key, lds_at + buffer * 2 * S::kTileBytes); };
  auto load_values = [&](int key, int buffer) {
    load_rows(vp, v_row, v_at, key, lds_at + (buffer * 2 + 1) * S::kTileBytes);
  };

  // The wave's query rows (behind the sequence: its last) come through LDS, where
  // the second values will be and on, so that a load is whole rows.
  const uint8_t *own_q = tile_of(1, 1) + member * (kWaveRows * kRowBytes);
#pragma unroll
  for (int i = 0; i < kWaveRows; i += S::kLoadRows) {
    const int rr = i + lane / S::kChunks;
    const int64_t at = (int64_t)(begin + min(wave0 + rr, len - 1)) * a.q_stride + head * D;
    load_to_lds(static_cast<const uint8_t *>(a.q) + at * 2 + 16 * (load_chunk ^ key_swizzle<D>(rr)),
                (uint32_t)(uintptr_t)(lds_ptr)own_q + i * kRowBytes);
  }
  // Group `part` has the tiles part, part + G, ... : its tile i is key_of(i).
  const int tiles = (tile_stop - tile_first + kKeys - 1) / kKeys;
  const int turns = (tiles + G - 1) / G, mine = (tiles - part + G - 1) / G;
  auto key_of = [&](int i) { return tile_first + (i * G + part) * kKeys; };
  if (mine > 0) {
    load_keys(key_of(0), 0);
    load_values(key_of(0), 0);
  }
  if (mine > 1) load_keys(key_of(1), 1);
  const float factor = a.scale * kLog2e;
  f32x16 acc[D / 32];
#pragma unroll
  for (int t = 0; t < D / 32; t++)
#pragma unroll
    for (int i = 0; i < 16; i++) acc[t][i] = 0.0f;
  float m = -kInf, l = 0.0f;
  constexpr float kBias = BF ? 0.0f : kBiasF16;
  // weigh's s * factor - m, in one rounding, is off from 0 at the maximum by what
  // m's own rounding lost: nothing that counts below 2^22, but past 2^24 whole
  // powers of two, at last an infinity or 0 for every key.  The scores of rows
  // that far out become differences of rounded products, over the factor, as
  // they are settled (on the way of the moving maximum, which costs every other
  // batch the least: 1 %; a test of its own a tile 1 to 4 %).
  float bar = -kInf;   // a score above it is settled apart: past m + kLazy, or any of such a row
  float m_use = 0.0f;  // what weigh takes off (a row without a key so far: exp2(-inf) whatever it is)

  u32x4 q[D / 16];
  // The steps of a tile.  scores: S^T of the keys in LDS.
  auto scores = [&](f32x16 (&s)[kSubs], int buffer) {
    const uint8_t *kt = tile_of(buffer, 0);
    f32x16 odd;  // a second chain of products where there is one subtile
#pragma unroll
    for (int i = 0; i < 16; i++) odd[i] = 0.0f;
#pragma unroll
    for (int u = 0; u < kSubs; u++) {
#pragma unroll
      for (int i = 0; i < 16; i++) s[u][i] = 0.0f;
      const int kr = 32 * u + n32;
#pragma unroll
      for (int i = 0; i < D / 16; i++) {
        const u32x4 kf =
            *reinterpret_cast<const u32x4 *>(kt + kr * kRowBytes + 16 * ((2 * i + h) ^ key_swizzle<D>(kr)));
        if (kSubs == 1 && (i & 1))
          odd = mfma32<BF>(kf, q[i], odd);
        else
          s[u] = mfma32<BF>(kf, q[i], s[u]);
      }
    }
    if (kSubs == 1) s[0] += odd;
  };
  // Whether a row of the wave has a masked key in the tile at `key` (the same for
  // the wave).
  auto edge_at = [&](int key) {
    return key + kKeys - 1 > wave0 || key < wave0 + kWaveRows - min(wave0 + kWaveRows, window);
  };
  // settle: masks them and moves the running maximum where they pass it.
  auto settle = [&](f32x16 (&s)[kSubs], int key, auto edge) {
    constexpr bool kMasked = decltype(edge)::value;
    if (kMasked && edge_at(key)) {
      // the lane's key 32 u + 8 (i / 4) + i % 4 of the tile, from its first
      const int to = row - key - 4 * h, from = first - key - 4 * h;
#pragma unroll
      for (int u = 0; u < kSubs; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int j = 32 * u + 8 * (i >> 2) + (i & 3);
          s[u][i] = j > to ? -kInf : s[u][i];
        }
      if (__any(from > 0)) {
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
    float x, y;
    halves(most, &x, &y);
    most = fmaxf(x, y) * factor;
    if (__any(most > bar)) {
      const float m_new = most > m + kLazy ? most : m;
      const float alpha = m_new == m ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int t = 0; t < D / 32; t++) acc[t] *= alpha;
      const bool far = fabsf(m) >= 0x1p22f && m != -kInf;
      bar = far ? -kInf : m + kLazy;
      m_use = far ? -kBias : m == -kInf ? 0.0f : m - kBias;
      if (__any(far)) {
        const float back = 1.0f / factor;
#pragma unroll
        for (int u = 0; u < kSubs; u++)
#pragma unroll
          for (int i = 0; i < 16; i++) s[u][i] = far ? (s[u][i] * factor - m) * back : s[u][i];
      }
    }
  };
  // weigh: the probabilities, as the B operand of the second product, of scores
  // that are settled.
  auto weigh = [&](const f32x16 (&s)[kSubs], u32x4 (&p)[2 * kSubs]) {
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
  };
  // gather: O^T += V^T P^T with the values in LDS (check: keys may be masked; the
  // tile is then the one at `key`).
  auto gather = [&](u32x4 (&p)[2 * kSubs], int buffer, bool check, int key, auto edge) {
    constexpr bool kMasked = decltype(edge)::value;
    const uint8_t *vt = tile_of(buffer, 1);
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
      if (kMasked && check) {  // (a weight of 0 times an infinity would be a NaN)
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
      // what infinities and NaNs come to in the rows that see them, as in a tile
      // without masked keys: themselves, or a NaN where a weight is 0.  Of a weight
      // its kind is enough, 1 for one above 0, -128 for a 0 that is seen (more than
      // all the tile's others), in a product for each of +inf, -inf and NaN
      int to = row - key - 4 * h, from = first - key - 4 * h;
      // (these formed here and the weights in l by now: kept, they would take
      // registers from the walk)
      asm volatile("" : "+v"(to), "+v"(from), "+v"(l));
#pragma unroll
      for (int jj = 0; jj < 2 * kSubs; jj++)
#pragma unroll
        for (int w = 0; w < 4; w++) {
          uint32_t of = 0;
#pragma unroll
          for (int b = 0; b < 2; b++) {
            const int j = 16 * jj + 8 * (w >> 1) + 2 * (w & 1) + b;
            const uint32_t one = BF ? 0x3f80u : 0x3c00u, none = BF ? 0xc300u : 0xd800u;
            of |= ((p[jj][w] >> (16 * b) & 0xffffu) != 0 ? one : j <= to && j >= from ? none : 0u) << (16 * b);
          }
          p[jj][w] = of;
        }
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
          for (int i = 0; i < 16; i++)
            acc[t][i] += weight[i] > 0.0f ? add : weight[i] < 0.0f ? __builtin_nanf("") : 0.0f;
        }
      }
    }
  };

  // The walk over the tiles: while tile i's weights and values are worked on,
  // the scores of tile i + 1 are formed, so that the matrix cores have work
  // during the exponentials, and keys i + 2 and values i + 1 are on their way
  // into the places of keys i and values i - 1, which no wave reads any more
  // after the barrier.
  auto sees = [&](int i) {  // whether any of the wave's rows has a key in tile i (the same for the wave)
    return i < mine && key_of(i) <= wave0 + kWaveRows - 1 &&
           key_of(i) + kKeys - 1 >= wave0 - min(wave0, window - 1);
  };
  auto next_loads = [&](int i) {
    __builtin_amdgcn_s_waitcnt(kWaitLoads);
    __syncthreads();
    if (i + 2 < mine) load_keys(key_of(i + 2), i & 1);
    if (i + 1 < mine) load_values(key_of(i + 1), (i + 1) & 1);
  };
  // Turns whose tiles every row of the workgroup sees whole.
  const int whole_first =
      (max(row0 + head_rows - min(row0 + head_rows, window) - tile_first + kKeys - 1, 0) / kKeys + G - 1) / G;
  const int whole_stop = (row0 + 1 - tile_first) / kKeys / G;
  f32x16 sa[kSubs], sb[kSubs];
  __builtin_amdgcn_s_waitcnt(kWaitLoads);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < D / 16; i++)
    q[i] = *reinterpret_cast<const u32x4 *>(own_q + n32 * kRowBytes + 16 * ((2 * i + h) ^ key_swizzle<D>(n32)));
  if (sees(0)) {
    scores(sa, 0);
    settle(sa, key_of(0), std::true_type{});
  }
  for (int i = 0; i < turns;) {
    // two at a time, so that each set of scores has its registers
    for (; i % 2 == 0 && i >= whole_first && i + 2 < whole_stop; i += 2) {
      u32x4 p[2 * kSubs];
      next_loads(i);
      scores(sb, 1);
      weigh(sa, p);
      gather(p, 0, false, 0, std::false_type{});
      settle(sb, 0, std::false_type{});
      next_loads(i + 1);
      scores(sa, 0);
      weigh(sb, p);
      gather(p, 1, false, 0, std::false_type{});
      settle(sa, 0, std::false_type{});
    }
    next_loads(i);
    const bool more = sees(i + 1);
    if (more) scores(sb, (i + 1) & 1);
    if (sees(i)) {
      u32x4 p[2 * kSubs];
      weigh(sa, p);
      gather(p, i & 1, edge_at(key_of(i)), key_of(i), std::true_type{});
    }
    if (more) {
      settle(sb, key_of(i + 1), std::true_type{});
#pragma unroll
      for (int u = 0; u < kSubs; u++) sa[u] = sb[u];
    }
    i++;
  }

  {
    float x, y;
    halves(l, &x, &y);
    l = x + y;
  }
  if (G > 1) {
    // the groups' parts of a row, through the tiles' place in LDS: the first
    // group's wave takes the others' in their order
    constexpr int kPart = 64 * (D / 2 + 2);  // floats of a wave: acc, m, l by lane
    float *place = reinterpret_cast<float *>(lds_all);
    static_assert((G - 1) * S::kGroupWaves * kPart * 4 <= (int)sizeof(lds_all), "the parts fit the tiles' place");
    __syncthreads();
    if (part > 0) {
      float *to = place + ((part - 1) * S::kGroupWaves + member) * kPart + lane;
#pragma unroll
      for (int t = 0; t < D / 32; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) to[64 * (16 * t + i)] = acc[t][i];
      to[64 * (D / 2)] = m;
      to[64 * (D / 2 + 1)] = l;
    }
    __syncthreads();
    if (part > 0) return;
#pragma unroll 1
    for (int g = 1; g < G; g++) {
      const float *from = place + ((g - 1) * S::kGroupWaves + member) * kPart + lane;
      const float mg = from[64 * (D / 2)], lg = from[64 * (D / 2 + 1)];
      const float m_new = fmaxf(m, mg);
      const float f = m == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
      const float e = mg == -kInf ? 0.0f : __builtin_amdgcn_exp2f(mg - m_new);
      m = m_new;
      l = l * f + lg * e;
#pragma unroll
      for (int t = 0; t < D / 32; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[t][i] = acc[t][i] * f + from[64 * (16 * t + i)] * e;
    }
  }
  // (every row of a prompt has a key, itself: a sum of 0 is scores of -inf only,
  // and 0 / 0 their softmax)
  const float inv = 1.0f / l;
  // With one group the wave's rows leave through LDS, so that a store is whole
  // rows and not 16 bytes of each: kSpan elements of them at a time, a row of 16
  // bits or half a row of f32, in chunks that are XORed as the keys' are.  With
  // two the launch is a few blocks whose end counts, and this costs more than it
  // gives (77 rows of 8 / 2 heads of 256: 10.2 and 10.9 us).
  if (G == 1) __syncthreads();  // no wave reads the tiles any more
  uint8_t *own = reinterpret_cast<uint8_t *>(lds_all) + wave * (kWaveRows * kRowBytes);
  static_assert(G > 1 || kWaves * kWaveRows * kRowBytes <= (int)sizeof(lds_all), "the rows fit the tiles' place");
  // (the lane anew: addresses that the loads share would take registers through the walk)
  int lane_now = lane;
  asm volatile("" : "+v"(lane_now));
  const int row_now = lane_now & 31, h_now = lane_now >> 5;
  auto store = [&](auto type) {
    constexpr int kType = decltype(type)::value, kE = kType == kElemF32 ? 4 : 2, kSpan = kRowBytes / kE;
    constexpr int kChunkMask = S::kChunks < 16 ? S::kChunks - 1 : 15;
    if (G > 1) {
      if (row >= len) return;
#pragma unroll
      for (int t = 0; t < D / 32; t++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const float v[4] = {acc[t][4 * b] * inv, acc[t][4 * b + 1] * inv, acc[t][4 * b + 2] * inv,
                              acc[t][4 * b + 3] * inv};
          store4(a.out, (int64_t)(begin + row) * a.out_stride + head * D + 32 * t + 8 * b + 4 * h, kType, v);
        }
      return;
    }
#pragma unroll
    for (int from = 0; from < D; from += kSpan) {
#pragma unroll
      for (int t = from / 32; t < (from + kSpan) / 32; t++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const float v[4] = {acc[t][4 * b] * inv, acc[t][4 * b + 1] * inv, acc[t][4 * b + 2] * inv,
                              acc[t][4 * b + 3] * inv};
          const int at = (32 * t + 8 * b + 4 * h_now - from) * kE;  // bytes of the row
          store4(own + row_now * kRowBytes + 16 * ((at >> 4) ^ (row_now & kChunkMask)) + (at & 15), 0, kType, v);
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // one lane's writes are another's reads
#pragma unroll
      for (int i = 0; i < kWaveRows; i += S::kLoadRows) {
        const int r = i + lane_now / S::kChunks, c = lane_now % S::kChunks;
        const u32x4 w = *reinterpret_cast<const u32x4 *>(own + r * kRowBytes + 16 * (c ^ (r & kChunkMask)));
        if (wave0 + r < len)
          *reinterpret_cast<u32x4 *>(static_cast<uint8_t *>(a.out) +
                                     ((int64_t)(begin + wave0 + r) * a.out_stride + head * D + from) * kE + 16 * c) = w;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  };
  if (a.out_type == kElemF32)
    store(std::integral_constant<int, kElemF32>{});
  else if (a.out_type == kElemF16)
    store(std::integral_constant<int, kElemF16>{});
  else
    store(std::integral_constant<int, kElemBf16>{});
}

// Groups of waves that the keys of a block are split over.  128 (row, head)
// pairs with the waves side by side read each key once for the most rows, which
// is best where the blocks fill the card.  Where they do not, the block with the
// most keys is what a launch takes, and blocks of 64 with two groups walk half of
// them each.  Blocks are counted from the rows, and two more for every further
// prompt: it ends inside a block, and makes the longest walk shorter, of which
// the split takes its half.  Measured with one group and two, us:
//   heads of 64: one prompt, 280 blocks 36.8 and 22.5, 512 31.7 and 31.5, 672
//     42.3 and 45.8; eight prompts, 704 9.1 and 10.2;
//   heads of 128, whose CU then has one workgroup: one prompt, 224 blocks 59.9
//     and 48.4 (8 heads) or 20.1 and 22.3 (32 heads), 288 77.1 and 79.3; three
//     prompts, 224 31.9 and 25.9; six prompts, 352 15.0 and 18.9;
//   heads of 256: one prompt, 256 blocks 132 and 102, 304 157 and 150, 352 186
//     and 194; ten prompts, 240 18.0 and 16.7, 304 25.2 and 27.9.
// Up to one tile of rows there is nothing to split (40 rows: heads of 128 6.3 and
// 7.6, of 256 8.8 and 9.4, but of 64 5.7 and 5.3).
int groups_of(const PackedAttnArgs &a, int num_cus) {
  const int64_t blocks = ((int64_t)a.tokens / (kWaveRows * kWaves) + 2 * (int64_t)a.sequences - 1) * a.nq;
  if (a.head_dim > 64 && a.tokens <= 64) return 1;
  return 8 * blocks < (a.head_dim == 64 ? 18 : a.head_dim == 128 ? 8 : 9) * (int64_t)num_cus ? 2 : 1;
}

// log2 of the heads that a workgroup has: as many as divide a KV head's and its
// waves (of a group of waves).
int heads_log2_of(const PackedAttnArgs &a, int groups) {
  const int group = a.nq / a.nkv;
  return group % 4 == 0 && groups == 1 ? 2 : group % 2 == 0 ? 1 : 0;
}
int64_t slots_of(const PackedAttnArgs &a, int groups) {
  return packed_blocks(a.tokens, a.sequences, (kWaveRows * kWaves / groups) >> heads_log2_of(a, groups));
}
int64_t grid_of(const PackedAttnArgs &a, int groups) {
  return (slots_of(a, groups) * a.nkv + kXcds - 1) / kXcds * kXcds * ((a.nq / a.nkv) >> heads_log2_of(a, groups));
}

template <int D, int G>
hipError_t launch(const PackedAttnArgs &a, hipStream_t s) {
  const unsigned grid = (unsigned)grid_of(a, G);
  const int slots = (int)slots_of(a, G);
  if (a.type == kElemBf16)
    hipLaunchKernelGGL((packed_attn_kernel<D, true, G>), dim3(grid), dim3(kThreads), 0, s, a, slots, heads_log2_of(a, G));
  else
    hipLaunchKernelGGL((packed_attn_kernel<D, false, G>), dim3(grid), dim3(kThreads), 0, s, a, slots, heads_log2_of(a, G));
  return hipGetLastError();
}

}  // namespace

// (a launch has fewer than 2^32 threads in a dimension; the shortest blocks
// are for batches far below it)
bool packed_attn_fits(const PackedAttnArgs &a) { return grid_of(a, 1) <= 0xffffffffll / kThreads / 8; }

hipError_t launch_packed_attn(const PackedAttnArgs &a, int num_cus, hipStream_t s) {
  if (a.tokens < 1 || a.sequences < 1 || a.nkv < 1 || a.nq % a.nkv != 0 || !packed_attn_fits(a))
    return hipErrorInvalidValue;
  const int groups = groups_of(a, num_cus);
  if (a.head_dim == 64) return groups == 1 ? launch<64, 1>(a, s) : launch<64, 2>(a, s);
  if (a.head_dim == 128) return groups == 1 ? launch<128, 1>(a, s) : launch<128, 2>(a, s);
  if (a.head_dim == 256) return groups == 1 ? launch<256, 1>(a, s) : launch<256, 2>(a, s);
  return hipErrorInvalidValue;
}

}  // namespace hp
