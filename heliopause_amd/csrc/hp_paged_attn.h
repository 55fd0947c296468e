// hp_paged_attn.h -- the kernels of the attention of one new token of every
// sequence over its pages, for paged_attn.hip (whole sequences, values as they
// are stored or times one scale) and block_attn.hip (a scale for each block of
// positions and KV head, a list of blocks to attend to).
//
// out_h = sum_j p_j v_j / sum_j p_j with p_j = exp(scale q_h . k_j - m) over the last min(length, window) positions j of the sequence.
//
// Every key and value is read once per KV head for up to eight query heads of its
// group (a larger group reads them once for each eight), so 2 (group) flop come on
// each 16-bit byte pair: the cache's bytes bound it, and the matrix cores, which a
// group of eight leaves at a few percent, are used because they hand every key to
// all heads of the group at once and leave the vector unit free.
//
// Products.  A wave takes 32 keys at a time, v_mfma_f32_16x16x32:
//   scores S^T = K Q^T, keys as the A rows, straight from the cache rows (a
//     lane's 8 consecutive elements of one key).  The B columns are the eight
//     query heads twice: column c < 8 holds the upper part of head c's query,
//     column c + 8 the rest of it, so one product gives both and their sum is
//     the score of the query to 22 bits (f16) or 16 (bf16; a query that came
//     as f32 has a third part there, in a second product into the same sums);
//   values O^T += V^T P^T, the lane's own scores as the B operand: lane (q4,
//     c) holds the scores of keys 4 q4 .. + 3 of both 16-key halves, and the
//     product's k index runs over just those, so the probabilities never
//     leave their registers; columns c and c + 8 hold the upper part and the
//     rest of p.  V^T's row index runs over the 16 lanes of a row, each with
//     D / 16 consecutive elements of a value row: 16 lanes load whole rows and
//     turn 8 keys x D / 16 elements into fragments with byte permutes.
// So results are those of f32 arithmetic to a few 2^-22 (f16, e4m3) or 2^-16
// (bf16) though the operands have 16 bits; sums, maximum and normaliser are
// f32.  p carries a factor 2^10, which cancels: it keeps p of 2^-24 and less
// out of f16's subnormal steps.  E4M3 elements become f16 exactly, and the
// cache's scales join the score's factor and the end.
//
// Masked keys (behind the length, before the window, on an absent page) get
// score -inf and value zero, whatever their slots hold.  A part of masked keys
// only has the maximum -inf; one whose other keys all score -inf themselves the
// lowest finite number: a row of nothing else is 0 / 0, not zeros.
//
// Split.  All (sequence, KV head) rows' steps of 128 keys (32 for each of the
// four waves; heads of 256 half as many) lie end to end, and each workgroup
// takes an equal share of that line with eight of a group's heads, whatever the
// lengths are: 48 ragged contexts and two of 131072 fill the card alike, and a
// captured launch serves every batch.  A workgroup finds its place by a scan of
// the lengths.  A row that one workgroup finishes is written at once; parts of
// the others go to scratch, at most two a workgroup, and the merge launch joins
// them in their order.  A group's further heads are workgroups beside one
// another on one XCD, whose L2 has the keys for the second (24 / 2 heads of 256
// over 20 contexts up to 6000: 26.2 us, with the blocks along the line 35.0).
// Not kept: parts joined by the workgroup that comes last, with stores and loads
// that cross the XCDs (one context of 4096 18.8 us for 13.9 then, larger batches
// the same).
//
// 48 contexts up to 8192, 32 / 8 heads of 128, bf16: 660 MB in 108 us, 6.1 TB/s,
// of which the merge launch is 5; two of 131072, f16: 419 MB in 69.5 us; 130
// windows of 1024 of 8 / 2 heads of 256, e4m3: 121 MB in 34 us, five of the merge
// and four until the first bytes come; one context of 4096: 8.4 MB in 12.4 us, two
// launches' latency.
#pragma once

#include <type_traits>

#include "hp_mfma.h"
#include "hp_serving.h"
#include "hp_wave.h"

namespace hp {

namespace {

// What a kernel knows of the cache besides its rows: a scale for each block of
// positions and KV head; a list of blocks for each sequence and KV head, to
// which the attention keeps.
constexpr int kWhole = 0, kScaled = 1, kSelected = 2;

constexpr int kWaves = kPagedWaves, kThreads = 64 * kWaves;
constexpr int kHeads = 8;  // query heads of a row

// 16-key tiles of a wave's step: heads of 256 take one where two would not fit
// the registers beside the sums (8 / 2 heads of 256 over 28 contexts up to 4096:
// f16 30.2 -> 27.9 us, bf16 pages with f32 queries 39.2 -> 29.0).
__host__ __device__ constexpr int tiles_of(int head_dim, int type) {
  return head_dim == 256 && elem_bytes(type) != 1 ? 1 : 2;
}
// Keys of a step of every wave.
__host__ __device__ constexpr int step_of(int head_dim, int type) { return 16 * tiles_of(head_dim, type) * kWaves; }
constexpr int kXcds = 8;  // workgroup i runs on XCD i % 8
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kBias = 10.0f;  // p carries 2^kBias
constexpr float kUnbias = 0x1p-10f;  // (with scales the normaliser does without it, and the sums lose it at the end)
constexpr float kNegInf = -__builtin_inff();
constexpr float kUnweighed = -3.40282346638528860e38f;  // the maximum of a part that has keys, all of which score -inf

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));

// The keys of line `row`: a sequence's, or the places in a (sequence, KV head)'s
// list of blocks.
template <int MODE>
__device__ __forceinline__ KeySpan span_of(const PagedAttnArgs &a, int row) {
  if (MODE & kSelected) {
    const int n = a.counts ? min(max(a.counts[row], 0), a.budget) : a.budget;
    return KeySpan{0, 0, n << a.block_shift};
  }
  return key_span(a.c.lengths[row], (int64_t)a.c.width << a.c.page_shift, a.window);
}

// Heads of a KV head's group in blocks of kHeads: rows of a sequence.
__host__ __device__ __forceinline__ int blocks_of(int nq, int nkv) { return (nq / nkv + kHeads - 1) / kHeads; }

// A part of a row: m and l of its heads, then the unnormalised sums; with scales
// what is left of m.
template <int D>
struct PartSums {
  float m[kHeads], l[kHeads];
  float o[kHeads][D];
};
template <bool SCALED>
struct PartLow {};
template <>
struct PartLow<true> {
  float low[kHeads];
};
template <int D, int MODE>
struct Part : PartSums<D>, PartLow<(MODE & kScaled) != 0> {};
// How far a maximum is from 2^24, in steps of f32: below kFar where it is that
// large (and finite), so that f32's steps are more than one and a scale's exponent
// needs `low`; other maxima have 0 there.
constexpr uint32_t kFar = 0x7f800000u - 0x4b800000u;
__device__ __forceinline__ uint32_t distance_of(float m) {
  return (__builtin_bit_cast(uint32_t, m) & 0x7fffffffu) - 0x4b800000u;
}
struct RowParts {
  int first, last;  // workgroups that hold the row's parts (the same: none)
};

template <int CT>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if (CT == kElemBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

// The same with the k index over 32 keys (four dwords) or 16 (two).
template <int CT, int N>
__device__ __forceinline__ f32x4 mfma_keys(const uint32_t (&a)[N], const uint32_t (&b)[N], f32x4 c) {
  if (N == 4)
    return mfma16<CT>((u32x4){a[0], a[1], a[2 % N], a[3 % N]}, (u32x4){b[0], b[1], b[2 % N], b[3 % N]}, c);
  const uint2 x = make_uint2(a[0], a[1]), y = make_uint2(b[0], b[1]);
  if (CT == kElemBf16)
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4v, x), __builtin_bit_cast(short4v, y), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(half4v, x), __builtin_bit_cast(half4v, y), c, 0, 0, 0);
}

// The operand type's bits of v, and the value they stand for.
template <int CT>
__device__ __forceinline__ uint32_t part_bits(float v) {
  return CT == kElemBf16 ? bf16_bits(v) : f16_bits(v);
}
template <int CT>
__device__ __forceinline__ float part_value(uint32_t b) {
  return CT == kElemBf16 ? bf16_value(b) : (float)__builtin_bit_cast(_Float16, (uint16_t)b);
}

// Bytes 2 i, 2 i + 1 of four fp8 values as two halves (exact: f16 holds every
// e4m3 value).  The results are taken as one dword; a bit cast of a vector's
// element reads element 0.
template <bool HI>
__device__ __forceinline__ uint32_t halves_of_e4m3(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
}
// The same of four i8 values: under the exponent byte 0x64 a byte b is the half
// 1024 + b, and q ^ 0x80 is q + 128.
template <int CT, bool HI>
__device__ __forceinline__ uint32_t halves_of(uint32_t w) {
  if (CT != kElemI8) return halves_of_e4m3<HI>(w);
  const half2v bias = {(_Float16)1152.0f, (_Float16)1152.0f};
  return as_u32(magic_pair<HI ? kSel23 : kSel01>(w ^ 0x80808080u) - bias);
}

// maximum / sum over the lanes c, c + 16, c + 32, c + 48
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// A row's 1 / l (times the cache's scale): 0 without a key, NaN where nothing has
// weight.
__device__ __forceinline__ float row_scale(float m, float l, float value_scale) {
  return m == kNegInf && l == 0.0f ? 0.0f : l == 0.0f ? __builtin_nanf("") : value_scale / l;
}

// 2^d, for a part's sums whose maximum is 2^d of the others'.  Under scales the
// sum l of a row's weights lies within 2^-100 and 2^100 n of its maximum's, whose
// scale counts there, and one maximum may be 2^200 above the next: 2^d by itself is
// 0 then, where its product with l is not, and l takes its root twice.
template <int MODE>
struct Exp2 {
  float root, all;
  __device__ __forceinline__ explicit Exp2(float d) {
    root = (MODE & kScaled) ? __builtin_amdgcn_exp2f(0.5f * d) : 0.0f;
    all = (MODE & kScaled) ? root * root : __builtin_amdgcn_exp2f(d);
  }
  __device__ __forceinline__ float of_sum(float l) const { return (MODE & kScaled) ? l * root * root : l * all; }
};

// A lane's elements of a key row of each tile (D / 32 operand fragments) and of
// the four value rows of each (D / 16 elements each), as loaded.
template <int D, int CT>
struct Tile {
  static constexpr int kE = elem_bytes(CT);            // bytes an element
  static constexpr int kTiles = tiles_of(D, CT), kKeys = 4 * kTiles;  // of a lane's values
  static constexpr int kKeyWords = D * kE / 4 / 4;     // dwords of a quarter key row
  static constexpr int kValueWords = D * kE / 16 / 4;  // dwords of a sixteenth of a value row
  uint32_t k[kTiles][kKeyWords];
  uint32_t v[kKeys][kValueWords];
};

// (STREAM: not to stay in the caches)
template <bool STREAM, int N>
__device__ __forceinline__ void load_words(uint32_t (&d)[N], const uint8_t *p) {
  constexpr int kWide = N < 4 ? N : 4;
  typedef uint32_t words __attribute__((ext_vector_type(kWide == 1 ? 2 : kWide)));
#pragma unroll
  for (int i = 0; i < N; i += kWide) {
    if (kWide == 1) {
      const uint32_t *q = reinterpret_cast<const uint32_t *>(p + 4 * i);
      d[i] = STREAM ? __builtin_nontemporal_load(q) : *q;
    } else {
      const words *q = reinterpret_cast<const words *>(p + 4 * i);
      const words w = STREAM ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
      for (int j = 0; j < kWide; j++) d[i + j] = w[j];
    }
  }
}

template <int D, int CT, int MODE, bool THIRD, bool STREAM>
__global__ __launch_bounds__(kThreads, 2) void paged_attn_kernel(const PagedAttnArgs a, RowParts *__restrict__ rows,
                                                                 Part<D, MODE> *__restrict__ parts, int groups) {
  using T = Tile<D, CT>;
  constexpr int kTiles = T::kTiles, kKeys = T::kKeys, kSub = 16 * kTiles, kStep = kSub * kWaves;
  constexpr int kE = T::kE, kFrags = D / 32, kRowBytes = D * kE, kT = D / 16;
  constexpr bool kList = (MODE & kSelected) != 0, kScales = (MODE & kScaled) != 0;
  __shared__ float4 sh_o[kWaves][kHeads][D / 4];
  __shared__ u32x4 sh_q[THIRD ? 2 : 1][kFrags][64];  // the query's operand fragments, the same for every wave
  __shared__ float sh_m[kWaves][kHeads], sh_l[kWaves][kHeads], sh_low[kScales ? kWaves : 1][kHeads];
  __shared__ alignas(4) bool sh_far[kWaves];  // waves whose maxima have a second part
  __shared__ float sh_most[kWaves][16];  // largest elements of the query rows
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q4 = lane >> 4, c16 = lane & 15;
  const int group = a.nq / a.c.nkv, blocks = blocks_of(a.nq, a.c.nkv);
  const int lines = kList ? a.c.sequences * a.c.nkv : a.c.sequences, units = kList ? 1 : a.c.nkv;
  // (share of the line, block of heads): a share's blocks, which read the same
  // keys, side by side on one XCD
  const int block = (int)blockIdx.x / kXcds % blocks;
  const uint32_t me = (int)blockIdx.x / (kXcds * blocks) * kXcds + (int)blockIdx.x % kXcds;

  // The line of steps, by each wave for itself (no barrier): a lane sums a run
  // of sequences, the runs are scanned, and the lane whose run has the
  // workgroup's first step tells its place.
  const int run = (lines + 63) >> 6;
  uint32_t mine = 0;
  for (int i = 0; i < run; i++) {
    const int s = lane * run + i;
    if (s < lines) mine += span_steps(span_of<MODE>(a, s), kStep);
  }
  uint32_t before = wave_scan(mine);
  const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)before, 63) * units;
  before = (before - mine) * units;
  mine *= units;
  const uint32_t shares = min((uint32_t)groups, total);
  if (me >= shares) return;
  uint32_t at = share_begin(total, me, shares);
  const uint32_t stop = share_begin(total, me + 1, shares);
  const bool mine_is = at >= before && at - before < mine;  // one lane
  int place = lane * run;
  uint32_t start = before;
  if (run > 1 && mine_is)
    for (; place < min(lane * run + run, lines) - 1; place++) {
      const uint32_t n = span_steps(span_of<MODE>(a, place), kStep) * units;
      if (at - start < n) break;
      start += n;
    }
  // (scalar registers from here on)
  const int holder = __builtin_ctzll(__ballot(mine_is));
  int line = __builtin_amdgcn_readlane(place, holder);
  uint32_t seq_start = (uint32_t)__builtin_amdgcn_readlane((int)start, holder);

  const uint8_t *keys = static_cast<const uint8_t *>(a.c.keys), *values = static_cast<const uint8_t *>(a.c.values);
  const int page_mask = (1 << a.c.page_shift) - 1;

  while (at < stop && line < lines) {
    const KeySpan span = span_of<MODE>(a, line);
    const uint32_t steps = span_steps(span, kStep);
    if (at - seq_start >= steps * units) {  // (also past sequences without a key)
      seq_start += steps * units;
      line++;
      continue;
    }
    const uint32_t unit = (at - seq_start) / steps, row_start = seq_start + unit * steps;
    const uint32_t i0 = at - row_start, n = min(stop - at, steps - i0);
    const int seq = kList ? line / a.c.nkv : line;
    const int kvh = kList ? line - seq * a.c.nkv : (int)unit, h0 = block * kHeads;  // KV head, first head of the group
    const int live = min(kHeads, group - h0);

    // the query: each wave takes a share of the fragments, lane c16 % 8's head
    // and the elements that the lane's keys have there
    constexpr int kMine = kFrags < kWaves ? 1 : kFrags / kWaves;
    const bool has = wave * kMine < kFrags;
    const int c8 = c16 & 7;
    uint4 raw[kMine][2];
    if (has) {
      const int64_t at_q = seq * a.q_stride + (int64_t)(kvh * group + h0 + min(c8, live - 1)) * D;
#pragma unroll
      for (int i = 0; i < kMine; i++) {
        const int f = wave * kMine + i, d = kE == 1 ? 64 * (f >> 1) + 16 * q4 + 8 * (f & 1) : 32 * f + 8 * q4;
        if (a.q_type == kElemF32) {
          const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const float *>(a.q) + at_q + d);
          raw[i][0] = p[0];
          raw[i][1] = p[1];
        } else {
          raw[i][0] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + at_q + d);
        }
      }
    }

    f32x4 acc[kT];
#pragma unroll
    for (int t = 0; t < kT; t++) acc[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = kNegInf, l_part = 0.0f;
    float m_low = 0.0f;  // (scales: the maximum is m_run + m_low)
    bool far = false;    // (the same for the wave)
    bool has_key = false;  // the lane has seen a key that is not masked

    // this wave's tiles: key .. key + kSub - 1 at key = begin + kStep i + kSub wave
    const int key0 = span.begin + (int)i0 * kStep + kSub * wave;
    const int key_stop = min(span.end, span.begin + (int)(i0 + n) * kStep);
    const int *table = a.c.pages + (int64_t)seq * a.c.width;
    const int64_t head_at = ((int64_t)kvh << a.c.page_shift) * D;
    // Table entry of the 16 keys from `key` on (the same for the wave), and the
    // page that it names or -1.  Only entries of pages that hold a key of the
    // sequence are read, a step ahead of their rows.  Here and below loads take
    // no branch: one that may not have been issued would make the next wait
    // one for all.
    // With a list of blocks, `key` counts the places of the list: its entries are
    // read a step ahead of the table's, and where[] has the position of a tile's
    // first key.
    const int table_keys = a.c.width << a.c.page_shift, length = kList ? min(a.c.lengths[seq], table_keys) : span.end;
    const int *list = kList ? a.selected + (int64_t)line * a.budget : nullptr;
    int entries[kTiles], page[kTiles], listed[kTiles], entry_at[kTiles], where[kTiles];
    auto load_listed = [&](int key) {
      if (!kList) return;
#pragma unroll
      for (int h = 0; h < kTiles; h++) listed[h] = list[min(key + 16 * h, span.end - 1) >> a.block_shift];
    };
    auto load_entries = [&](int key) {
#pragma unroll
      for (int h = 0; h < kTiles; h++) {
        int p = key + 16 * h;
        if (kList) {
          const int b = __builtin_amdgcn_readfirstlane(listed[h]);
          const bool is = p < span.end && b >= 0 && b < table_keys >> a.block_shift;
          p = is ? (b << a.block_shift) + (p & ((1 << a.block_shift) - 1)) : -1;
          entry_at[h] = p;
          entries[h] = table[max(p, 0) >> a.c.page_shift];
        } else {
          entries[h] = table[min(p, span.end - 1) >> a.c.page_shift];
        }
      }
    };
    auto pages_of = [&](int key, int (&pages)[kTiles], int (&at_key)[kTiles]) {
#pragma unroll
      for (int h = 0; h < kTiles; h++) {
        const int p = page_or_none(__builtin_amdgcn_readfirstlane(entries[h]), a.c.page_count);
        at_key[h] = kList ? max(entry_at[h], 0) : key + 16 * h;
        pages[h] = (kList && entry_at[h] < 0) || at_key[h] >= length ? -1 : p;
      }
    };
    // Bytes of the first of those keys' rows for this head; an absent page's
    // are page 0's, which are there and masked.
    auto tile_at = [&](int page, int key) -> int64_t {
      return (max(page, 0) * a.c.page_stride + head_at + (int64_t)(key & page_mask) * D) * kE;
    };
    T t;
    // (fp8: 16 bytes are the lane's elements of two fragments)
    auto load_keys = [&](const int (&at_key)[kTiles], const int (&pages)[kTiles]) {
#pragma unroll
      for (int h = 0; h < kTiles; h++) {
        const uint8_t *rows = keys + tile_at(pages[h], at_key[h]);
#pragma unroll
        for (int i = 0; i < T::kKeyWords / 4; i++) {
          uint32_t w[4];
          load_words<STREAM>(w, rows + c16 * kRowBytes + 64 * i + 16 * q4);
#pragma unroll
          for (int j = 0; j < 4; j++) t.k[h][4 * i + j] = w[j];
        }
      }
    };
    auto load_values = [&](const int (&at_key)[kTiles], const int (&pages)[kTiles]) {
#pragma unroll
      for (int j = 0; j < kKeys; j++)
        load_words<STREAM>(t.v[j], values + tile_at(pages[j >> 2], at_key[j >> 2]) +
                                       (4 * q4 + (j & 3)) * kRowBytes + c16 * kT * kE);
    };
    // the tiles' scales: 16 keys share a block
    float key_scale[kTiles], value_scale[kTiles];
    auto load_scales = [&](const int (&at_key)[kTiles], const int (&pages)[kTiles], float (&ks)[kTiles],
                           float (&vs)[kTiles]) {
      if (!kScales) return;
#pragma unroll
      for (int h = 0; h < kTiles; h++) {
        const int64_t i = (((int64_t)max(pages[h], 0) * a.c.nkv + kvh) << (a.c.page_shift - a.block_shift)) +
                          ((at_key[h] & page_mask) >> a.block_shift);
        ks[h] = a.key_scales[i];
        vs[h] = a.value_scales[i];
      }
    };

    // (a wave whose keys are all behind the end loads its first tile for nothing)
    int key = key0;
    load_listed(key);
    load_entries(key);
    load_listed(key + kStep);
    pages_of(key, page, where);
    load_entries(key + kStep);
    load_listed(key + 2 * kStep);
    load_scales(where, page, key_scale, value_scale);
    load_keys(where, page);
    load_values(where, page);

    // the query in parts, while the first keys are on their way
    float x[kMine][8];
    {
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < kMine; i++) {
        const uint32_t w[8] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w,
                               raw[i][1].x, raw[i][1].y, raw[i][1].z, raw[i][1].w};
        if (a.q_type == kElemF32) {
#pragma unroll
          for (int j = 0; j < 8; j++) x[i][j] = __builtin_bit_cast(float, w[j]);
        } else if (a.q_type == kElemF16) {
#pragma unroll
          for (int j = 0; j < 8; j++)
            x[i][j] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[j >> 1] >> (16 * (j & 1))));
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) x[i][j] = bf16_value(w[j >> 1] >> (16 * (j & 1)) & 0xffffu);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
          x[i][j] = c8 < live && has ? x[i][j] : 0.0f;
          most = fmaxf(most, fabsf(x[i][j]));
        }
      }
      most = column_max(most);
      if (q4 == 0) sh_most[wave][c16] = most;
    }
    __syncthreads();
    bool lifted;
    float factor, lift;  // of a score, to base 2: their product
    {
      float most = sh_most[0][c16];
#pragma unroll
      for (int w = 1; w < kWaves; w++) most = fmaxf(most, sh_most[w][c16]);
      // the row times the power of two that puts its largest element into
      // [16, 32): the parts' range is then no concern (not for zeros and
      // infinities, which stay)
      const int e = (int)(__builtin_bit_cast(uint32_t, most) >> 23) - 127;
      const int shift = most > 0.0f && e < 128 ? 4 - max(e, -100) : 0;
      const float up = __builtin_bit_cast(float, (uint32_t)(127 + shift) << 23);
      // (past f32's range where both the query and the scales are large: in two
      // steps, so that a score of 0 stays 0 and the others leave f32 only where
      // they do by themselves)
      const double whole = (double)a.scale * (kE == 1 ? a.c.key_scale : 1.0f) * kLog2e *
                           __builtin_bit_cast(float, (uint32_t)(127 - shift) << 23);
      const bool far = whole >= 0x1p126;
      factor = (float)(far ? whole * 0x1p-126 : whole);
      lift = far ? 0x1p126f : 1.0f;
      lifted = __any(far);
      const bool rest = c16 >= kHeads;
#pragma unroll
      for (int i = 0; i < kMine; i++) {
        u32x4 qa, qb;
#pragma unroll
        for (int w = 0; w < 4; w++) {
          uint32_t p0[2], p2[2];
#pragma unroll
          for (int b = 0; b < 2; b++) {
            const float v = x[i][2 * w + b] * up;
            const uint32_t hi = part_bits<CT>(v);
            const float r1 = v - part_value<CT>(hi);
            const uint32_t mid = part_bits<CT>(r1);
            p0[b] = rest ? mid : hi;
            p2[b] = rest ? 0u : part_bits<CT>(r1 - part_value<CT>(mid));
          }
          qa[w] = p0[0] | p0[1] << 16;
          qb[w] = p2[0] | p2[1] << 16;
        }
        if (has) {
          sh_q[0][wave * kMine + i][lane] = qa;
          if (THIRD) sh_q[THIRD ? 1 : 0][wave * kMine + i][lane] = qb;
        }
      }
    }
    __syncthreads();

    // One step: the scores of this tile, the next keys on their way, weights,
    // the products with the values, the next values on their way.
    auto step = [&](auto last) {
      constexpr bool kMore = !decltype(last)::value;
      // the query's fragments are read anew in every step where in registers they
      // would not fit
      if (D == 256 && THIRD) asm volatile("" ::: "memory");
      const int next = key + kStep;
      f32x4 s[kTiles];
#pragma unroll
      for (int h = 0; h < kTiles; h++) {
        s[h] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int f = 0; f < kFrags; f++) {
          u32x4 kf;
          if (kE == 1) {
            const uint32_t lo = t.k[h][2 * f], hi = t.k[h][2 * f + 1];
            kf = (u32x4){halves_of<CT, false>(lo), halves_of<CT, true>(lo), halves_of<CT, false>(hi),
                         halves_of<CT, true>(hi)};
          } else {
            constexpr int kN = T::kKeyWords;
            kf = (u32x4){t.k[h][4 * f % kN], t.k[h][(4 * f + 1) % kN], t.k[h][(4 * f + 2) % kN],
                         t.k[h][(4 * f + 3) % kN]};
          }
          s[h] = mfma16<CT>(kf, sh_q[0][f][lane], s[h]);
          if (THIRD) s[h] = mfma16<CT>(kf, sh_q[THIRD ? 1 : 0][f][lane], s[h]);
        }
      }
      // the next keys stream in while these are worked on
      int next_page[kTiles], next_where[kTiles];
      float next_key_scale[kTiles], next_value_scale[kTiles];
      if (kMore) {
        pages_of(next, next_page, next_where);
        load_entries(next + kStep);
        load_listed(next + 2 * kStep);
        load_scales(next_where, next_page, next_key_scale, next_value_scale);
        load_keys(next_where, next_page);
      }
      bool edge = !kList && (key < span.first || key + kSub > span.end);
#pragma unroll
      for (int h = 0; h < kTiles; h++) edge = edge || page[h] < 0 || (kList && where[h] + 16 > length);
      float x[kKeys];
#pragma unroll
      for (int j = 0; j < kKeys; j++) {
        const float v = s[j >> 2][j & 3];
        const float all = v + dpp_f32<kDppRor8>(v);
        x[j] = (kScales ? all * key_scale[j >> 2] : all) * factor;
        if (MODE == kWhole || lifted) x[j] *= lift;
      }
      has_key = has_key || !edge;
      if (edge) {  // the same for the wave
#pragma unroll
        for (int j = 0; j < kKeys; j++) {
          const int at_key = where[j >> 2] + 4 * q4 + (j & 3);
          const bool off = (!kList && at_key < span.first) || at_key >= length || page[j >> 2] < 0;
          x[j] = off ? kNegInf : x[j];
          has_key = has_key || !off;
#pragma unroll
          for (int w = 0; w < T::kValueWords; w++) t.v[j][w] = off ? 0u : t.v[j][w];
        }
      }
      // a value scale s >= 2^e: the maximum is that of x + e, so that the weights
      // s 2^(x - m) of the stored values are within range whatever the blocks' scales
      // are.  2^(x - m) itself is at most 2^100, and below f32 only where the weight
      // is less than 2^-26 of the largest, bias and all.  Where a step of x in f32 is
      // more than one the maximum has a second part, what x + e was rounded by:
      // without it equal scores under scales of 2^20 would weigh 2^30 (2^16 is past
      // f16).  Scores that large take this way alone
      auto exponent_of = [](float scale) -> float {
        const int e = (int)(__builtin_bit_cast(uint32_t, scale) >> 23 & 255) - 127;
        return e == 128 ? 0.0f : (float)max(e, -100);  // (an infinity or NaN)
      };
      auto most_of = [&](int h) -> float {
        float v = x[4 * h];
#pragma unroll
        for (int j = 1; j < 4; j++) v = fmaxf(v, x[4 * h + j]);
        return v;
      };
      float most = kNegInf;
      if (kScales) {
#pragma unroll
        for (int h = 0; h < kTiles; h++) {
          most = fmaxf(most, most_of(h) + exponent_of(value_scale[h]));
          if (page[h] < 0) value_scale[h] = 0.0f;  // (whatever is there; its keys' scores are -inf)
        }
      } else {
        most = x[0];
#pragma unroll
        for (int j = 1; j < kKeys; j++) most = fmaxf(most, x[j]);
      }
      most = column_max(most);
      if (__any(most > m_run) || (kScales && far)) {
        const float m_new = fmaxf(m_run, most);
        float drop = m_new == kNegInf ? 0.0f : m_run - m_new;
        if (kScales) {
          const bool were = far;
          far = __any(distance_of(m_new) < kFar);
          if (__builtin_expect(far || were, false)) {
            float low = m_run == m_new ? m_low : kNegInf;
#pragma unroll
            for (int h = 0; h < kTiles; h++) {
              const float v = most_of(h), e = exponent_of(value_scale[h]);
              if (v + e == m_new) low = fmaxf(low, (v - (v + e)) + e);
            }
            low = column_max(low);
            low = distance_of(m_new) < kFar ? low : 0.0f;
            drop += m_low - low;
            m_low = low;
          }
        }
        const Exp2<MODE> alpha(drop);
        m_run = m_new;
        l_part = alpha.of_sum(l_part);
#pragma unroll
        for (int i = 0; i < kT; i++) acc[i] *= alpha.all;
      }
      // a row without a key so far: exp2(-inf - 0) = 0.  From 2^27 on f32's steps
      // are as large as the bias, and what is left of it could be more: 2^16 is
      // past f16
      float m_use = m_run == kNegInf ? 0.0f : m_run - kBias;
      m_use = m_run - m_use > 15.0f ? m_run : m_use;
      if (kScales && __builtin_expect(far, false)) {
        m_use = m_run == kNegInf ? 0.0f : m_run;
#pragma unroll
        for (int j = 0; j < kKeys; j++) x[j] = (x[j] - m_use) - (m_low - kBias);
        m_use = 0.0f;
      }
      uint32_t pf[kKeys / 2];
      const bool rest = c16 >= kHeads;
      uint32_t pb[kKeys];
#pragma unroll
      for (int j = 0; j < kKeys; j++) {
        float p = __builtin_amdgcn_exp2f(x[j] - m_use);
        if (kScales) {
          l_part = fmaf(p, kUnbias, l_part);
          p *= value_scale[j >> 2];
        } else {
          l_part += p;
        }
        const uint32_t hi = part_bits<CT>(p), lo = part_bits<CT>(p - part_value<CT>(hi));
        pb[j] = rest ? lo : hi;
      }
#pragma unroll
      for (int w = 0; w < kKeys / 2; w++) pf[w] = pb[2 * w] | pb[2 * w + 1] << 16;
      // V^T fragments: element i of the lane's D / 16 from each of its keys
#pragma unroll
      for (int i = 0; i < kT; i++) {
        uint32_t vf[kKeys / 2];
#pragma unroll
        for (int w = 0; w < kKeys / 2; w++) {
          const uint32_t sel = (i & 1) ? 0x07060302u : 0x05040100u;
          if (kE == 1) {
            const uint32_t a0 = t.v[2 * w][i >> 2], a1 = t.v[2 * w + 1][i >> 2];
            const uint32_t x0 = (i & 2) ? halves_of<CT, true>(a0) : halves_of<CT, false>(a0);
            const uint32_t x1 = (i & 2) ? halves_of<CT, true>(a1) : halves_of<CT, false>(a1);
            vf[w] = __builtin_amdgcn_perm(x1, x0, sel);
          } else {
            constexpr int kN = T::kValueWords;
            vf[w] = __builtin_amdgcn_perm(t.v[2 * w + 1][(i >> 1) % kN], t.v[2 * w][(i >> 1) % kN], sel);
          }
        }
        acc[i] = mfma_keys<CT>(vf, pf, acc[i]);
      }
      if (kMore) {
        load_values(next_where, next_page);
#pragma unroll
        for (int h = 0; h < kTiles; h++) {
          page[h] = next_page[h];
          where[h] = next_where[h];
          if (kScales) {
            key_scale[h] = next_key_scale[h];
            value_scale[h] = next_value_scale[h];
          }
        }
      }
    };
    if (key < key_stop) {
      for (; key + kStep < key_stop; key += kStep) step(std::false_type{});
      step(std::true_type{});
    }

    // the four waves' parts, joined in LDS.  Lane (q4, c): head c, elements
    // kT (4 q4 + r) + i
    const float l_run = column_sum(l_part);
    if (__any(has_key)) m_run = fmaxf(m_run, kUnweighed);
#pragma unroll
    for (int i = 0; i < kT; i++)
#pragma unroll
      for (int r = 0; r < 4; r++) acc[i][r] += dpp_f32<kDppRor8>(acc[i][r]);
    if (c16 < kHeads) {
      if (q4 == 0) {
        sh_m[wave][c16] = m_run;
        sh_l[wave][c16] = l_run;
        if (kScales) sh_low[kScales ? wave : 0][c16] = m_low;
        if (kScales && c16 == 0) sh_far[wave] = far;
      }
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int i = 0; i < kT; i += 4)
          sh_o[wave][c16][(kT * (4 * q4 + r) + i) / 4] =
              make_float4(acc[i][r], acc[i + 1][r], acc[i + 2][r], acc[i + 3][r]);
    }
    __syncthreads();
    const bool whole = i0 == 0 && n == steps;
    static_assert(sizeof(sh_far) == sizeof(uint32_t), "one load");
    const bool any_far = kScales && __builtin_amdgcn_readfirstlane((int)*reinterpret_cast<const uint32_t *>(sh_far)) != 0;
    Part<D, MODE> *part = parts + 2 * ((int64_t)me * blocks + block) + (i0 == 0 ? 1 : 0);
    if (i0 == 0 && tid == 0) {
      rows[((int64_t)line * units + unit) * blocks + block] = RowParts{(int)me, (int)share_of(total, row_start + steps - 1, shares)};
    }
    for (int i = tid; i < kHeads * (D / 4); i += kThreads) {
      const int h = i / (D / 4), d = i - h * (D / 4);
      float m = kNegInf;
#pragma unroll
      for (int w = 0; w < kWaves; w++) m = fmaxf(m, sh_m[w][h]);
      float low = 0.0f;
      if (__builtin_expect(any_far, false)) {
        low = kNegInf;
#pragma unroll
        for (int w = 0; w < kWaves; w++) low = sh_m[w][h] == m ? fmaxf(low, sh_low[kScales ? w : 0][h]) : low;
      }
      float l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        const float mw = sh_m[w][h];
        float below = mw == kNegInf ? kNegInf : mw - m;
        if (__builtin_expect(any_far, false)) below += sh_low[kScales ? w : 0][h] - low;
        const Exp2<MODE> e(below);
        const float f = e.all;
        const float4 v = sh_o[w][h][d];
        l += e.of_sum(sh_l[w][h]);
        o[0] += f * v.x;
        o[1] += f * v.y;
        o[2] += f * v.z;
        o[3] += f * v.w;
      }
      if (h >= live) continue;
      if (whole) {
        const float inv = row_scale(m, l, kE == 1 ? a.c.value_scale : 1.0f);
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] *= inv;
        store4(a.out, seq * a.out_stride + (int64_t)(kvh * group + h0 + h) * D + 4 * d, a.out_type, o);
      } else {
        *reinterpret_cast<float4 *>(&part->o[h][4 * d]) = make_float4(o[0], o[1], o[2], o[3]);
        if (d == 0) {
          part->m[h] = m;
          part->l[h] = l;
          if constexpr (kScales) part->low[h] = low;
        }
      }
    }
    __syncthreads();  // the LDS is the next row's
    at += n;
  }
}

// One (sequence, head): the parts of its row in order, o = sum f o_c / sum f
// l_c with f = 2^(m_c - m); D / 4 threads a part, several parts at once.
template <int D, int MODE>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(const PagedAttnArgs a, const RowParts *__restrict__ rows,
                                                               const Part<D, MODE> *__restrict__ parts, int groups) {
  constexpr int kPer = D / 4, kAtOnce = kThreads / kPer;
  constexpr bool kScales = (MODE & kScaled) != 0;
  __shared__ float sh_m[kAtOnce], sh_l[kAtOnce];
  __shared__ alignas(4) bool sh_far[kWaves];
  __shared__ float4 sh_o[kAtOnce][kPer];
  const int group = a.nq / a.c.nkv, blocks = blocks_of(a.nq, a.c.nkv);
  const int head = blockIdx.x, seq = blockIdx.y;
  const int kvh = head / group, in_group = head - kvh * group, h = in_group % kHeads;
  const int tid = threadIdx.x, sub = tid / kPer, d = tid - sub * kPer;
  const int64_t out = seq * a.out_stride + (int64_t)head * D + 4 * d;
  // (left by the launch before; held to its workgroups, whatever a length that
  // changed under it would make of them)
  RowParts r = rows[((int64_t)seq * a.c.nkv + kvh) * blocks + in_group / kHeads];
  r.first = max(r.first, 0);
  r.last = min(r.last, groups - 1);
  if (span_of<MODE>(a, MODE & kSelected ? seq * a.c.nkv + kvh : seq).end == 0) {  // no key: zeros
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (sub == 0) store4(a.out, out, a.out_type, zero);
    return;
  }
  if (r.first >= r.last) return;  // written by the workgroup that had it whole
  float m = kNegInf, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  auto part_of = [&](int c) -> const Part<D, MODE> & {
    return parts[2 * ((int64_t)c * blocks + in_group / kHeads) + (c == r.first ? 1 : 0)];
  };
  uint32_t distance = ~0u;  // (the least of the parts')
  constexpr int kDeep = 8;  // parts that a thread has on their way
  for (int c0 = r.first + sub; c0 <= r.last; c0 += kAtOnce * kDeep) {
    float mc[kDeep], lc[kDeep];
    float4 v[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; i++) {
      const int c = min(c0 + i * kAtOnce, r.last);
      const Part<D, MODE> &p = part_of(c);
      mc[i] = p.m[h];
      lc[i] = p.l[h];
      v[i] = *reinterpret_cast<const float4 *>(&p.o[h][4 * d]);
    }
    float m_new = m;
#pragma unroll
    for (int i = 0; i < kDeep; i++) {
      if (c0 + i * kAtOnce > r.last) mc[i] = kNegInf;
      m_new = fmaxf(m_new, mc[i]);
    }
    if (kScales) {
#pragma unroll
      for (int i = 0; i < kDeep; i++) distance = min(distance, distance_of(mc[i]));
    }
    const Exp2<MODE> f(m == kNegInf ? kNegInf : m - m_new);
    l = f.of_sum(l);
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] *= f.all;
#pragma unroll
    for (int i = 0; i < kDeep; i++) {
      if (c0 + i * kAtOnce > r.last) continue;
      const Exp2<MODE> e(mc[i] == kNegInf ? kNegInf : mc[i] - m_new);
      const float g = e.all;
      l += e.of_sum(lc[i]);
      o[0] += v[i].x * g;
      o[1] += v[i].y * g;
      o[2] += v[i].z * g;
      o[3] += v[i].w * g;
    }
    m = m_new;
  }
  if (d == 0) {
    sh_m[sub] = m;
    sh_l[sub] = l;
  }
  if (kScales) sh_far[tid >> 6] = __any(distance < kFar);
  sh_o[sub][d] = make_float4(o[0], o[1], o[2], o[3]);
  __syncthreads();
  if (sub != 0) return;
  float most = kNegInf;
#pragma unroll
  for (int c = 0; c < kAtOnce; c++) most = fmaxf(most, sh_m[c]);
  l = o[0] = o[1] = o[2] = o[3] = 0.0f;
#pragma unroll
  for (int c = 0; c < kAtOnce; c++) {
    const Exp2<MODE> e(sh_m[c] == kNegInf ? kNegInf : sh_m[c] - most);
    const float f = e.all;
    const float4 v = sh_o[c][d];
    l += e.of_sum(sh_l[c]);
    o[0] += f * v.x;
    o[1] += f * v.y;
    o[2] += f * v.z;
    o[3] += f * v.w;
  }
  if constexpr (kScales) {
    if (__builtin_expect(*reinterpret_cast<const uint32_t *>(sh_far) != 0, false)) {
      // anew, with what is left of the maxima, one part after another
      float low = 0.0f;
      most = kNegInf;
      l = o[0] = o[1] = o[2] = o[3] = 0.0f;
#pragma unroll 1
      for (int c = r.first; c <= r.last; c++) {
        const Part<D, MODE> &p = part_of(c);
        const float pm = p.m[h], pl = p.low[h];
        const bool above = pm > most || (pm == most && pl > low);
        const float to = above ? pm : most, to_low = above ? pl : low;
        const Exp2<MODE> f(most == kNegInf ? kNegInf : (most - to) + (low - to_low));
        const Exp2<MODE> g(pm == kNegInf ? kNegInf : (pm - to) + (pl - to_low));
        const float4 v = *reinterpret_cast<const float4 *>(&p.o[h][4 * d]);
        l = f.of_sum(l) + g.of_sum(p.l[h]);
        o[0] = f.all * o[0] + g.all * v.x;
        o[1] = f.all * o[1] + g.all * v.y;
        o[2] = f.all * o[2] + g.all * v.z;
        o[3] = f.all * o[3] + g.all * v.w;
        most = to;
        low = to_low;
      }
    }
  }
  const float inv = row_scale(most, l, elem_bytes(a.c.type) == 1 ? a.c.value_scale : 1.0f);
#pragma unroll
  for (int j = 0; j < 4; j++) o[j] *= inv;
  store4(a.out, out, a.out_type, o);
}

template <int D, int CT, int MODE, bool THIRD, bool STREAM>
hipError_t launch_kernels(const PagedAttnArgs &a, int groups, hipStream_t s) {
  Part<D, MODE> *parts = reinterpret_cast<Part<D, MODE> *>(a.partials);
  const int blocks = blocks_of(a.nq, a.c.nkv), grid = (groups + kXcds - 1) / kXcds * kXcds * blocks;
  RowParts *row_parts = reinterpret_cast<RowParts *>(parts + 2 * (int64_t)groups * blocks);
  hipLaunchKernelGGL((paged_attn_kernel<D, CT, MODE, THIRD, STREAM>), dim3(grid), dim3(kThreads), 0, s, a, row_parts,
                     parts, groups);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((paged_merge_kernel<D, MODE>), dim3(a.nq, a.c.sequences), dim3(kThreads), 0, s, a,
                     row_parts, parts, groups);
  return hipGetLastError();
}

// Keys and values are read once where a group has one block of heads; what does
// not fit the L2s together (32 MB) then goes past them: 122 -> 110 us (5.4 ->
// 6.0 TB/s) on 48 contexts up to 8192, 80 -> 71 on two of 131072.  A batch that
// does fit is read from them in repeated calls: 13.7 us and 14.4 past them on
// one context of 4096.  The lengths are on the device, so it goes by the table.
template <int D, int CT, int MODE, bool THIRD>
hipError_t launch(const PagedAttnArgs &a, int groups, hipStream_t s) {
  uint64_t keys = MODE & kSelected ? (uint64_t)a.budget << a.block_shift : (uint64_t)a.c.width << a.c.page_shift;
  if (a.window > 0 && keys > (uint64_t)a.window) keys = a.window;
  const bool stream = blocks_of(a.nq, a.c.nkv) == 1 &&
                      keys * a.c.sequences * a.c.nkv * D * 2 * elem_bytes(CT) > (32u << 20);
  return stream ? launch_kernels<D, CT, MODE, THIRD, true>(a, groups, s)
                : launch_kernels<D, CT, MODE, THIRD, false>(a, groups, s);
}

}  // namespace

}  // namespace hp
