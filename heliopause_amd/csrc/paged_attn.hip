// paged_attn.hip -- attention of one new token of every sequence over its
// pages: out_h = sum_j p_j v_j / sum_j p_j with p_j = exp(scale q_h . k_j - m)
// over the last min(length, window) positions j of the sequence.
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
#include <type_traits>

#include "hp_mfma.h"
#include "hp_serving.h"
#include "hp_wave.h"

namespace hp {

namespace {

constexpr int kWaves = kPagedWaves, kThreads = 64 * kWaves;
constexpr int kHeads = 8;  // query heads of a row

// 16-key tiles of a wave's step: heads of 256 take one where two would not fit
// the registers beside the sums (8 / 2 heads of 256 over 28 contexts up to 4096:
// f16 30.2 -> 27.9 us, bf16 pages with f32 queries 39.2 -> 29.0).
__host__ __device__ constexpr int tiles_of(int head_dim, int type) { return head_dim == 256 && type != kElemE4m3 ? 1 : 2; }
// Keys of a step of every wave.
__host__ __device__ constexpr int step_of(int head_dim, int type) { return 16 * tiles_of(head_dim, type) * kWaves; }
constexpr int kXcds = 8;  // workgroup i runs on XCD i % 8
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kBias = 10.0f;  // p carries 2^kBias
constexpr float kNegInf = -__builtin_inff();
constexpr float kUnweighed = -3.40282346638528860e38f;  // the maximum of a part that has keys, all of which score -inf

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ KeySpan span_of(const PagedAttnArgs &a, int seq) {
  return key_span(a.c.lengths[seq], (int64_t)a.c.width << a.c.page_shift, a.window);
}

// Heads of a KV head's group in blocks of kHeads: rows of a sequence.
__host__ __device__ __forceinline__ int blocks_of(int nq, int nkv) { return (nq / nkv + kHeads - 1) / kHeads; }

// A part of a row: m and l of its heads, then the unnormalised sums.
template <int D>
struct Part {
  float m[kHeads], l[kHeads];
  float o[kHeads][D];
};
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

// Sum of v over the lanes up to this one.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v = dpp_add<0x111, 0xf>(v);         // row_shr 1, 2, 4, 8: within the 16 lanes
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);         // lane 15's into rows 1 and 3
  return dpp_add<0x143, 0xc>(v);      // lane 31's into rows 2 and 3
}

// A lane's elements of a key row of each tile (D / 32 operand fragments) and of
// the four value rows of each (D / 16 elements each), as loaded.
template <int D, int CT>
struct Tile {
  static constexpr int kE = CT == kElemE4m3 ? 1 : 2;   // bytes an element
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

template <int D, int CT, bool THIRD, bool STREAM>
__global__ __launch_bounds__(kThreads, 2) void paged_attn_kernel(const PagedAttnArgs a, RowParts *__restrict__ rows,
                                                                 Part<D> *__restrict__ parts, int groups) {
  using T = Tile<D, CT>;
  constexpr int kTiles = T::kTiles, kKeys = T::kKeys, kSub = 16 * kTiles, kStep = kSub * kWaves;
  constexpr int kE = T::kE, kFrags = D / 32, kRowBytes = D * kE, kT = D / 16;
  __shared__ float4 sh_o[kWaves][kHeads][D / 4];
  __shared__ u32x4 sh_q[THIRD ? 2 : 1][kFrags][64];  // the query's operand fragments, the same for every wave
  __shared__ float sh_m[kWaves][kHeads], sh_l[kWaves][kHeads];
  __shared__ float sh_most[kWaves][16];  // largest elements of the query rows
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q4 = lane >> 4, c16 = lane & 15;
  const int group = a.nq / a.c.nkv, blocks = blocks_of(a.nq, a.c.nkv), units = a.c.nkv;
  // (share of the line, block of heads): a share's blocks, which read the same
  // keys, side by side on one XCD
  const int block = (int)blockIdx.x / kXcds % blocks;
  const uint32_t me = (int)blockIdx.x / (kXcds * blocks) * kXcds + (int)blockIdx.x % kXcds;

  // The line of steps, by each wave for itself (no barrier): a lane sums a run
  // of sequences, the runs are scanned, and the lane whose run has the
  // workgroup's first step tells its place.
  const int run = (a.c.sequences + 63) >> 6;
  uint32_t mine = 0;
  for (int i = 0; i < run; i++) {
    const int s = lane * run + i;
    if (s < a.c.sequences) mine += span_steps(span_of(a, s), kStep);
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
    for (; place < min(lane * run + run, a.c.sequences) - 1; place++) {
      const uint32_t n = span_steps(span_of(a, place), kStep) * units;
      if (at - start < n) break;
      start += n;
    }
  // (scalar registers from here on)
  const int holder = __builtin_ctzll(__ballot(mine_is));
  int seq = __builtin_amdgcn_readlane(place, holder);
  uint32_t seq_start = (uint32_t)__builtin_amdgcn_readlane((int)start, holder);

  const uint8_t *keys = static_cast<const uint8_t *>(a.c.keys), *values = static_cast<const uint8_t *>(a.c.values);
  const int page_mask = (1 << a.c.page_shift) - 1;

  while (at < stop && seq < a.c.sequences) {
    const KeySpan span = span_of(a, seq);
    const uint32_t steps = span_steps(span, kStep);
    if (at - seq_start >= steps * units) {  // (also past sequences without a key)
      seq_start += steps * units;
      seq++;
      continue;
    }
    const uint32_t unit = (at - seq_start) / steps, row_start = seq_start + unit * steps;
    const uint32_t i0 = at - row_start, n = min(stop - at, steps - i0);
    const int kvh = (int)unit, h0 = block * kHeads;  // KV head, first head of the group
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
        const int f = wave * kMine + i, d = CT == kElemE4m3 ? 64 * (f >> 1) + 16 * q4 + 8 * (f & 1) : 32 * f + 8 * q4;
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
    auto entry_of = [&](int key) -> int { return table[min(key, span.end - 1) >> a.c.page_shift]; };
    auto page_of = [&](int key, int entry) -> int {
      const int p = page_or_none(__builtin_amdgcn_readfirstlane(entry), a.c.page_count);
      return key < span.end ? p : -1;
    };
    // Bytes of the first of those keys' rows for this head; an absent page's
    // are page 0's, which are there and masked.
    auto tile_at = [&](int page, int key) -> int64_t {
      return (max(page, 0) * a.c.page_stride + head_at + (int64_t)(key & page_mask) * D) * kE;
    };
    T t;
    // (fp8: 16 bytes are the lane's elements of two fragments)
    auto load_keys = [&](int key, const int (&pages)[kTiles]) {
#pragma unroll
      for (int h = 0; h < kTiles; h++) {
        const uint8_t *rows = keys + tile_at(pages[h], key + 16 * h);
#pragma unroll
        for (int i = 0; i < T::kKeyWords / 4; i++) {
          uint32_t w[4];
          load_words<STREAM>(w, rows + c16 * kRowBytes + 64 * i + 16 * q4);
#pragma unroll
          for (int j = 0; j < 4; j++) t.k[h][4 * i + j] = w[j];
        }
      }
    };
    auto load_values = [&](int key, const int (&pages)[kTiles]) {
#pragma unroll
      for (int j = 0; j < kKeys; j++)
        load_words<STREAM>(t.v[j], values + tile_at(pages[j >> 2], key + 16 * (j >> 2)) +
                                       (4 * q4 + (j & 3)) * kRowBytes + c16 * kT * kE);
    };
    int entries[kTiles], page[kTiles];
    auto load_entries = [&](int key) {
#pragma unroll
      for (int h = 0; h < kTiles; h++) entries[h] = entry_of(key + 16 * h);
    };
    auto pages_of = [&](int key, int (&pages)[kTiles]) {
#pragma unroll
      for (int h = 0; h < kTiles; h++) pages[h] = page_of(key + 16 * h, entries[h]);
    };

    // (a wave whose keys are all behind the end loads its first tile for nothing)
    int key = key0;
    load_entries(key);
    pages_of(key, page);
    load_entries(key + kStep);
    load_keys(key, page);
    load_values(key, page);

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
      const double whole = (double)a.scale * (CT == kElemE4m3 ? a.c.key_scale : 1.0f) * kLog2e *
                           __builtin_bit_cast(float, (uint32_t)(127 - shift) << 23);
      const bool far = whole >= 0x1p126;
      factor = (float)(far ? whole * 0x1p-126 : whole);
      lift = far ? 0x1p126f : 1.0f;
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
          if (CT == kElemE4m3) {
            const uint32_t lo = t.k[h][2 * f], hi = t.k[h][2 * f + 1];
            kf = (u32x4){halves_of_e4m3<false>(lo), halves_of_e4m3<true>(lo), halves_of_e4m3<false>(hi),
                         halves_of_e4m3<true>(hi)};
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
      int next_page[kTiles];
      if (kMore) {
        pages_of(next, next_page);
        load_entries(next + kStep);
        load_keys(next, next_page);
      }
      bool edge = key < span.first || key + kSub > span.end;
#pragma unroll
      for (int h = 0; h < kTiles; h++) edge = edge || page[h] < 0;
      float x[kKeys];
#pragma unroll
      for (int j = 0; j < kKeys; j++) {
        const float v = s[j >> 2][j & 3];
        x[j] = (v + dpp_f32<kDppRor8>(v)) * factor * lift;
      }
      has_key = has_key || !edge;
      if (edge) {  // the same for the wave
#pragma unroll
        for (int j = 0; j < kKeys; j++) {
          const int at_key = key + 16 * (j >> 2) + 4 * q4 + (j & 3);
          const bool off = at_key < span.first || at_key >= span.end || page[j >> 2] < 0;
          x[j] = off ? kNegInf : x[j];
          has_key = has_key || !off;
#pragma unroll
          for (int w = 0; w < T::kValueWords; w++) t.v[j][w] = off ? 0u : t.v[j][w];
        }
      }
      float most = x[0];
#pragma unroll
      for (int j = 1; j < kKeys; j++) most = fmaxf(most, x[j]);
      most = column_max(most);
      if (__any(most > m_run)) {
        const float m_new = fmaxf(m_run, most);
        const float alpha = m_new == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_part *= alpha;
#pragma unroll
        for (int i = 0; i < kT; i++) acc[i] *= alpha;
      }
      // a row without a key so far: exp2(-inf - 0) = 0.  From 2^27 on f32's steps
      // are as large as the bias, and what is left of it could be more: 2^16 is
      // past f16
      float m_use = m_run == kNegInf ? 0.0f : m_run - kBias;
      m_use = m_run - m_use > 15.0f ? m_run : m_use;
      uint32_t pf[kKeys / 2];
      const bool rest = c16 >= kHeads;
      uint32_t pb[kKeys];
#pragma unroll
      for (int j = 0; j < kKeys; j++) {
        const float p = __builtin_amdgcn_exp2f(x[j] - m_use);
        l_part += p;
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
          if (CT == kElemE4m3) {
            const uint32_t a0 = t.v[2 * w][i >> 2], a1 = t.v[2 * w + 1][i >> 2];
            const uint32_t x0 = (i & 2) ? halves_of_e4m3<true>(a0) : halves_of_e4m3<false>(a0);
            const uint32_t x1 = (i & 2) ? halves_of_e4m3<true>(a1) : halves_of_e4m3<false>(a1);
            vf[w] = __builtin_amdgcn_perm(x1, x0, sel);
          } else {
            constexpr int kN = T::kValueWords;
            vf[w] = __builtin_amdgcn_perm(t.v[2 * w + 1][(i >> 1) % kN], t.v[2 * w][(i >> 1) % kN], sel);
          }
        }
        acc[i] = mfma_keys<CT>(vf, pf, acc[i]);
      }
      if (kMore) {
        load_values(next, next_page);
#pragma unroll
        for (int h = 0; h < kTiles; h++) page[h] = next_page[h];
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
    Part<D> *part = parts + 2 * ((int64_t)me * blocks + block) + (i0 == 0 ? 1 : 0);
    if (i0 == 0 && tid == 0) {
      rows[((int64_t)seq * units + unit) * blocks + block] = RowParts{(int)me, (int)share_of(total, row_start + steps - 1, shares)};
    }
    for (int i = tid; i < kHeads * (D / 4); i += kThreads) {
      const int h = i / (D / 4), d = i - h * (D / 4);
      float m = kNegInf;
#pragma unroll
      for (int w = 0; w < kWaves; w++) m = fmaxf(m, sh_m[w][h]);
      float l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        const float mw = sh_m[w][h], f = mw == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(mw - m);
        const float4 v = sh_o[w][h][d];
        l += f * sh_l[w][h];
        o[0] += f * v.x;
        o[1] += f * v.y;
        o[2] += f * v.z;
        o[3] += f * v.w;
      }
      if (h >= live) continue;
      if (whole) {
        const float inv = row_scale(m, l, CT == kElemE4m3 ? a.c.value_scale : 1.0f);
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] *= inv;
        store4(a.out, seq * a.out_stride + (int64_t)(kvh * group + h0 + h) * D + 4 * d, a.out_type, o);
      } else {
        *reinterpret_cast<float4 *>(&part->o[h][4 * d]) = make_float4(o[0], o[1], o[2], o[3]);
        if (d == 0) {
          part->m[h] = m;
          part->l[h] = l;
        }
      }
    }
    __syncthreads();  // the LDS is the next row's
    at += n;
  }
}

// One (sequence, head): the parts of its row in order, o = sum f o_c / sum f
// l_c with f = 2^(m_c - m); D / 4 threads a part, several parts at once.
template <int D>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(const PagedAttnArgs a, const RowParts *__restrict__ rows,
                                                               const Part<D> *__restrict__ parts, int groups) {
  constexpr int kPer = D / 4, kAtOnce = kThreads / kPer;
  __shared__ float sh_m[kAtOnce], sh_l[kAtOnce];
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
  if (span_of(a, seq).end == 0) {  // no key: zeros
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (sub == 0) store4(a.out, out, a.out_type, zero);
    return;
  }
  if (r.first >= r.last) return;  // written by the workgroup that had it whole
  float m = kNegInf, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int kDeep = 8;  // parts that a thread has on their way
  for (int c0 = r.first + sub; c0 <= r.last; c0 += kAtOnce * kDeep) {
    float mc[kDeep], lc[kDeep];
    float4 v[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; i++) {
      const int c = min(c0 + i * kAtOnce, r.last);
      const Part<D> &p = parts[2 * ((int64_t)c * blocks + in_group / kHeads) + (c == r.first ? 1 : 0)];
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
    const float f = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - m_new);
    l *= f;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] *= f;
#pragma unroll
    for (int i = 0; i < kDeep; i++) {
      if (c0 + i * kAtOnce > r.last) continue;
      const float g = mc[i] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(mc[i] - m_new);
      l += lc[i] * g;
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
  sh_o[sub][d] = make_float4(o[0], o[1], o[2], o[3]);
  __syncthreads();
  if (sub != 0) return;
  float most = kNegInf;
#pragma unroll
  for (int c = 0; c < kAtOnce; c++) most = fmaxf(most, sh_m[c]);
  l = o[0] = o[1] = o[2] = o[3] = 0.0f;
#pragma unroll
  for (int c = 0; c < kAtOnce; c++) {
    const float f = sh_m[c] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(sh_m[c] - most);
    const float4 v = sh_o[c][d];
    l += f * sh_l[c];
    o[0] += f * v.x;
    o[1] += f * v.y;
    o[2] += f * v.z;
    o[3] += f * v.w;
  }
  const float inv = row_scale(most, l, a.c.type == kElemE4m3 ? a.c.value_scale : 1.0f);
#pragma unroll
  for (int j = 0; j < 4; j++) o[j] *= inv;
  store4(a.out, out, a.out_type, o);
}

template <int D, int CT, bool THIRD, bool STREAM>
hipError_t launch_kernels(const PagedAttnArgs &a, int groups, hipStream_t s) {
  Part<D> *parts = reinterpret_cast<Part<D> *>(a.partials);
  const int blocks = blocks_of(a.nq, a.c.nkv), grid = (groups + kXcds - 1) / kXcds * kXcds * blocks;
  RowParts *row_parts = reinterpret_cast<RowParts *>(parts + 2 * (int64_t)groups * blocks);
  hipLaunchKernelGGL((paged_attn_kernel<D, CT, THIRD, STREAM>), dim3(grid), dim3(kThreads), 0, s, a, row_parts, parts,
                     groups);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(paged_merge_kernel<D>, dim3(a.nq, a.c.sequences), dim3(kThreads), 0, s, a, row_parts, parts, groups);
  return hipGetLastError();
}

// Keys and values are read once where a group has one block of heads; what does
// not fit the L2s together (32 MB) then goes past them: 122 -> 110 us (5.4 ->
// 6.0 TB/s) on 48 contexts up to 8192, 80 -> 71 on two of 131072.  A batch that
// does fit is read from them in repeated calls: 13.7 us and 14.4 past them on
// one context of 4096.  The lengths are on the device, so it goes by the table.
template <int D, int CT, bool THIRD>
hipError_t launch(const PagedAttnArgs &a, int groups, hipStream_t s) {
  uint64_t keys = (uint64_t)a.c.width << a.c.page_shift;
  if (a.window > 0 && keys > (uint64_t)a.window) keys = a.window;
  const bool stream = blocks_of(a.nq, a.c.nkv) == 1 &&
                      keys * a.c.sequences * a.c.nkv * D * 2 * (CT == kElemE4m3 ? 1 : 2) > (32u << 20);
  return stream ? launch_kernels<D, CT, THIRD, true>(a, groups, s) : launch_kernels<D, CT, THIRD, false>(a, groups, s);
}

template <int D>
hipError_t launch_type(const PagedAttnArgs &a, int groups, hipStream_t s) {
  if (a.c.type == kElemF16) return launch<D, kElemF16, false>(a, groups, s);
  if (a.c.type == kElemE4m3) return launch<D, kElemE4m3, false>(a, groups, s);
  // two bf16 parts hold an f16 or bf16 query; an f32 one has a third
  return a.q_type == kElemF32 ? launch<D, kElemBf16, true>(a, groups, s) : launch<D, kElemBf16, false>(a, groups, s);
}

size_t part_bytes(int head_dim) { return (size_t)kHeads * (head_dim + 2) * sizeof(float); }

}  // namespace

uint64_t paged_attn_most_steps(const PagedAttnArgs &a) {
  uint64_t keys = (uint64_t)a.c.width << a.c.page_shift;
  if (a.window > 0 && keys > (uint64_t)a.window + 15) keys = (uint64_t)a.window + 15;
  const int step = step_of(a.c.head_dim, a.c.type);
  return (keys + step - 1) / step * a.c.sequences * a.c.nkv;
}

int paged_attn_groups(const PagedAttnArgs &a, int num_cus) {
  const uint64_t most = paged_attn_most_steps(a);
  const int room = 2 * num_cus / blocks_of(a.nq, a.c.nkv);  // two workgroups a CU
  return most < (uint64_t)room ? (int)most : room < 1 ? 1 : room;
}

size_t paged_attn_scratch_bytes(const PagedAttnArgs &a, int groups) {
  const size_t blocks = blocks_of(a.nq, a.c.nkv);
  return blocks * (2 * (size_t)groups * part_bytes(a.c.head_dim) +
                   (size_t)a.c.sequences * a.c.nkv * sizeof(RowParts));
}

hipError_t launch_paged_attn(const PagedAttnArgs &a, int groups, hipStream_t s) {
  if (groups < 1 || a.c.sequences < 1 || a.c.nkv < 1 || a.nq % a.c.nkv != 0 || !a.partials ||
      paged_attn_most_steps(a) >> 31)
    return hipErrorInvalidValue;
  switch (a.c.head_dim) {
    case 64: return launch_type<64>(a, groups, s);
    case 128: return launch_type<128>(a, groups, s);
    case 256: return launch_type<256>(a, groups, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace hp
