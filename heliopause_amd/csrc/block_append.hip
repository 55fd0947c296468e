// block_append.hip -- a batch's new tokens into pages of 8 bits whose blocks have
// a scale for each KV head: head norms and position rotation as
// paged_append.hip has them, then per block and head with A the largest
// magnitude among the call's rows in it
//   i8:   s' = A (1 / 127)      e4m3: s' = the least power of two with A <= 448 s'
// held within 2^-100 .. 2^100, and x is stored as round(x / s').  A block that
// was begun before the call keeps its scale s while A <= M s (M = 127 or 448);
// otherwise the scale grows to s' (i8: at least 1.25 s, so that growing again
// and again adds less than 5 half steps in all) and what it holds becomes
// round(stored * s / s').  e4m3's powers of two move its values without another
// rounding, but for those that become subnormal.  An infinity or NaN among the
// rows makes the block's scale NaN until the block is begun anew: 8 bits have no
// place for it, and what is read from the block then shows that.
//
// A workgroup takes the call's rows of one (block, KV head, key or value): they
// stay in registers from the load to the store, so that a row is read once
// though the scale needs all of them first.  Query rows, which need none, are
// workgroups of their own in the same launch.  D / 8 lanes have a row: lane l
// elements 4l .. 4l + 3 of both halves of the rotated part (or eight consecutive
// ones of the rest), so that a pair sits in one lane.
//
// The frequencies are formed in 64 bits, as the turns of an angle are; what is
// left of a turn, at most half of one, is 2^-25 off in f32, and its sine and
// cosine are series in f32 after the quarter turns are taken off.  A key's angles
// are its lanes' own, four each; a token's query rows share theirs through LDS
// (a quarter of the vector unit's work with every row's lanes forming them).
// 16000 tokens of 32 + 16 head rows of 128, 622 MB in and out: 124 us, 5.0 TB/s.
#include "hp_serving.h"
#include "hp_wave.h"

namespace hp {

namespace {

constexpr double kInvTwoPi = 0.15915494309189533577;
constexpr float kLeast = 0x1p-100f, kMost = 0x1p100f;  // of a scale
constexpr float kGrowth = 1.25f;
constexpr float kInf = __builtin_inff();

template <int CT>
constexpr float stored_most() {
  return CT == kElemI8 ? 127.0f : 448.0f;
}

// Sum over the L lanes that hold a row (L consecutive lanes, 8, 16 or 32).
template <int L>
__device__ __forceinline__ float row_sum(float v) {
  v += dpp_f32<kDppXor1>(v);
  v += dpp_f32<kDppXor2>(v);
  v += dpp_f32<kDppRowHalfMirror>(v);
  if (L >= 16) v += dpp_f32<kDppRowMirror>(v);
  if (L >= 32) v += __shfl_xor(v, 16);
  return v;
}

// The scale of a block whose largest element is `most`.  448 = 0.875 * 2^9.
template <int CT>
__device__ __forceinline__ float fresh_scale(float most) {
  float s;
  if (CT == kElemI8) {
    s = most * (1.0f / 127.0f);
  } else {
    int e;
    const float m = frexpf(most, &e);
    s = m > 0.0f ? ldexpf(1.0f, m <= 0.875f ? e - 9 : e - 8) : 0.0f;
  }
  return fminf(fmaxf(s, kLeast), kMost);
}

// Four values, already divided by the scale, in 8 bits: to nearest even and held
// within the range.
template <int CT>
__device__ __forceinline__ uint32_t stored4(const float (&v)[4]) {
  constexpr float most = stored_most<CT>();
  float s[4];
#pragma unroll
  for (int j = 0; j < 4; j++) s[j] = fminf(fmaxf(v[j], -most), most);
  if (CT == kElemI8) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) w |= ((uint32_t)(int)rintf(s[j]) & 255u) << (8 * j);
    return w;
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], w, true);
}
template <int CT>
__device__ __forceinline__ void values4(uint32_t w, float (&v)[4]) {
  if (CT == kElemI8) {
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = (float)(int8_t)(w >> (8 * j));
    return;
  }
  v[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
  v[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
  v[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
  v[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
}

// A lane's part of a row.
struct Lane {
  int u0, at0, at1;
  bool paired;
};
template <int D>
__device__ __forceinline__ Lane lane_of(int l, int rope_dims) {
  const int half = rope_dims >> 1, u0 = 4 * l;
  const bool paired = u0 < half;  // (half is a multiple of 4)
  const int at0 = paired ? u0 : rope_dims + 2 * (u0 - half);
  return Lane{u0, at0, paired ? u0 + half : at0 + 4, paired};
}

// The lane's weights of a norm; none: ones.
struct Weights {
  float x[4], y[4];
  __device__ __forceinline__ Weights(const float *w, const Lane &at) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[j] = w ? w[at.at0 + j] : 1.0f;
      y[j] = w ? w[at.at1 + j] : 1.0f;
    }
  }
};

// Norm of a row of which the lane has x and y.
template <int D>
__device__ __forceinline__ void norm_row(float (&x)[4], float (&y)[4], const Weights &w, float eps) {
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; j++) s += x[j] * x[j] + y[j] * y[j];
  const float scale = 1.0f / sqrtf(row_sum<D / 8>(s) / (float)D + eps);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    x[j] = x[j] * scale * w.x[j];
    y[j] = y[j] * scale * w.y[j];
  }
}

// Cosine and sine of a part of a turn, -1/2 .. 1/2: the quarter turns, then the
// series at x = -pi/4 .. pi/4, whose first terms left out are x^11 / 11! < 2^-28
// and x^12 / 12!.
__device__ __forceinline__ float2 cos_sin(float part) {
  const float quarters = part * 4.0f, k = rintf(quarters);
  const float x = (quarters - k) * 1.57079632679489662f, z = x * x;
  float s = fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
  s = fmaf(z, s, 1.0f / 120.0f);
  s = fmaf(z, s, -1.0f / 6.0f);
  s = fmaf(x * z, s, x);
  float c = fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  c = fmaf(z, c, -1.0f / 720.0f);
  c = fmaf(z, c, 1.0f / 24.0f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.0f);
  const int q = (int)k;
  const float cosine = q & 1 ? s : c, sine = q & 1 ? c : s;
  return make_float2(q + 1 & 2 ? -cosine : cosine, q & 2 ? -sine : sine);
}
__device__ __forceinline__ float2 angle_at(double turns_each, int position) {
  const double turns = (double)position * turns_each;
  return cos_sin((float)(turns - rint(turns)));
}
__device__ __forceinline__ void rotate_row(float (&x)[4], float (&y)[4], const float2 (&a)[4]) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const float p = x[j], q = y[j];
    x[j] = p * a[j].x - q * a[j].y;
    y[j] = p * a[j].y + q * a[j].x;
  }
}

__device__ __forceinline__ void load_row(const float *row, const Lane &at, float (&x)[4], float (&y)[4]) {
  const float4 a = *reinterpret_cast<const float4 *>(row + at.at0), b = *reinterpret_cast<const float4 *>(row + at.at1);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
  y[0] = b.x, y[1] = b.y, y[2] = b.z, y[3] = b.w;
}

// Tokens whose query rows a workgroup has: a thread an angle.
template <int D, int NT>
constexpr int query_tokens() {
  return NT / (D / 2) > 1 ? NT / (D / 2) : 1;
}

// NP: passes of a block's rows.  Workgroups 0 .. kv_units - 1 have keys and
// values, (block slot, KV head, key or value), the others tokens' query rows,
// (tokens, part).
template <int D, int CT, int NT, int NP>
__global__ __launch_bounds__(NT) void block_append_kernel(const PagedAppendArgs a, const CacheBlocks b, int kv_units,
                                                          int q_parts) {
  constexpr int kLanes = D / 8, kRows = NT / kLanes;  // of a row, rows at once
  constexpr int kTokens = query_tokens<D, NT>();
  __shared__ float2 sh_angle[kTokens][D / 2];  // a key's workgroup has its turns there
  __shared__ int sh_pos[kTokens];
  __shared__ float sh_most[NT / 64], sh_old;
  const int tid = threadIdx.x, sub = tid / kLanes;
  const Lane at = lane_of<D>(tid % kLanes, a.rope_dims);
  const int half = a.rope_dims >> 1;
  const int64_t table_keys = (int64_t)a.c.width << a.c.page_shift;
  auto turns_of = [&](int u) {
    const double turns = exp2(a.log2_base * (-2.0 * u / a.rope_dims)) * kInvTwoPi;
    return a.freq_factors ? turns / (double)a.freq_factors[u] : turns;
  };

  if ((int)blockIdx.x >= kv_units) {  // query rows
    const int unit = blockIdx.x - kv_units, t0 = unit / q_parts * kTokens, part = unit % q_parts;
    const int tokens = min(kTokens, a.tokens - t0);
    // row (t, h) of the thread, `step` rows on from one to the next; the first are on
    // their way before the positions are known
    const int step = q_parts * kRows, step_t = step / a.nq, step_h = step - step_t * a.nq;
    int t = (part * kRows + sub) / a.nq, h = part * kRows + sub - t * a.nq;
    float x[4], y[4], next_x[4], next_y[4];
    auto load = [&] {  // (behind the last row: another of the last token's)
      load_row(a.q + (t0 + min(t, tokens - 1)) * a.q_stride + (int64_t)h * D, at, next_x, next_y);
    };
    load();
    const Weights weights(a.q_norm, at);
    for (int i = tid >> 6; i < tokens; i += NT / 64) {  // a wave a token
      const int t = t0 + i;
      int seq = t, pos = -1;
      if (a.offsets) {
        seq = packed_sequence_of(a.offsets, a.c.sequences, t);
        if (seq < a.c.sequences) {
          const int begin = a.offsets[seq], end = a.offsets[seq + 1];
          if (t >= begin && t < end) pos = append_position(a.c.lengths[seq], (int64_t)end - t, a.c.page_shift, a.c.width);
        }
      } else {
        pos = append_position(a.c.lengths[seq], 1, a.c.page_shift, a.c.width);
      }
      if ((tid & 63) == 0) sh_pos[i] = pos;
    }
    __syncthreads();
    if (half > 0) {
      for (int i = tid; i < tokens * (D / 2); i += NT) {
        const int t = i / (D / 2), u = i - t * (D / 2);
        if (u < half) sh_angle[t][u] = angle_at(turns_of(u), sh_pos[t]);
      }
      __syncthreads();
    }
    while (t < tokens) {  // (the same for the lanes of a row)
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = next_x[j], y[j] = next_y[j];
      const int i = t;
      const int64_t o = ((int64_t)(t0 + t) * a.nq + h) * D;
      t += step_t;
      h += step_h;
      if (h >= a.nq) {
        t++;
        h -= a.nq;
      }
      load();
      if (sh_pos[i] < 0) continue;
      if (a.q_norm) norm_row<D>(x, y, weights, a.eps);
      if (at.paired) {
        const float2 angle[4] = {sh_angle[i][at.u0], sh_angle[i][at.u0 + 1], sh_angle[i][at.u0 + 2], sh_angle[i][at.u0 + 3]};
        rotate_row(x, y, angle);
      }
      store4(a.q_out, o + at.at0, a.out_type, x);
      store4(a.q_out, o + at.at1, a.out_type, y);
    }
    return;
  }

  // keys or values of a block
  const bool is_key = (blockIdx.x & 1) == 0;
  const int h = (int)(blockIdx.x >> 1) % a.c.nkv, slot = (int)(blockIdx.x >> 1) / a.c.nkv;
  int seq = slot, row_end;
  NewInBlock n;
  if (a.offsets) {
    seq = touched_sequence(a.offsets, a.c.sequences, slot, 1 << b.shift);
    const int begin = a.offsets[seq];
    row_end = a.offsets[seq + 1];
    n = new_in_block(a.c.lengths[seq], (int64_t)row_end - begin, slot - touched_first(begin, seq, 1 << b.shift), b.shift,
                     table_keys);
  } else {
    row_end = seq + 1;
    n = new_in_block(a.c.lengths[seq], 1, 0, b.shift, table_keys);
  }
  const int rows = n.end - n.first, behind = a.c.lengths[seq];  // row of position p: row_end - (behind - p)
  if (rows <= 0) return;  // (the same for the workgroup)
  const int page_mask = (1 << a.c.page_shift) - 1;
  const int page = page_or_none(a.c.pages[(int64_t)seq * a.c.width + (n.first >> a.c.page_shift)], a.c.page_count);
  const int64_t row0 = (int64_t)row_end - ((int64_t)behind - n.first);
  const float *src = is_key ? a.k : a.v ? a.v : a.k;
  const int64_t stride = is_key || !a.v ? a.k_stride : a.v_stride;
  float x[NP][4], y[NP][4];
#pragma unroll
  for (int i = 0; i < NP; i++) {  // (behind the last row: the first one's, which count for nothing)
    const int64_t t = row0 + (i * kRows + sub < rows ? i * kRows + sub : 0);
    const bool there = t >= 0 && t < a.tokens;
    load_row(src + (there ? t : 0) * stride + (int64_t)h * D, at, x[i], y[i]);
  }
  const bool old_block = (n.first & ((1 << b.shift) - 1)) != 0;
  const int64_t scale_at = (((int64_t)max(page, 0) * a.c.nkv + h) << (a.c.page_shift - b.shift)) +
                           ((n.first & page_mask) >> b.shift);
  float *scales = is_key ? b.key_scales : b.value_scales;
  float old = 0.0f;  // (read by the thread that writes it in the end)
  if (tid == 0) old = scales[scale_at];
  double *sh_turns = reinterpret_cast<double *>(&sh_angle[0][0]);
  if (is_key && half > 0) {
    for (int u = tid; u < half; u += NT) sh_turns[u] = turns_of(u);
    __syncthreads();
  }

  const bool norm = is_key ? a.k_norm != nullptr : a.norm_values != 0;
  const Weights weights(is_key ? a.k_norm : nullptr, at);
  void *out = is_key ? a.k_out : a.v_out;
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int64_t t = row0 + i * kRows + sub;
    if (norm) norm_row<D>(x[i], y[i], weights, a.eps);
    if (is_key && at.paired) {
      float2 angle[4];
#pragma unroll
      for (int j = 0; j < 4; j++) angle[j] = angle_at(sh_turns[at.u0 + j], n.first + i * kRows + sub);
      rotate_row(x[i], y[i], angle);
    }
    if (i * kRows + sub < rows && t >= 0 && t < a.tokens) {
      if (out) {
        const int64_t o = (t * a.c.nkv + h) * D;
        store4(out, o + at.at0, a.out_type, x[i]);
        store4(out, o + at.at1, a.out_type, y[i]);
      }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        most = fmaxf(most, fmaxf(fabsf(x[i][j]), fabsf(y[i][j])));
        if (!(fabsf(x[i][j]) < kInf) || !(fabsf(y[i][j]) < kInf)) most = kInf;
      }
    }
  }
  most = wave_max_f32(most);
  if (NT > 64) {
    if ((tid & 63) == 0) sh_most[tid >> 6] = most;
    if (tid == 0) sh_old = old;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; i++) most = fmaxf(most, sh_most[i]);
    old = sh_old;
  } else {
    old = readlane_f32(old, 0);
  }
  if (page < 0) return;  // rows of an absent page are dropped

  constexpr float kM = stored_most<CT>();
  const bool grows = old_block && most > old * kM;
  float scale = old;
  if (!old_block || grows) scale = fresh_scale<CT>(most);
  if (grows && CT == kElemI8) scale = fminf(fmaxf(scale, old * kGrowth), kMost);
  if (most == kInf) scale = __builtin_nanf("");
  uint8_t *pool = static_cast<uint8_t *>(is_key ? a.c.keys : a.c.values);
  uint8_t *head = pool + page * a.c.page_stride + ((int64_t)h << a.c.page_shift) * D;
  if (grows) {  // (the same for the workgroup) what the block holds moves to the new scale
    const int first = n.first & page_mask, begin = first & ~((1 << b.shift) - 1);
    const float ratio = old / scale;
    uint32_t *held = reinterpret_cast<uint32_t *>(head + (int64_t)begin * D);
    for (int i = tid; i < (first - begin) * (D / 4); i += NT) {
      float v[4];
      values4<CT>(held[i], v);
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] *= ratio;
      held[i] = stored4<CT>(v);
    }
  }
  const float inv = 1.0f / scale;
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const int64_t t = row0 + i * kRows + sub;
    if (i * kRows + sub >= rows || t < 0 || t >= a.tokens) continue;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[i][j] *= inv;
      y[i][j] *= inv;
    }
    uint8_t *row = head + (int64_t)((n.first & page_mask) + i * kRows + sub) * D;
    *reinterpret_cast<uint32_t *>(row + at.at0) = stored4<CT>(x[i]);
    *reinterpret_cast<uint32_t *>(row + at.at1) = stored4<CT>(y[i]);
  }
  if (tid == 0 && (!old_block || grows || most == kInf)) scales[scale_at] = scale;
}

template <int D, int CT, int NT, int NP>
hipError_t launch(const PagedAppendArgs &a, const CacheBlocks &b, int num_cus, hipStream_t s) {
  constexpr int kRows = NT / (D / 8);
  const int64_t slots = a.offsets ? touched_blocks(a.tokens, a.c.sequences, 1 << b.shift) : a.c.sequences;
  const int64_t kv_units = 2 * slots * a.c.nkv;
  constexpr int kTokens = query_tokens<D, NT>();
  const int q_groups = (a.tokens + kTokens - 1) / kTokens;
  int q_parts = (kTokens * a.nq + kRows - 1) / kRows;
  const int most = (4 * num_cus * 256 / NT + q_groups - 1) / q_groups;  // sixteen waves a CU
  q_parts = q_parts < 1 ? 1 : q_parts > most ? most : q_parts;
  const int64_t grid = kv_units + (a.nq > 0 ? (int64_t)q_groups * q_parts : 0);
  if (grid >> 31) return hipErrorInvalidValue;
  hipLaunchKernelGGL((block_append_kernel<D, CT, NT, NP>), dim3((unsigned)grid), dim3(NT), 0, s, a, b, (int)kv_units,
                     q_parts);
  return hipGetLastError();
}

template <int D, int CT>
hipError_t launch_type(const PagedAppendArgs &a, const CacheBlocks &b, int num_cus, hipStream_t s) {
  if (!a.offsets) return launch<D, CT, 64, 1>(a, b, num_cus, s);
  constexpr int kRows = 256 / (D / 8);
  switch (((1 << b.shift) + kRows - 1) / kRows) {
    case 1: return launch<D, CT, 256, 1>(a, b, num_cus, s);
    case 2: return launch<D, CT, 256, 2>(a, b, num_cus, s);
    case 4: return launch<D, CT, 256, 4>(a, b, num_cus, s);
    case 8: return launch<D, CT, 256, 8>(a, b, num_cus, s);
    case 16: return D == 256 ? launch<D, CT, 256, D == 256 ? 16 : 8>(a, b, num_cus, s) : hipErrorInvalidValue;
    default: return hipErrorInvalidValue;
  }
}

template <int D>
hipError_t launch_width(const PagedAppendArgs &a, const CacheBlocks &b, int num_cus, hipStream_t s) {
  return a.c.type == kElemI8 ? launch_type<D, kElemI8>(a, b, num_cus, s) : launch_type<D, kElemE4m3>(a, b, num_cus, s);
}

}  // namespace

bool block_append_fits(const PagedAppendArgs &a, const CacheBlocks &b) {
  const int64_t slots = a.offsets ? touched_blocks(a.tokens, a.c.sequences, 1 << b.shift) : a.c.sequences;
  return !((2 * slots * a.c.nkv + (int64_t)a.tokens * ((a.nq + 1) / 2)) >> 31);
}

hipError_t launch_block_append(const PagedAppendArgs &a, const CacheBlocks &b, int num_cus, hipStream_t s) {
  if (a.tokens < 1 || a.nq < 0 || a.c.nkv < 1 || a.rope_dims % 8 != 0 || a.rope_dims > a.c.head_dim ||
      elem_bytes(a.c.type) != 1 || !b.key_scales || !b.value_scales || b.shift < 4 || b.shift > 7 ||
      b.shift > a.c.page_shift || !block_append_fits(a, b))
    return hipErrorInvalidValue;
  switch (a.c.head_dim) {
    case 64: return launch_width<64>(a, b, num_cus, s);
    case 128: return launch_width<128>(a, b, num_cus, s);
    case 256: return launch_width<256>(a, b, num_cus, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace hp
