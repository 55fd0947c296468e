// paged_append.hip -- a batch's new tokens on their way from the projections
// to the attention: head norms, position rotation, and the keys and values
// into the sequences' pages.
//
// Per token at position p and head row x of D elements:
//   y = x / sqrt(mean(x^2) + eps) * w          (where the row has a norm)
//   angle_u = p * base^(-2u / R) / factor_u    (R = rope_dims, u < R / 2)
//   (y_u, y_{u + R/2}) -> (y_u cos - y_{u+R/2} sin, y_u sin + y_{u+R/2} cos)
// for query and key rows; value rows have the norm without a weight, or none.
// Elements from R on are not rotated.
//
// The angles are formed in 64 bits: at position 10^6 an f32 product is 0.06
// radians off.  The turns past the whole ones are taken off before the sine
// and cosine, which then need no reduction of their own; cosine and sine are
// used as f32, as the rest of the arithmetic (a row's sum of squares is a tree
// of f32 sums over the lanes that hold it).
//
// A workgroup takes a token, or where tokens are few a part of its rows.  Its
// threads first form the token's angles, one u each, into LDS -- every head row
// has the same -- and then take the rows, D / 8 lanes a row: lane l holds
// elements 4l .. 4l+3 of both halves of the rotated part (or eight consecutive
// ones of the rest), so that a pair sits in one lane and loads and stores are
// 16 and 8 bytes wide.  The first rows' loads go out before the position is
// known.  16000 tokens of 32 + 16 head rows of 128 (655 MB in and out): 121 us,
// 5.4 TB/s, which its bytes bound; with four tokens a workgroup 131 us, with
// loads past the caches 138.
#include "hp_serving.h"
#include "hp_wave.h"

namespace hp {

namespace {

constexpr int kThreads = 256;
constexpr float kE4m3Most = 448.0f;
constexpr double kInvTwoPi = 0.15915494309189533577;

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

// Four consecutive elements of a cache row.  E4M3 keeps x / scale, rounded to
// nearest even and held within the type's range (the conversion would make a
// NaN of what is past it); a NaN stays one.
template <int CT>
__device__ __forceinline__ void store_cache4(void *p, int64_t i, const float (&v)[4], float inv_scale) {
  if (CT != kElemE4m3) {
    store4(p, i, CT, v);
    return;
  }
  float s[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    s[j] = v[j] * inv_scale;
    s[j] = s[j] > kE4m3Most ? kE4m3Most : s[j] < -kE4m3Most ? -kE4m3Most : s[j];
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], w, true);
  *reinterpret_cast<int *>(static_cast<uint8_t *>(p) + i) = w;
}

template <int D, int CT>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(const PagedAppendArgs a) {
  constexpr int kLanes = D / 8;  // of a row
  constexpr int kRows = kThreads / kLanes;
  __shared__ float2 angle[D / 2];  // cos, sin
  const int tid = threadIdx.x, t = blockIdx.x, page_size = 1 << a.c.page_shift;

  // A thread's work: rows row0, row0 + step, ..., its elements at0 .. and at1 ..
  // of a row.  The next row's loads (the last row's again at the end) are on
  // their way while one is worked on.
  const int rows = a.nq + 2 * a.c.nkv, half = a.rope_dims >> 1;
  const int l = tid % kLanes, u0 = 4 * l;  // the lane's four pairs
  const bool paired = u0 < half;           // (half is a multiple of 4)
  const int at0 = paired ? u0 : a.rope_dims + 2 * (u0 - half), at1 = paired ? u0 + half : at0 + 4;
  const int row0 = blockIdx.y * kRows + tid / kLanes, step = gridDim.y * kRows;
  float4 next0, next1;
  auto load = [&](int row) {
    const int r = min(row, rows - 1), hk = r - a.nq, hv = hk - a.c.nkv;  // query, key, value head
    const float *src = hk < 0           ? a.q + t * a.q_stride + (int64_t)r * D
                       : hv < 0 || !a.v ? a.k + t * a.k_stride + (int64_t)(hv < 0 ? hk : hv) * D
                                        : a.v + t * a.v_stride + (int64_t)hv * D;
    next0 = *reinterpret_cast<const float4 *>(src + at0);
    next1 = *reinterpret_cast<const float4 *>(src + at1);
  };
  load(row0);

  // the token's sequence, position and page (each wave for itself)
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
  if (pos < 0) return;  // (the same for the workgroup) the token's rows stay as they were
  const int page = page_or_none(a.c.pages[(int64_t)seq * a.c.width + (pos >> a.c.page_shift)], a.c.page_count);
  const int64_t slot_at = page * a.c.page_stride + (int64_t)(pos & (page_size - 1)) * D;  // for head 0
  for (int u = tid; u < half; u += kThreads) {
    double turns = (double)pos * (exp2(a.log2_base * (-2.0 * u / a.rope_dims)) * kInvTwoPi);
    if (a.freq_factors) turns /= (double)a.freq_factors[u];
    double s, c;
    sincospi(2.0 * (turns - rint(turns)), &s, &c);
    angle[u] = make_float2((float)c, (float)s);
  }
  __syncthreads();

  const float inv_k = 1.0f / a.c.key_scale, inv_v = 1.0f / a.c.value_scale;
  for (int r = row0; r < rows; r += step) {  // (the same for the lanes of a row)
    float x[4] = {next0.x, next0.y, next0.z, next0.w}, y[4] = {next1.x, next1.y, next1.z, next1.w};
    load(r + step);
    const int kind = r < a.nq ? 0 : r < a.nq + a.c.nkv ? 1 : 2;  // query, key, value
    const int h = kind == 0 ? r : kind == 1 ? r - a.nq : r - a.nq - a.c.nkv;
    const float *w = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    if (w || (kind == 2 && a.norm_values)) {  // the same for the lanes of a row
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; j++) s += x[j] * x[j] + y[j] * y[j];
      const float scale = 1.0f / sqrtf(row_sum<kLanes>(s) / (float)D + a.eps);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        x[j] = x[j] * scale * (w ? w[at0 + j] : 1.0f);
        y[j] = y[j] * scale * (w ? w[at1 + j] : 1.0f);
      }
    }
    if (kind != 2 && paired) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float2 cs = angle[u0 + j];
        const float p = x[j], q = y[j];
        x[j] = p * cs.x - q * cs.y;
        y[j] = p * cs.y + q * cs.x;
      }
    }
    void *out = kind == 0 ? a.q_out : kind == 1 ? a.k_out : a.v_out;
    if (out) {
      const int64_t o = ((int64_t)t * (kind == 0 ? a.nq : a.c.nkv) + h) * D;
      store4(out, o + at0, a.out_type, x);
      store4(out, o + at1, a.out_type, y);
    }
    if (kind != 0 && page >= 0) {
      const int64_t o = slot_at + (int64_t)h * page_size * D;
      store_cache4<CT>(kind == 1 ? a.c.keys : a.c.values, o + at0, x, kind == 1 ? inv_k : inv_v);
      store_cache4<CT>(kind == 1 ? a.c.keys : a.c.values, o + at1, y, kind == 1 ? inv_k : inv_v);
    }
  }
}

template <int D>
hipError_t launch_width(const PagedAppendArgs &a, int num_cus, hipStream_t s) {
  const int passes = (a.nq + 2 * a.c.nkv + kThreads * 8 / D - 1) / (kThreads * 8 / D);
  int split = (4 * num_cus + a.tokens - 1) / a.tokens;  // four workgroups a CU
  split = split > passes ? passes : split;
  const dim3 grid(a.tokens, split);
  if (a.c.type == kElemF16)
    hipLaunchKernelGGL((paged_append_kernel<D, kElemF16>), grid, dim3(kThreads), 0, s, a);
  else if (a.c.type == kElemBf16)
    hipLaunchKernelGGL((paged_append_kernel<D, kElemBf16>), grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((paged_append_kernel<D, kElemE4m3>), grid, dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs &a, int num_cus, hipStream_t s) {
  if (a.tokens < 1 || a.nq < 0 || a.c.nkv < 1 || a.rope_dims % 8 != 0 || a.rope_dims > a.c.head_dim)
    return hipErrorInvalidValue;
  switch (a.c.head_dim) {
    case 64: return launch_width<64>(a, num_cus, s);
    case 128: return launch_width<128>(a, num_cus, s);
    case 256: return launch_width<256>(a, num_cus, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace hp
