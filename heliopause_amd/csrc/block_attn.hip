// block_attn.hip -- attention of one new token of every sequence over pages whose
// blocks have scales of their own, over listed blocks only, or both
// (hp_paged_attn.h).
#include "hp_paged_attn.h"

namespace hp {

namespace {

template <int D, int MODE>
hipError_t launch_scaled(const PagedAttnArgs &a, int groups, hipStream_t s) {
  return a.c.type == kElemI8 ? launch<D, kElemI8, MODE | kScaled, false>(a, groups, s)
                             : launch<D, kElemE4m3, MODE | kScaled, false>(a, groups, s);
}

template <int D>
hipError_t launch_type(const PagedAttnArgs &a, int groups, hipStream_t s) {
  if (!a.selected) return launch_scaled<D, kWhole>(a, groups, s);
  if (a.key_scales) return launch_scaled<D, kSelected>(a, groups, s);
  if (a.c.type == kElemF16) return launch<D, kElemF16, kSelected, false>(a, groups, s);
  if (a.c.type == kElemE4m3) return launch<D, kElemE4m3, kSelected, false>(a, groups, s);
  // two bf16 parts hold an f16 or bf16 query; an f32 one has a third
  return a.q_type == kElemF32 ? launch<D, kElemBf16, kSelected, true>(a, groups, s)
                              : launch<D, kElemBf16, kSelected, false>(a, groups, s);
}

}  // namespace

hipError_t launch_block_attn(const PagedAttnArgs &args, int groups, hipStream_t s) {
  PagedAttnArgs a = args;
  if (groups < 1 || a.c.sequences < 1 || a.c.nkv < 1 || a.nq % a.c.nkv != 0 || !a.partials ||
      paged_attn_most_steps(a) >> 31 || (!a.selected && !a.key_scales) || !a.key_scales != !a.value_scales)
    return hipErrorInvalidValue;
  if (a.key_scales) {
    if (elem_bytes(a.c.type) != 1) return hipErrorInvalidValue;
    a.c.key_scale = 1.0f;
    a.c.value_scale = kUnbias;
  }
  switch (a.c.head_dim) {
    case 64: return launch_type<64>(a, groups, s);
    case 128: return launch_type<128>(a, groups, s);
    case 256: return launch_type<256>(a, groups, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace hp
