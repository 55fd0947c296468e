// paged_attn.hip -- attention of one new token of every sequence over its whole
// pages (hp_paged_attn.h), and what its launches and those of block_attn.hip
// need: their shares and scratch.
#include "hp_paged_attn.h"

namespace hp {

namespace {

template <int D>
hipError_t launch_type(const PagedAttnArgs &a, int groups, hipStream_t s) {
  if (a.c.type == kElemF16) return launch<D, kElemF16, kWhole, false>(a, groups, s);
  if (a.c.type == kElemE4m3) return launch<D, kElemE4m3, kWhole, false>(a, groups, s);
  // two bf16 parts hold an f16 or bf16 query; an f32 one has a third
  return a.q_type == kElemF32 ? launch<D, kElemBf16, kWhole, true>(a, groups, s)
                                 : launch<D, kElemBf16, kWhole, false>(a, groups, s);
}

size_t part_bytes(int head_dim, bool scaled) { return (size_t)kHeads * (head_dim + 2 + scaled) * sizeof(float); }
static_assert(sizeof(Part<64, kWhole>) == kHeads * 66 * sizeof(float) && sizeof(Part<64, kScaled>) == kHeads * 67 * sizeof(float),
              "as the scratch has them");

}  // namespace

uint64_t paged_attn_most_steps(const PagedAttnArgs &a) {
  uint64_t keys = a.selected ? (uint64_t)a.budget << a.block_shift : (uint64_t)a.c.width << a.c.page_shift;
  if (a.window > 0 && keys > (uint64_t)a.window + 15) keys = (uint64_t)a.window + 15;
  const int step = step_of(a.c.head_dim, a.c.type);
  return (keys + step - 1) / step * a.c.sequences * a.c.nkv;
}

int paged_attn_groups(const PagedAttnArgs &a, int num_cus) {
  const uint64_t most = paged_attn_most_steps(a);
  // two workgroups a CU; block_attn.hip's of 8 bits, which have half the bytes on
  // their way in as many keys, as many as the registers hold
  const int each = elem_bytes(a.c.type) == 1 && (a.key_scales || a.selected) ? a.c.head_dim == 64 ? 4 : a.c.head_dim == 128 ? 3 : 2 : 2;
  const int room = each * num_cus / blocks_of(a.nq, a.c.nkv);
  return most < (uint64_t)room ? (int)most : room < 1 ? 1 : room;
}

size_t paged_attn_scratch_bytes(const PagedAttnArgs &a, int groups) {
  const size_t blocks = blocks_of(a.nq, a.c.nkv);
  return blocks * (2 * (size_t)groups * part_bytes(a.c.head_dim, a.key_scales != nullptr) +
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
