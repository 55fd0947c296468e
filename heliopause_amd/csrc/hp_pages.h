// hp_pages.h -- where the operators over several sequences find things: a
// position's page, a sequence's keys, the split of a batch's steps over
// workgroups, a packed block's sequence.  Plain integer rules without a device
// header, so that the CPU tests walk them over bad tables and odd batches
// before a kernel does.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define HP_PAGES_FN __host__ __device__ __forceinline__
#else
#define HP_PAGES_FN static inline
#endif

namespace hp {

// The page that a table's entry names, or -1.
HP_PAGES_FN int page_or_none(int entry, int page_count) { return entry >= 0 && entry < page_count ? entry : -1; }

// Position of the token `behind` places before the end of a sequence of
// `length` tokens (1: the last), or -1 where the table of `width` pages has
// no place for it.
HP_PAGES_FN int append_position(int length, int64_t behind, int page_shift, int width) {
  const int64_t p = (int64_t)length - behind;
  return p >= 0 && (p >> page_shift) < width ? (int)p : -1;
}

constexpr int kPagedWaves = 4;  // waves of a workgroup of the paged attention, side by side along the keys

// A sequence's keys first .. end - 1, and where the walk over them begins: at
// a multiple of 16, so that 16 keys on end share a page.
struct KeySpan {
  int first, begin, end;
};
HP_PAGES_FN KeySpan key_span(int length, int64_t table_keys, int window) {
  KeySpan s;
  s.end = length < 0 ? 0 : length < table_keys ? length : (int)table_keys;
  s.first = window > 0 && s.end > window ? s.end - window : 0;
  s.begin = s.first & ~15;
  return s;
}
// Steps of `step` keys (a power of two) that the walk takes.
HP_PAGES_FN uint32_t span_steps(const KeySpan &s, int step) { return (uint32_t)(s.end - s.begin + step - 1) / (uint32_t)step; }

// Share i of `shares` (<= total) of the steps 0 .. total - 1 begins here, and
// the share that step t is in: the first total % shares shares have one step
// more than the others.
HP_PAGES_FN uint32_t share_begin(uint32_t total, uint32_t i, uint32_t shares) {
  const uint32_t each = total / shares, more = total - each * shares;
  return i * each + (i < more ? i : more);
}
HP_PAGES_FN uint32_t share_of(uint32_t total, uint32_t t, uint32_t shares) {
  const uint32_t each = total / shares, more = total - each * shares, long_part = more * (each + 1);
  return t < long_part ? t / (each + 1) : more + (t - long_part) / each;
}

// A packed batch in blocks of `rows` query rows: sequence s has the blocks from
// this one up to the next sequence's, at least as many as its rows fill, with
// no sum over the sequences before it.
HP_PAGES_FN int64_t packed_first_block(int offset, int s, int rows) { return (offset > 0 ? offset : 0) / rows + (int64_t)s; }
HP_PAGES_FN int64_t packed_blocks(int64_t tokens, int64_t sequences, int rows) { return tokens / rows + 1 + sequences; }

}  // namespace hp
