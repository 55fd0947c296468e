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

// Blocks of `block` positions (a power of two) that new tokens lie in.  Sequence
// s's slots begin here and end where the next one's begin: rows offset .. end -
// 1 of it touch at most (rows - 1) / block + 2 blocks, whatever position they
// begin at, and with no sum over the sequences before it there are that many.
HP_PAGES_FN int64_t touched_first(int offset, int s, int block) { return (offset > 0 ? offset : 0) / block + 2 * (int64_t)s; }
HP_PAGES_FN int64_t touched_blocks(int64_t tokens, int64_t sequences, int block) { return tokens / block + 2 * sequences; }

// The new tokens of a sequence of `length` tokens, the last `rows` of them, in
// the i-th block that they touch: positions first .. end - 1, none where the
// block is behind the last or outside the table.
struct NewInBlock {
  int block, first, end;
};
HP_PAGES_FN NewInBlock new_in_block(int length, int64_t rows, int64_t i, int block_shift, int64_t table_keys) {
  NewInBlock n = {0, 0, 0};
  const int64_t all = length > 0 ? length : 0, begin = rows >= all ? 0 : rows > 0 ? all - rows : all;
  const int64_t b = (begin >> block_shift) + i, at = b << block_shift;
  const int64_t first = at > begin ? at : begin, stop = at + ((int64_t)1 << block_shift), end = stop < all ? stop : all;
  if (i < 0 || first >= end || at >= table_keys) return n;
  n.block = (int)b;
  n.first = (int)first;
  n.end = (int)end;
  return n;
}

// A step's plan for one sequence: table entries 0 .. back - 1 are given back;
// the new tokens' positions begin at `old`, and of the entries first .. last -
// 1, whose positions are all new, those that name no page get one.
struct PlanSpan {
  int old, back, first, last;
  int64_t fresh;  // new tokens
};
HP_PAGES_FN PlanSpan plan_span(int length, int64_t fresh, int keep_from, int page_shift, int width) {
  PlanSpan p;
  p.old = keep_from < 0 || length < 0 ? 0 : length;
  const int64_t gone = keep_from < 0 ? width : keep_from >> page_shift, page = (int64_t)1 << page_shift;
  p.back = gone < width ? (int)gone : width;
  p.fresh = fresh > 0 ? fresh : 0;
  const int64_t first = ((int64_t)p.old + page - 1) >> page_shift, last = ((int64_t)p.old + p.fresh + page - 1) >> page_shift;
  p.first = first < width ? (int)first : width;
  p.last = last < width ? (int)last : width;
  return p;
}

// The other pages that the new tokens lie in: entry `begun` of the table (-1:
// none), whose first positions are older, and `beyond` that are past its end.
struct PlanRest {
  int begun, beyond;
};
HP_PAGES_FN PlanRest plan_rest(int old, int64_t fresh, int page_shift, int width) {
  PlanRest r = {-1, 0};
  if (fresh <= 0) return r;
  const int64_t page = (int64_t)1 << page_shift, end = ((int64_t)old + fresh + page - 1) >> page_shift;
  const int first = old >> page_shift;
  if ((old & (page - 1)) != 0 && first < width) r.begun = first;
  if (end > width) r.beyond = (int)(end - (first > width ? first : width));
  return r;
}

}  // namespace hp
