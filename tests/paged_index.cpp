// Walks the index rules of hp_pages.h over bad tables, odd batches and uneven
// shares; prints "ok" or the first rule that fails.
#include <stdio.h>
#include <stdlib.h>

#include <random>
#include <vector>

#include "../heliopause_amd/csrc/hp_pages.h"

#define CHECK(c)                                          \
  do {                                                    \
    if (!(c)) {                                           \
      printf("failed: %s (line %d)\n", #c, __LINE__);     \
      exit(1);                                            \
    }                                                     \
  } while (0)

using namespace hp;

int main() {
  // bad pages and positions
  for (int e : {-2147483647 - 1, -1, 5, 6, 2147483647}) CHECK(page_or_none(e, 5) == -1);
  for (int e = 0; e < 5; e++) CHECK(page_or_none(e, 5) == e);
  CHECK(append_position(0, 1, 4, 3) == -1 && append_position(1, 1, 4, 3) == 0);
  CHECK(append_position(48, 1, 4, 3) == 47 && append_position(49, 1, 4, 3) == -1);
  CHECK(append_position(-2147483647 - 1, 2147483647ll, 4, 3) == -1);
  CHECK(append_position(2147483647, 1, 4, 3) == -1);

  // spans: the keys that count, walked from a tile's start, never past the table
  for (int length : {-5, 0, 1, 15, 16, 17, 127, 128, 129, 300, 511, 512, 513, 2147483647})
    for (int window : {0, 1, 15, 16, 17, 100, 512, 2147483647}) {
      const KeySpan s = key_span(length, 512, window);
      const int end = length < 0 ? 0 : length > 512 ? 512 : length;
      CHECK(s.end == end && s.first == (window > 0 && end > window ? end - window : 0));
      CHECK(s.begin <= s.first && s.first - s.begin < 16 && s.begin % 16 == 0);
      for (int step : {64, 128}) {
        CHECK((span_steps(s, step) == 0) == (end == 0));
        CHECK((uint64_t)s.begin + span_steps(s, step) * (uint64_t)step >= (uint64_t)end);
        if (window > 0) CHECK(span_steps(s, step) <= ((uint64_t)window + 15 + step - 1) / step);
      }
    }

  // shares: together every step once, none empty, and each step's share is found
  std::mt19937 rng(1);
  for (int round = 0; round < 2000; round++) {
    const uint32_t total = 1 + rng() % (round < 1000 ? 200 : 5000), groups = 1 + rng() % 600;
    const uint32_t shares = groups < total ? groups : total;
    CHECK(share_begin(total, 0, shares) == 0 && share_begin(total, shares, shares) == total);
    for (uint32_t i = 0; i < shares; i++) {
      const uint32_t b = share_begin(total, i, shares), e = share_begin(total, i + 1, shares);
      CHECK(b < e);
      CHECK(share_of(total, b, shares) == i && share_of(total, e - 1, shares) == i);
    }
    // a row's parts: the share of its first step writes slot 2 i + 1, later
    // ones slot 2 i, and no slot has two writers
    std::vector<int> writer(2 * shares, -1);
    uint32_t at = 0;
    for (int row = 0; at < total; row++) {
      uint32_t n = 1 + rng() % 40;
      if (n > total - at) n = total - at;
      const uint32_t first = share_of(total, at, shares), last = share_of(total, at + n - 1, shares);
      if (first != last)
        for (uint32_t i = first; i <= last; i++) {
          const uint32_t slot = 2 * i + (i == first ? 1 : 0);
          CHECK(writer[slot] == -1);
          writer[slot] = row;
        }
      at += n;
    }
  }
  const uint32_t big = 0x7fffffffu;
  CHECK(share_begin(big, 511, 512) < big && share_of(big, big - 1, 512) == 511);

  // packed blocks: in order, and enough for every sequence
  for (int round = 0; round < 3000; round++) {
    const int n = 1 + rng() % 20, rows = 32 << (round % 3);
    std::vector<int> offset(n + 1);
    offset[0] = rng() % 200;
    for (int s = 0; s < n; s++) offset[s + 1] = offset[s] + (rng() % 4 ? rng() % 400 : 0);
    const int64_t blocks = packed_blocks(offset[n], n, rows);
    for (int s = 0; s < n; s++) {
      const int64_t b = packed_first_block(offset[s], s, rows);
      const int64_t e = s + 1 < n ? packed_first_block(offset[s + 1], s + 1, rows) : blocks;
      CHECK(b < e && e <= blocks);
      CHECK((e - b) * rows >= offset[s + 1] - offset[s]);
    }
  }
  CHECK(packed_first_block(-7, 3, 128) == 3);
  puts("ok");
  return 0;
}
