// Walks the index rules of hp_pages.h that blocks and page plans go by over bad
// lengths, odd batches and full tables; prints "ok" or the first rule that fails.
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <random>
#include <set>
#include <utility>
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
  std::mt19937 rng(3);
  const int extremes[] = {-2147483647 - 1, -5, 0, 1, 15, 16, 17, 63, 64, 65, 1000, 1 << 30, 2147483647};

  // every new position of a sequence is in exactly one touched block, and only they are
  for (int round = 0; round < 4000; round++) {
    const int shift = 4 + rng() % 4, n = 1 + rng() % 12, keys = (1 << shift) * (1 + rng() % 9);  // (a page holds whole blocks)
    std::vector<int> offset(n + 1), length(n);
    offset[0] = rng() % 3 ? 0 : rng() % 100;
    for (int s = 0; s < n; s++) {
      const int rows = rng() % 4 ? rng() % 300 : 0;
      offset[s + 1] = offset[s] + rows;
      length[s] = rng() % 5 ? rows + rng() % 200 : (int)(rng() % 40);
    }
    const int64_t slots = touched_blocks(offset[n], n, 1 << shift);
    std::set<std::pair<int, int>> seen;
    for (int s = 0; s < n; s++) {
      const int64_t begin = touched_first(offset[s], s, 1 << shift), next = touched_first(offset[s + 1], s + 1, 1 << shift);
      CHECK(begin < next && next <= slots);
      const int rows = offset[s + 1] - offset[s];
      for (int64_t slot = begin; slot < next; slot++) {
        const NewInBlock b = new_in_block(length[s], rows, slot - begin, shift, keys);
        CHECK(b.first <= b.end && b.end - b.first <= 1 << shift);
        if (b.first < b.end) CHECK(b.first >> shift == b.block && (b.end - 1) >> shift == b.block && b.first < keys && b.end <= length[s]);
        for (int p = b.first; p < b.end; p++) CHECK(seen.insert({s, p}).second);
      }
      // as the rows' own rule places them
      for (int t = 0; t < rows; t++) {
        const int p = append_position(length[s], rows - t, shift, keys >> shift);
        if (p >= 0) CHECK(seen.count({s, p}));
      }
    }
  }
  for (int length : extremes)
    for (int64_t rows : {(int64_t)-2147483648ll, (int64_t)-1, (int64_t)0, (int64_t)1, (int64_t)70, (int64_t)4294967295ll})
      for (int64_t i : {(int64_t)-3, (int64_t)0, (int64_t)1, (int64_t)1 << 26}) {
        const NewInBlock b = new_in_block(length, rows, i, 4, 4096);
        CHECK(b.first <= b.end && b.end - b.first <= 16);
        if (b.first < b.end) CHECK(b.first >= 0 && b.block < 256 && length > 0 && rows > 0);
      }

  // plans stay within the table and name new positions' pages only
  for (int length : extremes)
    for (int64_t fresh : {(int64_t)-7, (int64_t)0, (int64_t)1, (int64_t)33, (int64_t)2147483647})
      for (int keep : extremes)
        for (int shift : {4, 6, 12})
          for (int width : {1, 3, 100}) {
            const PlanSpan p = plan_span(length, fresh, keep, shift, width);
            CHECK(p.old >= 0 && p.fresh >= 0 && p.back >= 0 && p.back <= width);
            CHECK(p.first >= 0 && p.first <= width && p.last <= width && p.first <= p.last);
            CHECK(p.old == (keep < 0 || length < 0 ? 0 : length) && (keep >= 0 || p.back == width));
            if (keep >= 0) CHECK(p.back == std::min(width, keep >> shift));
            for (int64_t e = p.first; e < p.last; e++) CHECK(e << shift >= p.old && e << shift < p.old + p.fresh);
            if (p.last < width) CHECK(((int64_t)p.last << shift) >= p.old + p.fresh);
          }
  puts("ok");
  return 0;
}
