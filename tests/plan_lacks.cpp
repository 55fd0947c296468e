// Walks the rule of hp_pages.h for the pages that a step's new tokens lie in and
// that the step does not deal, against a walk over the tokens; prints "ok" or the
// first check that fails.
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <set>

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
  for (int shift : {4, 5})
    for (int width : {1, 2, 5})
      for (int old = 0; old < 130; old++)
        for (int64_t fresh = 0; fresh < 70; fresh++) {
          const PlanSpan p = plan_span(old, fresh, 0, shift, width);
          const PlanRest r = plan_rest(old, fresh, shift, width);
          std::set<int64_t> pages;
          for (int64_t i = old; i < old + fresh; i++) pages.insert(i >> shift);
          int beyond = 0, begun = -1;
          for (int64_t page : pages) {
            if (page >= width)
              beyond++;
            else if (page < p.first)
              begun = (int)page;
            else
              CHECK(page < p.last);
          }
          CHECK(r.beyond == beyond && r.begun == begun);
          CHECK((int)pages.size() == (p.last - p.first) + beyond + (begun >= 0));
        }
  const int most = 2147483647;
  for (int width : {1, 100, 1 << 26}) {
    PlanRest r = plan_rest(most, most, 4, width);
    CHECK(r.begun == -1 && r.beyond == (1 << 28) - (most >> 4));
    r = plan_rest(0, most, 4, width);
    CHECK(r.begun == -1 && r.beyond == std::max(0, (1 << 27) - width));
    r = plan_rest(most, 0, 4, width);
    CHECK(r.begun == -1 && r.beyond == 0);
  }
  puts("ok");
  return 0;
}
