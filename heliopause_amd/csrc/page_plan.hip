// page_plan.hip -- a step's page tables, lengths, row offsets and slot maps
// from the requests' lengths.
//
// The free pages are a stack.  In order of sequence and position: pages that a
// sequence no longer needs go on top, then the entries that the new tokens need
// and that name no page take theirs from the top.  So a step is two counts of
// each sequence, their sums over the sequences before it, and copies:
//   stack = free[0 .. f) ++ (named entries given back),  T = its size
//   entry of rank r among those wanted: stack[T - 1 - r], -1 from r = T on
// A page that was begun without one gets none, since its first positions are not
// in the cache; it is among those missing as long as new tokens lie in it, as what
// lies past the table's end is.
// and the outcome does not depend on which workgroup comes first.
#include "hp_serving.h"
#include "hp_wave.h"

namespace hp {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kScanThreads = 1024;
constexpr int kAtOnce = 8;  // entries that a lane has on their way

// Scratch: what one launch leaves for the next.
struct PlanState {
  int free_with, free_after;  // entries of the stack, with those given back and in the end
  int pad[2];
};
struct PlanRow {
  int old, fresh, back, want;  // pages that go back, that are wanted
};
struct PlanAt {
  int back, want;  // the same of the sequences before
};
// In `old` and `fresh`, which are not negative: some of the new pages' entries want
// a page and some have one; all have one.
constexpr int kGaps = 1 << 31, kNamed = 1 << 31;
__device__ __forceinline__ PlanRow *rows_of(PlanState *s) { return reinterpret_cast<PlanRow *>(s + 1); }
__device__ __forceinline__ PlanAt *places_of(PlanState *s, int sequences) {
  return reinterpret_cast<PlanAt *>(rows_of(s) + sequences);
}
__device__ __forceinline__ int *offsets_of(PlanState *s, int sequences) {
  return reinterpret_cast<int *>(places_of(s, sequences) + sequences);
}
__device__ __forceinline__ int free_before(const PagePlanArgs &a) { return min(max(*a.free_count, 0), a.page_count); }

__device__ __forceinline__ PlanSpan span_of(const PagePlanArgs &a, int s) {
  const int length = a.lengths[s], keep = a.keep_from ? a.keep_from[s] : 0;
  return plan_span(length, a.fresh ? a.fresh[s] : (length > 0 && keep >= 0 ? 1 : 0), keep, a.page_shift, a.width);
}

// Sum of v over the lanes up to this one.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t o = __shfl_up(v, d);
    v += lane >= d ? o : 0;
  }
  return v;
}

// One sequence, by a wave: how many pages go back, how many are wanted.
__device__ __forceinline__ void count_sequence(const PagePlanArgs &a, PlanState *st, int s) {
  const int lane = threadIdx.x & 63;
  const PlanSpan p = span_of(a, s);
  const int *table = a.pages + (int64_t)s * a.width;
  int back = 0, want = 0;
  for (int i0 = lane; i0 < p.back; i0 += 64 * kAtOnce) {
#pragma unroll
    for (int j = 0; j < kAtOnce; j++) {
      const int i = i0 + 64 * j, entry = table[min(i, p.back - 1)];
      back += i < p.back && page_or_none(entry, a.page_count) >= 0;
    }
  }
  for (int i0 = p.first + lane; i0 < p.last; i0 += 64 * kAtOnce) {
#pragma unroll
    for (int j = 0; j < kAtOnce; j++) {
      const int i = i0 + 64 * j, entry = table[min(i, p.last - 1)];
      want += i < p.last && (i < p.back || page_or_none(entry, a.page_count) < 0);
    }
  }
  const uint64_t both = wave_scan((uint64_t)(uint32_t)back << 32 | (uint32_t)want);
  if (lane == 63) {
    want = (int)(uint32_t)both;
    rows_of(st)[s] = PlanRow{p.old | (want > 0 && want < p.last - p.first ? kGaps : 0),
                             (int)(p.fresh > 0x7fffffff ? 0x7fffffff : p.fresh) | (want == 0 ? kNamed : 0),
                             (int)(both >> 32), want};
  }
}

// Sums over the sequences before, by one workgroup; a thread has a run of them.
template <int THREADS>
__device__ void scan_sequences(const PagePlanArgs &a, PlanState *st) {
  __shared__ uint64_t sh_pages[THREADS / 64], sh_tokens[THREADS / 64];
  const PlanRow *rows = rows_of(st);
  PlanAt *places = places_of(st, a.sequences);
  int *offsets = offsets_of(st, a.sequences);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int run = (a.sequences + THREADS - 1) / THREADS, begin = min(tid * run, a.sequences), end = min(begin + run, a.sequences);
  uint64_t pages = 0, tokens = 0;  // (given back, wanted) of 2^31 at most each
  for (int s = begin; s < end; s++) {
    pages += (uint64_t)(uint32_t)rows[s].back << 32 | (uint32_t)rows[s].want;
    tokens += (uint32_t)(rows[s].fresh & ~kNamed);
  }
  const uint64_t pages_to = wave_scan(pages), tokens_to = wave_scan(tokens);
  if (lane == 63) {
    sh_pages[wave] = pages_to;
    sh_tokens[wave] = tokens_to;
  }
  __syncthreads();
  uint64_t p = pages_to - pages, t = tokens_to - tokens, all = 0, rows_all = 0;
  for (int w = 0; w < THREADS / 64; w++) {
    p += w < wave ? sh_pages[w] : 0;
    t += w < wave ? sh_tokens[w] : 0;
    all += sh_pages[w];
    rows_all += sh_tokens[w];
  }
  for (int s = begin; s < end; s++) {
    const PlanRow r = rows[s];
    places[s] = PlanAt{(int)(p >> 32), (int)(uint32_t)p};
    const int at = (int)(t < 0x7fffffff ? t : 0x7fffffff);
    offsets[s] = at;
    if (a.offsets) a.offsets[s] = at;
    const int fresh = r.fresh & ~kNamed;
    const int64_t length = (int64_t)(r.old & ~kGaps) + fresh;
    a.lengths_out[s] = (int)(length < 0x7fffffff ? length : 0x7fffffff);
    p += (uint64_t)(uint32_t)r.back << 32 | (uint32_t)r.want;
    t += (uint32_t)fresh;
  }
  if (tid == 0) {
    const int at = (int)(rows_all < 0x7fffffff ? rows_all : 0x7fffffff);
    offsets[a.sequences] = at;
    if (a.offsets) a.offsets[a.sequences] = at;
    const int64_t with = free_before(a) + (int64_t)(all >> 32), want = (int64_t)(uint32_t)all;
    const int top = (int)(with < a.page_count ? with : a.page_count);
    st->free_with = top;
    st->free_after = want < top ? top - (int)want : 0;
  }
}

__global__ __launch_bounds__(kThreads) void plan_count_kernel(const PagePlanArgs a, PlanState *__restrict__ st) {
  const int s = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (s < a.sequences) count_sequence(a, st, s);
}

__global__ __launch_bounds__(kScanThreads) void plan_scan_kernel(const PagePlanArgs a, PlanState *__restrict__ st) {
  scan_sequences<kScanThreads>(a, st);
}

// One sequence's pages onto the stack behind `at` others, by a wave.
__device__ __forceinline__ void give_back(const PagePlanArgs &a, int64_t at, int s) {
  const int lane = threadIdx.x & 63;
  const int keep = a.keep_from[s], back = plan_span(0, 0, keep, a.page_shift, a.width).back;
  int *table = a.pages + (int64_t)s * a.width;
  at += free_before(a);
  for (int i0 = lane; i0 - lane < back; i0 += 64 * kAtOnce) {
    int entry[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; j++) entry[j] = table[min(i0 + 64 * j, back - 1)];
#pragma unroll
    for (int j = 0; j < kAtOnce; j++) {
      const bool in = i0 + 64 * j < back;
      const int page = in ? page_or_none(entry[j], a.page_count) : -1;
      const uint64_t named = __ballot(page >= 0);
      const int64_t to = at + __popcll(named & ((1ull << lane) - 1));
      if (page >= 0 && to < a.page_count) a.free[to] = page;
      if (in && entry[j] != -1) table[i0 + 64 * j] = -1;
      at += __popcll(named);
    }
  }
}

// SUM: the sums are not there yet; each workgroup adds up what the sequences
// before its own give back, and one more has the scan for the next launch.
template <bool SUM>
__global__ __launch_bounds__(kThreads) void plan_back_kernel(const PagePlanArgs a, PlanState *__restrict__ st) {
  const int s0 = blockIdx.x * kWaves, s = s0 + (threadIdx.x >> 6);
  if (!SUM) {
    if (s < a.sequences) give_back(a, places_of(st, a.sequences)[s].back, s);
    return;
  }
  if (blockIdx.x == gridDim.x - 1) {
    scan_sequences<kThreads>(a, st);
    return;
  }
  __shared__ uint64_t sh_sum[kWaves];
  const PlanRow *rows = rows_of(st);
  uint64_t before = 0;
  for (int i = threadIdx.x; i < s0; i += kThreads) before += (uint32_t)rows[i].back;
  before = wave_scan(before);
  if ((threadIdx.x & 63) == 63) sh_sum[threadIdx.x >> 6] = before;
  __syncthreads();
  before = 0;
  for (int w = 0; w < kWaves; w++) before += sh_sum[w];
  for (int i = s0; i < s && i < a.sequences; i++) before += (uint32_t)rows[i].back;
  if (s < a.sequences) give_back(a, (int64_t)before, s);
}

// A row's place: position p of sequence s (-1: none) on `page`.
__device__ __forceinline__ void put_row(const PagePlanArgs &a, int t, int s, int64_t p, int page) {
  if (p > 0x7fffffff) s = -1;
  if (a.sequence_of) a.sequence_of[t] = s;
  if (a.positions) a.positions[t] = s >= 0 ? (int)p : -1;
  if (a.slots) a.slots[t] = s >= 0 && page >= 0 ? ((int64_t)page << a.page_shift) + (p & ((1 << a.page_shift) - 1)) : -1;
}
__device__ __forceinline__ int page_at(const PagePlanArgs &a, int s, int64_t p) {
  const int64_t i = p >> a.page_shift;
  return i < a.width ? page_or_none(a.pages[(int64_t)s * a.width + i], a.page_count) : -1;
}

// Pages that a sequence's new tokens lie in and lack, other than the new ones.
__device__ __forceinline__ int missing_of(const PagePlanArgs &a, int s, int old, int64_t fresh) {
  const PlanRest r = plan_rest(old, fresh, a.page_shift, a.width);
  const bool begun = r.begun >= 0 && page_or_none(a.pages[(int64_t)s * a.width + r.begun], a.page_count) < 0;
  return r.beyond + begun;
}

// One sequence's new pages off the stack, by a wave; where some entries have
// theirs already, its rows too.
__device__ __forceinline__ void deal(const PagePlanArgs &a, const PlanState *st, const int *offsets, PlanRow r, int want_at, int s) {
  const int lane = threadIdx.x & 63;
  const bool gaps = (r.old & kGaps) != 0, named = (r.fresh & kNamed) != 0;
  r.old &= ~kGaps;
  r.fresh &= ~kNamed;
  const int rest = lane == 63 && a.missing ? missing_of(a, s, r.old, r.fresh) : 0;
  if (named) {
    if (lane == 63 && a.missing) a.missing[s] = rest;
    return;
  }
  const PlanSpan p = plan_span(r.old, r.fresh, 0, a.page_shift, a.width);
  int *table = a.pages + (int64_t)s * a.width;
  int64_t at = (int64_t)st->free_with - 1 - (uint32_t)want_at;
  int missing = 0;
  for (int i0 = p.first + lane; i0 - lane < p.last; i0 += 64 * kAtOnce) {
    int entry[kAtOnce], page[kAtOnce];
    bool want[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; j++) entry[j] = gaps ? table[min(i0 + 64 * j, p.last - 1)] : -1;
#pragma unroll
    for (int j = 0; j < kAtOnce; j++) {
      want[j] = i0 + 64 * j < p.last && page_or_none(entry[j], a.page_count) < 0;
      const uint64_t wanted = __ballot(want[j]);
      const int64_t from = at - __popcll(wanted & ((1ull << lane) - 1));
      page[j] = want[j] && from >= 0 ? a.free[from] : -1;
      at -= __popcll(wanted);
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; j++) {
      page[j] = page_or_none(page[j], a.page_count);
      if (want[j]) table[i0 + 64 * j] = page[j];
      missing += want[j] && page[j] < 0;
    }
  }
  const uint64_t all = wave_scan((uint64_t)(uint32_t)missing);
  if (lane == 63 && a.missing) a.missing[s] = (int)all + rest;
  if (!gaps || a.rows == 0) return;
  __threadfence_block();  // (the wave's own entries)
  const int row0 = a.fresh ? offsets[s] : s;
  for (int64_t i = lane; i < r.fresh && row0 + i < a.rows; i += 64)
    put_row(a, (int)(row0 + i), s, r.old + i, page_at(a, s, r.old + i));
}

// Row t's sequence, from that of a row before it: mostly the same, or the next.
__device__ __forceinline__ int sequence_from(const PagePlanArgs &a, const int *offsets, int lo, int t) {
  for (int step = 0; lo < a.sequences && offsets[lo + 1] <= t; step++) {
    lo++;
    if (step < 2) continue;
    int n = a.sequences;  // lo .. n: the first whose end is past the row
    while (lo < n) {
      const int mid = (lo + n) >> 1;
      if (offsets[mid + 1] <= t)
        lo = mid + 1;
      else
        n = mid;
    }
    break;
  }
  return lo;
}

constexpr int kRowsEach = 4;

// The first workgroups deal, a wave a sequence; the others have the rows.  Where
// all of a sequence's new pages come off the stack the i-th is known without the
// table, so that its rows need not wait for it.
__global__ __launch_bounds__(kThreads) void plan_deal_kernel(const PagePlanArgs a, const PlanState *__restrict__ st_in,
                                                             int deals) {
  PlanState *st = const_cast<PlanState *>(st_in);
  const int *offsets = offsets_of(st, a.sequences);
  const PlanAt *places = places_of(st, a.sequences);
  if ((int)blockIdx.x < deals) {
    const int s = blockIdx.x * kWaves + (threadIdx.x >> 6);
    if (s < a.sequences) deal(a, st, offsets, rows_of(st)[s], places[s].want, s);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.free_count = st->free_after;
    return;
  }
  // a wave has 64 * kRowsEach rows
  const int t0 = ((blockIdx.x - deals) * kWaves + (threadIdx.x >> 6)) * 64 * kRowsEach, lane = threadIdx.x & 63;
  if (t0 >= a.rows) return;
  int at = a.fresh ? packed_sequence_of(offsets, a.sequences, t0) : 0;
  // the place of row t of sequence s
  auto put = [&](int t, int s, const PlanRow &r, int want_at, int offset) {
    const int fresh = r.fresh & ~kNamed;
    const int64_t p = (int64_t)(r.old & ~kGaps) + (a.fresh ? t - offset : 0), i = p >> a.page_shift;
    const int first = plan_span(r.old & ~kGaps, 0, 0, a.page_shift, a.width).first;
    // (one load, of the table or of the stack)
    const int64_t from = (int64_t)st->free_with - 1 - (uint32_t)want_at - (i - first);
    const bool in_table = (r.fresh & kNamed) != 0 || i < first, there = i < a.width && (in_table || from >= 0);
    const int *entry = in_table ? a.pages + (int64_t)s * a.width + i : a.free + from;
    const int page = there && fresh > 0 ? page_or_none(*entry, a.page_count) : -1;
    if (!(r.old & kGaps) && t < a.rows) put_row(a, t, fresh > 0 ? s : -1, p, page);  // (gaps: the dealing wave's)
  };
  if (a.fresh && at < a.sequences && offsets[at + 1] >= min(t0 + 64 * kRowsEach, a.rows)) {  // mostly: one sequence's
    const PlanRow r = rows_of(st)[at];
    const int want_at = places[at].want, offset = offsets[at];
#pragma unroll
    for (int j = 0; j < kRowsEach; j++) put(t0 + 64 * j + lane, at, r, want_at, offset);
    return;
  }
  for (int j = 0; j < kRowsEach; j++) {
    const int t = t0 + 64 * j + lane;
    if (t >= a.rows) continue;
    int s = t;
    if (a.fresh) {
      at = sequence_from(a, offsets, at, t);
      s = at;
    }
    if (s < a.sequences)
      put(t, s, rows_of(st)[s], places[s].want, offsets[s]);
    else
      put_row(a, t, -1, 0, -1);
  }
}

// ---- small batches: everything in one workgroup ----------------------------------

constexpr int kOneThreads = 1024, kOneWaves = kOneThreads / 64, kOneAtOnce = 4;

// Two sums over the threads before, and over all.
__device__ __forceinline__ void block_scan(uint64_t x, uint64_t y, uint64_t (*sh)[2], uint64_t (&before)[2], uint64_t (&all)[2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t x_to = wave_scan(x), y_to = wave_scan(y);
  if (lane == 63) {
    sh[wave][0] = x_to;
    sh[wave][1] = y_to;
  }
  __syncthreads();
  before[0] = x_to - x;
  before[1] = y_to - y;
  all[0] = all[1] = 0;
#pragma unroll
  for (int w = 0; w < kOneWaves; w++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      before[i] += w < wave ? sh[w][i] : 0;
      all[i] += sh[w][i];
    }
}

// The largest s in 0 .. n - 1 with at[s] <= i (at[0] = 0; n <= 1024).
__device__ __forceinline__ int find(const int *at, int n, int i) {
  int lo = 0;
#pragma unroll
  for (int step = 512; step > 0; step >>= 1)
    if (lo + step < n && at[lo + step] <= i) lo += step;
  return lo;
}

// The entries of all sequences' ranges lie end to end, thread after thread, so
// that one count over them ranks them all: f(j, index) says whether one counts,
// g(j, whether, rank) has what becomes of it.
struct RankShared {
  int counts[kOneAtOnce][kOneWaves];
};
template <class F, class G>
__device__ __forceinline__ int ranked(RankShared &sh, int n, F f, G g) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int total = 0;
  for (int i0 = 0; i0 < n; i0 += kOneThreads * kOneAtOnce) {
    uint64_t mask[kOneAtOnce];
#pragma unroll
    for (int j = 0; j < kOneAtOnce; j++) mask[j] = __ballot(i0 + j * kOneThreads + tid < n && f(j, i0 + j * kOneThreads + tid));
    __syncthreads();
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < kOneAtOnce; j++) sh.counts[j][wave] = __popcll(mask[j]);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kOneAtOnce; j++) {
      int rank = total + __popcll(mask[j] & ((1ull << lane) - 1));
#pragma unroll
      for (int w = 0; w < kOneWaves; w++) {
        rank += w < wave ? sh.counts[j][w] : 0;
        total += sh.counts[j][w];
      }
      if (i0 + j * kOneThreads + tid < n) g(j, (mask[j] >> lane & 1) != 0, rank);
    }
  }
  return total;
}

// All sequences' pages onto the stack of `before`; sh_back: where their ranges
// begin among `back` entries.  The entries of the stack with them.
__device__ __forceinline__ int give_all_back(const PagePlanArgs &a, RankShared &sh, const int *sh_back, int back, int before) {
  if (back == 0) return before;
  int *at[kOneAtOnce];
  int entry[kOneAtOnce];
  const int n = ranked(
      sh, back,
      [&](int j, int i) {
        const int s = find(sh_back, a.sequences, i);
        at[j] = a.pages + (int64_t)s * a.width + (i - sh_back[s]);
        entry[j] = *at[j];
        return page_or_none(entry[j], a.page_count) >= 0;
      },
      [&](int j, bool named, int rank) {
        if (named && rank < a.page_count - before) a.free[before + rank] = entry[j];
        if (entry[j] != -1) *at[j] = -1;
      });
  __syncthreads();  // (the stack and the table are read next)
  return min(n, a.page_count - before) + before;
}

// One token each: a sequence's thread has its position, its page and its row.
__global__ __launch_bounds__(kOneThreads) void plan_step_kernel(const PagePlanArgs a) {
  __shared__ RankShared sh;
  __shared__ int sh_back[kOneThreads], sh_sum[kOneWaves], sh_more[kOneWaves];
  __shared__ int sh_free;  // (read by the thread that writes it in the end)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint64_t below = (1ull << lane) - 1;
  PlanSpan p = {0, 0, 0, 0, 0};
  if (tid < a.sequences) p = span_of(a, tid);
  // the position's entry, read ahead of what goes back
  const int i = p.old >> a.page_shift;
  int *entry = a.pages + (int64_t)tid * a.width + i;
  const bool has = p.fresh > 0 && i < a.width;
  int page = has ? page_or_none(*entry, a.page_count) : -1;
  page = i < p.back ? -1 : page;
  const uint32_t back_to = wave_scan((uint32_t)p.back);
  const uint64_t rows = __ballot(p.fresh > 0);
  if (tid == 0) sh_free = free_before(a);
  if (lane == 63) sh_sum[wave] = (int)back_to;
  if (lane == 0) sh_more[wave] = __popcll(rows);
  __syncthreads();
  int back_at = (int)back_to - p.back, back = 0, row_at = __popcll(rows & below), row_all = 0;
#pragma unroll
  for (int w = 0; w < kOneWaves; w++) {
    back_at += w < wave ? sh_sum[w] : 0;
    back += sh_sum[w];
    row_at += w < wave ? sh_more[w] : 0;
    row_all += sh_more[w];
  }
  sh_back[tid] = back_at;
  __syncthreads();
  const int top = give_all_back(a, sh, sh_back, back, sh_free);

  const bool want = has && p.first < p.last && page < 0;
  const uint64_t wants = __ballot(want);
  if (lane == 0) sh_sum[wave] = __popcll(wants);
  __syncthreads();
  int rank = __popcll(wants & below), wanted = 0;
#pragma unroll
  for (int w = 0; w < kOneWaves; w++) {
    rank += w < wave ? sh_sum[w] : 0;
    wanted += sh_sum[w];
  }
  if (want) {
    page = rank < top ? page_or_none(a.free[top - 1 - rank], a.page_count) : -1;
    *entry = page;
  }
  if (tid < a.sequences) {
    const int64_t length = (int64_t)p.old + p.fresh;
    a.lengths_out[tid] = (int)(length < 0x7fffffff ? length : 0x7fffffff);
    if (a.missing) a.missing[tid] = p.fresh > 0 && page < 0;
    if (a.offsets) a.offsets[tid] = row_at;
  }
  if (tid < a.rows) put_row(a, tid, p.fresh > 0 ? tid : -1, p.old, page);
  if (tid == 0) {
    if (a.offsets) a.offsets[a.sequences] = row_all;
    *a.free_count = wanted < top ? top - wanted : 0;
  }
}

// Any number of tokens each.
__global__ __launch_bounds__(kOneThreads) void plan_one_kernel(const PagePlanArgs a) {
  __shared__ uint64_t sh_scan[kOneWaves][2];
  __shared__ int sh_old[kOneThreads], sh_first[kOneThreads], sh_back[kOneThreads], sh_want[kOneThreads],
      sh_rows[kOneThreads + 1], sh_missing[kOneThreads];
  __shared__ RankShared sh;
  __shared__ int sh_free;
  const int tid = threadIdx.x, S = a.sequences;
  PlanSpan p = {0, 0, 0, 0, 0};
  if (tid < S) p = span_of(a, tid);
  const int fresh = (int)(p.fresh > 0x7fffffff ? 0x7fffffff : p.fresh);
  uint64_t before[2], all[2];
  block_scan((uint64_t)(uint32_t)p.back << 32 | (uint32_t)(p.last - p.first), (uint32_t)fresh, sh_scan, before, all);
  const uint64_t range_at = before[0], row_at = before[1], ranges = all[0], tokens = all[1];
  sh_old[tid] = p.old;
  sh_first[tid] = p.first;
  sh_back[tid] = (int)(range_at >> 32);
  sh_want[tid] = (int)(uint32_t)range_at;
  sh_rows[tid] = (int)(row_at < 0x7fffffff ? row_at : 0x7fffffff);
  if (tid == 0) sh_rows[S] = (int)(tokens < 0x7fffffff ? tokens : 0x7fffffff);
  sh_missing[tid] = 0;
  if (tid == 0) sh_free = free_before(a);
  __syncthreads();

  const int want = (int)(uint32_t)ranges, top = give_all_back(a, sh, sh_back, (int)(ranges >> 32), sh_free);
  int wanted = 0;
  if (want > 0) {
    int *at[kOneAtOnce];
    int seq[kOneAtOnce];
    wanted = ranked(
        sh, want,
        [&](int j, int i) {
          const int s = find(sh_want, S, i);
          seq[j] = s;
          at[j] = a.pages + (int64_t)s * a.width + sh_first[s] + (i - sh_want[s]);
          return page_or_none(*at[j], a.page_count) < 0;
        },
        [&](int j, bool is, int rank) {
          if (!is) return;
          const int page = rank < top ? page_or_none(a.free[top - 1 - rank], a.page_count) : -1;
          *at[j] = page;
          if (page < 0) atomicAdd(&sh_missing[seq[j]], 1);
        });
    __syncthreads();
  }
  if (tid < S) {
    const int64_t length = (int64_t)p.old + fresh;
    a.lengths_out[tid] = (int)(length < 0x7fffffff ? length : 0x7fffffff);
    if (a.missing) a.missing[tid] = sh_missing[tid] + missing_of(a, tid, p.old, fresh);
    if (a.offsets) a.offsets[tid] = sh_rows[tid];
  }
  if (tid == 0) {
    *a.free_count = wanted < top ? top - wanted : 0;
    if (a.offsets) a.offsets[S] = sh_rows[S];
  }
  for (int t = tid; t < a.rows; t += kOneThreads) {
    const int s = t < sh_rows[S] ? find(sh_rows, S, t) : S;
    const bool is = s < S;
    const int64_t p = is ? (int64_t)sh_old[s] + t - sh_rows[s] : 0;
    put_row(a, t, is ? s : -1, p, is ? page_at(a, s, p) : -1);
  }
}

}  // namespace

int page_plan_launches(const PagePlanArgs &a) {
  if (a.sequences <= kOneThreads && (int64_t)a.sequences * a.width <= 1 << 16 && a.rows <= 1 << 13) return 1;
  return a.keep_from && a.sequences > 4096 ? 4 : 3;
}

size_t page_plan_scratch_bytes(const PagePlanArgs &a) {
  return sizeof(PlanState) + (size_t)a.sequences * (sizeof(PlanRow) + sizeof(PlanAt)) + ((size_t)a.sequences + 1) * sizeof(int);
}

hipError_t launch_page_plan(const PagePlanArgs &a, void *scratch, hipStream_t s) {
  if (a.sequences < 1 || a.width < 1 || a.page_count < 1 || (!scratch && page_plan_launches(a) > 1) || (!a.fresh && a.rows > a.sequences))
    return hipErrorInvalidValue;
  // one launch where one workgroup has a few turns of work (a token each of 201
  // sequences, 2700 entries to look through: 6.4 us a call, in several launches 18.6;
  // as one of several tokens 8.9)
  if (page_plan_launches(a) == 1) {
    if (a.fresh)
      hipLaunchKernelGGL(plan_one_kernel, dim3(1), dim3(kOneThreads), 0, s, a);
    else
      hipLaunchKernelGGL(plan_step_kernel, dim3(1), dim3(kOneThreads), 0, s, a);
    return hipGetLastError();
  }
  PlanState *st = static_cast<PlanState *>(scratch);
  const int by_sequence = (a.sequences + kWaves - 1) / kWaves,
            by_row = (int)(((int64_t)a.rows + kThreads * kRowsEach - 1) / (kThreads * kRowsEach));
  hipLaunchKernelGGL(plan_count_kernel, dim3(by_sequence), dim3(kThreads), 0, s, a, st);
  // (to 4096 sequences the sums are a launch's overhead: 4 us of the 18 of 256
  // sequences and 700001 rows)
  if (page_plan_launches(a) == 3 && a.keep_from) {
    hipLaunchKernelGGL(plan_back_kernel<true>, dim3(by_sequence + 1), dim3(kThreads), 0, s, a, st);
  } else {
    hipLaunchKernelGGL(plan_scan_kernel, dim3(1), dim3(kScanThreads), 0, s, a, st);
    if (a.keep_from) hipLaunchKernelGGL(plan_back_kernel<false>, dim3(by_sequence), dim3(kThreads), 0, s, a, st);
  }
  hipLaunchKernelGGL(plan_deal_kernel, dim3(by_sequence + by_row), dim3(kThreads), 0, s, a, st, by_sequence);
  return hipGetLastError();
}

}  // namespace hp
