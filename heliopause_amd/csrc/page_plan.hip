// page_plan.hip -- a step's page tables, lengths, row offsets and slot maps
// from the requests' lengths.
//
// The free pages are a stack.  In order of sequence and position: pages that a
// sequence no longer needs go on top, then the entries that the new tokens need
// and that name no page take theirs from the top.  So a step is two counts of
// each sequence, their sums over the sequences before it, and copies:
//   stack = free[0 .. f) ++ (named entries given back),  T = its size
//   entry of rank r among those wanted: stack[T - 1 - r], -1 from r = T on
// and the outcome does not depend on which workgroup comes first.
#include "hp_serving.h"
#include "hp_wave.h"

namespace hp {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kScanThreads = 1024;

// Scratch: what one launch leaves for the next.
struct PlanState {
  int free_before, free_with;  // entries of the stack, before and with those given back
  int pad[2];
};
struct PlanRow {
  int old, fresh, back_at, want_at;  // (counts until they are summed up)
};
__device__ __forceinline__ PlanRow *rows_of(PlanState *s) { return reinterpret_cast<PlanRow *>(s + 1); }
__device__ __forceinline__ int *offsets_of(PlanState *s, int sequences) {
  return reinterpret_cast<int *>(rows_of(s) + sequences);
}

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
  for (int i = lane; i < p.back; i += 64) back += page_or_none(table[i], a.page_count) >= 0;
  for (int i = p.first + lane; i < p.last; i += 64) want += i < p.back || page_or_none(table[i], a.page_count) < 0;
  const uint64_t both = wave_scan((uint64_t)(uint32_t)back << 32 | (uint32_t)want);
  if (lane == 63)
    rows_of(st)[s] = PlanRow{p.old, (int)(p.fresh > 0x7fffffff ? 0x7fffffff : p.fresh), (int)(both >> 32), (int)(uint32_t)both};
}

__global__ __launch_bounds__(kThreads) void plan_count_kernel(const PagePlanArgs a, PlanState *__restrict__ st) {
  const int s = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (s < a.sequences) count_sequence(a, st, s);
}

// Sums over the sequences before, by one workgroup; a thread has a run of them.
template <int THREADS>
__device__ void scan_sequences(const PagePlanArgs &a, PlanState *st) {
  __shared__ uint64_t sh_pages[THREADS / 64], sh_tokens[THREADS / 64];
  PlanRow *rows = rows_of(st);
  int *offsets = offsets_of(st, a.sequences);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int run = (a.sequences + THREADS - 1) / THREADS, begin = min(tid * run, a.sequences), end = min(begin + run, a.sequences);
  uint64_t pages = 0, tokens = 0;  // (given back, wanted) of 2^31 at most each
  for (int s = begin; s < end; s++) {
    pages += (uint64_t)(uint32_t)rows[s].back_at << 32 | (uint32_t)rows[s].want_at;
    tokens += (uint32_t)rows[s].fresh;
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
    rows[s].back_at = (int)(p >> 32);
    rows[s].want_at = (int)(uint32_t)p;
    const int at = (int)(t < 0x7fffffff ? t : 0x7fffffff);
    offsets[s] = at;
    if (a.offsets) a.offsets[s] = at;
    const int64_t length = (int64_t)r.old + r.fresh;
    a.lengths_out[s] = (int)(length < 0x7fffffff ? length : 0x7fffffff);
    p += (uint64_t)(uint32_t)r.back_at << 32 | (uint32_t)r.want_at;
    t += (uint32_t)r.fresh;
  }
  if (tid == 0) {
    const int at = (int)(rows_all < 0x7fffffff ? rows_all : 0x7fffffff);
    offsets[a.sequences] = at;
    if (a.offsets) a.offsets[a.sequences] = at;
    const int before = min(max(*a.free_count, 0), a.page_count);
    const int64_t with = (int64_t)before + (int64_t)(all >> 32), want = (int64_t)(uint32_t)all;
    const int top = (int)(with < a.page_count ? with : a.page_count);
    st->free_before = before;
    st->free_with = top;
    *a.free_count = want < top ? top - (int)want : 0;
  }
}

__global__ __launch_bounds__(kScanThreads) void plan_scan_kernel(const PagePlanArgs a, PlanState *__restrict__ st) {
  scan_sequences<kScanThreads>(a, st);
}

// One sequence's pages onto the stack, by a wave.
__device__ __forceinline__ void give_back(const PagePlanArgs &a, const PlanState *st, const PlanRow &r, int s) {
  const int lane = threadIdx.x & 63;
  const int keep = a.keep_from[s], back = plan_span(0, 0, keep, a.page_shift, a.width).back;
  int *table = a.pages + (int64_t)s * a.width;
  int64_t at = (int64_t)st->free_before + r.back_at;
  for (int i0 = 0; i0 < back; i0 += 64) {
    const int i = i0 + lane;
    const int entry = i < back ? table[i] : -1, page = page_or_none(entry, a.page_count);
    const uint64_t named = __ballot(page >= 0);
    const int64_t to = at + __popcll(named & ((1ull << lane) - 1));
    if (page >= 0 && to < a.page_count) a.free[to] = page;
    if (i < back && entry != -1) table[i] = -1;
    at += __popcll(named);
  }
}

__global__ __launch_bounds__(kThreads) void plan_back_kernel(const PagePlanArgs a, PlanState *__restrict__ st) {
  const int s = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (s < a.sequences) give_back(a, st, rows_of(st)[s], s);
}

// One sequence's new pages off the stack, by a wave.
__device__ __forceinline__ void deal(const PagePlanArgs &a, const PlanState *st, const PlanRow &r, int s) {
  const int lane = threadIdx.x & 63;
  const PlanSpan p = plan_span(r.old, r.fresh, 0, a.page_shift, a.width);
  int *table = a.pages + (int64_t)s * a.width;
  int64_t at = (int64_t)st->free_with - 1 - (uint32_t)r.want_at;
  int missing = 0;
  for (int i0 = p.first; i0 < p.last; i0 += 64) {
    const int i = i0 + lane;
    const bool want = i < p.last && page_or_none(table[min(i, p.last - 1)], a.page_count) < 0;
    const uint64_t wanted = __ballot(want);
    const int64_t from = at - __popcll(wanted & ((1ull << lane) - 1));
    if (want) {
      const int page = from >= 0 ? page_or_none(a.free[from], a.page_count) : -1;
      table[i] = page;
      missing += page < 0;
    }
    at -= __popcll(wanted);
  }
  const uint64_t all = wave_scan((uint64_t)(uint32_t)missing);
  if (lane == 63 && a.missing) a.missing[s] = (int)all;
}

__global__ __launch_bounds__(kThreads) void plan_deal_kernel(const PagePlanArgs a, PlanState *__restrict__ st) {
  const int s = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (s < a.sequences) deal(a, st, rows_of(st)[s], s);
}

// A row's place.
__device__ __forceinline__ void map_row(const PagePlanArgs &a, const PlanRow *rows, const int *offsets, int t, int s) {
  int seq = -1, position = -1;
  int64_t slot = -1;
  if (s < a.sequences) {
    const PlanRow r = rows[s];
    const int64_t p = (int64_t)r.old + (a.fresh ? t - offsets[s] : 0);
    if (r.fresh > 0 && p <= 0x7fffffff) {
      seq = s;
      position = (int)p;
      const int64_t i = p >> a.page_shift;
      if (i < a.width) {
        const int page = page_or_none(a.pages[(int64_t)s * a.width + i], a.page_count);
        if (page >= 0) slot = ((int64_t)page << a.page_shift) + (p & ((1 << a.page_shift) - 1));
      }
    }
  }
  if (a.sequence_of) a.sequence_of[t] = seq;
  if (a.positions) a.positions[t] = position;
  if (a.slots) a.slots[t] = slot;
}

// The row's sequence: 64 rows of a wave mostly have one.
__device__ __forceinline__ int sequence_of(const PagePlanArgs &a, const int *offsets, int t0, int t) {
  if (!a.fresh) return t;
  int lo = packed_sequence_of(offsets, a.sequences, t0);
  if (__any(lo < a.sequences && offsets[min(lo, a.sequences - 1) + 1] <= t)) {
    int n = a.sequences;  // lo .. n: the first whose end is past the row
    while (lo < n) {
      const int mid = (lo + n) >> 1;
      if (offsets[mid + 1] <= t)
        lo = mid + 1;
      else
        n = mid;
    }
  }
  return lo;
}

__global__ __launch_bounds__(kThreads) void plan_rows_kernel(const PagePlanArgs a, PlanState *__restrict__ st) {
  const int t = blockIdx.x * kThreads + threadIdx.x, t0 = t & ~63;
  if (t0 >= a.rows) return;
  const int *offsets = offsets_of(st, a.sequences);
  const int s = sequence_of(a, offsets, t0, t);
  if (t < a.rows) map_row(a, rows_of(st), offsets, t, s);
}

}  // namespace

size_t page_plan_scratch_bytes(const PagePlanArgs &a) {
  return sizeof(PlanState) + (size_t)a.sequences * sizeof(PlanRow) + ((size_t)a.sequences + 1) * sizeof(int);
}

hipError_t launch_page_plan(const PagePlanArgs &a, void *scratch, hipStream_t s) {
  if (a.sequences < 1 || a.width < 1 || a.page_count < 1 || !scratch || (!a.fresh && a.rows > a.sequences))
    return hipErrorInvalidValue;
  PlanState *st = static_cast<PlanState *>(scratch);
  const dim3 by_sequence((a.sequences + kWaves - 1) / kWaves);
  hipLaunchKernelGGL(plan_count_kernel, by_sequence, dim3(kThreads), 0, s, a, st);
  hipLaunchKernelGGL(plan_scan_kernel, dim3(1), dim3(kScanThreads), 0, s, a, st);
  if (a.keep_from) hipLaunchKernelGGL(plan_back_kernel, by_sequence, dim3(kThreads), 0, s, a, st);
  hipLaunchKernelGGL(plan_deal_kernel, by_sequence, dim3(kThreads), 0, s, a, st);
  if (a.rows > 0)
    hipLaunchKernelGGL(plan_rows_kernel, dim3((a.rows + kThreads - 1) / kThreads), dim3(kThreads), 0, s, a, st);
  return hipGetLastError();
}

}  // namespace hp
