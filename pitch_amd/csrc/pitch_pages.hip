// The pages of a paged cache: handing out, giving back, sharing and compacting them, with tables, lengths and counts of references in
// device memory, so that a captured graph serves every step.
//
// Free pages are ranked, not listed: a pool's references are counted in segments by one launch, and the next gives page number k
// among the free ones to the k-th place that needs a page. Every order is that of the numbers, never that of arrival: the same state
// gives the same pages. Counts of references change by atomic additions, whose order does not matter.
//
// What bounds it. Bookkeeping is a chain of dependent reads of a few KB: a launch takes 3 to 8 us on the device, and a call of one or
// two of them the 8 to 10 us of the host. 64 sequences of about 3,000 tokens that reserve up to 2,000 each in pages of 16, of 40,000,
// and give some back: 13.7 us (plan 3.4, places 7.8, trim 3.0). 64 beams of 1,000 tokens, 32 layers: 26 us, 14 of them the copies of
// their last pages. A pool of 2,000 pages of 32 layers, 1.1 GB of which move: 410 to 475 us on different cards, the copies at the rate
// of a large copy (4.7 to 5.5 TB/s), and 10 us for the bookkeeping.
#include "pitch_pages.h"

namespace pitch {
namespace {

constexpr uint32_t kThreads = 256, kOneThreads = 1024, kMostWaves = kOneThreads / 64;
constexpr uint32_t kMostSequences = 2048;
// The largest calls whose bookkeeping one workgroup does, in one launch: it costs the host about 2 us less for each launch saved, but
// a workgroup's wave turns to one row, or to 64 pages, after the other. Kernels' times, one workgroup against several launches: reserve of
// 4,096 pages 5.0 us against 5.9 and a launch more; a fork of 64 rows 17.0 against 10.3 (so the limit on rows), of 8 rows a call of 9.8
// against 15.8; a compaction of 2,000 pages 9.5 against 13.8.
constexpr uint32_t kReserveOnePages = 4096, kReserveOneRows = 256, kReserveOneTokens = 4096;
constexpr uint32_t kForkOnePages = 4096, kForkOneRows = 16;
constexpr uint32_t kCompactOnePages = 4096, kCompactOneRows = 64;

__device__ __forceinline__ uint32_t lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}
__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, uint32_t page) { return tokens / page + (tokens % page != 0); }
// A sequence's length as it is taken: within its row of the table.
__device__ __forceinline__ uint32_t length_of(const PagesTables& t, int32_t x) { return min((uint32_t)max(x, 0), t.most_tokens); }
__device__ __forceinline__ bool in_pool(const PagesTables& t, int32_t page) { return (uint32_t)page < t.pages; }

// The workgroup's threads: 256, or 1,024 where one does all of a call's work.
__device__ __forceinline__ uint32_t group_waves() { return blockDim.x >> 6; }

// Sums over the workgroup, in every thread.
__device__ __forceinline__ uint32_t group_sum(uint32_t x, uint32_t* lds) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  uint32_t sum = 0;
  for (uint32_t w = 0; w < group_waves(); ++w) sum += lds[w];
  return sum;
}
// The sum over the lanes before this one; *total gets the wave's.
template <typename T>
__device__ __forceinline__ T wave_before(T x, T* total) {
  const uint32_t lane = threadIdx.x & 63;
  T sum = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T up = __shfl_up(sum, d);
    if (lane >= (uint32_t)d) sum += up;
  }
  *total = __shfl(sum, 63);
  return sum - x;
}
// The same over the workgroup's threads.
template <typename T>
__device__ __forceinline__ T group_before(T x, T* lds, T* total) {
  const uint32_t wave = threadIdx.x >> 6;
  T own;
  T before = wave_before(x, &own), all = 0;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[wave] = own;
  __syncthreads();
  for (uint32_t w = 0; w < group_waves(); ++w) {
    const T n = lds[w];
    before += w < wave ? n : 0;
    all += n;
  }
  *total = all;
  return before;
}

// A page's count of references. With PAST_CACHE it is read past the compute unit's cache, which may hold what the line was before
// this workgroup's own atomics changed it in L2.
template <bool PAST_CACHE>
__device__ __forceinline__ int32_t references_of(const PagesTables& t, uint32_t page) {
  if constexpr (PAST_CACHE) return __hip_atomic_load(t.references + page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return t.references[page];
}

// Counts a segment's pages with (USED) or without references.
template <bool USED, bool PAST_CACHE = false>
__device__ __forceinline__ void count_segment(const PagesTables& t, uint32_t segment, uint32_t* lds) {
  const uint32_t from = segment * t.segment, to = min(from + t.segment, t.pages);
  uint32_t n = 0;
#pragma unroll 4
  for (uint32_t p = from + threadIdx.x; p < to; p += blockDim.x) n += (references_of<PAST_CACHE>(t, p) > 0) == USED;
  n = group_sum(n, lds);
  if (threadIdx.x == 0) t.counts[segment] = n;
}
// The counted pages before a segment, and of the pool.
__device__ __forceinline__ uint32_t counted_before(const PagesTables& t, uint32_t segment, uint32_t* lds, uint32_t* total) {
  if (t.segments == 1) {
    *total = t.counts[0];
    return 0;
  }
  uint32_t before = 0, all = 0;
  for (uint32_t i = threadIdx.x; i < t.segments; i += blockDim.x) {
    const uint32_t n = t.counts[i];
    all += n;
    before += i < segment ? n : 0;
  }
  *total = group_sum(all, lds);
  return group_sum(before, lds);
}
// Calls f(page, counted, rank) for every page of a segment, all lanes of a wave together (page t.pages for lanes behind the segment):
// counted says whether it is one of the counted pages, rank is their number before it in the pool. Stops behind the page of rank `last`.
template <bool USED, bool PAST_CACHE = false, typename F>
__device__ __forceinline__ void for_segment(const PagesTables& t, uint32_t segment, uint32_t before, uint32_t last, uint32_t* lds, F f) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, each = t.segment / group_waves();
  const uint32_t from = segment * t.segment + wave * each, end = min((segment + 1) * t.segment, t.pages), to = min(from + each, end);
  uint32_t n = 0;
  for (uint32_t p = from + lane; p < to; p += 64) n += (references_of<PAST_CACHE>(t, p) > 0) == USED;
#pragma unroll
  for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
  __syncthreads();
  if (lane == 0) lds[wave] = n;
  __syncthreads();
  uint32_t rank = before;
  for (uint32_t w = 0; w < wave; ++w) rank += lds[w];
  for (uint32_t p = from; p < to && rank < last; p += 64) {
    const bool inside = p + lane < to, counted = inside && (references_of<PAST_CACHE>(t, p + lane) > 0) == USED;
    const uint64_t mask = __ballot(counted);
    f(inside ? p + lane : t.pages, counted, rank + lanes_below(mask));
    rank += __popcll(mask);
  }
}

// ------------------------------------------------------------------------------------------------ reserve
// plan: [0] tokens of the call, [1] pages needed; arrays: the rows' first tokens, their tokens, the pages needed before them, their
// lengths before the call.
struct ReservePlan {
  uint32_t *words, *start, *tokens, *first, *length;
  __device__ explicit ReservePlan(const PagesTables& t) : ReservePlan(t.plan, t.sequences) {}
  __device__ ReservePlan(uint32_t* at, uint32_t rows)
      : words(at), start(at + 8), tokens(start + rows), first(tokens + rows), length(first + rows) {}
};

// The plan, by a workgroup or by one wave (whose sums take no barrier).
template <bool WAVE>
__device__ __forceinline__ void reserve_plan(const PagesReserveArgs& a, const ReservePlan& plan, uint32_t* lds, uint64_t* wide) {
  const PagesTables& t = a.t;
  const uint32_t width = WAVE ? 64 : blockDim.x, me = WAVE ? threadIdx.x & 63 : threadIdx.x;
  uint64_t tokens = 0;
  uint32_t pages = 0;
  for (uint32_t base = 0; base < t.sequences; base += width) {
    const uint32_t b = base + me;
    const bool row = b < t.sequences;
    const uint32_t asked = row ? (uint32_t)max(a.new_tokens[b], 0) : 0, length = row ? length_of(t, t.lengths[b]) : 0;
    uint64_t all;
    const uint64_t at = tokens + (WAVE ? wave_before<uint64_t>(asked, &all) : group_before<uint64_t>(asked, wide, &all));
    tokens += all;
    const uint32_t start = (uint32_t)min(at, (uint64_t)a.capacity), n = min(asked, a.capacity - start);
    const uint32_t need = pages_of(length + min(n, t.most_tokens - length), t.page_size) - pages_of(length, t.page_size);
    uint32_t sum;
    const uint32_t first = pages + (WAVE ? wave_before<uint32_t>(need, &sum) : group_before<uint32_t>(need, lds, &sum));
    pages += sum;
    if (row) {
      plan.start[b] = start;
      plan.tokens[b] = n;
      plan.first[b] = first;
      plan.length[b] = length;
    }
  }
  if (me == 0) {
    plan.words[0] = (uint32_t)min(tokens, (uint64_t)a.capacity);
    plan.words[1] = pages;
  }
}
// A row's tokens end where the free pages do.
__device__ __forceinline__ uint32_t reserve_end(const PagesTables& t, const ReservePlan& plan, uint32_t b, uint32_t free) {
  const uint32_t page = t.page_size, length = plan.length[b], fits = min(plan.tokens[b], t.most_tokens - length);
  const uint32_t held = pages_of(length, page), need = pages_of(length + fits, page) - held, at = plan.first[b];
  const uint32_t got = min(need, free - min(free, at));
  return got == need ? length + fits : min(length + fits, (held + got) * page);
}

// A page that is handed out: its first token's place in the call, its tokens, its number, its first token's position.
struct Handed {
  uint32_t from, tokens, page, position;
};

// Gives a wave's free ones of 64 pages to the rows that need them, and writes their tokens. `first` is the plan's, in LDS.
__device__ __forceinline__ void reserve_pages(const PagesReserveArgs& a, const ReservePlan& plan, const uint32_t* first, Handed* handed,
                                              uint32_t p, bool is_free, uint32_t rank, uint32_t needed, uint32_t free) {
  const PagesTables& t = a.t;
  const uint32_t lane = threadIdx.x & 63, page = t.page_size;
  const bool given = is_free && rank < needed;
  const uint64_t mask = __ballot(given);
  if (given) {
    uint32_t lo = 0, hi = t.sequences;   // the last row whose pages begin at this rank or before it
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      (first[mid] <= rank ? lo : hi) = mid;
    }
    const uint32_t length = plan.length[lo], end = reserve_end(t, plan, lo, free);
    const uint32_t at = pages_of(length, page) + rank - first[lo], pos = at * page, tokens = min(page, end - min(end, pos));
    t.tables[(uint64_t)lo * t.width + at] = (int32_t)p;
    t.references[p] = 1;
    // (a new page begins at the length or behind it)
    handed[lanes_below(mask)] = Handed{plan.start[lo] + pos - length, tokens, p, pos};
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  // the pages' tokens, 64 at a time whatever the page's size
  const uint32_t all = __popcll(mask) * page;   // (at most 64 pages of 65,536)
  for (uint32_t i = lane; i < all; i += 64) {
    const uint32_t k = i / page, at = i - k * page;
    const Handed h = handed[k];
    if (at >= h.tokens) continue;
    a.slots[h.from + at] = (int64_t)((uint64_t)h.page * page + at);
    if (a.positions) a.positions[h.from + at] = h.position + at;
  }
  __builtin_amdgcn_wave_barrier();
}

// The rows' tokens in pages that they held before, those without a page, the entries behind the last token, the lengths.
__device__ __forceinline__ void reserve_rows(const PagesReserveArgs& a, const ReservePlan& plan, uint32_t free, uint32_t wave,
                                             uint32_t waves) {
  const PagesTables& t = a.t;
  const uint32_t lane = threadIdx.x & 63, page = t.page_size, needed = plan.words[1];
  for (uint32_t b = wave; b < t.sequences; b += waves) {
    const uint32_t length = plan.length[b], start = plan.start[b], n = plan.tokens[b], end = reserve_end(t, plan, b, free);
    const uint32_t full = min(end, pages_of(length, page) * page);
    for (uint32_t i = lane; i < full - length; i += 64) {
      const uint32_t pos = length + i;
      const int32_t entry = t.tables[(uint64_t)b * t.width + pos / page];
      a.slots[start + i] = in_pool(t, entry) ? (int64_t)((uint64_t)entry * page + pos % page) : -1;
      if (a.positions) a.positions[start + i] = pos;
    }
    for (uint32_t i = end - length + lane; i < n; i += 64) {
      a.slots[start + i] = -1;
      if (a.positions) a.positions[start + i] = -1;
    }
    if (lane == 0) t.lengths[b] = (int32_t)end;
  }
  for (uint32_t i = plan.words[0] + wave * 64 + lane; i < a.capacity; i += waves * 64) {
    a.slots[i] = -1;
    if (a.positions) a.positions[i] = -1;
  }
  if (wave == 0 && lane == 0 && t.missing) *t.missing = (int32_t)(needed - min(needed, free));
}

__global__ __launch_bounds__(kThreads) void pages_reserve_plan(PagesReserveArgs a) {
  __shared__ uint32_t lds[kMostWaves];
  __shared__ uint64_t wide[kMostWaves];
  if (blockIdx.x < a.t.segments)
    count_segment<false>(a.t, blockIdx.x, lds);
  else
    reserve_plan<false>(a, ReservePlan(a.t), lds, wide);
}

__global__ __launch_bounds__(kThreads) void pages_reserve_place(PagesReserveArgs a) {
  __shared__ uint32_t lds[kMostWaves];
  __shared__ uint32_t first[kMostSequences];
  __shared__ Handed handed[kThreads / 64][64];
  const PagesTables& t = a.t;
  const ReservePlan plan(t);
  const bool rows = blockIdx.x >= t.segments;
  uint32_t free;
  const uint32_t before = counted_before(t, rows ? 0 : blockIdx.x, lds, &free), needed = plan.words[1];
  if (rows) {
    reserve_rows(a, plan, free, (blockIdx.x - t.segments) * 4 + (threadIdx.x >> 6), (gridDim.x - t.segments) * 4);
  } else if (before < needed) {
    for (uint32_t b = threadIdx.x; b < t.sequences; b += blockDim.x) first[b] = plan.first[b];
    __syncthreads();
    for_segment<false>(t, blockIdx.x, before, needed, lds, [&](uint32_t p, bool is_free, uint32_t rank) {
      reserve_pages(a, plan, first, handed[threadIdx.x >> 6], p, is_free, rank, needed, free);
    });
  }
}

// All of it by one workgroup: a wave holds which of its 256 pages are free while the first wave makes the plan, in LDS.
__global__ __launch_bounds__(kOneThreads) void pages_reserve_one(PagesReserveArgs a) {
  constexpr uint32_t kTurns = kReserveOnePages / kOneThreads;
  __shared__ uint32_t counts[kMostWaves], room[8 + 4 * kReserveOneRows];
  __shared__ Handed handed[kMostWaves][64];
  const PagesTables& t = a.t;
  const ReservePlan plan(room, t.sequences);
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, from = wave * (64 * kTurns) + lane;
  bool is_free[kTurns];
  uint32_t found = 0;
#pragma unroll
  for (uint32_t i = 0; i < kTurns; ++i) is_free[i] = from + i * 64 < t.pages && t.references[from + i * 64] <= 0;
#pragma unroll
  for (uint32_t i = 0; i < kTurns; ++i) found += __popcll(__ballot(is_free[i]));
  if (lane == 0) counts[wave] = found;
  if (wave == 0) reserve_plan<true>(a, plan, nullptr, nullptr);
  __syncthreads();
  uint32_t free = 0, rank = 0;
  for (uint32_t w = 0; w < kMostWaves; ++w) {
    free += counts[w];
    rank += w < wave ? counts[w] : 0;
  }
  reserve_rows(a, plan, free, wave, kMostWaves);
  const uint32_t needed = plan.words[1];
#pragma unroll
  for (uint32_t i = 0; i < kTurns; ++i) {
    const uint64_t mask = __ballot(is_free[i]);
    if (rank < needed)
      reserve_pages(a, plan, plan.first, handed[wave], from + i * 64, is_free[i], rank + lanes_below(mask), needed, free);
    rank += __popcll(mask);
  }
}

// ------------------------------------------------------------------------------------------------ trim
__global__ __launch_bounds__(kThreads) void pages_trim(PagesTrimArgs a) {
  const PagesTables& t = a.t;
  const uint32_t lane = threadIdx.x & 63, b = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= t.sequences) return;
  const uint32_t length = length_of(t, t.lengths[b]), end = min(length, (uint32_t)max(a.keep[b], 0));
  for (uint32_t i = pages_of(end, t.page_size) + lane; i < pages_of(length, t.page_size); i += 64) {
    const int32_t page = t.tables[(uint64_t)b * t.width + i];
    if (in_pool(t, page)) atomicSub(t.references + page, 1);
  }
  if (lane == 0) t.lengths[b] = (int32_t)end;
}

// ------------------------------------------------------------------------------------------------ fork
// plan: [0] rows that need a copy, [1] pages copied; arrays: lengths before the call, each row's number among those that need a copy
// (kNone: none), and the copies' sources, targets and tokens. room: the tables as they were, of the rows' lengths.
constexpr uint32_t kNone = 0xFFFFFFFFu;
struct ForkPlan {
  uint32_t *words, *length, *rank, *source, *target, *tokens, *old;
  __device__ explicit ForkPlan(const PagesTables& t)
      : words(t.plan), length(t.plan + 8), rank(length + t.sequences), source(rank + t.sequences), target(source + t.sequences),
        tokens(target + t.sequences), old(t.room) {}
};

// Counts of references as they will be, by one wave for each row.
__device__ __forceinline__ void fork_row(const PagesForkArgs& a, uint32_t b) {
  const PagesTables& t = a.t;
  const ForkPlan plan(t);
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t length = length_of(t, t.lengths[b]), parent = (uint32_t)a.parents[b];
  const int32_t* const row = t.tables + (uint64_t)b * t.width;
  const bool changed = parent != b;
  for (uint32_t i = lane; i < pages_of(length, t.page_size); i += 64) {
    const int32_t page = row[i];
    plan.old[(uint64_t)b * t.width + i] = (uint32_t)page;
    if (changed && in_pool(t, page)) atomicSub(t.references + page, 1);
  }
  bool copy = false;
  if (changed && parent < t.sequences) {
    const uint32_t tokens = length_of(t, t.lengths[parent]), whole = tokens / t.page_size;
    const int32_t* const from = t.tables + (uint64_t)parent * t.width;
    // the parent's own row keeps its last page, or the first of its children does
    bool keeps = (uint32_t)a.parents[parent] != parent;
    for (uint32_t i = 0; i < b && keeps; i += 64)
      keeps = !__ballot(i + lane < b && (uint32_t)a.parents[min(i + lane, b)] == parent);
    const bool part = tokens % t.page_size != 0;
    for (uint32_t i = lane; i < whole + (part && keeps); i += 64)
      if (in_pool(t, from[i])) atomicAdd(t.references + from[i], 1);
    copy = part && !keeps && in_pool(t, from[whole]);
  }
  if (lane == 0) {
    plan.length[b] = length;
    plan.rank[b] = copy ? 0 : kNone;
  }
}

// Numbers the rows that need a copy.
__device__ __forceinline__ void fork_plan(const PagesForkArgs& a, uint32_t* lds) {
  const PagesTables& t = a.t;
  const ForkPlan plan(t);
  uint32_t copies = 0;
  for (uint32_t base = 0; base < t.sequences; base += blockDim.x) {
    const uint32_t b = base + threadIdx.x;
    const bool copy = b < t.sequences && plan.rank[b] != kNone;
    uint32_t all;
    const uint32_t rank = copies + group_before<uint32_t>(copy, lds, &all);
    copies += all;
    if (!copy) continue;
    const uint32_t parent = (uint32_t)a.parents[b], tokens = plan.length[parent], whole = tokens / t.page_size;
    plan.rank[b] = rank;
    plan.source[rank] = plan.old[(uint64_t)parent * t.width + whole];
    plan.target[rank] = b;       // the row, until the page is known
    plan.tokens[rank] = tokens % t.page_size;
  }
  if (threadIdx.x == 0) plan.words[0] = copies;
}

// Gives a segment's free pages to the rows that need a copy.
template <bool PAST_CACHE>
__device__ __forceinline__ void fork_segment(const PagesForkArgs& a, uint32_t segment, uint32_t before, uint32_t* lds) {
  const PagesTables& t = a.t;
  const ForkPlan plan(t);
  const uint32_t copies = plan.words[0];
  if (before >= copies) return;
  for_segment<false, PAST_CACHE>(t, segment, before, copies, lds, [&](uint32_t p, bool is_free, uint32_t rank) {
    if (!is_free || rank >= copies) return;
    const uint32_t b = plan.target[rank], whole = plan.length[(uint32_t)a.parents[b]] / t.page_size;
    t.tables[(uint64_t)b * t.width + whole] = (int32_t)p;
    t.references[p] = 1;
    plan.target[rank] = p;
  });
}

// A changed row's entries and length, by one wave.
__device__ __forceinline__ void fork_entries(const PagesForkArgs& a, uint32_t b, uint32_t free) {
  const PagesTables& t = a.t;
  const ForkPlan plan(t);
  const uint32_t lane = threadIdx.x & 63, copies = plan.words[0];
  if (b == 0 && lane == 0) {
    plan.words[1] = min(copies, free);
    if (t.missing) *t.missing = (int32_t)(copies - min(copies, free));
  }
  const uint32_t parent = (uint32_t)a.parents[b], rank = plan.rank[b];
  if (parent == b) return;
  uint32_t end = 0;
  if (parent < t.sequences) {
    end = plan.length[parent];
    const uint32_t whole = end / t.page_size, n = rank == kNone ? pages_of(end, t.page_size) : whole;
    for (uint32_t i = lane; i < n; i += 64) t.tables[(uint64_t)b * t.width + i] = (int32_t)plan.old[(uint64_t)parent * t.width + i];
    if (rank != kNone && rank >= free) end = whole * t.page_size;   // no page is left for the last tokens
  }
  if (lane == 0) t.lengths[b] = (int32_t)end;
}

__global__ __launch_bounds__(kThreads) void pages_fork_rows(PagesForkArgs a) {
  const uint32_t b = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b < a.t.sequences) fork_row(a, b);
}

__global__ __launch_bounds__(kThreads) void pages_fork_plan(PagesForkArgs a) {
  __shared__ uint32_t lds[kMostWaves];
  if (blockIdx.x < a.t.segments)
    count_segment<false>(a.t, blockIdx.x, lds);
  else
    fork_plan(a, lds);
}

__global__ __launch_bounds__(kThreads) void pages_fork_place(PagesForkArgs a) {
  __shared__ uint32_t lds[kMostWaves];
  const bool rows = blockIdx.x >= a.t.segments;
  uint32_t free;
  const uint32_t before = counted_before(a.t, rows ? 0 : blockIdx.x, lds, &free);
  if (!rows) {
    fork_segment<false>(a, blockIdx.x, before, lds);
    return;
  }
  const uint32_t b = (blockIdx.x - a.t.segments) * 4 + (threadIdx.x >> 6);
  if (b < a.t.sequences) fork_entries(a, b, free);
}

// All of it by one workgroup (the pool is one segment).
__global__ __launch_bounds__(kOneThreads) void pages_fork_one(PagesForkArgs a) {
  __shared__ uint32_t lds[kMostWaves];
  for (uint32_t b = threadIdx.x >> 6; b < a.t.sequences; b += kMostWaves) fork_row(a, b);
  __syncthreads();
  count_segment<false, true>(a.t, 0, lds);
  fork_plan(a, lds);
  __syncthreads();
  const uint32_t free = a.t.counts[0];
  for (uint32_t b = threadIdx.x >> 6; b < a.t.sequences; b += kMostWaves) fork_entries(a, b, free);
  fork_segment<true>(a, 0, 0, lds);
}

// ------------------------------------------------------------------------------------------------ compact
// U pages are in use. Those at U and above (movers) go to the free ones below U (holes), as many, the k-th to the k-th. plan: [0] U,
// [1] movers; room: the holes, the movers counted from the last, and for each page at U or above its number among these (kNone: free).
struct CompactPlan {
  uint32_t *words, *holes, *movers, *number;
  __device__ explicit CompactPlan(const PagesTables& t)
      : words(t.plan), holes(t.room), movers(t.room + t.pages), number(t.room + 2ull * t.pages) {}
};

__device__ __forceinline__ void compact_segment(const PagesCompactArgs& a, uint32_t segment, uint32_t* lds) {
  const PagesTables& t = a.t;
  const CompactPlan plan(t);
  uint32_t used;
  const uint32_t before = counted_before(t, segment, lds, &used);
  for_segment<true>(t, segment, before, kNone, lds, [&](uint32_t p, bool in_use, uint32_t rank) {
    if (p >= t.pages) return;
    if (p == used) plan.words[1] = used - rank;   // as many lie at U and above as are missing below
    if (p < used) {
      if (!in_use) plan.holes[p - rank] = p;
    } else {
      plan.number[p] = in_use ? used - 1 - rank : kNone;
      if (in_use) plan.movers[used - 1 - rank] = p;
    }
    if (a.mapping && !(in_use && p >= used)) a.mapping[p] = in_use ? (int32_t)p : -1;
  });
  if (segment == 0 && threadIdx.x == 0) {
    plan.words[0] = used;
    if (used == t.pages) plan.words[1] = 0;
    if (a.used) *a.used = (int32_t)used;
  }
}

// The tables' entries, and the references and mapping of the pages that move.
__device__ __forceinline__ void compact_tables(const PagesCompactArgs& a, uint32_t at, uint32_t all) {
  const PagesTables& t = a.t;
  const CompactPlan plan(t);
  const uint32_t used = plan.words[0], moves = plan.words[1];
  for (uint32_t i = at; i < moves; i += all) {
    const uint32_t from = plan.movers[moves - 1 - i], to = plan.holes[i];
    t.references[to] = t.references[from];
    t.references[from] = 0;
    if (a.mapping) a.mapping[from] = (int32_t)to;
  }
  for (uint32_t b = at / 64; b < t.sequences; b += all / 64) {
    const uint32_t n = pages_of(length_of(t, t.lengths[b]), t.page_size);
    for (uint32_t i = at % 64; i < n; i += 64) {
      int32_t* const entry = t.tables + (uint64_t)b * t.width + i;
      const int32_t page = *entry;
      if (!in_pool(t, page) || (uint32_t)page < used) continue;
      const uint32_t number = plan.number[page];
      if (number != kNone) *entry = (int32_t)plan.holes[moves - 1 - number];
    }
  }
}

__global__ __launch_bounds__(kThreads) void pages_compact_count(PagesCompactArgs a) {
  __shared__ uint32_t lds[kMostWaves];
  count_segment<true>(a.t, blockIdx.x, lds);
}
__global__ __launch_bounds__(kThreads) void pages_compact_list(PagesCompactArgs a) {
  __shared__ uint32_t lds[kMostWaves];
  compact_segment(a, blockIdx.x, lds);
}
__global__ __launch_bounds__(kThreads) void pages_compact_tables(PagesCompactArgs a) {
  compact_tables(a, blockIdx.x * kThreads + threadIdx.x, gridDim.x * kThreads);
}

// All of it by one workgroup (the pool is one segment).
__global__ __launch_bounds__(kOneThreads) void pages_compact_one(PagesCompactArgs a) {
  __shared__ uint32_t lds[kMostWaves];
  count_segment<true>(a.t, 0, lds);
  __syncthreads();
  compact_segment(a, 0, lds);
  __syncthreads();
  compact_tables(a, threadIdx.x, kOneThreads);
}

// ------------------------------------------------------------------------------------------------ copies
typedef uint32_t w4 __attribute__((ext_vector_type(4)));
typedef w4 w4_any __attribute__((aligned(4)));   // (buffers are aligned to 4 bytes)

// Copies pieces [first, last) of 16 bytes of `runs` runs, `run` bytes apart, `used` bytes of each (a multiple of 4).
__device__ __forceinline__ void copy_runs(const uint8_t* from, uint8_t* to, uint32_t runs, uint32_t run, uint32_t used, uint32_t first,
                                          uint32_t last) {
  const uint32_t each = (used + 15) / 16;
  for (uint32_t i = first + threadIdx.x; i < last; i += kThreads) {
    const uint32_t r = runs > 1 ? i / each : 0, at = (i - r * each) * 16, left = used - at;
    const uint8_t* const f = from + (uint64_t)r * run + at;
    uint8_t* const g = to + (uint64_t)r * run + at;
    if (left >= 16) {
      *(w4_any*)g = *(const w4_any*)f;
    } else {
      for (uint32_t j = 0; j < left; j += 4) *(uint32_t*)(g + j) = *(const uint32_t*)(f + j);
    }
  }
}

// A unit of work is a slice of a page of a layer, all four buffers one behind the other, or one of them.
__global__ __launch_bounds__(kThreads) void pages_copy(PagesCopyArgs a) {
  const uint32_t count = min(*a.count, a.most);
  const uint64_t units = (uint64_t)count * a.layers * a.slices * a.parts;
  for (uint64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    uint64_t rest = unit / a.parts;
    const uint32_t only = (uint32_t)(unit % a.parts), slice = (uint32_t)(rest % a.slices);
    rest /= a.slices;
    const uint32_t l = (uint32_t)(rest % a.layers), i = (uint32_t)(rest / a.layers);
    const uint32_t source = a.source[a.backwards ? count - 1 - i : i], target = a.target[i];
    const PagesLayer& layer = a.layer[l];
    const uint32_t tokens = a.tokens ? a.tokens[i] : a.page_size;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (a.parts > 1 && only != (uint32_t)b) continue;
      const uint32_t row = b & 1 ? 4u : layer.row_bytes[b >> 1];
      const uint64_t stride = (uint64_t)layer.page_stride * row;
      // whole pages and token-major ones are one run
      const bool split = layer.head_major && tokens != a.page_size;
      const uint32_t runs = split ? layer.kv_heads : 1, used = tokens * row * (split ? 1 : layer.kv_heads), run = a.page_size * row;
      const uint32_t pieces = runs * ((used + 15) / 16), each = (pieces + a.slices - 1) / a.slices;
      copy_runs(layer.base[b] + source * stride, layer.base[b] + target * stride, runs, run, used, min(slice * each, pieces),
                min((slice + 1) * each, pieces));
    }
  }
}

}  // namespace

// The pool as one segment, for one workgroup.
static void as_one_segment(PagesTables& t) {
  t.segment = (t.pages + kOneThreads - 1) / kOneThreads * kOneThreads;
  t.segments = 1;
}

hipError_t launch_pages_reserve(const PagesReserveArgs& a, hipStream_t s) {
  if (a.t.pages <= kReserveOnePages && a.t.sequences <= kReserveOneRows && a.capacity <= kReserveOneTokens) {
    pages_reserve_one<<<dim3(1), dim3(kOneThreads), 0, s>>>(a);
    return hipGetLastError();
  }
  pages_reserve_plan<<<dim3(a.t.segments + 1), dim3(kThreads), 0, s>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  pages_reserve_place<<<dim3(a.t.segments + (a.t.sequences + 3) / 4), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_pages_trim(const PagesTrimArgs& a, hipStream_t s) {
  pages_trim<<<dim3((a.t.sequences + 3) / 4), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_pages_fork(const PagesForkArgs& call, PagesCopyArgs* copies, hipStream_t s) {
  PagesForkArgs a = call;
  const uint32_t rows = (a.t.sequences + 3) / 4;
  copies->count = a.t.plan + 1;
  copies->source = a.t.plan + 8 + 2ull * a.t.sequences;
  copies->target = copies->source + a.t.sequences;
  copies->tokens = copies->target + a.t.sequences;
  copies->backwards = 0;
  copies->most = a.t.sequences;
  if (a.t.pages <= kForkOnePages && a.t.sequences <= kForkOneRows) {
    as_one_segment(a.t);
    pages_fork_one<<<dim3(1), dim3(kOneThreads), 0, s>>>(a);
    return hipGetLastError();
  }
  pages_fork_rows<<<dim3(rows), dim3(kThreads), 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  pages_fork_plan<<<dim3(a.t.segments + 1), dim3(kThreads), 0, s>>>(a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  pages_fork_place<<<dim3(a.t.segments + rows), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_pages_compact(const PagesCompactArgs& call, PagesCopyArgs* copies, hipStream_t s) {
  PagesCompactArgs a = call;
  copies->count = a.t.plan + 1;
  copies->target = a.t.room;
  copies->source = a.t.room + a.t.pages;
  copies->tokens = nullptr;
  copies->backwards = 1;
  copies->most = a.t.pages / 2;
  if (a.t.pages <= kCompactOnePages && a.t.sequences <= kCompactOneRows) {
    as_one_segment(a.t);
    pages_compact_one<<<dim3(1), dim3(kOneThreads), 0, s>>>(a);
    return hipGetLastError();
  }
  pages_compact_count<<<dim3(a.t.segments), dim3(kThreads), 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  pages_compact_list<<<dim3(a.t.segments), dim3(kThreads), 0, s>>>(a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  pages_compact_tables<<<dim3((a.t.sequences + 3) / 4), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_pages_copy(const PagesCopyArgs& call, uint32_t cus, hipStream_t s) {
  PagesCopyArgs a = call;
  const uint64_t slices = (uint64_t)a.most * a.layers * a.slices, most = 8ull * cus;
  if (slices == 0) return hipSuccess;
  // Where there are few slices, a workgroup takes one buffer of a slice: the four do not wait for each other (two pages of 12 layers
  // 4.0 us instead of 5.4). Where there are many, a unit of all four costs fewer divisions and looks at its pages' numbers once.
  a.parts = slices < 2ull * cus ? 4 : 1;
  const uint64_t units = slices * a.parts;
  pages_copy<<<dim3((uint32_t)(units < most ? units : most)), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace pitch
