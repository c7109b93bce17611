// The pages of a paged cache beyond a step's own: requests that go on in several ways, pages given back, pages moved
// together, and the copy of what is in them.
//
// A page's holders are the block table rows that name it: shares[page] + 1 of them, 0 where it is free or has one.
// Pages that nobody holds are free_pages[free_start ..). Everything here is decided by integers in a fixed order,
// whatever order the threads run in.
#pragma once

#include "common.h"
#include "paged_args.h"
#include "paged_cache.h"

namespace aoto {

constexpr int kPageSteps = 8, kPageBatch = 1024 * kPageSteps;  // pages that a block looks at in one round trip

// Of a batch of flags in the order of their pages (thread tid has those of pages 1024 i + tid, bit i of `bits`): how
// many lie before each. before[i] for this thread's, `total` for the block. `scratch`: kPageRanks values.
constexpr int kPageRanks = 16 * kPageSteps + 2;
AOTO_DEVICE void page_ranks(uint32_t bits, int (&before)[kPageSteps], int& total, int* scratch) {
  constexpr int ALL = 16 * kPageSteps;  // waves of flags: two waves sum them
  static_assert(ALL == 128, "two waves");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int i = 0; i < kPageSteps; ++i) {
    const unsigned long long lanes = __ballot(bits >> i & 1);
    before[i] = __popcll(lanes & ((1ull << lane) - 1));
    if (lane == 0) scratch[16 * i + wave] = __popcll(lanes);
  }
  __syncthreads();
  int own = 0, sum = 0;
  if (tid < ALL) {
    own = sum = scratch[tid];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    if (lane == 63) scratch[ALL + wave] = sum;
  }
  __syncthreads();
  if (tid < ALL) scratch[tid] = sum - own + (wave ? scratch[ALL] : 0);
  total = scratch[ALL] + scratch[ALL + 1];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPageSteps; ++i) before[i] += scratch[16 * i + wave];
  __syncthreads();
}

// Entry j of request r is its parent's, whose page has one holder more.
AOTO_DEVICE void share_page(const PagedForkArgs& a, int r, int j) {
  const int page = a.block_tables[(size_t)a.parents[r] * a.table_stride + j];
  a.block_tables[(size_t)r * a.table_stride + j] = page;
  if ((unsigned)page < (unsigned)a.pages) atomicAdd(a.shares + page, 1);
}

// Four neighbours of a list, 0 past its end.
struct __attribute__((packed, aligned(4))) PageFour {
  int v[4];
};
AOTO_DEVICE PageFour page_four(const int* values, int from, int count) {
  if (from + 4 <= count) return *reinterpret_cast<const PageFour*>(values + from);
  PageFour four;
#pragma unroll
  for (int e = 0; e < 4; ++e) four.v[e] = from + e < count ? values[from + e] : 0;
  return four;
}

// f(row, place, page) for the table entries of all rows (those past a row's count too), by one block: eight entries a
// thread on their way at a time.
template <typename F>
AOTO_DEVICE void each_entry(const int* tables, long long stride, int requests, int max_blocks, F f) {
  const int all = requests * max_blocks, tid = threadIdx.x;
  for (int base = 0; base < all; base += kPageBatch) {
    int page[kPageSteps];
#pragma unroll
    for (int i = 0; i < kPageSteps; ++i) {
      const int k = min(base + 1024 * i + tid, all - 1), r = k / max_blocks;
      page[i] = tables[(size_t)r * stride + (k - r * max_blocks)];
    }
#pragma unroll
    for (int i = 0; i < kPageSteps; ++i) {
      const int k = base + 1024 * i + tid, r = k / max_blocks;
      if (k < all) f(r, k - r * max_blocks, page[i]);
    }
  }
}

}  // namespace aoto

// Which rows go on from which, which of the others end inside a page that is not theirs alone, the pages taken for them
// and what is to be copied (formulas at the entry point's declaration). One block: everything hangs on a running sum
// over the requests. Where `fill` is set it also enters the full pages, which aoto_paged_share does otherwise. Bound by
// round trips: a row, the row that it goes on from, the page in progress, its holders, the writes (8 rows 4.3 us, 900
// and the second launch 8.2).
extern "C" __global__ __launch_bounds__(1024) void aoto_paged_fork(PagedForkArgs a, int fill) {
  using namespace aoto;
  __shared__ long long s_scan[16];
  __shared__ int s_ends[1024];   // the shared page that a row of this pass ends in, -1 without
  __shared__ int s_spare[1024];  // the free list's next
  __shared__ int s_error;
  const int tid = threadIdx.x;
  if (tid == 0) s_error = 0;
  const int start = a.free_start[0];
  const long long first_free = max(start, 0);
  long long taken = 0;
  int error = 0;
  __syncthreads();
  for (int base = 0; base < a.requests; base += 1024) {
    const int r = base + tid, mine = min(r, a.requests - 1);
    // asked for together: the row as one that stays, and the pages that this pass may take
    int parent = a.parents[mine], count = a.page_counts[mine], length = a.context_lens[mine];
    const long long next = first_free + taken + tid;
    const int spare = next < a.free_count ? a.free_pages[next] : -1;
    if (r >= a.requests) parent = -1, count = 0;
    if (parent >= a.requests) error |= AOTO_PAGED_BAD_ROW, parent = -1;
    if (parent >= 0 && count > 0) error |= AOTO_PAGED_ROW_HELD, parent = -1;
    const int of = parent >= 0 ? parent : mine;
    if (parent >= 0) count = a.page_counts[parent], length = a.context_lens[parent];
    count = min(max(count, 0), a.max_blocks);
    length = (int)min((long long)max(length, 0), (long long)count * a.page);
    const int full = length / a.page;
    const int page = length > full * a.page ? a.block_tables[(size_t)of * a.table_stride + full] : -1;
    // Holders of the page that a row which stays ends in, beside it. What the passes before took from them is past the
    // first cache.
    int others = 0;
    if (parent < 0 && (unsigned)page < (unsigned)a.pages)
      others = base ? __hip_atomic_load(a.shares + page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                    : a.shares[page];
    s_spare[tid] = spare, s_ends[tid] = others > 0 ? page : -1;
    __syncthreads();
    if (others > 0)
      for (int i = 0; i < tid; ++i) others -= s_ends[i] == page;  // those of rows before are gone
    const bool leaves = others > 0, part = leaves || (parent >= 0 && length > full * a.page);
    long long total = 0;
    const int at = (int)block_scan_1024(part ? 1 : 0, s_scan, total) - 1;
    if (r < a.requests) {
      int source = -1, target = -1, plan = parent >= 0 ? full : -1;
      if (part) {
        const bool some = first_free + taken + at < a.free_count;
        if (some) source = page, target = s_spare[at];
        if (!some) error |= AOTO_PAGED_NO_PAGES, length = full * a.page;
        if (leaves) {
          if ((unsigned)target < (unsigned)a.pages) {
            plan = -2 - full;
            if (atomicSub(a.shares + page, 1) <= 0) error |= AOTO_PAGED_BAD_SHARE;
          } else {
            source = target = -1, error |= AOTO_PAGED_NO_PAGES | AOTO_PAGED_ROW_SHARED;
          }
        }
      }
      a.source[r] = source, a.target[r] = target;
      a.plan[2 * r] = plan, a.plan[2 * r + 1] = length;
    }
    taken += total;
    if (base + 1024 < a.requests) __syncthreads();  // s_spare and s_ends are read
  }
  if (error) atomicOr(&s_error, error);
  __syncthreads();
  // only now: a row may be the parent of another, and the outputs may be the inputs
  for (int r = tid; r < a.requests; r += 1024) {
    const int full = a.plan[2 * r], length = a.plan[2 * r + 1];
    const bool part = full >= 0 && length > full * a.page;
    if (part || full < -1) a.block_tables[(size_t)r * a.table_stride + (part ? full : -2 - full)] = a.target[r];
    a.context_lens_out[r] = full >= 0 ? length : a.context_lens[r];
    a.page_counts_out[r] = full >= 0 ? full + (part ? 1 : 0) : a.page_counts[r];
  }
  if (fill)
    for (int k = tid; k < a.requests * a.max_blocks; k += 1024) {
      const int r = k / a.max_blocks, j = k - r * a.max_blocks;
      if (j < a.plan[2 * r]) share_page(a, r, j);
    }
  if (tid == 0) {
    const long long available = max(0LL, a.free_count - first_free);
    a.free_start_out[0] = taken ? (int)(first_free + min(taken, available)) : start;
    if (s_error && a.error) atomicOr(a.error, s_error);
  }
}

// The full pages of the rows that go on: entered in their own rows, one holder more each.
extern "C" __global__ __launch_bounds__(256) void aoto_paged_share(PagedForkArgs a) {
  const int r = blockIdx.x, full = a.plan[2 * r];
  for (int j = threadIdx.x; j < full; j += 256) aoto::share_page(a, r, j);
}

namespace aoto {
// The pages that a request holds, and those of them that it keeps.
AOTO_DEVICE int pages_held(const PagedReleaseArgs& a, int held) { return min(max(held, 0), a.max_blocks); }
AOTO_DEVICE int pages_kept(const PagedReleaseArgs& a, int count, int keep) {
  return keep < 0 ? count : min(count, (int)(((unsigned)keep + (unsigned)a.page - 1) / (unsigned)a.page));
}
// While a pool's pages are given back, what stands in `shares` of a page of the free list has kPageMark added, once for
// each of its entries. A page's shares and the holders that go are below 2^27, so that the upper four bits tell the
// mark; the lower ones are the shares that are left, -1 where nobody holds the page.
constexpr int kPageMark = 1 << 28;
AOTO_DEVICE int page_mark(int v) { return ((unsigned)v + kPageMark / 2) >> 28; }
AOTO_DEVICE int page_share(int v) { return (int)((unsigned)v << 4) >> 4; }
AOTO_DEVICE bool page_gone(int v) { return page_share(v) < 0 && !page_mark(v); }
}  // namespace aoto

// Requests' pages past what they keep lose a holder each, and pages of the free list are marked: additions, in any
// order, from which aoto::page_mark and page_share tell both. Blocks 0 .. requests - 1: a row of the tables each; the
// others: the free list.
extern "C" __global__ __launch_bounds__(256) void aoto_paged_drop(PagedReleaseArgs a) {
  const int r = blockIdx.x;
  if (r >= a.requests) {
    const int first = min(max(a.free_start[0], 0), a.free_count);
    for (long long j = first + (r - a.requests) * 256LL + threadIdx.x; j < a.free_count; j += a.list_blocks * 256LL) {
      const int page = a.free_pages[j];
      if ((unsigned)page < (unsigned)a.pages) atomicAdd(a.shares + page, aoto::kPageMark);
    }
    return;
  }
  const int held = a.page_counts[r], keep = a.keep_lens[r];
  const int count = aoto::pages_held(a, held), stays = aoto::pages_kept(a, count, keep);
  __syncthreads();  // the counts written may be the counts read
  if (threadIdx.x == 0) a.page_counts_out[r] = keep < 0 ? held : stays;
  const int* table = a.block_tables + (size_t)r * a.table_stride;
  for (int j = stays + threadIdx.x; j < count; j += 256) {
    const int page = table[j];
    if ((unsigned)page < (unsigned)a.pages) atomicSub(a.shares + page, 1);
  }
}

// The pages left without a holder, in the order of their numbers, to the places before the free list's first: their
// number in each 1024 pages, then their places. (In one launch a block would have to read the whole pool for its own
// place, at a single CU's 20 GB/s: 15 us for 41000 pages instead of 2.2 + 2.8.) A page that the list holds already
// was given back more often than held and is not entered again.
extern "C" __global__ __launch_bounds__(256) void aoto_paged_gone(PagedReleaseArgs a) {
  using namespace aoto;
  __shared__ int s_count[4];
  const int wave = threadIdx.x >> 6, chunk = blockIdx.x;
  const PageFour share = page_four(a.shares, kPageChunk * chunk + 4 * threadIdx.x, a.pages);
  int count = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) count += __popcll(__ballot(page_gone(share.v[e])));
  if ((threadIdx.x & 63) == 0) s_count[wave] = count;
  __syncthreads();
  if (threadIdx.x != 0) return;
  a.scratch[1 + chunk] = s_count[0] + s_count[1] + s_count[2] + s_count[3];
  if (chunk == 0) a.scratch[0] = a.free_start[0];  // the start written may be the start read
}

extern "C" __global__ __launch_bounds__(256) void aoto_paged_reclaim(PagedReleaseArgs a) {
  using namespace aoto;
  __shared__ int s_count[4], s_before[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, chunk = blockIdx.x;
  const int from = kPageChunk * chunk + 4 * tid;
  const PageFour share = page_four(a.shares, from, a.pages);
  int before = 0;
  for (int i = tid; i < chunk; i += 256) before += a.scratch[1 + i];
  const int start = a.scratch[0], first = min(max(start, 0), a.free_count);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) before += __shfl_xor(before, d);
  int count = 0, rank = 0;
  const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const unsigned long long lanes = __ballot(page_gone(share.v[e]));
    count += __popcll(lanes), rank += __popcll(lanes & below);
  }
  if (lane == 0) s_count[wave] = count, s_before[wave] = before;
  __syncthreads();
  before = s_before[0] + s_before[1] + s_before[2] + s_before[3];
  int total = before;
#pragma unroll
  for (int w = 0; w < 4; ++w) rank += w < wave ? s_count[w] : 0, total += s_count[w];
  int error = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int left = page_share(share.v[e]), now = max(left, 0);
    if (now != share.v[e]) a.shares[from + e] = now;
    if (left < -1 || (left < 0 && page_mark(share.v[e]))) error |= AOTO_PAGED_BAD_SHARE;
    if (page_gone(share.v[e])) {
      const int at = first - 1 - before - rank++;
      if (at >= 0) a.free_pages[at] = from + e;
      else error |= AOTO_PAGED_LIST_FULL;
    }
  }
  if (error && a.error) atomicOr(a.error, error);
  if (tid == 0 && chunk == (a.pages - 1) / kPageChunk) a.free_start_out[0] = total ? max(0, first - total) : start;
}

// All of it by one block, which counts the holders that go in LDS: pools of up to kPagesFew pages. What bounds it is
// one CU's reading, so it gains by its two launches fewer (2 to 3 us each where they are not captured) and only as long
// as the GPU is hardly slower. In a graph, for entries of tables and pages of the pool: 512 and 600 5.5 us and 5.7 in
// three launches, 2048 and 2500 6.7 and 6.3, 4096 and 4000 7.7 and 6.1; in an instance for 8192 pages 8192 and 8000 9.8
// and 6.6.
extern "C" __global__ __launch_bounds__(1024) void aoto_paged_release_few(PagedReleaseArgs a) {
  using namespace aoto;
  constexpr uint32_t LISTED = 0x80000000u;
  __shared__ uint32_t s_gone[kPagesFew];  // of each page: the holders that go, and whether the free list holds it
  __shared__ int s_scratch[kPageRanks];
  const int tid = threadIdx.x;
  const int start = a.free_start[0], first = min(max(start, 0), a.free_count);
  for (int page = tid; page < a.pages; page += 1024) s_gone[page] = 0;
  __syncthreads();
  each_entry(a.block_tables, a.table_stride, a.requests, a.max_blocks, [&](int r, int j, int page) {
    const int count = pages_held(a, a.page_counts[r]);
    if (j < count && j >= pages_kept(a, count, a.keep_lens[r]) && (unsigned)page < (unsigned)a.pages)
      atomicAdd(&s_gone[page], 1u);
  });
  for (int j = first + tid; j < a.free_count; j += 1024) {
    const int page = a.free_pages[j];
    if ((unsigned)page < (unsigned)a.pages) atomicOr(&s_gone[page], LISTED);
  }
  __syncthreads();  // also: the counts written may be the counts read
  for (int r = tid; r < a.requests; r += 1024) {
    const int held = a.page_counts[r], keep = a.keep_lens[r];
    a.page_counts_out[r] = keep < 0 ? held : pages_kept(a, pages_held(a, held), keep);
  }
  static_assert(kPagesFew <= kPageBatch, "one look at each page");
  int left[kPageSteps], rank[kPageSteps], total, error = 0;
  uint32_t none = 0;
#pragma unroll
  for (int i = 0; i < kPageSteps; ++i) {
    const int page = 1024 * i + tid;
    left[i] = page < a.pages ? a.shares[page] : 0;
  }
#pragma unroll
  for (int i = 0; i < kPageSteps; ++i) {
    const int page = 1024 * i + tid;
    const uint32_t of = page < a.pages ? s_gone[page] : 0;
    const int gone = (int)(of & ~LISTED);
    left[i] -= gone;
    none |= (uint32_t)(left[i] < 0 && !(of & LISTED)) << i;
    if (gone || left[i] < 0) a.shares[page] = max(left[i], 0);
    if (left[i] < -1 || (left[i] < 0 && of & LISTED)) error |= AOTO_PAGED_BAD_SHARE;
  }
  page_ranks(none, rank, total, s_scratch);
#pragma unroll
  for (int i = 0; i < kPageSteps; ++i)
    if (none >> i & 1) {
      const int at = first - 1 - rank[i];
      if (at >= 0) a.free_pages[at] = 1024 * i + tid;
      else error |= AOTO_PAGED_LIST_FULL;
    }
  if (error && a.error) atomicOr(a.error, error);
  if (tid == 0) a.free_start_out[0] = total ? max(0, first - total) : start;
}

// What each page is: 0, and then (aoto_paged_mark) 1 where a request holds it, 2 where it is in the free list.
extern "C" __global__ __launch_bounds__(256) void aoto_paged_clear(PagedCompactArgs a) {
  const int page = blockIdx.x * 256 + threadIdx.x;
  if (page < a.pages) a.state[page] = 0;
}

// Blocks 0 .. requests - 1: a row of the tables each; the others: the free list.
extern "C" __global__ __launch_bounds__(256) void aoto_paged_mark(PagedCompactArgs a) {
  const int r = blockIdx.x;
  if (r < a.requests) {
    const int count = min(max(a.page_counts[r], 0), a.max_blocks);
    for (int j = threadIdx.x; j < count; j += 256) {
      const int page = a.block_tables[(size_t)r * a.table_stride + j];
      if ((unsigned)page < (unsigned)a.pages) atomicOr(a.state + page, 1);
    }
    return;
  }
  const int first = max(a.free_start[0], 0), others = a.list_blocks;
  for (long long j = first + (long long)(r - a.requests) * 256 + threadIdx.x; j < a.free_count; j += others * 256LL) {
    const int page = a.free_pages[j];
    if ((unsigned)page < (unsigned)a.pages) atomicOr(a.state + page, 2);
  }
}

// The moves. With m pages held, and the pages held or free in the order of their numbers: held ones past the first m
// go, in order, to the free ones among the first m, and the rest is the free list. One block: 8192 pages a round trip,
// once for m and once for the places. `state_of`: what each page is, then its new number.
namespace aoto {
AOTO_DEVICE void page_moves(const PagedCompactArgs& a, int* state_of) {
  __shared__ int s_scratch[kPageRanks];
  __shared__ int s_low;
  const int tid = threadIdx.x;
  const int first = min(max(a.free_start[0], 0), a.free_count);
  int own = 0, both = 0;
  for (int base = 0; base < a.pages; base += kPageBatch) {
    int state[kPageSteps];
#pragma unroll
    for (int i = 0; i < kPageSteps; ++i) {
      const int page = base + 1024 * i + tid;
      state[i] = page < a.pages ? state_of[page] : 0;
    }
#pragma unroll
    for (int i = 0; i < kPageSteps; ++i) own += state[i] & 1, both += state[i] == 3;
  }
  int error = both ? AOTO_PAGED_BAD_SHARE : 0;
  __shared__ long long s_scan[16];
  long long total_held;
  block_scan_1024(own, s_scan, total_held);
  const int m = (int)total_held;
  if (tid == 0) s_low = 0;
  __syncthreads();
  int places = 0, held = 0;  // of the pages before
  for (int base = 0; base < a.pages; base += kPageBatch) {
    int state[kPageSteps];
#pragma unroll
    for (int i = 0; i < kPageSteps; ++i) {
      const int page = base + 1024 * i + tid;
      state[i] = page < a.pages ? state_of[page] : 0;
    }
    uint32_t any = 0, is_held = 0;
#pragma unroll
    for (int i = 0; i < kPageSteps; ++i) {
      any |= (uint32_t)(state[i] != 0) << i;
      is_held |= (uint32_t)(state[i] & 1) << i;
    }
    int place[kPageSteps], held_before[kPageSteps], some, some_held;
    page_ranks(any, place, some, s_scratch);
    page_ranks(is_held, held_before, some_held, s_scratch);
#pragma unroll
    for (int i = 0; i < kPageSteps; ++i) {
      place[i] += places, held_before[i] += held;
      const int page = base + 1024 * i + tid;
      if (any >> i & 1 && place[i] < m) {
        if (!(is_held >> i & 1)) a.target[place[i] - held_before[i]] = page;
        if (place[i] == m - 1) s_low = held_before[i] + (is_held >> i & 1);  // held pages that stay
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPageSteps; ++i) {
      const int page = base + 1024 * i + tid;
      if (page >= a.pages) continue;
      int now = page;
      if (any >> i & 1 && place[i] >= m) {
        if (is_held >> i & 1) {
          const int k = held_before[i] - s_low;
          a.source[k] = page;
          now = a.target[k];
          a.shares[now] = a.shares[page];
          a.shares[page] = 0;
        }
        const int at = first + place[i] - m;
        if (at < a.free_count) a.free_pages[at] = page;
      }
      state_of[page] = now;
    }
    places += some, held += some_held;
    __syncthreads();
  }
  const int moved = m - s_low;
  for (int k = moved + tid; k < a.pages; k += 1024) a.source[k] = a.target[k] = -1;
  // entries of the list that named no page, or one twice
  const int rest = first + places - m;
  if (rest < a.free_count) error |= AOTO_PAGED_BAD_SHARE;
  for (int j = rest + tid; j < a.free_count; j += 1024) a.free_pages[j] = -1;
  if (error && a.error) atomicOr(a.error, error);
  if (tid == 0) a.count[0] = moved;
}
}  // namespace aoto

extern "C" __global__ __launch_bounds__(1024) void aoto_paged_moves(PagedCompactArgs a) {
  aoto::page_moves(a, a.state);
}

extern "C" __global__ __launch_bounds__(256) void aoto_paged_remap(PagedCompactArgs a) {
  const int r = blockIdx.x, count = min(max(a.page_counts[r], 0), a.max_blocks);
  for (int j = threadIdx.x; j < count; j += 256) {
    int* entry = a.block_tables + (size_t)r * a.table_stride + j;
    const int page = *entry;
    if ((unsigned)page < (unsigned)a.pages) *entry = a.state[page];
  }
}

// All of it by one block, with the pages' states in LDS: pools of up to kPagesFew pages. As in aoto_paged_release_few,
// the gain is three launches: 512 entries of tables and 600 pages 9.5 us and 11.0 in four, 2048 and 2500 11.1 and 11.4,
// 4096 and 4000 12.5 and 11.9; in an instance for 8192 pages 8192 and 8000 15.8 and 12.9.
extern "C" __global__ __launch_bounds__(1024) void aoto_paged_compact_few(PagedCompactArgs a) {
  using namespace aoto;
  __shared__ int s_state[kPagesFew];
  const int tid = threadIdx.x;
  for (int page = tid; page < a.pages; page += 1024) s_state[page] = 0;
  __syncthreads();
  auto mark = [&](int page, int as) {
    if ((unsigned)page < (unsigned)a.pages) atomicOr(&s_state[page], as);
  };
  each_entry(a.block_tables, a.table_stride, a.requests, a.max_blocks, [&](int r, int j, int page) {
    if (j < a.page_counts[r]) mark(page, 1);
  });
  for (long long j = max(a.free_start[0], 0) + tid; j < a.free_count; j += 1024) mark(a.free_pages[j], 2);
  __syncthreads();
  page_moves(a, s_state);
  __syncthreads();
  each_entry(a.block_tables, a.table_stride, a.requests, a.max_blocks, [&](int r, int j, int page) {
    if (j < a.page_counts[r] && (unsigned)page < (unsigned)a.pages)
      a.block_tables[(size_t)r * a.table_stride + j] = s_state[page];
  });
}

// Pages' contents from source[i] to target[i], in every plane of every tensor. Every wave looks at 64 pairs at a time,
// a lane each, and the block takes its share of the chunks (16 KB of a page of a plane) of those that are to be copied:
// pairs without a copy cost a 64th of a look. The grid's size comes as an argument, and a thread's 64 bytes have names
// of their own: what makes the compiler ask for the dispatch packet (gridDim, an array that it moves to LDS) is a read
// of host memory by every block, 40 ns each one after the other (384 blocks without a page to copy: 15.6 us). Bound by
// the read and the write: 470 MB in 93 us (5.05 TB/s; a copy of a gigabyte reaches 5.10), 201 MB in 30.
extern "C" __global__ __launch_bounds__(256) void aoto_paged_copy(PagedCopyArgs a) {
  const int lane = threadIdx.x & 63;
  const int pairs = a.count ? min(max(a.count[0], 0), a.pairs) : a.pairs;
  const unsigned each = (unsigned)a.planes * a.chunks;  // chunks of a pair
  int error = 0;
  unsigned next = blockIdx.x;  // this block's next chunk, counted from the present pairs' first
  for (int base = 0; base < pairs; base += 64) {
    const int mine = min(base + lane, pairs - 1);
    const int source = a.source[mine], target = a.target[mine];
    const bool inside = (unsigned)source < (unsigned)a.pages && (unsigned)target < (unsigned)a.pages;
    const unsigned long long some = __ballot(inside && source != target && base + lane < pairs);
    if (source < -1 || source >= a.pages || target < -1 || target >= a.pages) error = AOTO_PAGED_BAD_SLOT;
    const unsigned long long chunks = (unsigned long long)__popcll(some) * each;
    const int rank = __popcll(some & ((1ull << lane) - 1));
    unsigned long long item = next;
    for (; item < chunks; item += a.blocks) {
      const int pair = (int)(item < 0x80000000ull ? (unsigned)item / each : item / each);
      const unsigned within = (unsigned)(item - (unsigned long long)pair * each);
      const int at_lane = __ffsll(__ballot(some >> lane & 1 && rank == pair)) - 1;
      const int from_page = __builtin_amdgcn_readlane(source, at_lane);
      const int to_page = __builtin_amdgcn_readlane(target, at_lane);
      const int plane = a.chunks == 1 ? within : within / a.chunks, chunk = within - plane * a.chunks;
      int t = 0;
      while (t + 1 < a.tensors && a.at[t + 1].first <= plane) ++t;
      const PagedCopyTensor& at = a.at[t];
      if (chunk >= at.chunks) continue;
      uint8_t* first = at.base + (plane - at.first) * at.plane_stride + (long long)chunk * kPagedCopyChunk;
      const uint8_t* from = first + from_page * at.page_stride;
      uint8_t* to = first + to_page * at.page_stride;
      const int bytes = (int)min(at.bytes - (long long)chunk * kPagedCopyChunk, (long long)kPagedCopyChunk);
      if (a.wide && bytes == kPagedCopyChunk) {
        const uint4* f = reinterpret_cast<const uint4*>(from) + threadIdx.x;
        uint4* t4 = reinterpret_cast<uint4*>(to) + threadIdx.x;
        const uint4 v0 = f[0], v1 = f[256], v2 = f[512], v3 = f[768];
        t4[0] = v0, t4[256] = v1, t4[512] = v2, t4[768] = v3;
      } else if (a.wide) {
        for (int b = threadIdx.x; b < bytes / 16; b += 256)
          reinterpret_cast<uint4*>(to)[b] = reinterpret_cast<const uint4*>(from)[b];
      } else {
        for (int b = threadIdx.x; b < bytes; b += 256) to[b] = from[b];
      }
    }
    next = (unsigned)(item - chunks);
  }
  if (error && a.error && blockIdx.x == 0) atomicOr(a.error, error);
}
