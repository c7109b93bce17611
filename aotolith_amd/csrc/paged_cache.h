// The paged key/value cache that requests of different lengths share: a step's bookkeeping and the write of its
// new keys and values.
//
// Cache of one layer: keys and values of a page, bf16 [Hkv][page][D] at any page / head / slot strides; slot number
// s is row s % page of page s / page. A request's logical rows lie in the pages its block table row names, in order.
#pragma once

#include "common.h"
#include "paged_args.h"

namespace aoto {

// Inclusive sum over a 1024-thread block; the block's total in `total`. `scratch` holds 16 values.
AOTO_DEVICE long long block_scan_1024(long long v, long long* scratch, long long& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const long long up = __shfl_up(v, d);
    if (lane >= d) v += up;
  }
  if (lane == 63) scratch[wave] = v;
  __syncthreads();
  total = 0;
  long long before = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    before += w < wave ? scratch[w] : 0;
    total += scratch[w];
  }
  __syncthreads();
  return v + before;
}

// The first i of [0, n) with sums[i] > k (sums not decreasing, sums[n - 1] > k).
AOTO_DEVICE int first_above(const int* sums, int n, int k) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] > k) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Whether a token may not be written to a page because others read it there.
AOTO_DEVICE bool page_of_others(const PagedTablesArgs& a, int page) {
  return a.shares && (unsigned)page < (unsigned)a.pages && a.shares[page] > 0;
}

}  // namespace aoto

// A step's pages, block tables and token maps from the requests' lengths (formulas at the entry point's declaration).
// One block: everything hangs on two running sums over the requests (tokens, taken pages), taken 1024 requests at a
// time with the sums so far carried in registers; the entries taken and, where `fill` is set, the tokens are then
// shared out over the threads by a search of those sums in LDS. Bound by latency: three round trips to memory a pass
// of 1024 requests (lengths, free pages, stores); 5.9 us for 8 requests, 5.2 and 3.2 (the maps' own launch) for 256.
extern "C" __global__ __launch_bounds__(1024) void aoto_paged_tables(PagedTablesArgs a, int fill) {
  using namespace aoto;
  __shared__ long long s_scan[16];
  __shared__ int s_tokens[1024], s_taken[1024];   // inclusive sums of this pass's requests
  __shared__ int s_count[1024], s_context[1024];
  __shared__ int s_error;
  const int tid = threadIdx.x;
  if (tid == 0) s_error = 0;
  const int start = a.free_start[0];
  const long long first_free = max(start, 0);
  const long long available = max(0LL, (long long)a.free_count - first_free);
  long long tokens = 0, taken = 0;
  int error = 0;
  __syncthreads();
  for (int base = 0; base < a.requests; base += 1024) {
    const int r = base + tid, live = min(1024, a.requests - base);
    int context = 0, count = 0;
    long long fresh = 0;
    if (tid < live) {
      context = min(max(a.context_lens[r], 0), kPagedMostContext);
      count = min(max(a.page_counts[r], 0), a.max_blocks);
      fresh = max(a.new_lens[r], 0);
    }
    long long total = 0;
    const long long end_all = tokens + block_scan_1024(fresh, s_scan, total);
    // rows past max_tokens are not there: a request that meets the end is cut
    const long long end = min(end_all, (long long)a.max_tokens);
    const long long begin = min(end_all - fresh, (long long)a.max_tokens);
    if (end_all > a.max_tokens) error |= AOTO_PAGED_TOKENS_CUT;
    const int kv = context + (int)(end - begin);
    const int full = (int)(((unsigned)kv + a.page - 1) / (unsigned)a.page);
    if (full > a.max_blocks) error |= AOTO_PAGED_TABLE_FULL;
    const int need = max(count, min(full, a.max_blocks));
    long long total_taken = 0;
    const long long taken_end = taken + block_scan_1024(need - count, s_scan, total_taken);
    const long long taken_begin = taken_end - (need - count);
    const int got = (int)max(0LL, min(taken_end, available) - min(taken_begin, available));
    if (got < need - count) error |= AOTO_PAGED_NO_PAGES;
    if (tid < live) {
      a.query_start[r + 1] = (int)end;
      a.kv_lens[r] = kv;
      a.page_counts_out[r] = count + got;
    }
    s_tokens[tid] = (int)(end - min(tokens, (long long)a.max_tokens));
    s_taken[tid] = (int)(taken_end - taken);
    s_count[tid] = tid < live ? count : 0;
    s_context[tid] = context;
    __syncthreads();
    for (int k = tid; k < (int)total_taken; k += 1024) {
      const int i = first_above(s_taken, 1024, k);
      const int j = k - (i ? s_taken[i - 1] : 0);
      const long long at = taken + k;
      a.block_tables[(size_t)(base + i) * a.table_stride + s_count[i] + j] =
          at < available ? a.free_pages[first_free + at] : -1;
    }
    if (fill) {
      // the entries just written are read below by other threads of the block
      __syncthreads();
      const int here = s_tokens[1023];
      const int offset = (int)min(tokens, (long long)a.max_tokens);
      for (int k = tid; k < here; k += 1024) {
        const int i = first_above(s_tokens, 1024, k);
        const int position = s_context[i] + k - (i ? s_tokens[i - 1] : 0);
        const int block = position / a.page;
        const int begin_taken = i ? s_taken[i - 1] : 0;
        int page = -1;
        if (block < s_count[i] + s_taken[i] - begin_taken)
          page = a.block_tables[(size_t)(base + i) * a.table_stride + block];
        if (page_of_others(a, page)) page = -1, error |= AOTO_PAGED_ROW_SHARED;
        a.positions[offset + k] = position;
        a.slots[offset + k] = page < 0 ? -1 : (long long)page * a.page + (position - block * a.page);
      }
    }
    tokens += total;
    taken += total_taken;
    __syncthreads();
  }
  if (error) atomicOr(&s_error, error);
  const int rows = (int)min(tokens, (long long)a.max_tokens);
  if (fill)
    for (int t = rows + tid; t < a.max_tokens; t += 1024) {
      a.positions[t] = 0;
      a.slots[t] = -1;
    }
  __syncthreads();
  if (tid == 0) {
    a.query_start[0] = 0;
    a.free_start_out[0] = taken ? (int)(first_free + min(taken, available)) : start;
    if (s_error && a.error) atomicOr(a.error, s_error);
  }
}

// The tokens' positions and slots after aoto_paged_tables, where they are too many for its one block: block (r, y)
// takes every gridDim.y-th 256 tokens of request r; the blocks of r == requests those behind the last.
extern "C" __global__ __launch_bounds__(256) void aoto_paged_slots(PagedTablesArgs a) {
  const int r = blockIdx.x;
  const int begin = a.query_start[r];
  const int end = r < a.requests ? a.query_start[r + 1] : a.max_tokens;
  const int context = r < a.requests ? a.kv_lens[r] - (end - begin) : 0;
  const int count = r < a.requests ? a.page_counts_out[r] : 0;
  for (int t = begin + blockIdx.y * 256 + threadIdx.x; t < end; t += gridDim.y * 256) {
    int position = 0;
    long long slot = -1;
    if (r < a.requests) {
      position = context + t - begin;
      const int block = position / a.page;
      const int page = block < count ? a.block_tables[(size_t)r * a.table_stride + block] : -1;
      if (aoto::page_of_others(a, page)) {
        if (a.error) atomicOr(a.error, AOTO_PAGED_ROW_SHARED);
      } else if (page >= 0) {
        slot = (long long)page * a.page + (position - block * a.page);
      }
    }
    a.positions[t] = position;
    a.slots[t] = slot;
  }
}

// RoPE of a step's q and k rows, q to a dense [T][Hq][D], the rotated keys and the values to their cache slots.
// A thread takes 8 dims of a head's first half and their partners in the second: two 16-byte loads, four of the
// table rows (f32 arithmetic, one rounding), two stores. Bound by HBM for a chunk (2048 rows of 32 + 16 heads of 128:
// 10.4 us, 4.9 TB/s), by its launch for a decode step (3.1 us).
extern "C" __global__ __launch_bounds__(256) void aoto_paged_rope_append(PagedAppendArgs a) {
  using namespace aoto;
  const int half = a.head_dim >> 1, lanes = half >> 3;
  const int heads = a.query_heads + 2 * a.kv_heads;
  const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
  const int per_token = heads * lanes;
  const long long t = item / per_token;
  if (t >= a.tokens) return;
  const int within = (int)(item - t * per_token);
  const int h = within / lanes, d = 8 * (within - h * lanes);
  const long long slot = a.slots[t], position = a.positions[t];
  const bool stored = slot >= 0 && slot < a.slot_count;
  if (!stored || position < 0 || position >= a.table_rows) {
    if (a.error && slot != -1 && within == 0) atomicOr(a.error, stored ? AOTO_PAGED_BAD_POSITION : AOTO_PAGED_BAD_SLOT);
    return;
  }
  const uint16_t* src = a.qkv + t * a.row_stride + (size_t)h * a.head_dim + d;
  uint4 lo = *reinterpret_cast<const uint4*>(src), hi = *reinterpret_cast<const uint4*>(src + half);
  if (h < a.query_heads + a.kv_heads) {
    const uint16_t* cos_row = a.cos_table + position * a.head_dim + d;
    const uint16_t* sin_row = a.sin_table + position * a.head_dim + d;
    const uint4 c0 = *reinterpret_cast<const uint4*>(cos_row), c1 = *reinterpret_cast<const uint4*>(cos_row + half);
    const uint4 s0 = *reinterpret_cast<const uint4*>(sin_row), s1 = *reinterpret_cast<const uint4*>(sin_row + half);
    const uint32_t la[4] = {lo.x, lo.y, lo.z, lo.w}, ha[4] = {hi.x, hi.y, hi.z, hi.w};
    const uint32_t ca[4] = {c0.x, c0.y, c0.z, c0.w}, cb[4] = {c1.x, c1.y, c1.z, c1.w};
    const uint32_t sa[4] = {s0.x, s0.y, s0.z, s0.w}, sb[4] = {s1.x, s1.y, s1.z, s1.w};
    uint32_t ol[4], oh[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float l0 = bf16_lo(la[i]), l1 = bf16_hi(la[i]), h0 = bf16_lo(ha[i]), h1 = bf16_hi(ha[i]);
      ol[i] = cvt_pk_bf16(l0 * bf16_lo(ca[i]) - h0 * bf16_lo(sa[i]), l1 * bf16_hi(ca[i]) - h1 * bf16_hi(sa[i]));
      oh[i] = cvt_pk_bf16(h0 * bf16_lo(cb[i]) + l0 * bf16_lo(sb[i]), h1 * bf16_hi(cb[i]) + l1 * bf16_hi(sb[i]));
    }
    lo = make_uint4(ol[0], ol[1], ol[2], ol[3]);
    hi = make_uint4(oh[0], oh[1], oh[2], oh[3]);
  }
  uint16_t* dst;
  if (h < a.query_heads) {
    dst = a.q_out + (t * a.query_heads + h) * a.head_dim + d;
  } else {
    const int kh = (h - a.query_heads) % a.kv_heads;
    const long long page = slot / a.page, row = slot - page * a.page;
    dst = (h < a.query_heads + a.kv_heads ? a.keys : a.values) + page * a.page_stride + kh * a.head_stride +
          row * a.slot_stride + d;
  }
  *reinterpret_cast<uint4*>(dst) = lo;
  *reinterpret_cast<uint4*>(dst + half) = hi;
}
