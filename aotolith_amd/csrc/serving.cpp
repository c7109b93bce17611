// Host side of the C ABI's entry points over a 4-bit paged cache, for its pages' upkeep and for logits
// (include/aoto_hip.h): checks, launch choices, launches.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "aoto_hip.h"
#include "internal.h"
#include "paged_args.h"
#include "paged_host.h"

namespace {

using aoto::aligned;
using aoto::attention_plan;
using aoto::AttentionPlan;
using aoto::kWideRows;
using aoto::launch;
using aoto::set_error;

int check_cache(const char* what, const aoto_mx4_cache* c, int page, int kv_heads, int head_dim, PagedMx4Cache& to) {
  if (!c || !c->keys || !c->values || !c->key_scales || !c->value_scales)
    return set_error(AOTO_ERR_ARGUMENT, "%s: null pointer", what);
  if (c->pages <= 0 || page <= 0 || page > (1 << 20) || kv_heads <= 0 || head_dim <= 0)
    return set_error(AOTO_ERR_ARGUMENT, "%s: bad cache shape", what);
  if (head_dim % 64)
    return set_error(AOTO_ERR_UNSUPPORTED, "%s: head_dim %d is not a multiple of 64", what, head_dim);
  if (!aligned(c->keys, 16) || !aligned(c->values, 16) || c->page_stride % 16 || c->head_stride % 16 ||
      c->slot_stride % 16)
    return set_error(AOTO_ERR_ARGUMENT, "%s: codes 16-byte aligned with strides of multiples of 16", what);
  to.keys = static_cast<uint8_t*>(c->keys), to.values = static_cast<uint8_t*>(c->values);
  to.key_scales = static_cast<uint8_t*>(c->key_scales), to.value_scales = static_cast<uint8_t*>(c->value_scales);
  to.page_stride = c->page_stride, to.head_stride = c->head_stride, to.slot_stride = c->slot_stride;
  to.scale_page_stride = c->scale_page_stride, to.scale_head_stride = c->scale_head_stride;
  to.scale_slot_stride = c->scale_slot_stride;
  return AOTO_OK;
}

// An array of an entry point on pages: `rows` of `bytes` each, `stride` bytes apart. Those that are written are one row
// and have the one input that they may be, at the same address.
struct Array {
  const void* at;
  long long bytes;
  const void* with = nullptr;
  long long rows = 1, stride = 1;
};
Array table_array(const int32_t* tables, int requests, int max_blocks, int64_t stride) {
  return {tables, 4LL * max_blocks, nullptr, requests, 4 * stride};
}
// Whether one row meets any of another array's.
bool meet(const Array& one, const Array& other) {
  if (!one.at || !other.at) return false;
  long long from = (long long)(reinterpret_cast<uintptr_t>(one.at) - reinterpret_cast<uintptr_t>(other.at));
  const long long to = from + one.bytes;
  from = std::max(from, 0LL);
  // the last row that begins before `from` ends behind it, or the next one begins before `to`
  const long long row = std::min(from / other.stride, other.rows - 1);
  return from < to && (from < row * other.stride + other.bytes ||
                       (row + 1 < other.rows && (row + 1) * other.stride < to));
}
template <size_t N, size_t M>
bool overlap(const Array (&written)[N], const Array (&read)[M]) {
  for (size_t i = 0; i < N; ++i) {
    for (const Array& b : read)
      if (meet(written[i], b) && !(written[i].at == b.at && b.at == written[i].with)) return true;
    for (size_t j = 0; j < i; ++j)
      if (meet(written[i], written[j])) return true;
  }
  return false;
}

// GPU blocks of the attention's narrow tiles of 16 rows that a CU holds. A tile's rows are a quarter of what they are
// in bf16, so that two do not ask for enough at a time (345000 keys of 64 requests, 8 kv heads of 128: 88 us with two,
// 84 with three, 93 with four, whose registers are too few).
constexpr int kMx4NarrowBlocks = 3;

// Entries of all block tables up to which the fork's one block enters the pages itself instead of a second launch (8 x
// 64 entries 4.2 us and 6.1 with two launches, 32 x 64 5.5 and 6.0, 64 x 64 7.7 and 6.4, 64 x 256 16.4 and 6.7).
constexpr long long kForkFill = 2048;

// Entries of all block tables (and of the free list) up to which one block releases the pages of a pool of up to
// kPagesFew, or compacts it (paged_pages.h).
constexpr long long kEntriesFew = 4096;

}  // namespace

extern "C" {

int aoto_hip_paged_rope_append_mx4(const void* qkv, int64_t row_stride, const int64_t* positions, const int64_t* slots,
                                   const void* cos_table, const void* sin_table, int table_rows,
                                   const aoto_mx4_cache* cache, int page, int tokens, int query_heads, int kv_heads,
                                   int head_dim, void* q_out, int32_t* error, void* stream) {
  if (!qkv || !positions || !slots || !cos_table || !sin_table || !q_out)
    return set_error(AOTO_ERR_ARGUMENT, "paged_rope_append_mx4: null pointer");
  PagedMx4AppendArgs a{};
  if (int s = check_cache("paged_rope_append_mx4", cache, page, kv_heads, head_dim, a.cache)) return s;
  if (tokens <= 0 || query_heads <= 0 || table_rows <= 0)
    return set_error(AOTO_ERR_ARGUMENT, "paged_rope_append_mx4: bad shape");
  if (!aligned(qkv, 16) || row_stride % 8 || !aligned(cos_table, 16) || !aligned(sin_table, 16) || !aligned(q_out, 16))
    return set_error(AOTO_ERR_ARGUMENT, "paged_rope_append_mx4: rows, tables and q_out 16-byte aligned");
  const long long per_token = (query_heads + 2LL * kv_heads) * (head_dim / 16);
  if (per_token > (1 << 24)) return set_error(AOTO_ERR_UNSUPPORTED, "paged_rope_append_mx4: rows too long");
  a.qkv = static_cast<const uint16_t*>(qkv), a.row_stride = row_stride;
  a.positions = reinterpret_cast<const long long*>(positions), a.slots = reinterpret_cast<const long long*>(slots);
  a.cos_table = static_cast<const uint16_t*>(cos_table), a.sin_table = static_cast<const uint16_t*>(sin_table);
  a.q_out = static_cast<uint16_t*>(q_out), a.error = error;
  a.slot_count = (long long)cache->pages * page, a.tokens = tokens, a.query_heads = query_heads;
  a.kv_heads = kv_heads, a.head_dim = head_dim, a.page = page, a.table_rows = table_rows;
  return launch("aoto_paged_rope_append_mx4", (tokens * per_token + 255) / 256, 1, 256, stream, a);
}

int aoto_hip_paged_unpack_mx4(const aoto_mx4_cache* cache, int page, int kv_heads, int head_dim, void* keys_out,
                              void* values_out, void* stream) {
  if (!keys_out || !values_out) return set_error(AOTO_ERR_ARGUMENT, "paged_unpack_mx4: null pointer");
  PagedMx4UnpackArgs a{};
  if (int s = check_cache("paged_unpack_mx4", cache, page, kv_heads, head_dim, a.cache)) return s;
  if (!aligned(keys_out, 16) || !aligned(values_out, 16))
    return set_error(AOTO_ERR_ARGUMENT, "paged_unpack_mx4: outputs 16-byte aligned");
  a.keys_out = static_cast<uint16_t*>(keys_out), a.values_out = static_cast<uint16_t*>(values_out);
  a.page = page, a.kv_heads = kv_heads, a.head_dim = head_dim;
  const long long rows = (long long)kv_heads * page;
  if (rows >= (1 << 24) || head_dim > (1 << 10))
    return set_error(AOTO_ERR_UNSUPPORTED, "paged_unpack_mx4: pages too large");
  return launch("aoto_paged_unpack_mx4", cache->pages, (rows * (head_dim / 16) + 255) / 256, 256, stream, a);
}

size_t aoto_hip_paged_attention_mx4_workspace(int tokens, int requests, int max_blocks, int page, int query_heads,
                                              int kv_heads, int head_dim, int max_query_len, int max_kv_len) {
  if (tokens <= 0 || requests <= 0 || max_blocks <= 0 || page <= 0 || query_heads <= 0 || kv_heads <= 0 ||
      query_heads % kv_heads || head_dim <= 0 || max_query_len < 0 || max_kv_len < 0)
    return 0;
  return attention_plan(tokens, requests, max_blocks, page, query_heads, kv_heads, head_dim, max_query_len, max_kv_len,
                        kMx4NarrowBlocks)
      .workspace;
}

int aoto_hip_paged_attention_mx4(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                 const aoto_mx4_cache* cache, int page, const int32_t* block_tables,
                                 int64_t table_stride, int max_blocks, const int32_t* query_start,
                                 const int32_t* kv_lens, int tokens, int requests, int query_heads, int kv_heads,
                                 int head_dim, int causal, float scale, int max_query_len, int max_kv_len,
                                 void* workspace, void* out, void* stream) {
  if (!q || !block_tables || !query_start || !kv_lens || !out)
    return set_error(AOTO_ERR_ARGUMENT, "paged_attention_mx4: null pointer");
  PagedMx4AttentionArgs args{};
  if (int s = check_cache("paged_attention_mx4", cache, page, kv_heads, head_dim, args.cache)) return s;
  if (tokens <= 0 || requests <= 0 || max_blocks <= 0 || query_heads <= 0 || query_heads % kv_heads ||
      table_stride < max_blocks || max_query_len < 0 || max_kv_len < 0)
    return set_error(AOTO_ERR_ARGUMENT, "paged_attention_mx4: bad shape");
  if (head_dim != 64 && head_dim != 128)
    return set_error(AOTO_ERR_UNSUPPORTED, "paged_attention_mx4: head_dim %d (64 or 128)", head_dim);
  if (!aligned(q, 16) || q_token_stride % 8 || q_head_stride % 8 || !aligned(out, 16))
    return set_error(AOTO_ERR_ARGUMENT, "paged_attention_mx4: q and out 16-byte aligned, strides of multiples of 8");
  if ((long long)max_blocks * page > (1 << 28))
    return set_error(AOTO_ERR_UNSUPPORTED, "paged_attention_mx4: block tables of more than 2^28 keys");
  for (const int64_t* stride : {&cache->page_stride, &cache->scale_page_stride})
    if (stride[0] < 0 || stride[0] > 0xFFFFFFFFLL || stride[2] < 0 || stride[2] > 0x3FFFFFFFLL / page)
      return set_error(AOTO_ERR_UNSUPPORTED, "paged_attention_mx4: pages 2^32 bytes apart, or rows 2^30");
  if (!(scale > 0.f) || !std::isfinite(scale))
    return set_error(AOTO_ERR_ARGUMENT, "paged_attention_mx4: scale %g is not a positive number", (double)scale);
  if (query_heads / kv_heads > kWideRows)
    return set_error(AOTO_ERR_UNSUPPORTED, "paged_attention_mx4: %d query heads a kv head (at most %d)",
                     query_heads / kv_heads, kWideRows);
  const AttentionPlan plan = attention_plan(tokens, requests, max_blocks, page, query_heads, kv_heads, head_dim,
                                            max_query_len, max_kv_len, kMx4NarrowBlocks);
  if (plan.workspace && (!workspace || !aligned(workspace, 16)))
    return set_error(AOTO_ERR_ARGUMENT, "paged_attention_mx4: needs a 16-byte aligned workspace of %zu bytes",
                     plan.workspace);
  PagedAttentionArgs& a = args.base;
  a.q = static_cast<const uint16_t*>(q), a.block_tables = block_tables, a.query_start = query_start;
  a.kv_lens = kv_lens, a.out = static_cast<uint16_t*>(out), a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride, a.table_stride = table_stride, a.tokens = tokens, a.requests = requests;
  a.pages = cache->pages, a.page = page, a.query_heads = query_heads, a.kv_heads = kv_heads;
  a.causal = causal != 0, a.scale = scale;
  aoto::attention_launch(plan, max_blocks, workspace, a);
  // Tiles not cut, a chunk's longest first, two GPU blocks a CU: the second ones shortest first, so that a CU's two are
  // as long together as another's (one request of 32 / 8 heads of 128: 2048 tokens over 6000 keys 236 -> 229 us, 4096
  // over themselves 160 -> 149; 14 / 2 of 64, both sides in turn, five calls after a pause: 4096 over 2000 134.9 ->
  // 134.3, 8192 over themselves 228.0 -> 219.9, three of 2000 62.7 -> 61.6; 32 / 8 of 64, 2048 over 6000: 207 -> 202).
  // What comes after them goes to whoever ends first.
  if (!plan.target && plan.wide_rows) {
    args.turn_from = std::max(1, aoto::device_cu_count() / kv_heads);
    args.turn_to = (int)std::min(plan.units, 2LL * args.turn_from);
  }
  char name[64];
  snprintf(name, sizeof(name), "aoto_paged_attention_mx4_d%d_%s", head_dim,
           plan.wide_rows ? "w" : plan.narrow_rows == 16 ? "n1" : "n2");
  if (int s = launch(name, (plan.target ? plan.target : plan.units) * kv_heads, 1, 256, stream, args)) return s;
  if (!plan.target) return AOTO_OK;
  return launch(head_dim == 64 ? "aoto_paged_attention_join_d64" : "aoto_paged_attention_join_d128",
                ((long long)tokens * query_heads + 3) / 4, 1, 256, stream, a);
}

int aoto_hip_paged_fork(const int32_t* parents, const int32_t* context_lens, int32_t* block_tables,
                        int64_t table_stride, const int32_t* page_counts, int32_t* shares, const int32_t* free_pages,
                        const int32_t* free_start, int requests, int max_blocks, int free_count, int pages, int page,
                        int32_t* context_lens_out, int32_t* page_counts_out, int32_t* free_start_out, int32_t* source,
                        int32_t* target, int32_t* plan, int32_t* error, void* stream) {
  if (!parents || !context_lens || !block_tables || !page_counts || !shares || (!free_pages && free_count) ||
      !free_start || !context_lens_out || !page_counts_out || !free_start_out || !source || !target || !plan)
    return set_error(AOTO_ERR_ARGUMENT, "paged_fork: null pointer");
  if (requests <= 0 || max_blocks <= 0 || free_count < 0 || pages <= 0 || page <= 0 || table_stride < max_blocks)
    return set_error(AOTO_ERR_ARGUMENT, "paged_fork: bad shape");
  if (max_blocks > (1 << 20) || page > (1 << 20) || requests > (1 << 28))
    return set_error(AOTO_ERR_UNSUPPORTED, "paged_fork: at most 2^20 blocks a request and tokens a page");
  // what is written is read by other threads than those that read the inputs
  const long long row = 4LL * requests;
  const Array written[] = {{context_lens_out, row, context_lens}, {page_counts_out, row, page_counts},
                           {free_start_out, 4, free_start}, {source, row}, {target, row}, {plan, 2 * row}};
  const Array read[] = {{parents, row}, {context_lens, row}, {page_counts, row}, {free_start, 4}, {error, 4},
                        {shares, 4LL * pages}, {free_pages, 4LL * free_count},
                        table_array(block_tables, requests, max_blocks, table_stride)};
  if (overlap(written, read)) return set_error(AOTO_ERR_ARGUMENT, "paged_fork: its outputs overlap other arrays");
  PagedForkArgs a{};
  a.parents = parents, a.context_lens = context_lens, a.block_tables = block_tables, a.page_counts = page_counts;
  a.shares = shares, a.free_pages = free_pages, a.free_start = free_start, a.context_lens_out = context_lens_out;
  a.page_counts_out = page_counts_out, a.free_start_out = free_start_out, a.source = source, a.target = target;
  a.plan = plan, a.error = error, a.table_stride = table_stride, a.requests = requests, a.max_blocks = max_blocks;
  a.free_count = free_count, a.pages = pages, a.page = page;
  const int fill = (long long)requests * max_blocks <= kForkFill;
  if (int s = launch("aoto_paged_fork", 1, 1, 1024, stream, a, fill)) return s;
  if (fill) return AOTO_OK;
  return launch("aoto_paged_share", requests, 1, 256, stream, a);
}

int aoto_hip_paged_release(const int32_t* keep_lens, const int32_t* block_tables, int64_t table_stride,
                           const int32_t* page_counts, int32_t* shares, int32_t* free_pages,
                           const int32_t* free_start, int requests, int max_blocks, int free_count, int pages,
                           int page, int32_t* page_counts_out, int32_t* free_start_out, int32_t* scratch,
                           int32_t* error, void* stream) {
  if (!keep_lens || !block_tables || !page_counts || !shares || (!free_pages && free_count) || !free_start ||
      !page_counts_out || !free_start_out || !scratch)
    return set_error(AOTO_ERR_ARGUMENT, "paged_release: null pointer");
  if (requests <= 0 || max_blocks <= 0 || free_count < 0 || pages <= 0 || page <= 0 || table_stride < max_blocks)
    return set_error(AOTO_ERR_ARGUMENT, "paged_release: bad shape");
  if (max_blocks > (1 << 20) || page > (1 << 20) || pages > (1 << 30))
    return set_error(AOTO_ERR_UNSUPPORTED,
                     "paged_release: at most 2^20 blocks a request and tokens a page, 2^30 pages");
  PagedReleaseArgs a{};
  a.keep_lens = keep_lens, a.block_tables = block_tables, a.page_counts = page_counts, a.shares = shares;
  a.free_pages = free_pages, a.free_start = free_start, a.page_counts_out = page_counts_out;
  a.free_start_out = free_start_out, a.error = error, a.table_stride = table_stride, a.requests = requests;
  a.max_blocks = max_blocks, a.free_count = free_count, a.pages = pages, a.page = page, a.scratch = scratch;
  if (pages <= kPagesFew && (long long)requests * max_blocks <= kEntriesFew && free_count <= kEntriesFew)
    return launch("aoto_paged_release_few", 1, 1, 1024, stream, a);
  const int chunks = (pages - 1) / kPageChunk + 1;
  a.list_blocks = (int)std::min(256LL, std::max(1LL, (free_count + 255LL) / 256));
  if (int s = launch("aoto_paged_drop", (long long)requests + a.list_blocks, 1, 256, stream, a)) return s;
  if (int s = launch("aoto_paged_gone", chunks, 1, 256, stream, a)) return s;
  return launch("aoto_paged_reclaim", chunks, 1, 256, stream, a);
}

int aoto_hip_paged_compact(int32_t* block_tables, int64_t table_stride, const int32_t* page_counts, int32_t* shares,
                           int32_t* free_pages, const int32_t* free_start, int requests, int max_blocks,
                           int free_count, int pages, int32_t* source, int32_t* target, int32_t* count,
                           int32_t* state, int32_t* error, void* stream) {
  if (!block_tables || !page_counts || !shares || (!free_pages && free_count) || !free_start || !source || !target ||
      !count || !state)
    return set_error(AOTO_ERR_ARGUMENT, "paged_compact: null pointer");
  if (requests <= 0 || max_blocks <= 0 || free_count < 0 || pages <= 0 || table_stride < max_blocks)
    return set_error(AOTO_ERR_ARGUMENT, "paged_compact: bad shape");
  if (max_blocks > (1 << 20) || pages > (1 << 30) || requests > (1 << 28))
    return set_error(AOTO_ERR_UNSUPPORTED, "paged_compact: at most 2^20 blocks a request, 2^30 pages");
  const long long all = 4LL * pages;
  const Array written[] = {{source, all}, {target, all}, {count, 4}, {state, all}};
  const Array read[] = {{page_counts, 4LL * requests}, {free_start, 4}, {error, 4}, {shares, all},
                        {free_pages, 4LL * free_count}, table_array(block_tables, requests, max_blocks, table_stride)};
  if (overlap(written, read)) return set_error(AOTO_ERR_ARGUMENT, "paged_compact: its outputs overlap other arrays");
  PagedCompactArgs a{};
  a.block_tables = block_tables, a.page_counts = page_counts, a.shares = shares, a.free_pages = free_pages;
  a.free_start = free_start, a.source = source, a.target = target, a.count = count, a.state = state, a.error = error;
  a.table_stride = table_stride, a.requests = requests, a.max_blocks = max_blocks, a.free_count = free_count;
  a.pages = pages;
  if (pages <= kPagesFew && (long long)requests * max_blocks <= kEntriesFew && free_count <= kEntriesFew)
    return launch("aoto_paged_compact_few", 1, 1, 1024, stream, a);
  if (int s = launch("aoto_paged_clear", (pages + 255LL) / 256, 1, 256, stream, a)) return s;
  a.list_blocks = (int)std::min(256LL, std::max(1LL, (free_count + 255LL) / 256));
  if (int s = launch("aoto_paged_mark", (long long)requests + a.list_blocks, 1, 256, stream, a)) return s;
  if (int s = launch("aoto_paged_moves", 1, 1, 1024, stream, a)) return s;
  return launch("aoto_paged_remap", requests, 1, 256, stream, a);
}

int aoto_hip_paged_copy(const aoto_page_tensor* tensors, int tensor_count, int pages, const int32_t* source,
                        const int32_t* target, int pairs, const int32_t* count, int32_t* error, void* stream) {
  if (!tensors || !source || !target) return set_error(AOTO_ERR_ARGUMENT, "paged_copy: null pointer");
  if (tensor_count <= 0 || pages <= 0 || pairs <= 0) return set_error(AOTO_ERR_ARGUMENT, "paged_copy: bad shape");
  // all of them looked at before the first launch: a refused call has copied nothing
  for (const bool run : {false, true})
    for (int from = 0; from < tensor_count; from += kPagedCopyTensors) {
      PagedCopyArgs a{};
      a.source = source, a.target = target, a.count = count, a.error = from ? nullptr : error;
      a.pairs = pairs, a.pages = pages, a.tensors = std::min(kPagedCopyTensors, tensor_count - from), a.wide = 1;
      long long planes = 0;
      for (int i = 0; i < a.tensors; ++i) {
        const aoto_page_tensor& t = tensors[from + i];
        if (!t.data || t.planes <= 0 || t.page_bytes <= 0)
          return set_error(AOTO_ERR_ARGUMENT, "paged_copy: tensor %d: bad shape", from + i);
        const long long chunks = (t.page_bytes - 1) / kPagedCopyChunk + 1;
        if (chunks > (1 << 20)) return set_error(AOTO_ERR_UNSUPPORTED, "paged_copy: pages of more than 16 GB");
        a.at[i].base = static_cast<uint8_t*>(t.data), a.at[i].page_stride = t.page_stride;
        a.at[i].plane_stride = t.plane_stride, a.at[i].bytes = t.page_bytes, a.at[i].first = (int)planes;
        a.at[i].chunks = (int)chunks, a.chunks = std::max(a.chunks, (int)chunks);
        if (!aligned(t.data, 16) || t.page_stride % 16 || t.plane_stride % 16 || t.page_bytes % 16) a.wide = 0;
        planes += t.planes;
        if (planes > (1 << 20)) return set_error(AOTO_ERR_UNSUPPORTED, "paged_copy: more than 2^20 planes");
      }
      a.planes = (int)planes;
      if (planes * a.chunks > 0x7FFFFFFFLL) return set_error(AOTO_ERR_UNSUPPORTED, "paged_copy: pages too large");
      const long long items = planes * a.chunks * (long long)pairs;
      a.blocks = (int)std::min(items, 8LL * aoto::device_cu_count());  // what the chip holds at a time
      if (run)
        if (int s = launch("aoto_paged_copy", a.blocks, 1, 256, stream, a)) return s;
    }
  return AOTO_OK;
}

int aoto_hip_adjust_logits(const void* logits, int logits_f32, int64_t row_stride, int rows, int vocab, int requests,
                           const aoto_adjustments* adjust, void* out, int64_t out_stride, void* stream) {
  if (!logits || !adjust || !out) return set_error(AOTO_ERR_ARGUMENT, "adjust_logits: null pointer");
  if (rows <= 0 || vocab <= 0 || requests <= 0) return set_error(AOTO_ERR_ARGUMENT, "adjust_logits: bad shape");
  const aoto_adjustments& j = *adjust;
  if (j.history_len < 0 || j.drafts < 0 || j.biases < 0 || (j.history_len && !j.history) ||
      (j.drafts && !j.draft_tokens) || (j.biases && (!j.bias_tokens || !j.bias_values)))
    return set_error(AOTO_ERR_ARGUMENT, "adjust_logits: null pointer");
  if (vocab > 1 << 30) return set_error(AOTO_ERR_UNSUPPORTED, "adjust_logits: %d tokens (at most 2^30)", vocab);
  if (j.history_len >= 1 << 30) return set_error(AOTO_ERR_UNSUPPORTED, "adjust_logits: texts of 2^30 tokens");
  if (requests > 65535) return set_error(AOTO_ERR_UNSUPPORTED, "adjust_logits: %d requests (at most 65535)", requests);
  const size_t size = logits_f32 ? 4 : 2;
  if (!aligned(logits, size) || !aligned(out, size))
    return set_error(AOTO_ERR_ARGUMENT, "adjust_logits: logits aligned to their type");
  if (rows > 1 && out_stride < vocab) return set_error(AOTO_ERR_ARGUMENT, "adjust_logits: rows of out overlap");
  if (rows > 1 && out == logits && out_stride != row_stride)
    return set_error(AOTO_ERR_ARGUMENT, "adjust_logits: out is logits at another stride");
  AdjustArgs a{};
  a.logits = logits, a.out = out, a.query_start = j.query_start;
  a.history = reinterpret_cast<const long long*>(j.history), a.history_lens = j.history_lens;
  a.prompt_lens = j.prompt_lens, a.draft_tokens = reinterpret_cast<const long long*>(j.draft_tokens);
  a.repetition = j.repetition, a.presence = j.presence, a.frequency = j.frequency;
  a.bias_tokens = reinterpret_cast<const long long*>(j.bias_tokens), a.bias_values = j.bias_values;
  a.allowed = reinterpret_cast<const uint8_t*>(j.allowed), a.row_stride = row_stride, a.out_stride = out_stride;
  a.history_stride = j.history_stride, a.draft_stride = j.draft_stride, a.bias_stride = j.bias_stride;
  a.value_stride = j.value_stride, a.allowed_stride = 4 * j.allowed_stride;
  a.rows = rows, a.requests = requests, a.vocab = vocab, a.history_len = j.history_len, a.drafts = j.drafts;
  a.biases = j.biases;
  // tokens a thread, by the logits that there are room for; how long the texts are is known on the GPU alone (adjust.h)
  const long long most = (long long)rows * vocab;
  const int per = most <= 1 << 21 ? 2 : logits_f32 || most <= 1 << 23 ? 4 : 8, threads = per == 2 ? 512 : 256;
  char name[64];
  snprintf(name, sizeof(name), "aoto_adjust_logits_%s_%d", logits_f32 ? "f32" : "bf16", per);
  return launch(name, (vocab - 1) / (per * threads) + 1, requests, threads, stream, a);
}

}  // extern "C"
