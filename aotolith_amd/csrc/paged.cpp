// Host side of the C ABI's paged-cache entry points (include/aoto_hip.h): checks, launch choices, launches.
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

// Strides and bases of a layer's pages, as every kernel that touches them assumes.
int check_pages(const char* what, const void* keys, const void* values, int64_t page_stride, int64_t head_stride,
                int64_t slot_stride, int pages, int page) {
  if (!keys || !values) return set_error(AOTO_ERR_ARGUMENT, "%s: null pointer", what);
  if (pages <= 0 || page <= 0 || page > (1 << 20)) return set_error(AOTO_ERR_ARGUMENT, "%s: bad cache shape", what);
  if (!aligned(keys, 16) || !aligned(values, 16) || page_stride % 8 || head_stride % 8 || slot_stride % 8)
    return set_error(AOTO_ERR_ARGUMENT, "%s: keys/values 16-byte aligned with strides of multiples of 8", what);
  return AOTO_OK;
}

// Tokens up to which the tables' one block writes the maps itself: a second launch costs more than it saves.
constexpr int kTablesFill = 4096;

}  // namespace

extern "C" {

int aoto_hip_paged_tables(const int32_t* context_lens, const int32_t* new_lens, int32_t* block_tables,
                          int64_t table_stride, const int32_t* page_counts, const int32_t* free_pages,
                          const int32_t* free_start, int requests, int max_blocks, int free_count, int page,
                          int max_tokens, int32_t* query_start, int32_t* kv_lens, int64_t* positions, int64_t* slots,
                          int32_t* page_counts_out, int32_t* free_start_out, int32_t* error, void* stream) {
  return aoto_hip_paged_tables_shared(context_lens, new_lens, block_tables, table_stride, page_counts, free_pages,
                                      free_start, nullptr, requests, max_blocks, free_count, 0, page, max_tokens,
                                      query_start, kv_lens, positions, slots, page_counts_out, free_start_out, error,
                                      stream);
}

int aoto_hip_paged_tables_shared(const int32_t* context_lens, const int32_t* new_lens, int32_t* block_tables,
                                 int64_t table_stride, const int32_t* page_counts, const int32_t* free_pages,
                                 const int32_t* free_start, const int32_t* shares, int requests, int max_blocks,
                                 int free_count, int pages, int page, int max_tokens, int32_t* query_start,
                                 int32_t* kv_lens, int64_t* positions, int64_t* slots, int32_t* page_counts_out,
                                 int32_t* free_start_out, int32_t* error, void* stream) {
  if (!context_lens || !new_lens || !block_tables || !page_counts || (!free_pages && free_count) || !free_start ||
      !query_start || !kv_lens || ((!positions || !slots) && max_tokens) || !page_counts_out || !free_start_out)
    return set_error(AOTO_ERR_ARGUMENT, "paged_tables: null pointer");
  if (requests <= 0 || max_blocks <= 0 || free_count < 0 || page <= 0 || max_tokens < 0 || table_stride < max_blocks ||
      pages < (shares ? 1 : 0))
    return set_error(AOTO_ERR_ARGUMENT, "paged_tables: bad shape");
  if (max_blocks > (1 << 20) || page > (1 << 20) || max_tokens >= (1 << 30))
    return set_error(AOTO_ERR_UNSUPPORTED,
                     "paged_tables: at most 2^20 blocks a request and tokens a page, 2^30 - 1 rows");
  PagedTablesArgs a{};
  a.context_lens = context_lens, a.new_lens = new_lens, a.block_tables = block_tables, a.page_counts = page_counts;
  a.free_pages = free_pages, a.free_start = free_start, a.query_start = query_start, a.kv_lens = kv_lens;
  a.positions = reinterpret_cast<long long*>(positions), a.slots = reinterpret_cast<long long*>(slots);
  a.page_counts_out = page_counts_out, a.free_start_out = free_start_out, a.error = error;
  a.table_stride = table_stride, a.requests = requests, a.max_blocks = max_blocks, a.free_count = free_count;
  a.page = page, a.max_tokens = max_tokens, a.shares = shares, a.pages = pages;
  const int fill = max_tokens <= kTablesFill;
  if (int s = launch("aoto_paged_tables", 1, 1, 1024, stream, a, fill)) return s;
  if (fill) return AOTO_OK;
  const long long y = std::min<long long>(16, std::max<long long>(1, max_tokens / 1024));
  return launch("aoto_paged_slots", requests + 1LL, y, 256, stream, a);
}

int aoto_hip_paged_rope_append(const void* qkv, int64_t row_stride, const int64_t* positions, const int64_t* slots,
                               const void* cos_table, const void* sin_table, int table_rows, void* keys, void* values,
                               int64_t page_stride, int64_t head_stride, int64_t slot_stride, int pages, int page,
                               int tokens, int query_heads, int kv_heads, int head_dim, void* q_out, int32_t* error,
                               void* stream) {
  if (!qkv || !positions || !slots || !cos_table || !sin_table || !q_out)
    return set_error(AOTO_ERR_ARGUMENT, "paged_rope_append: null pointer");
  if (int s = check_pages("paged_rope_append", keys, values, page_stride, head_stride, slot_stride, pages, page))
    return s;
  if (tokens <= 0 || query_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || table_rows <= 0)
    return set_error(AOTO_ERR_ARGUMENT, "paged_rope_append: bad shape");
  if (head_dim % 16)
    return set_error(AOTO_ERR_UNSUPPORTED, "paged_rope_append: head_dim %d is not a multiple of 16", head_dim);
  if (!aligned(qkv, 16) || row_stride % 8 || !aligned(cos_table, 16) || !aligned(sin_table, 16) || !aligned(q_out, 16))
    return set_error(AOTO_ERR_ARGUMENT, "paged_rope_append: rows, tables and q_out 16-byte aligned");
  PagedAppendArgs a{};
  a.qkv = static_cast<const uint16_t*>(qkv);
  a.positions = reinterpret_cast<const long long*>(positions), a.slots = reinterpret_cast<const long long*>(slots);
  a.cos_table = static_cast<const uint16_t*>(cos_table), a.sin_table = static_cast<const uint16_t*>(sin_table);
  a.keys = static_cast<uint16_t*>(keys), a.values = static_cast<uint16_t*>(values);
  a.q_out = static_cast<uint16_t*>(q_out), a.error = error;
  a.row_stride = row_stride, a.page_stride = page_stride, a.head_stride = head_stride, a.slot_stride = slot_stride;
  a.slot_count = (long long)pages * page, a.tokens = tokens, a.query_heads = query_heads, a.kv_heads = kv_heads;
  a.head_dim = head_dim, a.page = page, a.table_rows = table_rows;
  const long long items = (long long)tokens * (query_heads + 2LL * kv_heads) * (head_dim / 16);
  return launch("aoto_paged_rope_append", (items + 255) / 256, 1, 256, stream, a);
}

size_t aoto_hip_paged_attention_workspace(int tokens, int requests, int max_blocks, int page, int query_heads,
                                          int kv_heads, int head_dim, int max_query_len, int max_kv_len) {
  if (tokens <= 0 || requests <= 0 || max_blocks <= 0 || page <= 0 || query_heads <= 0 || kv_heads <= 0 ||
      query_heads % kv_heads || head_dim <= 0 || max_query_len < 0 || max_kv_len < 0)
    return 0;
  return attention_plan(tokens, requests, max_blocks, page, query_heads, kv_heads, head_dim, max_query_len, max_kv_len)
      .workspace;
}

int aoto_hip_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* keys,
                             const void* values, int64_t page_stride, int64_t head_stride, int64_t slot_stride,
                             int pages, int page, const int32_t* block_tables, int64_t table_stride, int max_blocks,
                             const int32_t* query_start, const int32_t* kv_lens, int tokens, int requests,
                             int query_heads, int kv_heads, int head_dim, int causal, float scale, int max_query_len,
                             int max_kv_len, void* workspace, void* out, void* stream) {
  if (!q || !block_tables || !query_start || !kv_lens || !out)
    return set_error(AOTO_ERR_ARGUMENT, "paged_attention: null pointer");
  if (int s = check_pages("paged_attention", keys, values, page_stride, head_stride, slot_stride, pages, page))
    return s;
  if (tokens <= 0 || requests <= 0 || max_blocks <= 0 || query_heads <= 0 || kv_heads <= 0 ||
      query_heads % kv_heads || table_stride < max_blocks || max_query_len < 0 || max_kv_len < 0)
    return set_error(AOTO_ERR_ARGUMENT, "paged_attention: bad shape");
  if (head_dim != 64 && head_dim != 128)
    return set_error(AOTO_ERR_UNSUPPORTED, "paged_attention: head_dim %d (64 or 128)", head_dim);
  if (!aligned(q, 16) || q_token_stride % 8 || q_head_stride % 8 || !aligned(out, 16))
    return set_error(AOTO_ERR_ARGUMENT, "paged_attention: q and out 16-byte aligned, strides of multiples of 8");
  if ((long long)max_blocks * page > (1 << 28))
    return set_error(AOTO_ERR_UNSUPPORTED, "paged_attention: block tables of more than 2^28 keys");
  if (page_stride < 0 || page_stride > 0xFFFFFFFFLL || slot_stride < 0 || slot_stride > 0x3FFFFFFFLL / page)
    return set_error(AOTO_ERR_UNSUPPORTED, "paged_attention: pages of more than 2^32 elements, or rows 2^30 apart");
  if (!(scale > 0.f) || !std::isfinite(scale))
    return set_error(AOTO_ERR_ARGUMENT, "paged_attention: scale %g is not a positive number", (double)scale);
  if (query_heads / kv_heads > kWideRows)
    return set_error(AOTO_ERR_UNSUPPORTED, "paged_attention: %d query heads a kv head (at most %d)",
                     query_heads / kv_heads, kWideRows);
  const AttentionPlan plan = attention_plan(tokens, requests, max_blocks, page, query_heads, kv_heads, head_dim,
                                            max_query_len, max_kv_len);
  if (plan.workspace && (!workspace || !aligned(workspace, 16)))
    return set_error(AOTO_ERR_ARGUMENT, "paged_attention: needs a 16-byte aligned workspace of %zu bytes",
                     plan.workspace);
  PagedAttentionArgs a{};
  a.q = static_cast<const uint16_t*>(q), a.keys = static_cast<const uint16_t*>(keys);
  a.values = static_cast<const uint16_t*>(values), a.block_tables = block_tables, a.query_start = query_start;
  a.kv_lens = kv_lens, a.out = static_cast<uint16_t*>(out), a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride, a.page_stride = page_stride, a.head_stride = head_stride;
  a.slot_stride = slot_stride, a.table_stride = table_stride, a.tokens = tokens, a.requests = requests;
  a.pages = pages, a.page = page, a.query_heads = query_heads, a.kv_heads = kv_heads;
  a.causal = causal != 0, a.scale = scale;
  aoto::attention_launch(plan, max_blocks, workspace, a);
  char name[64];
  snprintf(name, sizeof(name), "aoto_paged_attention_d%d_%s", head_dim,
           plan.wide_rows ? "w" : plan.narrow_rows == 16 ? "n1" : "n2");
  if (int s = launch(name, (plan.target ? plan.target : plan.units) * kv_heads, 1, 256, stream, a)) return s;
  if (!plan.target) return AOTO_OK;
  return launch(head_dim == 64 ? "aoto_paged_attention_join_d64" : "aoto_paged_attention_join_d128",
                ((long long)tokens * query_heads + 3) / 4, 1, 256, stream, a);
}

size_t aoto_hip_verify_draft_workspace(int requests, int drafts, int vocab) {
  if (requests <= 0 || drafts < 0 || vocab <= 0) return 0;
  const size_t chunks = ((size_t)vocab + kVerifyChunk - 1) / kVerifyChunk;
  return (size_t)requests *
         (chunks * ((2 * (size_t)drafts + 1) * kVerifyChunkBytes + sizeof(double)) + kVerifyLawBytes);
}

int aoto_hip_verify_draft(const void* logits, int logits_f32, int64_t row_stride, int rows, int vocab,
                          const int64_t* draft_tokens, const void* draft_logits, int64_t draft_request_stride,
                          int64_t draft_row_stride, const int32_t* query_start, const float* uniforms,
                          const float* temperature, int requests, int drafts, void* workspace, int64_t* tokens_out,
                          int32_t* accepted, void* stream) {
  if (!logits || (!draft_tokens && drafts) || !query_start || (temperature && !uniforms) || !workspace || !tokens_out ||
      !accepted)
    return set_error(AOTO_ERR_ARGUMENT, "verify_draft: null pointer");
  if (rows <= 0 || vocab <= 0 || requests <= 0 || drafts < 0)
    return set_error(AOTO_ERR_ARGUMENT, "verify_draft: bad shape");
  if (drafts > 62) return set_error(AOTO_ERR_UNSUPPORTED, "verify_draft: %d drafts a request (at most 62)", drafts);
  if (vocab > 1 << 30) return set_error(AOTO_ERR_UNSUPPORTED, "verify_draft: %d tokens (at most 2^30)", vocab);
  const size_t size = logits_f32 ? 4 : 2;
  if (!aligned(logits, size) || (draft_logits && !aligned(draft_logits, size)) || !aligned(workspace, 8))
    return set_error(AOTO_ERR_ARGUMENT, "verify_draft: logits aligned to their type, workspace to 8 bytes");
  VerifyArgs a{};
  a.logits = logits, a.draft_logits = drafts ? draft_logits : nullptr;
  a.draft_tokens = reinterpret_cast<const long long*>(draft_tokens), a.query_start = query_start;
  a.uniforms = uniforms, a.temperature = temperature, a.tokens_out = reinterpret_cast<long long*>(tokens_out);
  a.accepted = accepted, a.workspace = workspace, a.row_stride = row_stride;
  a.draft_request_stride = draft_request_stride, a.draft_row_stride = draft_row_stride, a.rows = rows;
  a.requests = requests, a.drafts = drafts, a.vocab = vocab, a.chunks = (vocab - 1) / kVerifyChunk + 1;
  a.judged = temperature && a.draft_logits ? 2 * drafts + 1 : drafts + 1;
  if ((long long)requests * a.judged > 65535)
    return set_error(AOTO_ERR_UNSUPPORTED, "verify_draft: %d requests of %d drafts", requests, drafts);
  if (int s = launch(logits_f32 ? "aoto_verify_stats_f32" : "aoto_verify_stats_bf16", (a.chunks + 3) / 4,
                     (long long)requests * a.judged, 256, stream, a))
    return s;
  if (!temperature || !a.draft_logits)
    return launch(logits_f32 ? "aoto_verify_follow_f32" : "aoto_verify_follow_bf16", requests, 1, kVerifyChunk / 8,
                  stream, a);
  if (int s = launch(logits_f32 ? "aoto_verify_law_f32" : "aoto_verify_law_bf16", requests, 1, 256, stream, a))
    return s;
  if (int s = launch(logits_f32 ? "aoto_verify_mass_f32" : "aoto_verify_mass_bf16", a.chunks, requests, 256, stream, a))
    return s;
  return launch(logits_f32 ? "aoto_verify_pick_f32" : "aoto_verify_pick_bf16", requests, 1, kVerifyChunk / 8, stream,
                a);
}

}  // extern "C"
