// Host side of the C ABI's paged-cache entry points (include/aoto_hip.h): checks, launch choices, launches.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "aoto_hip.h"
#include "internal.h"
#include "paged_args.h"

namespace {

using aoto::set_error;

bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

template <typename Args, typename... More>
int launch(const char* name, long long gx, long long gy, unsigned block, void* stream, Args& args, More... more) {
  if (gx > 0x7FFFFFFFLL || gy > 65535) return set_error(AOTO_ERR_UNSUPPORTED, "%s: grid too large", name);
  void* params[] = {static_cast<void*>(&args), static_cast<void*>(&more)...};
  const unsigned grid[3] = {(unsigned)gx, (unsigned)gy, 1};
  return aoto::launch_kernel(name, grid, block, stream, params);
}

// Strides and bases of a layer's pages, as every kernel that touches them assumes.
int check_pages(const char* what, const void* keys, const void* values, int64_t page_stride, int64_t head_stride,
                int64_t slot_stride, int pages, int page) {
  if (!keys || !values) return set_error(AOTO_ERR_ARGUMENT, "%s: null pointer", what);
  if (pages <= 0 || page <= 0 || page > (1 << 20)) return set_error(AOTO_ERR_ARGUMENT, "%s: bad cache shape", what);
  if (!aligned(keys, 16) || !aligned(values, 16) || page_stride % 8 || head_stride % 8 || slot_stride % 8)
    return set_error(AOTO_ERR_ARGUMENT, "%s: keys/values 16-byte aligned with strides of multiples of 8", what);
  return AOTO_OK;
}

// Rows of a wide tile of the attention.
constexpr int kWideRows = 128;

struct AttentionPlan {
  int wide_rows;      // of a wide tile, 0 where no chunk of a prompt is among the requests: the narrow instances
  int narrow_rows;    // of a narrow tile (16 or 32)
  int target;         // GPU blocks a kv head among which the keys are dealt, 0 where each takes one tile
  long long units;    // tiles and cuts of them, a kv head, at most
  size_t workspace;
};

// From what the host knows: shapes and the caller's bounds. The lengths are on the GPU.
AttentionPlan attention_plan(int tokens, int requests, int max_blocks, int page, int query_heads, int kv_heads,
                             int head_dim, int max_query_len, int max_kv_len) {
  const int group = query_heads / kv_heads, cus = aoto::device_cu_count();
  const long long rows = (long long)(max_query_len ? std::min(max_query_len, tokens) : tokens) * group;
  const long long some = std::min(requests, tokens);
  auto tiles = [&](int of) { return some + (tokens - some) / std::max(of / group, 1); };
  AttentionPlan p{};
  p.narrow_rows = rows <= 16 || rows > 32 ? 16 : 32;
  p.wide_rows = rows > 32 ? kWideRows : 0;
  p.units = tiles(p.wide_rows ? p.wide_rows : p.narrow_rows);
  const long long full = 2LL * cus;  // GPU blocks that the chip holds at a time
  long long keys = std::min<long long>((long long)max_blocks * page, 1 << 28);
  const long long most = keys / 128 + 8;  // key blocks of a tile
  if (max_kv_len) keys = std::min<long long>(keys, max_kv_len);
  // Not worth the join: narrow tiles of up to 256 keys, wide ones of up to 1024 (512 tokens over themselves: 28 us
  // whole and 35 cut at 128 dims, 19.5 and 24 at 64), wide ones that give every CU a block (32 / 8 heads of 128, 1024
  // tokens over 1 / 1000 / 4000 keys before them: 41 / 62 / 127 us whole, 56 / 76 / 128 cut; 14 / 2 heads of 64, 4096
  // over 2000 / 6000: 113 / 191 and 153 / 231). Those are tiles of equal length; the count says nothing of lengths, so
  // where it ends the cutting (256 single tokens of 8 kv heads, say) one request far longer than the rest ends late.
  if (keys > (p.wide_rows ? 1024 : 256) && 2 * p.units * kv_heads < (p.wide_rows ? 1 : 8) * full &&
      p.units * most < (1 << 30)) {
    p.target = (int)((full + kv_heads - 1) / kv_heads);
    p.units += p.target;
    p.workspace = (size_t)tokens * 16 + (size_t)p.units * kv_heads * (p.wide_rows ? p.wide_rows : p.narrow_rows) *
                                            (head_dim + 2) * sizeof(float);
  }
  return p;
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
  if (!context_lens || !new_lens || !block_tables || !page_counts || (!free_pages && free_count) || !free_start ||
      !query_start || !kv_lens || ((!positions || !slots) && max_tokens) || !page_counts_out || !free_start_out)
    return set_error(AOTO_ERR_ARGUMENT, "paged_tables: null pointer");
  if (requests <= 0 || max_blocks <= 0 || free_count < 0 || page <= 0 || max_tokens < 0 || table_stride < max_blocks)
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
  a.page = page, a.max_tokens = max_tokens;
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
  a.table_keys = max_blocks * page;
  unsigned log2 = 0;
  while ((1u << log2) < (unsigned)page) ++log2;
  a.page_magic = (unsigned)(((1ull << (31 + log2)) + page - 1) / page), a.page_shift = log2 ? log2 - 1 : 0;
  a.narrow_tokens = plan.narrow_rows / (query_heads / kv_heads);
  a.wide_tokens = plan.wide_rows / (query_heads / kv_heads);
  a.target = plan.target, a.least_blocks = 2;
  a.record_rows = plan.wide_rows ? plan.wide_rows : plan.narrow_rows, a.units = (int)std::min(plan.units, 0x3FFFFFFFLL);
  a.joins = static_cast<int*>(workspace);
  a.records = reinterpret_cast<float*>(static_cast<char*>(workspace) + (size_t)tokens * 16);
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
