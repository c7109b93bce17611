// Arguments of the paged-cache kernels, shared by host and device.
#pragma once

#include <stdint.h>

#include "aoto_hip.h"

// Longer contexts are taken as this long: with fewer than 2^30 rows a step, lengths stay within 31 bits.
constexpr int kPagedMostContext = 1 << 30;

struct PagedTablesArgs {
  const int* context_lens;
  const int* new_lens;
  int* block_tables;
  const int* page_counts;
  const int* free_pages;
  const int* free_start;
  int* query_start;
  int* kv_lens;
  long long* positions;
  long long* slots;
  int* page_counts_out;
  int* free_start_out;
  int* error;
  long long table_stride;
  int requests, max_blocks, free_count, page, max_tokens;
};

struct PagedAppendArgs {
  const uint16_t* qkv;
  const long long* positions;
  const long long* slots;
  const uint16_t* cos_table;
  const uint16_t* sin_table;
  uint16_t* keys;
  uint16_t* values;
  uint16_t* q_out;
  int* error;
  long long row_stride, page_stride, head_stride, slot_stride, slot_count;
  int tokens, query_heads, kv_heads, head_dim, page, table_rows;
};

struct PagedAttentionArgs {
  const uint16_t* q;
  const uint16_t* keys;
  const uint16_t* values;
  const int* block_tables;
  const int* query_start;
  const int* kv_lens;
  uint16_t* out;
  float* records;   // partial results of requests whose keys are split over blocks
  int* joins;       // per token: where its records begin and how many there are
  long long q_token_stride, q_head_stride, page_stride, head_stride, slot_stride, table_stride;
  int tokens, requests, pages, page, query_heads, kv_heads, causal;
  int table_keys;      // max_blocks * page, at most 2^28
  unsigned page_magic, page_shift;  // key / page = (key * page_magic) >> 32 >> page_shift for keys below 2^31
  int narrow_tokens, wide_tokens;   // of a request, that a narrow / wide tile holds
  int target;          // GPU blocks a kv head among which the key blocks (128 keys) are dealt; 0: one a tile
  int least_blocks;    // key blocks that make a GPU block worth its while
  int record_rows;     // rows of a record
  int units;           // records a kv head that the workspace holds
  float scale;
};

// Tokens of a vocabulary that one wave of the verification takes, and the bytes of what it leaves of a row of them.
constexpr int kVerifyChunk = 2048;
constexpr int kVerifyChunkBytes = 16;
constexpr int kVerifyLawBytes = 96;  // what stands of a request's drafts, and where its token comes from

struct VerifyArgs {
  const void* logits;
  const void* draft_logits;
  const long long* draft_tokens;
  const int* query_start;
  const float* uniforms;
  const float* temperature;
  long long* tokens_out;
  int* accepted;
  void* workspace;
  long long row_stride, draft_request_stride, draft_row_stride;
  int rows, requests, drafts, vocab, chunks;
  int judged;  // rows of a request that have statistics: the target's drafts + 1, and the drafts' where they matter
};
