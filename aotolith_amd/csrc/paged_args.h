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
  const int* shares;  // of each of `pages` pages, holders beyond the first, or NULL: not looked at
  int pages;
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

// A layer's cache in 4 bits: codes and scale bytes, each with strides (bytes) of its own.
struct PagedMx4Cache {
  uint8_t* keys;
  uint8_t* values;
  uint8_t* key_scales;
  uint8_t* value_scales;
  long long page_stride, head_stride, slot_stride;
  long long scale_page_stride, scale_head_stride, scale_slot_stride;
};

struct PagedMx4AppendArgs {
  PagedMx4Cache cache;
  const uint16_t* qkv;
  const long long* positions;
  const long long* slots;
  const uint16_t* cos_table;
  const uint16_t* sin_table;
  uint16_t* q_out;
  int* error;
  long long row_stride, slot_count;
  int tokens, query_heads, kv_heads, head_dim, page, table_rows;
};

struct PagedMx4UnpackArgs {
  PagedMx4Cache cache;
  uint16_t* keys_out;
  uint16_t* values_out;
  int page, kv_heads, head_dim;
};

struct PagedMx4AttentionArgs {
  PagedAttentionArgs base;  // its pages' addresses and strides are not used
  PagedMx4Cache cache;
  int turn_from, turn_to;  // items taken in the opposite order
};

struct PagedForkArgs {
  const int* parents;
  const int* context_lens;
  int* block_tables;
  const int* page_counts;
  int* shares;
  const int* free_pages;
  const int* free_start;
  int* context_lens_out;
  int* page_counts_out;
  int* free_start_out;
  int* source;
  int* target;
  // Two entries a request: the full pages that it takes over, -1 where it stays as it is, -2 - j where it gets entry j
  // of its own; its length.
  int* plan;
  int* error;
  long long table_stride;
  int requests, max_blocks, free_count, pages, page;
};

// Pages that a block of paged_release looks at, and pages of a pool that one block does all of it for.
constexpr int kPageChunk = 1024, kPagesFew = 4096;

struct PagedReleaseArgs {
  const int* keep_lens;
  const int* block_tables;
  const int* page_counts;
  int* shares;
  int* free_pages;
  const int* free_start;
  int* page_counts_out;
  int* free_start_out;
  int* scratch;  // the list's start as it was, then the pages given back in each kPageChunk
  int* error;
  long long table_stride;
  int requests, max_blocks, free_count, pages, page;
  int list_blocks;  // of aoto_paged_drop, that go over the free list
};

struct PagedCompactArgs {
  int* block_tables;
  const int* page_counts;
  int* shares;
  int* free_pages;
  const int* free_start;
  int* source;
  int* target;
  int* count;
  int* state;  // of each page: what it is, then its new number
  int* error;
  long long table_stride;
  int requests, max_blocks, free_count, pages;
  int list_blocks;  // of aoto_paged_mark, that go over the free list
};

// What a copy of pages moves: planes of pages of one size.
constexpr int kPagedCopyTensors = 64;
constexpr int kPagedCopyChunk = 16384;  // bytes that a block moves at a time

struct PagedCopyTensor {
  uint8_t* base;
  long long page_stride, plane_stride;  // bytes
  long long bytes;                      // of a page
  int first;                            // planes of the tensors before it
  int chunks;                           // of a page
};

struct PagedCopyArgs {
  const int* source;
  const int* target;
  const int* count;  // pairs in use, or NULL: all
  int* error;
  int pairs, pages, tensors, planes, chunks;  // planes of all tensors, chunks of the longest page
  int blocks;                                 // of the launch
  int wide;                                   // everything a multiple of 16 bytes
  PagedCopyTensor at[kPagedCopyTensors];
};

struct AdjustArgs {
  const void* logits;
  void* out;
  const int* query_start;   // NULL: a row a request
  const long long* history;
  const int* history_lens;
  const int* prompt_lens;
  const long long* draft_tokens;
  const float* repetition;
  const float* presence;
  const float* frequency;
  const long long* bias_tokens;
  const float* bias_values;
  const uint8_t* allowed;
  long long row_stride, out_stride, history_stride, draft_stride, bias_stride, value_stride, allowed_stride;
  int rows, requests, vocab, history_len, drafts, biases;
};
