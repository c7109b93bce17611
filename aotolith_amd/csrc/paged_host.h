// Host-side helpers of the paged-cache entry points: launches, and how the attention's work is laid out.
#pragma once

#include <algorithm>
#include <cstdint>

#include "aoto_hip.h"
#include "internal.h"
#include "paged_args.h"

namespace aoto {

inline bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

template <typename Args, typename... More>
int launch(const char* name, long long gx, long long gy, unsigned block, void* stream, Args& args, More... more) {
  if (gx > 0x7FFFFFFFLL || gy > 65535) return set_error(AOTO_ERR_UNSUPPORTED, "%s: grid too large", name);
  void* params[] = {static_cast<void*>(&args), static_cast<void*>(&more)...};
  const unsigned grid[3] = {(unsigned)gx, (unsigned)gy, 1};
  return launch_kernel(name, grid, block, stream, params);
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

// From what the host knows: shapes and the caller's bounds. The lengths are on the GPU. narrow_blocks: GPU blocks of the
// narrow tiles of 16 rows that a CU holds.
inline AttentionPlan attention_plan(int tokens, int requests, int max_blocks, int page, int query_heads, int kv_heads,
                                    int head_dim, int max_query_len, int max_kv_len, int narrow_blocks = 2) {
  const int group = query_heads / kv_heads, cus = device_cu_count();
  const long long rows = (long long)(max_query_len ? std::min(max_query_len, tokens) : tokens) * group;
  const long long some = std::min(requests, tokens);
  auto tiles = [&](int of) { return some + (tokens - some) / std::max(of / group, 1); };
  AttentionPlan p{};
  p.narrow_rows = rows <= 16 || rows > 32 ? 16 : 32;
  p.wide_rows = rows > 32 ? kWideRows : 0;
  p.units = tiles(p.wide_rows ? p.wide_rows : p.narrow_rows);
  // GPU blocks that the chip holds at a time
  const long long full = (p.wide_rows || p.narrow_rows > 16 ? 2LL : narrow_blocks) * cus;
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

// The arguments that follow from the plan, a's shapes and the workspace.
inline void attention_launch(const AttentionPlan& plan, int max_blocks, void* workspace, PagedAttentionArgs& a) {
  const int group = a.query_heads / a.kv_heads;
  a.table_keys = max_blocks * a.page;
  unsigned log2 = 0;
  while ((1u << log2) < (unsigned)a.page) ++log2;
  a.page_magic = (unsigned)(((1ull << (31 + log2)) + a.page - 1) / a.page), a.page_shift = log2 ? log2 - 1 : 0;
  a.narrow_tokens = plan.narrow_rows / group;
  a.wide_tokens = plan.wide_rows / group;
  a.target = plan.target, a.least_blocks = 2;
  a.record_rows = plan.wide_rows ? plan.wide_rows : plan.narrow_rows, a.units = (int)std::min(plan.units, 0x3FFFFFFFLL);
  a.joins = static_cast<int*>(workspace);
  a.records = reinterpret_cast<float*>(static_cast<char*>(workspace) + (size_t)a.tokens * 16);
}

}  // namespace aoto
