// Attention of requests' new tokens over their pages of a shared key/value cache.
//
//   out[t][h] = sum_j softmax_j(scale * q[t][h] . k_j) v_j
// over the keys j of token t's request r that it may see: with n_r = query_start[r + 1] - query_start[r] rows and
// kv_r keys, row i sees j < kv_r - n_r + i + 1 (causal) or j < kv_r, as far as the block table row goes and where its
// entry names a page of the cache; a row that sees none gives 0. Key j of head h / (Hq / Hkv) is row j % page of page
// block_tables[r][j / page]. Scores, maxima and sums in f32, one pass over the keys with a running maximum. P goes
// into its product with V as bf16, the matrix instructions' operands being of one type: as two of them in narrow tiles,
// rounded to one in wide tiles (as the prefill attention does), which is off by as much as the result's own rounding.
//
// NaN and infinities are the softmax's, in every tile and however an item is cut: a NaN score or one of +inf makes its
// row NaN, scores of -inf weigh nothing beside others and give NaN alone, a NaN or infinite value that a row sees is in
// its dim of the row however small its weight (one that f32 or a score of -inf makes 0, too), and what a row does not
// see weighs exactly 0 and leaves nothing.
//
// Work is cut on the GPU, from the lengths as they are there. An item is one tile of a request's rows (all query heads
// of a kv head that share its keys, token after token) against all the keys they see, counted in blocks of 128 keys.
// With `target` blocks a kv head, the items' key blocks, one item after the other, are dealt out evenly: every GPU
// block takes the same number of them, wherever that begins and ends, so that requests of very different lengths end
// together (an item cut among several leaves records, maximum, sum and unnormalized row, that
// aoto_paged_attention_join_* combines). Without a target, where the host counts tiles enough for the chip, every GPU
// block takes one item, and the longest ends last. A GPU block finds its place by running sums over the requests.
//   narrow tiles (16 NT rows, decodes and drafted tokens): the four waves take 32 keys each of every 128; K goes
//     straight from the pages to operand registers, V through the wave's own LDS; no barrier in the loop
//   wide tiles (128 rows, chunks of prompts): the four waves take 32 rows each, 64-key tiles of K and V staged once for
//     all of them
#pragma once

#include "common.h"
#include "flash_attention.h"
#include "paged_args.h"

namespace aoto {

typedef short pa_s16x4 __attribute__((ext_vector_type(4)));
typedef short pa_s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) pa_s16x4 pa_lds_s16x4;

typedef __attribute__((address_space(3))) fa_bf16x8 paged_lds_bf16x8;

AOTO_DEVICE uint32_t paged_lds(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

constexpr int kPagedUnitKeys = 128;  // keys of a key block
// What starting on an item costs (its rows, table entries and first keys are three round trips to memory), in key
// blocks: a GPU block that goes from one item to another takes so many fewer. (1, 2, 4: 16 requests' drafted rows 44.9,
// 43.3, 44.3 us; a chunk of 500 beside 24 tokens 34.6, 32.3, 32.1; 32 tokens over 88000 keys 76.6, 77.5, 79.8.)
constexpr int kPagedLead = 2;

struct PagedUnit {
  int request, begin, rows;  // its first row and how many
  int keys;                  // that the tile's rows see, as far as the block table reaches
  int first;                 // keys that the request's first row sees (causal; else more than there are)
  int token, tokens;         // of the request: the tile's first and count
  int from, to;              // key blocks of this part
  int record, part, parts;   // the first part's record, which part this is of how many
  bool narrow;
};

struct PagedRequest {
  int begin, rows, keys, first, tiles, tokens;  // tokens a tile
  bool narrow;
};

template <bool MIXED>
AOTO_DEVICE PagedRequest paged_request(const PagedAttentionArgs& a, int r) {
  PagedRequest q;
  q.begin = min(max(a.query_start[r], 0), a.tokens);
  q.rows = min(max(a.query_start[r + 1], q.begin), a.tokens) - q.begin;
  const int keys = max(a.kv_lens[r], 0);
  q.keys = min(keys, a.table_keys);
  q.first = a.causal ? keys - q.rows + 1 : 0x3FFFFFFF;
  q.narrow = !MIXED || q.rows <= a.narrow_tokens;
  q.tokens = max(1, q.narrow ? a.narrow_tokens : a.wide_tokens);  // more than 16 heads: only rowless ones are narrow
  q.tiles = (q.rows + q.tokens - 1) / q.tokens;
  return q;
}

// Keys that the rows of a tile see, and the blocks of them (one where there are none: the rows are written all the
// same).
AOTO_DEVICE int paged_tile_keys(const PagedRequest& q, int tile) {
  return min(q.keys, max(0, q.first + min(q.rows, (tile + 1) * q.tokens) - 1));
}
AOTO_DEVICE int paged_tile_blocks(const PagedRequest& q, int tile) {
  return max(1, (paged_tile_keys(q, tile) + kPagedUnitKeys - 1) / kPagedUnitKeys);
}

// The parts that one GPU block goes through.
template <bool MIXED>
struct PagedWalk {
  int request, tile, item, from;  // where it stands: the tile's number among all, its next place
  int left;                       // places to go, those of whole items counted as they come (target 0: one item)
  int block;                      // which of the `target`
  int each, more;                 // places a GPU block takes; the first `more` take one more
  PagedRequest q;                 // the request it stands at

  // 256 threads, all of them; false where nothing is left for this one.
  AOTO_DEVICE bool start(const PagedAttentionArgs& a, int u) {
    __shared__ int s_sum[2][4];
    __shared__ int s_at[8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // a thread's requests; where there are few of them, 1 / 2^share of one's tiles (a chunk of a prompt has many)
    const int share = a.requests <= 8 ? 5 : a.requests <= 32 ? 3 : a.requests <= 128 ? 1 : 0;
    const int per = (a.requests + 255) / 256;
    const int lo = min((tid >> share) * per, a.requests), hi = min(lo + per, a.requests);
    auto tiles_of = [&](const PagedRequest& q, int& begin, int& end) {
      const int some = (q.tiles + (1 << share) - 1) >> share;
      begin = min((tid & ((1 << share) - 1)) * some, q.tiles), end = min(begin + some, q.tiles);
    };
    int items = 0, work = 0;
    PagedRequest only = {};  // a thread's request, where it has but one
    for (int r = lo; r < hi; ++r) {
      const PagedRequest q = only = paged_request<MIXED>(a, r);
      int begin, end;
      tiles_of(q, begin, end);
      items += end - begin;
      if (a.target > 0)
        for (int t = begin; t < end; ++t) work += kPagedLead + paged_tile_blocks(q, t);
    }
    int items_to = items, work_to = work;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int i = __shfl_up(items_to, d), w = __shfl_up(work_to, d);
      if (lane >= d) items_to += i, work_to += w;
    }
    if (lane == 63) s_sum[0][wave] = items_to, s_sum[1][wave] = work_to;
    if (tid == 0) s_at[0] = -1;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) items_to += s_sum[0][w], work_to += s_sum[1][w];
      total += s_sum[1][w];
    }
    int at = u;  // of the items, or of the key blocks
    block = u, each = 1, more = 0, left = 1;
    if (a.target > 0) {
      const int blocks = max(1, min(a.target, total / a.least_blocks));
      each = __builtin_amdgcn_readfirstlane(total / blocks);
      more = __builtin_amdgcn_readfirstlane(total - each * blocks);
      at = u * each + min(u, more);
      left = u < blocks ? each + (u < more ? 1 : 0) : 0;
    }
    const int upto = a.target > 0 ? work_to : items_to, mine = a.target > 0 ? work : items;
    if (left > 0 && at < upto && at >= upto - mine) {
      int before = upto - mine, item_before = items_to - items;
      for (int r = lo; r < hi; ++r) {
        const PagedRequest q = per == 1 ? only : paged_request<MIXED>(a, r);
        int begin, end, t;
        tiles_of(q, begin, end);
        if (a.target > 0) {
          for (t = begin; t < end; ++t) {
            const int n = kPagedLead + paged_tile_blocks(q, t);
            if (at < before + n) break;
            before += n;
          }
        } else {
          t = min(begin + at - item_before, end);
        }
        if (t < end) {
          // without a target the longest rows of a causal chunk first
          s_at[0] = r, s_at[1] = a.target > 0 ? t : q.tiles - 1 - t, s_at[2] = item_before + t - begin;
          s_at[3] = a.target > 0 ? at - before : 0;
          s_at[4] = q.begin, s_at[5] = q.rows, s_at[6] = q.keys, s_at[7] = q.first;
          break;
        }
        item_before += end - begin;
      }
    }
    __syncthreads();
    request = __builtin_amdgcn_readfirstlane(s_at[0]), tile = __builtin_amdgcn_readfirstlane(s_at[1]);
    item = __builtin_amdgcn_readfirstlane(s_at[2]), from = __builtin_amdgcn_readfirstlane(s_at[3]);
    q.begin = s_at[4], q.rows = s_at[5], q.keys = s_at[6], q.first = s_at[7];
    settle(a);
    return request >= 0;
  }
  // The request's numbers in scalar registers, which loads do not go to, and what follows from them.
  AOTO_DEVICE void settle(const PagedAttentionArgs& a) {
    q.begin = __builtin_amdgcn_readfirstlane(q.begin), q.rows = __builtin_amdgcn_readfirstlane(q.rows);
    q.keys = __builtin_amdgcn_readfirstlane(q.keys), q.first = __builtin_amdgcn_readfirstlane(q.first);
    q.narrow = !MIXED || q.rows <= a.narrow_tokens;
    q.tokens = max(1, q.narrow ? a.narrow_tokens : a.wide_tokens);
    q.tiles = (q.rows + q.tokens - 1) / q.tokens;
  }

  // The next part; false at the end. Uniform.
  AOTO_DEVICE bool next(const PagedAttentionArgs& a, PagedUnit& unit) {
    if (left <= 0) return false;
    while (tile >= q.tiles) {
      if (++request >= a.requests) return false;
      tile = 0;
      q = paged_request<MIXED>(a, request);
      settle(a);
    }
    const int n = paged_tile_blocks(q, tile);
    unit.request = request, unit.begin = q.begin, unit.rows = q.rows, unit.first = q.first;
    unit.keys = paged_tile_keys(q, tile);
    unit.token = tile * q.tokens, unit.tokens = min(q.tokens, q.rows - unit.token);
    unit.narrow = q.narrow;
    unit.from = 0, unit.to = n, unit.record = unit.part = 0, unit.parts = 1;
    if (a.target > 0) {
      // of the item's places the first kPagedLead stand for its start
      const int place = block * each + min(block, more) + (each + (block < more ? 1 : 0) - left) - from + kPagedLead;
      left -= max(0, kPagedLead - from);
      if (left <= 0) return false;
      unit.from = max(0, from - kPagedLead), unit.to = min(n, unit.from + left);
      left -= unit.to - unit.from;
      // the GPU blocks that hold the item's first and last key block
      const int head = owner(place), tail = owner(place + n - 1);
      unit.record = head + item, unit.part = block - head, unit.parts = tail - head + 1;
      // only where query_start decreases and requests share rows: more tiles than rows make
      if (unit.record < 0 || unit.part < 0 || unit.record > a.units - unit.parts) return false;
    } else {
      left = 0;
    }
    from = 0, ++tile, ++item;
    return true;
  }
  AOTO_DEVICE int owner(int at) const {
    const int longer = more * (each + 1);
    return __builtin_amdgcn_readfirstlane(at < longer ? at / (each + 1) : more + (at - longer) / each);
  }
};

// The block table entry of a key.
AOTO_DEVICE int paged_block(const PagedAttentionArgs& a, int key) {
  return a.page == 1 ? key : (int)(__umulhi((unsigned)key, a.page_magic) >> a.page_shift);
}

// Element offset of a key's row in the pages of kv head 0, -1 where its entry names no page.
AOTO_DEVICE long long paged_row(const PagedAttentionArgs& a, const int* __restrict__ table, int key) {
  const int block = paged_block(a, key);
  const int page = table[block];
  const int row = key - block * a.page;
  return (unsigned)page < (unsigned)a.pages ? page * a.page_stride + row * a.slot_stride : -1;
}

// 1 / sum of a row's weights, whose maximum is `big`: 0 where no key was seen, NaN where every score is one (they have
// no maximum, but a sum of NaN) or is -inf (kPagedNoWeight).
AOTO_DEVICE float paged_inverse(float big, float sum) {
  return sum == 0.f ? (big == -INFINITY ? 0.f : NAN) : 1.f / sum;
}
// The maximum of a row that sees keys, their scores all -inf: beside other keys it weighs nothing, but it is not that
// of a row without keys.
constexpr float kPagedNoWeight = -0x1.fffffep127f;

AOTO_DEVICE bool bf16_pair_special(uint32_t w) {
  return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
}
AOTO_DEVICE uint32_t bf16_pair_finite(uint32_t w) {
  if ((w & 0x7F80u) == 0x7F80u) w &= 0xFFFF0000u;
  if ((w & 0x7F800000u) == 0x7F800000u) w &= 0xFFFFu;
  return w;
}
// Whether a 16-byte chunk of V holds an infinity or a NaN; the chunk without them.
AOTO_DEVICE bool chunk_special(const uint4& v) {
  return bf16_pair_special(v.x) || bf16_pair_special(v.y) || bf16_pair_special(v.z) || bf16_pair_special(v.w);
}
AOTO_DEVICE uint4 chunk_finite(const uint4& v) {
  return make_uint4(bf16_pair_finite(v.x), bf16_pair_finite(v.y), bf16_pair_finite(v.z), bf16_pair_finite(v.w));
}
// The infinity or NaN in the upper or lower half of w, else 0.
AOTO_DEVICE float special_lo(uint32_t w) { return (w & 0x7F80u) == 0x7F80u ? bf16_lo(w) : 0.f; }
AOTO_DEVICE float special_hi(uint32_t w) { return (w & 0x7F800000u) == 0x7F800000u ? bf16_hi(w) : 0.f; }


// Whether one of keys k0 .. limit - 1 (k0 < limit) has a page.
AOTO_DEVICE bool paged_sees(const PagedAttentionArgs& a, const int* __restrict__ table, int k0, int limit) {
  bool sees = false;
#pragma unroll 1
  for (int b = paged_block(a, k0); !sees && b * a.page < limit; ++b) sees = (unsigned)table[b] < (unsigned)a.pages;
  return sees;
}

// The sum of the infinities and NaN among four dims of keys k0 .. limit - 1 that have a page, 0 where there are none.
// A weight of 0 (2^-118 of the row's largest and less; 2^-95 for the second term of narrow tiles) makes a NaN of an
// infinite value, which the result should be: a row that has one, though none of its scores is, takes this sum there.
// Seldom called, so kept short: one round trip to memory for four keys (2048 rows over 32000 keys, a value infinite in
// one dim and without weight: 13 ms instead of 1.2; 32 tokens over 8000 each: 2.9 instead of 0.2).
AOTO_DEVICE f32x4_t paged_special(const PagedAttentionArgs& a, const int* __restrict__ table,
                                  const uint16_t* __restrict__ values, int k0, int limit) {
  f32x4_t sum{};
#pragma unroll 4
  for (int k = k0; k < limit; ++k) {
    const long long row = paged_row(a, table, k);
    const uint2 w = *reinterpret_cast<const uint2*>(values + max(row, 0LL));
    const bool there = row >= 0;
    sum[0] += there ? special_lo(w.x) : 0.f, sum[1] += there ? special_hi(w.x) : 0.f;
    sum[2] += there ? special_lo(w.y) : 0.f, sum[3] += there ? special_hi(w.y) : 0.f;
  }
  return sum;
}
AOTO_DEVICE bool paged_any_nan(const f32x4_t& v) {
  return v[0] != v[0] || v[1] != v[1] || v[2] != v[2] || v[3] != v[3];
}
// v with the sums of special values (not 0 where there are some) in the place of its NaN.
AOTO_DEVICE f32x4_t paged_with_special(f32x4_t v, const f32x4_t& special) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = v[i] != v[i] && special[i] != 0.f ? special[i] : v[i];
  return v;
}
// An infinite value of a part stays one under any factor, 0 too.
AOTO_DEVICE float paged_scaled(float x, float by) { return fabsf(x) < INFINITY ? x * by : x; }

AOTO_DEVICE float* paged_record(const PagedAttentionArgs& a, int unit, int kvh, int row, int head_dim) {
  return a.records + (((size_t)unit * a.kv_heads + kvh) * a.record_rows + row) * (head_dim + 2);
}

// What a joined token needs: its tile's first record, how many there are, its first row in them.
AOTO_DEVICE void paged_note(const PagedAttentionArgs& a, const PagedUnit& unit, int kvh) {
  if (a.target <= 0 || kvh != 0 || unit.part != 0) return;
  const int group = a.query_heads / a.kv_heads;
  for (int i = threadIdx.x; i < unit.tokens; i += 256)
    reinterpret_cast<int4*>(a.joins)[unit.begin + unit.token + i] = make_int4(unit.record, unit.parts, i * group, 0);
}

// ---------------------------------------------------------------------------------------------------- narrow tiles
template <int D, int NT>
struct PagedNarrowShared {
  static constexpr int STR = D + 16;  // bf16 of a staged V row: the transposing reads' four rows start 8 banks apart
  union {
    uint16_t v[4][32 * STR];
    float o[4][16 * NT][D];
  };
  float m[4][16 * NT], l[4][16 * NT];
};

// v_mfma_f32_16x16x32_bf16: S^T [16 keys x 16 rows] = K . Q^T, O^T [16 d x 16 rows] += V^T . P^T. Lane l owns row
// l % 16 of a tile in both; the k slots of the second product hold the keys in the order S^T leaves them in a lane:
// slot 8 q + j is key 4 q + j of the first 16 (j < 4), 4 q + j - 4 of the second.
//
// Bound by the read of K and V: 88000 keys of 32 requests, 8 kv heads of 128, in 72 us, 5.0 TB/s. Each wave keeps a
// tile's K and V on their way while it works on the one before, and waits for nobody.
template <int D, int NT>
AOTO_DEVICE void paged_narrow(const PagedAttentionArgs& a, const PagedUnit& unit, int kvh,
                              PagedNarrowShared<D, NT>& s) {
  constexpr int DC = D / 32, DT = D / 16, STR = PagedNarrowShared<D, NT>::STR;
  // P keeps 16 bits, as its upper half cut off and the rest rounded: two products, which cost nothing with 16 rows
  // (78.7 us with and without for 32 requests' 88000 keys) and 4% with 32 (16 requests' five rows 44.5 us, 42.7 rounded
  // to bf16: a single token may run in either tile, by the bound its caller gives).
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int group = a.query_heads / a.kv_heads;
  const int live = unit.tokens * group;  // rows in use; the others repeat the last
  const int* table = a.block_tables + unit.request * a.table_stride;
  const uint16_t* keys = a.keys + kvh * a.head_stride + 8 * quad;
  const uint16_t* values = a.values + kvh * a.head_stride + 8 * quad;
  uint16_t* vs = s.v[wave];

  const int k0 = unit.from * kPagedUnitKeys, k1 = min(unit.keys, unit.to * kPagedUnitKeys);
  // this wave's 32-key tiles: k0 + 32 wave + 128 i
  const int mine = k0 + 32 * wave;
  const int trips = k1 > mine ? (k1 - mine + 127) / 128 : 0;

  fa_bf16x8 qf[NT][DC];
  int limit[NT];  // keys that this lane's row sees
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = min(16 * t + col, live - 1), i = unit.token + row / group, g = row % group;
    const uint16_t* q = a.q + (unit.begin + i) * a.q_token_stride + (kvh * group + g) * a.q_head_stride + 8 * quad;
#pragma unroll
    for (int c = 0; c < DC; ++c) qf[t][c] = *reinterpret_cast<const fa_bf16x8*>(q + 32 * c);
    limit[t] = min(k1, unit.first + i);
  }
  const int least = min(k1, unit.first + unit.token);  // keys that every row sees

  float run_max[NT], run_sum[NT];
  f32x4_t o[NT][DT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    run_max[t] = -INFINITY, run_sum[t] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[t][d] = f32x4_t{};
  }
  const float c2 = a.scale * 1.4426950408889634f;

  // This lane loads keys col and 16 + col of a tile. Their pages are looked up two tiles ahead, their offsets known one
  // tile ahead: a lookup inside the tile that needs it is a round trip to memory in which nothing else is asked for.
  struct Rows {
    int page[2], row[2];
  };
  auto look = [&](int base) {
    Rows of;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int key = min(base + 16 * g + col, k1 - 1), block = paged_block(a, key);
      of.page[g] = table[block];
      of.row[g] = key - block * a.page;
    }
    return of;
  };
  auto place = [&](const Rows& of, long long (&to)[2]) {
#pragma unroll
    for (int g = 0; g < 2; ++g)
      to[g] = (unsigned)of.page[g] < (unsigned)a.pages
                  ? (long long)((unsigned long long)(unsigned)of.page[g] * (unsigned)a.page_stride) +
                        of.row[g] * (int)a.slot_stride
                  : -1;
  };
  long long at[2], next[2];
  uint4 kq[2][DC], vq[2][DC];
  Rows ahead;
  if (trips > 0) {
    const Rows now = look(mine), then = look(mine + 128);
    ahead = look(mine + 256);
    place(now, at);
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int c = 0; c < DC; ++c) kq[g][c] = *reinterpret_cast<const uint4*>(keys + max(at[g], 0LL) + 32 * c);
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int c = 0; c < DC; ++c) vq[g][c] = *reinterpret_cast<const uint4*>(values + max(at[g], 0LL) + 32 * c);
    place(then, next);
  }
  for (int trip = 0; trip < trips; ++trip) {
    const int base = mine + 128 * trip;
    f32x4_t sc[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        sc[t][g] = f32x4_t{};
#pragma unroll
        for (int c = 0; c < DC; ++c)
          sc[t][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(fa_bf16x8, kq[g][c]), qf[t][c],
                                                             sc[t][g], 0, 0, 0);
      }
    // the keys of this tile that exist, one bit each; their values to LDS, zeros for the others
    bool there[2];
    uint32_t exist = 0;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      there[g] = at[g] >= 0 && base + 16 * g + col < k1;
      exist |= (uint32_t)(__ballot(there[g]) & 0xFFFFu) << (16 * g);
    }
    const bool whole = exist == 0xFFFFFFFFu && base + 32 <= least;
    uint32_t special = 0;  // keys, not seen by every row, whose values are not finite: added row by row below
    if (!whole && least < k1 && base + 32 > least) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        bool odd = false;
#pragma unroll
        for (int c = 0; c < DC; ++c) odd |= chunk_special(vq[g][c]);
        unsigned long long lanes = __ballot(odd && there[g]);
        lanes |= lanes >> 32;
        special |= (uint32_t)((lanes | lanes >> 16) & 0xFFFFu) << (16 * g);
      }
    }
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        uint4 v = there[g] ? vq[g][c] : make_uint4(0, 0, 0, 0);
        if (special) v = chunk_finite(v);
        *reinterpret_cast<uint4*>(vs + (16 * g + col) * STR + 32 * c + 8 * quad) = v;
      }
    // the next tile's loads, K first, then the tile after it
    const long long old[2] = {at[0], at[1]};
#pragma unroll
    for (int g = 0; g < 2; ++g) at[g] = next[g];
    place(ahead, next);
    ahead = look(base + 384);
    if (trip + 1 < trips) {
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int c = 0; c < DC; ++c) kq[g][c] = *reinterpret_cast<const uint4*>(keys + max(at[g], 0LL) + 32 * c);
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int c = 0; c < DC; ++c) vq[g][c] = *reinterpret_cast<const uint4*>(values + max(at[g], 0LL) + 32 * c);
    }
    fa_bf16x8 pb[NT], pr[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (!whole) {
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = 16 * g + 4 * quad + e;
            if (!(exist >> k & 1) || base + k >= limit[t]) sc[t][g][e] = -INFINITY;
          }
      }
      float top = -INFINITY;
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, sc[t][g][e]);
      top = xor32_max(xor16_max(top)) * c2;
      // the exponentials' reference moves only where a score passes it, and then 2^8 ahead: no weight is above 1, which
      // a value near the largest number would not bear
      const float moved = top > run_max[t] ? top + 8.f : run_max[t];
      const float keep = moved == run_max[t] ? 1.f : __builtin_amdgcn_exp2f(run_max[t] - moved);
      run_max[t] = moved;
      const float ref = moved == -INFINITY ? 0.f : moved;
      if (__any(keep != 1.f)) {
        run_sum[t] *= keep;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] *= keep;
      }
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // 0 for a key that is not there or hidden from the row, whose value here is finite
        p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][j >> 2][j & 3], c2, -ref));
        run_sum[t] += p[j];
      }
      uint32_t high[4], low[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        high[j] = __builtin_amdgcn_perm(__float_as_uint(p[2 * j + 1]), __float_as_uint(p[2 * j]), 0x07060302u);
        // the rest, and 2^-23 of the weight, which is lost beside it but keeps the term from 0 where nothing is left: 0
        // would make a NaN of every infinite value
        constexpr float kMore = 1.f + 0x1p-23f;
        low[j] = cvt_pk_bf16(__builtin_fmaf(p[2 * j], kMore, -bf16_lo(high[j])),
                             __builtin_fmaf(p[2 * j + 1], kMore, -bf16_hi(high[j])));
      }
      pb[t] = __builtin_bit_cast(fa_bf16x8, high);
      pr[t] = __builtin_bit_cast(fa_bf16x8, low);
    }
    const uint16_t* vp = vs + (4 * quad + (col >> 2)) * STR + 4 * (col & 3);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const pa_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s16x4*)(vp + 16 * d));
      const pa_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s16x4*)(vp + 16 * STR + 16 * d));
      const pa_s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(fa_bf16x8, both), pb[t], o[t][d], 0, 0, 0);
        o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(fa_bf16x8, both), pr[t], o[t][d], 0, 0, 0);
      }
    }
    while (special) {
      const int k = __ffs(special) - 1;
      special &= special - 1;
      const long long row = __shfl(k < 16 ? old[0] : old[1], k & 15);
      const uint16_t* v = a.values + kvh * a.head_stride + row + 4 * quad;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const uint2 w = *reinterpret_cast<const uint2*>(v + 16 * d);
#pragma unroll
        for (int t = 0; t < NT; ++t)
          if (base + k < limit[t]) {
            o[t][d][0] += special_lo(w.x), o[t][d][1] += special_hi(w.x);
            o[t][d][2] += special_lo(w.y), o[t][d][3] += special_hi(w.y);
          }
      }
    }
  }

  // the waves' shares of each row, combined as the join combines chunks
#pragma unroll
  for (int t = 0; t < NT; ++t) run_sum[t] = xor32_sum(xor16_sum(run_sum[t]));
  __syncthreads();  // every wave is through with its V
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<f32x4_t*>(&s.o[wave][16 * t + col][16 * d + 4 * quad]) = o[t][d];
    if (quad == 0) s.m[wave][16 * t + col] = run_max[t], s.l[wave][16 * t + col] = run_sum[t];
  }
  __syncthreads();
  constexpr int PER_ROW = D / 4;
  for (int c = threadIdx.x; c < live * PER_ROW; c += 256) {
    const int row = c / PER_ROW, d = 4 * (c % PER_ROW);
    float big = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) big = fmaxf(big, s.m[w][row]);
    float sum = 0.f;
    f32x4_t v{};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = s.m[w][row] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s.m[w][row] - big);
      sum += f * s.l[w][row];
      // a wave without keys holds zeros: 0 * 0
      v += f * *reinterpret_cast<const f32x4_t*>(&s.o[w][row][d]);
    }
    // what is rare, out of the way: fetched with the code around it, it took 0.2 of a small call's 7.2 us
    if (__builtin_expect(__any(!(fabsf(v[0] + v[1] + v[2] + v[3]) < INFINITY && sum > 0.f)), 0)) {
      const int sees = min(k1, unit.first + unit.token + row / group);
      if (paged_any_nan(v) && sum == sum)
        v = paged_with_special(v, paged_special(a, table, a.values + kvh * a.head_stride + d, k0, sees));
      if (big == -INFINITY && sum == 0.f && k0 < sees && paged_sees(a, table, k0, sees)) big = kPagedNoWeight;
    }
    if (unit.parts > 1) {
      float* rec = paged_record(a, unit.record + unit.part, kvh, row, D);
      if (d == 0) rec[0] = big, rec[1] = sum;
      *reinterpret_cast<float2*>(rec + 2 + d) = make_float2(v[0], v[1]);
      *reinterpret_cast<float2*>(rec + 4 + d) = make_float2(v[2], v[3]);
    } else {
      const float inv = paged_inverse(big, sum);
      const size_t token = unit.begin + unit.token + row / group;
      *reinterpret_cast<uint2*>(a.out + (token * a.query_heads + kvh * group + row % group) * D + d) =
          make_uint2(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv));
    }
  }
}

// ------------------------------------------------------------------------------------------------------ wide tiles
template <int D>
struct PagedWideShared {
  uint16_t k[5][32 * D];  // halves of tiles: tile t's are slots 2 t and 2 t + 1, mod 5
  uint16_t v[2][64 * D];
  uint32_t exist[4][4];  // by tile (mod 4) and staging wave: which of its 16 rows exist (a page, and not past the end)
  uint32_t known[4][4];  // and which have a page
  uint32_t special[4];   // which of the V tile's rows hold a value that is not finite and not seen by every row
};

// 16 bytes a lane from global memory to 1 KB of LDS. Not the builtin: the compiler's wait counts lose track of which
// buffer such a load writes; the loop below waits for all of them before its barrier.
AOTO_DEVICE void paged_dma(const uint16_t* from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory", "m0");
}

// Waits for all loads in flight, those to LDS among them: the builtin, so that the compiler knows it too and does not
// wait, inside the loop, for loads it thinks are still out.
AOTO_DEVICE void paged_landed() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0) alone
  asm volatile("" ::: "memory");
}

// Changes of an accumulator that the tile loop makes seldom, in place: as plain arithmetic they make the compiler hold
// O in the ordinary registers and move all of it (128 registers) to the accumulation registers and back in every tile.
// It does not see that these read what products wrote, so acc_settle() stands before the first and after the last: the
// 64 cycles that a product's result takes, with room.
AOTO_DEVICE void acc_scale(float& x, float by) {
  float y;
  asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
               : "+a"(x), "=&v"(y) : "v"(by));
}
AOTO_DEVICE void acc_add(float& x, float by) {
  float y;
  asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_add_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
               : "+a"(x), "=&v"(y) : "v"(by));
}
AOTO_DEVICE void acc_settle() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// v_mfma_f32_32x32x16_bf16: S^T [32 keys x 32 rows] = K . Q^T, O^T [32 d x 32 rows] += V^T . P^T (layouts and slot
// order as in the prefill attention). A wave has 32 rows; two waves, of two blocks, share a SIMD and its 512 registers.
// A step holds, in this order and spread out between its products, the scores of the next 32 keys (with three quarters
// of the present keys' exponentials) and the product of the present keys' weights with V (with the other exponentials,
// the next scores out of their accumulators and their maximum). Operands are read from LDS two products ahead. K and V
// go from memory to LDS without registers, K up to two tiles ahead and V one; K in five slots of half a tile, so that
// two blocks' tiles fit the LDS. The 16-byte pieces of a row are permuted by a function of the row (the lanes fetch
// them so) that spreads each phase of the reads over all banks. Rows' addresses advance by 64 keys a tile without a
// division or a product but the page's.
//
// Bound by issue, every part with its share: 2048 rows over 8048 keys, 32 / 8 heads of 128, run at 0.85 PFLOP/s in
// 276 us (263 to 283, by the card), the matrix units busy for 37% of it and the vector units for 64%; without its loads
// to LDS it would take 35 us less, without the reads of K 34, of V 11, without half of the products 32, without the
// exponentials 17. Reading operands one or three products ahead, no fences between the products, and the packing of
// weights one product later changed it by less than 1%. One wave a SIMD with 64 rows, half the reads from LDS and 512
// registers took 297 us there, 96 us (73 here) for 2048 rows over themselves and 61 us (41) for 1024, its tiles being
// too few for the chip.
template <int D>
AOTO_DEVICE void paged_wide(const PagedAttentionArgs& a, const PagedUnit& unit, int kvh, PagedWideShared<D>& s) {
  constexpr int DS = D / 16, DT = D / 32, LPR = D / 8;  // lanes (16-byte pieces) a row
  constexpr int RPL = 64 / LPR;                         // rows a wave's load covers
  constexpr int LOADS = 16 / RPL;                       // loads of K (and V) a thread does for a 64-key tile
  constexpr int ROWB = 2 * D, HALFB = 32 * ROWB, TILEB = 64 * ROWB;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int group = a.query_heads / a.kv_heads;
  const int live = unit.tokens * group;
  const int* table = a.block_tables + unit.request * a.table_stride;
  const int k0 = unit.from * kPagedUnitKeys, k1 = min(unit.keys, unit.to * kPagedUnitKeys);
  const int tiles = k1 > k0 ? (k1 - k0 + 63) / 64 : 0;
  const bool active = 32 * wave < live;  // a wave of none of the rows only stages

  // this lane's row: its token of the request and head of the group, and the keys it sees
  const int row = 32 * wave + col, token = unit.token + min(row, live - 1) / group, head = min(row, live - 1) % group;
  const uint16_t* q = a.q + (unit.begin + token) * a.q_token_stride + (kvh * group + head) * a.q_head_stride + 8 * half;
  fa_bf16x8 qf[DS];
#pragma unroll
  for (int d = 0; d < DS; ++d) qf[d] = *reinterpret_cast<const fa_bf16x8*>(q + 16 * d);
  const int limit = min(k1, unit.first + token);
  const int least = min(k1, unit.first + unit.token);  // keys that every row of the block sees
  const float c2 = a.scale * 1.4426950408889634f;

  // The permutation of a row's pieces: piece c of row r lies at c ^ swizzle(r).
  auto swizzle = [](int r) { return D == 128 ? (r & 3) << 2 | (r >> 2 & 3) : (r >> 1 & 1) << 2 | (r >> 2 & 3); };
  // Staging: load i of a tile takes row 4 RPL i + stage_row, its piece lane % LPR.
  const int stage_row = wave * RPL + lane / LPR;
  const int piece = 8 * ((lane % LPR) ^ swizzle(stage_row));
  const uint16_t* keys = a.keys + kvh * a.head_stride + piece;
  const uint16_t* values = a.values + kvh * a.head_stride + piece;
  const uint32_t last_entry = 4 * paged_block(a, max(k1 - 1, 0));
  const uint32_t page_span = a.page * (uint32_t)a.slot_stride;
  const int step_blocks = paged_block(a, 64);
  const uint32_t step_off = (64 - step_blocks * a.page) * (uint32_t)a.slot_stride;
  // of the tile looked up last: the rows' table entries (bytes in the table), their offsets in their pages, the pages
  uint32_t entry[LOADS], off[LOADS];
  int ahead[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int key = k0 + 4 * RPL * i + stage_row, block = paged_block(a, key);
    entry[i] = 4 * block;
    off[i] = (key - block * a.page) * (uint32_t)a.slot_stride;
  }
  auto look_row = [&](int i, int (&page)[LOADS]) __attribute__((always_inline)) {
    page[i] = *reinterpret_cast<const int*>(reinterpret_cast<const char*>(table) + min(entry[i], last_entry));
  };
  auto look = [&](int (&page)[LOADS]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) look_row(i, page);
  };
  // to the next tile's entries and offsets
  auto advance = [&] {
    if (step_off == 0) {  // whole pages a tile
#pragma unroll
      for (int i = 0; i < LOADS; ++i) entry[i] += 4 * step_blocks;
      return;
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      off[i] += step_off;
      const bool over = off[i] >= page_span;
      off[i] -= over ? page_span : 0;
      entry[i] += 4 * (step_blocks + (over ? 1 : 0));
    }
  };
  auto place = [&](int tile, const int (&page)[LOADS], const uint32_t (&row)[LOADS], long long (&at)[LOADS])
      __attribute__((always_inline)) {
    uint32_t most = page[0];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      most = max(most, (uint32_t)page[i]);
      at[i] = (long long)((unsigned long long)(unsigned)page[i] * (unsigned)a.page_stride + row[i]);
    }
    uint32_t exist = 0xFFFFu, paged = 0xFFFFu;
    if (k0 + 64 * tile + 64 > k1 || __any(most >= (unsigned)a.pages)) {
      exist = paged = 0;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const bool known = (unsigned)page[i] < (unsigned)a.pages;
        if (!known) at[i] = row[i];  // of page 0, and not looked at
        const unsigned long long pages = __ballot(known);
        const unsigned long long lanes = __ballot(known && k0 + 64 * tile + 4 * RPL * i + stage_row < k1);
#pragma unroll
        for (int j = 0; j < RPL; ++j) {
          exist |= (uint32_t)(lanes >> (j * LPR) & 1) << (i * RPL + j);
          paged |= (uint32_t)(pages >> (j * LPR) & 1) << (i * RPL + j);
        }
      }
    }
    if (lane == 0) s.exist[tile & 3][wave] = exist, s.known[tile & 3][wave] = paged;
  };
  const uint32_t lds_k0 = paged_lds(s.k[0]), lds_v0 = paged_lds(s.v[0]);
  auto slot = [](int n) { return n >= 5 ? n - 5 : n; };
  auto fetch_k_row = [&](const long long (&at)[LOADS], int kb, int i) __attribute__((always_inline)) {
    const uint32_t to = lds_k0 + (i < LOADS / 2 ? kb : slot(kb + 1)) * HALFB;
    paged_dma(keys + at[i], __builtin_amdgcn_readfirstlane(to + (4 * (i % (LOADS / 2)) + wave) * 1024));
  };
  auto fetch_v_row = [&](const long long (&at)[LOADS], uint32_t to, int i) __attribute__((always_inline)) {
    paged_dma(values + at[i], __builtin_amdgcn_readfirstlane(to + (4 * i + wave) * 1024));
  };
  auto fetch_k = [&](const long long (&at)[LOADS], int kb) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) fetch_k_row(at, kb, i);
  };
  auto fetch_v = [&](const long long (&at)[LOADS], uint32_t to) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) fetch_v_row(at, to, i);
  };
  // Operands: byte addresses in a tile, XORed with a constant per 16 (K) or 32 (V) dims.
  const uint32_t lds_k = lds_k0 + col * ROWB + ((half ^ swizzle(col)) << 4);
  const int r = lane & 15, v_row = 4 * half + (r >> 2);
  const uint32_t lds_v =
      lds_v0 + v_row * ROWB + (((2 * (lane >> 4 & 1) + (r & 3) / 2) ^ swizzle(v_row)) << 4) + (r & 1) * 8;
  auto read_k = [&](uint32_t base, int d) { return *(const paged_lds_bf16x8*)(uintptr_t)(base ^ (d << 5)); };
  auto read_v = [&](uint32_t base, int kt, int d) {  // keys 16 kt .. of the tile
    const pa_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s16x4*)((base ^ (d << 6)) + kt * (16 * ROWB)));
    const pa_s16x4 hi =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s16x4*)((base ^ (32 | d << 6)) + kt * (16 * ROWB) + 8 * ROWB));
    const pa_s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(fa_bf16x8, both);
  };

  float run_max = -INFINITY, run_sum = 0.f, ref = 0.f;
  fa_f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    o[d] = fa_f32x16{};
    asm("" : "+a"(o[d]));  // in the accumulation registers, here and wherever else than a product changes it
  }
  fa_f32x16 sc;                            // scores of the present 32 keys
  float top;                               // their maximum, over this lane's
  constexpr int AHEAD = 2;                 // products that operands are read ahead; 3 measured the same
  fa_bf16x8 kf[AHEAD + 1], vf[AHEAD + 1];  // operands on their way

  auto top_of = [&] {
    top = sc[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, sc[e]);
  };
  // Whether every row sees every key of tile t.
  auto whole = [&](int t) {
    const uint32_t exist = s.exist[t & 3][0] & s.exist[t & 3][1] & s.exist[t & 3][2] & s.exist[t & 3][3];
    return __builtin_amdgcn_readfirstlane(exist == 0xFFFFu && k0 + 64 * t + 64 <= least) != 0;
  };
  // The scores that a row may not see, or that are of no page, leave; then the maximum.
  auto mask = [&](int t, int sub) {
    if (whole(t)) return;
    const int j0 = k0 + 64 * t + 32 * sub + 4 * half;
    const int sees = limit - j0;
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = 8 * (e >> 2) + (e & 3) < sees ? sc[e] : -INFINITY;
    const uint32_t known = s.known[t & 3][0] & s.known[t & 3][1] & s.known[t & 3][2] & s.known[t & 3][3];
    if (__builtin_amdgcn_readfirstlane(known) != 0xFFFFu) {
      uint32_t hidden = 0;  // of this lane's 16 keys
#pragma unroll 1
      for (int e = 0; e < 16; ++e) {
        const int k = 32 * sub + 8 * (e >> 2) + 4 * half + (e & 3);
        hidden |= (~s.known[t & 3][k / RPL % 4] >> (k / (4 * RPL) * RPL + k % RPL) & 1) << e;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = hidden >> e & 1 ? -INFINITY : sc[e];
    }
    top_of();
  };
  // the exponentials' reference moves only where a score passes it, and then 2^8 ahead; O and the sum follow
  auto move = [&] {
    const float most = xor32_max(top) * c2;
    const float moved = most > run_max ? most + 8.f : run_max;
    // (nothing to scale yet where there was no reference)
    const float keep = moved == run_max || run_max == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(run_max - moved);
    run_max = moved;
    ref = moved == -INFINITY ? 0.f : moved;
    if (__any(keep != 1.f)) {
      acc_settle();
      run_sum *= keep;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x = o[d][e];
          acc_scale(x, keep);
          o[d][e] = x;
        }
      acc_settle();
    }
  };
  // Keys 32 sub .. of tile t (their scores in sc); then, with K of 32 keys at k_base (operands 0 and 1 in kf), the
  // scores of those; the first operands at kn_base follow into kf.
  // `beside(i)`: what else goes among the products, i of DS + 2 DT times.
  auto step = [&](uint32_t v_base, int sub, uint32_t k_base, uint32_t kn_base, auto beside)
      __attribute__((always_inline)) {
    constexpr int START = DS == 8 ? 2 : 1;           // products after which the reference is settled
    constexpr int PER = 6 / (DS - START);            // pairs of exponentials after each of the others
    uint32_t pk[2][4];
    auto pair = [&](int u) {  // pair u of 8: k-step u / 4
      const int e = 8 * (u >> 2) + 2 * (u & 3);
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], c2, -ref));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e + 1], c2, -ref));
      pk[u >> 2][u & 3] = cvt_pk_bf16(p0, p1);
      run_sum = dot2_bf16(pk[u >> 2][u & 3], 0x3F803F80u, run_sum);  // the rounded weights' sum
    };
    fa_f32x16 next = fa_f32x16{};
#pragma unroll
    for (int d = 0; d < DS; ++d) {
      constexpr int RING = AHEAD + 1;
      if (d + AHEAD < DS) kf[(d + AHEAD) % RING] = read_k(k_base, d + AHEAD);
      else vf[d + AHEAD - DS] = read_v(v_base, 2 * sub + (d + AHEAD - DS) / DT, (d + AHEAD - DS) % DT);
      next = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[d % RING], qf[d], next, 0, 0, 0);
      if (d >= START)
#pragma unroll
        for (int u = (d - START) * PER; u < (d - START + 1) * PER; ++u) pair(u);
      beside(d);
      if (d == START - 1) {
        move();
        __builtin_amdgcn_s_setprio(1);  // ahead of the SIMD's other wave where that stages or waits (284 -> 277 us)
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    float most = -INFINITY;
#pragma unroll
    for (int m = 0; m < 2 * DT; ++m) {
      const int kt = m / DT, d = m % DT;
      constexpr int RING = AHEAD + 1;
      if (m + AHEAD < 2 * DT) vf[(m + AHEAD) % RING] = read_v(v_base, 2 * sub + (m + AHEAD) / DT, (m + AHEAD) % DT);
      else kf[m + AHEAD - 2 * DT] = read_k(kn_base, m + AHEAD - 2 * DT);
      const uint32_t w[4] = {pk[kt][0], pk[kt][1], pk[kt][2], pk[kt][3]};
      o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[m % RING], __builtin_bit_cast(fa_bf16x8, w), o[d], 0, 0, 0);
      if (kt == 0)
#pragma unroll
        for (int u = 6 + 2 * d / DT; u < 6 + 2 * (d + 1) / DT; ++u) pair(u);
      // 8 / DT of the first (second) eight of the next scores
#pragma unroll
      for (int i = 0; i < 8 / DT; ++i) {
        const int e = 8 * kt + d * (8 / DT) + i;
        float x = next[e];
        asm("" : "+v"(x));  // out of its accumulator once, here
        sc[e] = x;
        most = fmaxf(most, x);
      }
      beside(DS + m);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    // what the next step needs is done in this one, among its products
    top = most;
    asm volatile("" : "+v"(run_sum), "+v"(top));
  };
  // V of tile t in LDS, where some of its rows do not exist or are not seen by every row: zeros for the former; for the
  // latter what is not finite goes (0 * inf) and is added at the end of the tile, row by row
  auto tidy = [&](int t) {
    const uint32_t exist = s.exist[t & 3][wave];
    const bool partial = least < k1 && k0 + 64 * t + 64 > least;
    uint32_t special = 0;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      uint4* at = reinterpret_cast<uint4*>(s.v[t & 1] + (4 * i + wave) * 512 + 8 * lane);
      uint4 v = *at;
      if (!(exist >> (i * RPL + lane / LPR) & 1)) v = make_uint4(0, 0, 0, 0);
      if (partial) {
        const unsigned long long lanes = __ballot(chunk_special(v));
        v = chunk_finite(v);
#pragma unroll
        for (int j = 0; j < RPL; ++j)
          special |= (uint32_t)((lanes >> (j * LPR) & ((1ull << LPR) - 1)) != 0) << (i * RPL + j);
      }
      *at = v;
    }
    if (lane == 0) s.special[wave] = special;
  };
  auto add_special = [&](int t) {
    acc_settle();
    for (int w = 0; w < 4; ++w) {
      uint32_t special = __builtin_amdgcn_readfirstlane(s.special[w]);
      while (special) {
        const int b = __ffs(special) - 1;
        special &= special - 1;
        const int k = k0 + 64 * t + (4 * (b / RPL) + w) * RPL + b % RPL;
        const uint16_t* v = a.values + kvh * a.head_stride + paged_row(a, table, k) + 4 * half;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint2 x = *reinterpret_cast<const uint2*>(v + 32 * d + 8 * g);
            const float add[4] = {special_lo(x.x), special_hi(x.x), special_lo(x.y), special_hi(x.y)};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float y = o[d][4 * g + i];
              acc_add(y, k < limit ? add[i] : 0.f);
              o[d][4 * g + i] = y;
            }
          }
      }
    }
    acc_settle();
  };

  // At tile t: K of tile t's second half and of tile t + 1 and V of tile t are in LDS, the scores of tile t's first 32
  // keys in sc; K of tile t + 2 goes to the two free slots and V of tile t + 1 to the buffer of tile t - 1 while it
  // runs, and the rows of tile t + 3 are looked up.
  long long at_k[LOADS], at_v[LOADS];
  if (tiles > 0) {
    int now[LOADS], then[LOADS];
    uint32_t row_now[LOADS], row_then[LOADS];
    look(now);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) row_now[i] = off[i];
    advance();
    look(then);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) row_then[i] = off[i];
    advance();
    look(ahead);
    place(0, now, row_now, at_v);
    fetch_k(at_v, 0);
    fetch_v(at_v, lds_v0);
    place(1, then, row_then, at_v);
    fetch_k(at_v, 2);
    place(2, ahead, off, at_k);
    advance();
    paged_landed();
    __syncthreads();
    if (active) {
      sc = fa_f32x16{};
#pragma unroll
      for (int d = 0; d < DS; ++d) {
        const fa_bf16x8 k = read_k(lds_k, d);
        sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, qf[d], sc, 0, 0, 0);
      }
      top_of();
      mask(0, 0);
#pragma unroll
      for (int d = 0; d < AHEAD; ++d) kf[d] = read_k(lds_k + HALFB, d);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float x = sc[e];
        asm("" : "+v"(x));
        sc[e] = x;
      }
    }
    __syncthreads();  // the first half has been read by all: tile 2 goes there
  }
  auto stage = [&](int t, int kb) {
    fetch_k(at_k, slot(kb + 4));
    fetch_v(at_v, lds_v0 + ((t + 1) & 1) * TILEB);
    look(ahead);
  };
  auto staged = [&](int t) {
    paged_landed();
#pragma unroll
    for (int i = 0; i < LOADS; ++i) at_v[i] = at_k[i];
    place(t + 3, ahead, off, at_k);
    advance();
    __syncthreads();
  };
  // The two steps of a tile. `edge` (a compile-time bool): keys that a row may not see or that are of no page may be
  // among those of this tile and the next one's; without it there is no branch but the reference's move.
  auto tile = [&](int t, int kb, auto edge) __attribute__((always_inline)) {
    const uint32_t vb = lds_v + (t & 1) * TILEB, to_v = lds_v0 + ((t + 1) & 1) * TILEB;
    const uint32_t kn = lds_k + slot(kb + 2) * HALFB;
    step(vb, 0, lds_k + slot(kb + 1) * HALFB, kn, [&](int i) __attribute__((always_inline)) {
      if (i < LOADS) fetch_k_row(at_k, slot(kb + 4), i);
      else if (i < 2 * LOADS) fetch_v_row(at_v, to_v, i - LOADS);
      else if (i < 3 * LOADS) look_row(i - 2 * LOADS, ahead);
    });
    if constexpr (decltype(edge)::value) mask(t, 1);
    step(vb, 1, kn, lds_k + slot(kb + 3) * HALFB, [](int) {});
    if constexpr (decltype(edge)::value)
      if (t + 1 < tiles) mask(t + 1, 0);
  };
  auto after = [&](int kb) { return slot(kb + 2); };
  paged_landed();     // on the way past the block above too
  int t = 0, kb = 0;  // kb = 2 t % 5
  if (!active) {
    for (; t < tiles; ++t, kb = after(kb)) {
      stage(t, kb);
      if (!whole(t)) {
        tidy(t);
        __syncthreads();
      }
      staged(t);
    }
    return;
  }
  for (bool easy = tiles > 1 && whole(0) && whole(1); easy; ++t, kb = after(kb)) {
    // written before the last barrier, for the next tile
    const uint4 one = *reinterpret_cast<const uint4*>(s.exist[(t + 1) & 3]);
    const uint4 two = *reinterpret_cast<const uint4*>(s.exist[(t + 2) & 3]);
    tile(t, kb, std::false_type{});
    const uint32_t exist = one.x & one.y & one.z & one.w & two.x & two.y & two.z & two.w;
    easy = t + 2 < tiles && k0 + 64 * t + 192 <= least && __builtin_amdgcn_readfirstlane(exist) == 0xFFFFu;
    staged(t);
  }
  for (; t < tiles; ++t, kb = after(kb)) {  // the last tiles, and all from one on that has a row without a page
    const bool care = !whole(t);
    if (care) {
      tidy(t);
      __syncthreads();
    }
    tile(t, kb, std::true_type{});
    if (care) add_special(t);
    staged(t);
  }

  const float sum = xor32_sum(run_sum);
  if (row >= live) return;
  const bool none = run_max == -INFINITY && sum == 0.f && k0 < limit;
  if (__builtin_expect(__any(none), 0))
    if (none && paged_sees(a, table, k0, limit)) run_max = kPagedNoWeight;
  float probe = 0.f;  // NaN where an element of O is not finite
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) probe = __builtin_fmaf(o[d][e], 0.f, probe);
  float* rec = unit.parts > 1 ? paged_record(a, unit.record + unit.part, kvh, row, D) : nullptr;
  uint16_t* to = a.out + ((size_t)(unit.begin + token) * a.query_heads + kvh * group + head) * D + 4 * half;
  if (unit.parts > 1) {
    if (half == 0) rec[0] = run_max, rec[1] = sum;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float2* at = reinterpret_cast<float2*>(rec + 2 + 32 * d + 8 * g + 4 * half);
        at[0] = make_float2(o[d][4 * g], o[d][4 * g + 1]);
        at[1] = make_float2(o[d][4 * g + 2], o[d][4 * g + 3]);
        __builtin_amdgcn_sched_barrier(0);
      }
  } else {
    const float inv = paged_inverse(run_max, sum);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        *reinterpret_cast<uint2*>(to + 32 * d + 8 * g) =
            make_uint2(cvt_pk_bf16(o[d][4 * g] * inv, o[d][4 * g + 1] * inv),
                       cvt_pk_bf16(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv));
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  if (__builtin_expect(__any(probe != probe && sum == sum), 0)) {
    // special values in the place of NaN, in what this lane has just written
#pragma unroll 1
    for (int c = 0; c < D / 8; ++c) {
      float2* at = reinterpret_cast<float2*>(rec + 2 + 8 * c + 4 * half);
      uint2* out = reinterpret_cast<uint2*>(to + 8 * c);
      f32x4_t v;
      if (unit.parts > 1) v = f32x4_t{at[0].x, at[0].y, at[1].x, at[1].y};
      else v = f32x4_t{bf16_lo(out->x), bf16_hi(out->x), bf16_lo(out->y), bf16_hi(out->y)};
      if (!paged_any_nan(v) || sum != sum) continue;
      v = paged_with_special(v, paged_special(a, table, a.values + kvh * a.head_stride + 8 * c + 4 * half, k0, limit));
      if (unit.parts > 1) at[0] = make_float2(v[0], v[1]), at[1] = make_float2(v[2], v[3]);
      else *out = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    }
  }
}

// ------------------------------------------------------------------------------------------------------- the blocks
template <int D, int NT>
__device__ void paged_attention_narrow(const PagedAttentionArgs& a) {
  __shared__ __attribute__((aligned(16))) PagedNarrowShared<D, NT> s;
  const int kvh = blockIdx.x % a.kv_heads;
  PagedWalk<false> walk;
  if (!walk.start(a, blockIdx.x / a.kv_heads)) return;
  for (PagedUnit unit; walk.next(a, unit); __syncthreads()) {
    paged_note(a, unit, kvh);
    paged_narrow<D, NT>(a, unit, kvh, s);
  }
}

template <int D>
__device__ void paged_attention_mixed(const PagedAttentionArgs& a) {
  __shared__ __attribute__((aligned(256))) union {  // the wide form's addresses are XORed within a row
    PagedNarrowShared<D, 1> narrow;
    PagedWideShared<D> wide;
  } s;
  const int kvh = blockIdx.x % a.kv_heads;
  PagedWalk<true> walk;
  if (!walk.start(a, blockIdx.x / a.kv_heads)) return;
  for (PagedUnit unit; walk.next(a, unit); __syncthreads()) {
    paged_note(a, unit, kvh);
    if (unit.narrow) paged_narrow<D, 1>(a, unit, kvh, s.narrow);
    else paged_wide<D>(a, unit, kvh, s.wide);
  }
}

// A wave joins the parts of one row (32 to 80 tokens of 32 heads: 5 us with its launch): with m the largest maximum,
// out = sum 2^(m_s - m) o_s / sum 2^(m_s - m) l_s. Bound by latency: the note, then eight records at a time in one
// round trip.
template <int D>
__device__ void paged_attention_join(const PagedAttentionArgs& a) {
  constexpr int PER = D / 64, SOME = 8;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int t = row / a.query_heads, h = row % a.query_heads;
  if (t >= a.tokens) return;
  const int4 note = reinterpret_cast<const int4*>(a.joins)[t];
  if (t < a.query_start[0] || t >= a.query_start[a.requests] || note.y <= 1) return;
  // no note where query_start decreases
  if (note.x < 0 || note.y > a.units || note.x > a.units - note.y || (unsigned)note.z >= (unsigned)a.record_rows)
    return;
  const int group = a.query_heads / a.kv_heads, kvh = h / group, at = note.z + h % group;
  const size_t step = (size_t)a.kv_heads * a.record_rows * (D + 2);
  const float* rec = paged_record(a, note.x, kvh, at, D);
  float big = -INFINITY, sum = 0.f, acc[PER] = {};
  for (int s0 = 0; s0 < note.y; s0 += SOME) {
    float m[SOME], l[SOME], o[SOME][PER];
#pragma unroll
    for (int i = 0; i < SOME; ++i) {
      const float* from = rec + min(s0 + i, note.y - 1) * step;
      m[i] = from[0], l[i] = from[1];
#pragma unroll
      for (int e = 0; e < PER; ++e) o[i][e] = from[2 + PER * lane + e];
    }
    float top = big;
#pragma unroll
    for (int i = 0; i < SOME; ++i) {
      if (s0 + i >= note.y) {
        m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < PER; ++e) o[i][e] = 0.f;
      }
      top = fmaxf(top, m[i]);
    }
    const float keep = big == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(big - top);
    big = top;
    sum *= keep;
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = paged_scaled(acc[e], keep);
#pragma unroll
    for (int i = 0; i < SOME; ++i) {
      const float f = m[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[i] - big);
      sum += f * l[i];  // NaN of a part whose scores are all NaN, too
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[e] += paged_scaled(o[i][e], f);
    }
  }
  const float inv = paged_inverse(big, sum);
  uint16_t* out = a.out + ((size_t)t * a.query_heads + h) * D + PER * lane;
  if constexpr (PER == 2) *reinterpret_cast<uint32_t*>(out) = cvt_pk_bf16(acc[0] * inv, acc[1] * inv);
  else out[0] = (uint16_t)f32_to_bf16(acc[0] * inv);
}

}  // namespace aoto

#define AOTO_PAGED_ATTENTION(D)                                                                                    \
  extern "C" __global__ __launch_bounds__(256, 2) void aoto_paged_attention_d##D##_n1(PagedAttentionArgs a) {      \
    aoto::paged_attention_narrow<D, 1>(a);                                                                         \
  }                                                                                                                \
  extern "C" __global__ __launch_bounds__(256, 2) void aoto_paged_attention_d##D##_n2(PagedAttentionArgs a) {      \
    aoto::paged_attention_narrow<D, 2>(a);                                                                         \
  }                                                                                                                \
  extern "C" __global__ __launch_bounds__(256, 2) void aoto_paged_attention_d##D##_w(PagedAttentionArgs a) {       \
    aoto::paged_attention_mixed<D>(a);                                                                             \
  }                                                                                                                \
  extern "C" __global__ __launch_bounds__(256) void aoto_paged_attention_join_d##D(PagedAttentionArgs a) {         \
    aoto::paged_attention_join<D>(a);                                                                              \
  }
