// Attention of requests' new tokens over their pages of a cache held in 4 bits (paged_mx4.h). What is computed, how the
// work is cut and how parts are joined is the bf16 cache's (paged_attention.h); a row of 128 dims is 68 bytes here
// instead of 256, and there are no infinities among the values.
//
// Narrow tiles (decodes, drafted tokens) are bound by the read: codes become bf16, exactly, in registers. Wide tiles
// (chunks of prompts) are bound by issue: their K stays in 4 bits up to the matrix units, which take it beside an 8-bit
// Q (v_mfma_scale_f32_32x32x64_f8f6f4). A bf16 q is two 8-bit numbers: its upper four bits of mantissa and the rest,
// with a scale for each 32 dims (to 2^-22 of the largest of them), in two products, at the rate of one in bf16. V
// becomes bf16 on its way to LDS, once for the four waves.
//
// Roundings of wide tiles. The weights are rounded once to bf16, for the product and for the sum alike, as the bf16
// cache's: one product with V instead of two, half of which takes 35 of 229 us. That unit brings eight products to the
// exponent of the largest of them and keeps 13 bits below it (and adds to f32), so a score is off by at most 2^-13 of
// those largest products, eight each. Beside the codes' own half steps that is little: against 64 bits the outputs are
// as far off as the bf16 cache's wide tiles are on the same values, for single products (0.0023 each, relative, all
// elements), for heads sharpened 4 and 16 times (0.0018, 0.0013) and with a dim 100 x 30 in every key and row (0.0022
// to 0.0023); with one of 30 x 20 0.0024 and 0.0023 to 0.0024.
#pragma once

#include "paged_attention.h"
#include "paged_mx4.h"

namespace aoto {

typedef int mx4_i32x8 __attribute__((ext_vector_type(8)));

// Where a page's row begins. The host sees to page strides below 2^32 and pages that span less than 2^30 bytes.
AOTO_DEVICE long long mx4_at(unsigned page, long long page_stride, int row, long long slot_stride) {
  return (long long)((unsigned long long)page * (unsigned)page_stride + (unsigned)(row * (int)slot_stride));
}

// ---------------------------------------------------------------------------------------------------- narrow tiles
// As paged_narrow, whose layouts and softmax these are. A lane has D / 4 neighbouring dims of the keys it loads, 16 (8)
// bytes and one scale byte: the k slots of the first product hold the dims in that order, in K and in Q.
//
// Single tokens of 64 requests, 32 / 8 heads of 128, 345000 keys: 375 MB in 82 us (4.6 TB/s), 79 where only the loads
// are left (in bf16 the keys and values are 1.41 GB). Two tiles of loads on their way instead of one gave nothing.
template <int D, int NT>
AOTO_DEVICE void paged_mx4_narrow(const PagedMx4AttentionArgs& args, const PagedUnit& unit, int kvh,
                                  PagedNarrowShared<D, NT>& s) {
  const PagedAttentionArgs& a = args.base;
  const PagedMx4Cache& cache = args.cache;
  constexpr int DC = D / 32, DT = D / 16, STR = PagedNarrowShared<D, NT>::STR;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int group = a.query_heads / a.kv_heads;
  const int live = unit.tokens * group;  // rows in use; the others repeat the last
  const int* table = a.block_tables + unit.request * a.table_stride;
  const uint8_t* keys = cache.keys + kvh * cache.head_stride + quad * (D / 8);
  const uint8_t* values = cache.values + kvh * cache.head_stride + quad * (D / 8);
  const int scale_of = quad * (D / 4) / 32;
  const uint8_t* key_scales = cache.key_scales + kvh * cache.scale_head_stride + scale_of;
  const uint8_t* value_scales = cache.value_scales + kvh * cache.scale_head_stride + scale_of;
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
    const uint16_t* q =
        a.q + (unit.begin + i) * a.q_token_stride + (kvh * group + g) * a.q_head_stride + quad * (D / 4);
#pragma unroll
    for (int c = 0; c < DC; ++c) qf[t][c] = *reinterpret_cast<const fa_bf16x8*>(q + 8 * c);
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

  // This lane loads keys col and 16 + col of a tile. Their pages are looked up two tiles ahead, their rows one.
  struct Rows {
    int page[2], row[2];
  };
  struct Tile {
    uint32_t k[2][DC], v[2][DC];
    uint8_t ks[2], vs[2];
    bool paged[2];
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
  auto words = [](const uint8_t* from, uint32_t (&to)[DC]) {
    if constexpr (D == 128) {
      const uint4 w = *reinterpret_cast<const uint4*>(from);
      to[0] = w.x, to[1] = w.y, to[2] = w.z, to[3] = w.w;
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(from);
      to[0] = w.x, to[1] = w.y;
    }
  };
  auto fetch = [&](const Rows& of, Tile& to) {
    long long at[2], scale_at[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      to.paged[g] = (unsigned)of.page[g] < (unsigned)a.pages;
      const unsigned page = to.paged[g] ? of.page[g] : 0;
      at[g] = mx4_at(page, cache.page_stride, of.row[g], cache.slot_stride);
      scale_at[g] = mx4_at(page, cache.scale_page_stride, of.row[g], cache.scale_slot_stride);
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) words(keys + at[g], to.k[g]), to.ks[g] = key_scales[scale_at[g]];
#pragma unroll
    for (int g = 0; g < 2; ++g) words(values + at[g], to.v[g]), to.vs[g] = value_scales[scale_at[g]];
  };
  Rows ahead;
  Tile tile;
  if (trips > 0) {
    const Rows now = look(mine);
    ahead = look(mine + 128);
    fetch(now, tile);
  }
  for (int trip = 0; trip < trips; ++trip) {
    const int base = mine + 128 * trip;
    f32x4_t sc[NT][2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const float scale = mx4_scale(tile.ks[g]);
#pragma unroll
      for (int t = 0; t < NT; ++t) sc[t][g] = f32x4_t{};
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        const fa_bf16x8 k = __builtin_bit_cast(fa_bf16x8, mx4_unpack(tile.k[g][c], scale));
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[t][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, qf[t][c], sc[t][g], 0, 0, 0);
      }
    }
    // the keys of this tile that exist, one bit each; their values to LDS, zeros for the others
    bool there[2];
    uint32_t exist = 0;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      there[g] = tile.paged[g] && base + 16 * g + col < k1;
      exist |= (uint32_t)(__ballot(there[g]) & 0xFFFFu) << (16 * g);
    }
    const bool whole = exist == 0xFFFFFFFFu && base + 32 <= least;
    // by lane: groups of keys, not seen by every row, that stand for NaN; added row by row below
    unsigned long long special[2] = {0, 0};
    if (!whole && least < k1 && base + 32 > least) {
#pragma unroll
      for (int g = 0; g < 2; ++g) special[g] = __ballot(there[g] && tile.vs[g] > 252);
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const bool none = !there[g] || (special[g] && tile.vs[g] > 252);
      const float scale = mx4_scale(none ? 0 : tile.vs[g]);
#pragma unroll
      for (int c = 0; c < DC; ++c)
        *reinterpret_cast<uint4*>(vs + (16 * g + col) * STR + quad * (D / 4) + 8 * c) =
            mx4_unpack(none ? 0u : tile.v[g][c], scale);
    }
    // the next tile's loads, then the lookup of the tile after it
    if (trip + 1 < trips) {
      fetch(ahead, tile);
      ahead = look(base + 256);
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
      // The exponentials' reference moves only where a weight is above 1 (or NaN, as a row's without a reference are),
      // and then 2^8 ahead of the largest score: in most tiles no maximum stands before the exponentials.
      float p[8];
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][j >> 2][j & 3], c2, -run_max[t]));
        most = max(most, __float_as_uint(p[j]));
      }
      if (__any(most > 0x3F800000u)) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, sc[t][j >> 2][j & 3]);
        top = xor32_max(xor16_max(top)) * c2;
        const float moved = top > run_max[t] ? top + 8.f : run_max[t];
        const bool kept = moved == run_max[t] || run_max[t] == -INFINITY;
        const float keep = kept ? 1.f : __builtin_amdgcn_exp2f(run_max[t] - moved);
        run_max[t] = moved;
        run_sum[t] *= keep;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] *= keep;
        const float by = moved == -INFINITY ? 0.f : moved;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][j >> 2][j & 3], c2, -by));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) run_sum[t] += p[j];
      // 16 bits of a weight: its upper half cut off and the rest rounded, in two products
      uint32_t high[4], low[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        high[j] = __builtin_amdgcn_perm(__float_as_uint(p[2 * j + 1]), __float_as_uint(p[2 * j]), 0x07060302u);
        low[j] = cvt_pk_bf16(p[2 * j] - bf16_lo(high[j]), p[2 * j + 1] - bf16_hi(high[j]));
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
#pragma unroll
    for (int g = 0; g < 2; ++g)
      while (special[g]) {
        const int from = __ffsll(special[g]) - 1;  // the lane: key 16 g + from % 16, dims (from / 16) D / 4 ..
        special[g] &= special[g] - 1;
        const int k = base + 16 * g + (from & 15), first = (from >> 4) * (D / 4);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int t = 0; t < NT; ++t)
            if (k < limit[t] && 16 * d >= first && 16 * d < first + D / 4) o[t][d] += NAN;
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
    if (__builtin_expect(__any(big == -INFINITY && sum == 0.f), 0)) {
      const int sees = min(k1, unit.first + unit.token + row / group);
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
// 64 keys at a time, their scores 32 by 32: the products of the next 32 keys' scores and the exponentials of the
// present ones are written in turns, as the matrix units and the others then work side by side (one after the other:
// 273 us instead of 242 for what follows).
//
// 2048 tokens over the 6000 before them, 32 / 8 heads of 128, 236 GFLOP: 230 us among 200 calls without a pause, 1020
// TFLOP/s, where a large matrix product of bf16 reaches 1400; 270 to 290 us for single calls after pauses, 820 to 870
// TFLOP/s, and the product 1250 to 1320. Left out for the timing, of 229 us q's low parts take 20, the exponentials 30,
// half of the products with V 35, reading V from LDS 11, V's conversion nothing.
template <int D>
struct PagedMx4WideShared {
  uint16_t v[2][64 * D];       // pieces of 16 bytes of a row in the order of paged_wide
  uint8_t k[3][64 * D / 2];    // codes
  uint8_t ks[3][64 * D / 32];  // scale bytes
  uint32_t exist[4][4];        // by tile and staging wave: which of its 16 rows exist (a page, and not past the end)
  unsigned long long special[2][4];  // groups, not seen by every row, that stand for NaN, by lane of the staging wave
};

// Two 8-bit numbers for each of 16 dims of q, x = high + low / 32, before the group's scale 2^(byte - 127).
AOTO_DEVICE void mx4_split(const uint32_t (&w)[8], uint32_t byte, int* high, int* low) {
  // the group's largest magnitude becomes one of 128 .. 256; high is off by 8 at most
  const float by = __uint_as_float((254u - byte) << 23);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[4] = {bf16_lo(w[2 * i]) * by, bf16_hi(w[2 * i]) * by, bf16_lo(w[2 * i + 1]) * by,
                  bf16_hi(w[2 * i + 1]) * by};
    int h = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    h = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], h, true);
    const float r[4] = {(x[0] - __builtin_amdgcn_cvt_f32_fp8(h, 0)) * 32.f,
                        (x[1] - __builtin_amdgcn_cvt_f32_fp8(h, 1)) * 32.f,
                        (x[2] - __builtin_amdgcn_cvt_f32_fp8(h, 2)) * 32.f,
                        (x[3] - __builtin_amdgcn_cvt_f32_fp8(h, 3)) * 32.f};
    int l = __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false);
    l = __builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], l, true);
    high[i] = h, low[i] = l;
  }
}

// 32 keys' scores over 64 dims of one of q's parts. KEY, Q: which byte of a lane's scales is the product's.
template <int KEY, int Q>
AOTO_DEVICE fa_f32x16 mx4_product(const uint4& k, uint32_t ks, const mx4_i32x8& q, int qs, const fa_f32x16& sum) {
  constexpr int FP4 = 4, FP8 = 0;
  const mx4_i32x8 codes = {(int)k.x, (int)k.y, (int)k.z, (int)k.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(codes, q, sum, FP4, FP8, KEY, (int)ks, Q, qs);
}

// The larger of two pairs of positive bf16: their bits are in the order of their values.
AOTO_DEVICE uint32_t mx4_larger(uint32_t a, uint32_t b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

template <int D>
AOTO_DEVICE void paged_mx4_wide(const PagedMx4AttentionArgs& args, const PagedUnit& unit, int kvh,
                                PagedMx4WideShared<D>& s) {
  const PagedAttentionArgs& a = args.base;
  const PagedMx4Cache& cache = args.cache;
  constexpr int KS = D / 64, DT = D / 32, ROWB = 2 * D, TILEB = 64 * ROWB;
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
  const int limit = min(k1, unit.first + token);
  const int least = min(k1, unit.first + unit.token);  // keys that every row of the block sees
  const float c2 = a.scale * 1.4426950408889634f;

  // Q: the matrix units take dims 64 s + 16 half .. and 64 s + 32 + 16 half .. of step s from this lane, and the scale
  // of the 32 dims from 64 s + 32 half on.
  mx4_i32x8 qh[KS], ql[KS];
  int q_scale[KS];
  {
    const uint16_t* q =
        a.q + (unit.begin + token) * a.q_token_stride + (kvh * group + head) * a.q_head_stride + 16 * half;
#pragma unroll
    for (int st = 0; st < KS; ++st) {
      uint32_t byte[2];
      int high[8], low[8];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint4 x = *reinterpret_cast<const uint4*>(q + 64 * st + 32 * b);
        const uint4 y = *reinterpret_cast<const uint4*>(q + 64 * st + 32 * b + 8);
        const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, max(w[i] << 16 & 0x7FFFFFFFu, w[i] & 0x7FFF0000u));
        const auto both = __builtin_amdgcn_permlane32_swap(most, most, false, false);
        most = max((uint32_t)both[0], (uint32_t)both[1]);
        // the low numbers' scale is 2^-5 of it
        byte[b] = (uint32_t)max((int)(most >> 23) - 7, 6);
        mx4_split(w, byte[b], high + 4 * b, low + 4 * b);
        if (most >= 0x7F800000u) byte[b] = 255u;  // an infinity or NaN in q: its scores are NaN
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) qh[st][i] = high[i], ql[st][i] = low[i];
      const uint32_t mine = half ? byte[1] : byte[0];
      q_scale[st] = (int)(mine | (mine == 255u ? 255u : mine - 5u) << 8);
    }
  }

  // Staging: this thread has D / 4 neighbouring dims of row 16 wave + lane % 16 of a tile (the conversions' writes of
  // eight lanes then spread over all banks).
  const int srow = 16 * wave + (lane & 15), part = lane >> 4;
  auto swizzle = [](int r) { return D == 128 ? (r & 3) << 2 | (r >> 2 & 3) : (r >> 1 & 1) << 2 | (r >> 2 & 3); };
  const uint8_t* keys = cache.keys + kvh * cache.head_stride + part * (D / 8);
  const uint8_t* values = cache.values + kvh * cache.head_stride + part * (D / 8);
  const int scale_of = part * (D / 4) / 32;
  const uint8_t* key_scales = cache.key_scales + kvh * cache.scale_head_stride + scale_of;
  const uint8_t* value_scales = cache.value_scales + kvh * cache.scale_head_stride + scale_of;
  constexpr int W = D / 32;  // words of codes
  struct Row {               // of a tile: where it is
    long long at, scale_at;
    bool paged;
  };
  struct Codes {
    uint32_t w[W];
    uint32_t scale;
  };
  int ahead_page, ahead_row;
  auto look = [&](int t) {
    const int key = min(k0 + 64 * t + srow, k1 - 1), block = paged_block(a, key);
    ahead_page = table[block];
    ahead_row = key - block * a.page;
  };
  auto place = [&](Row& to) {
    to.paged = (unsigned)ahead_page < (unsigned)a.pages;
    const unsigned page = to.paged ? ahead_page : 0;
    to.at = mx4_at(page, cache.page_stride, ahead_row, cache.slot_stride);
    to.scale_at = mx4_at(page, cache.scale_page_stride, ahead_row, cache.scale_slot_stride);
  };
  auto fetch = [&](const uint8_t* codes, const uint8_t* scales, const Row& of, Codes& to) {
    if constexpr (D == 128) {
      const uint4 w = *reinterpret_cast<const uint4*>(codes + of.at);
      to.w[0] = w.x, to.w[1] = w.y, to.w[2] = w.z, to.w[3] = w.w;
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(codes + of.at);
      to.w[0] = w.x, to.w[1] = w.y;
    }
    to.scale = scales[of.scale_at];
  };
  auto store_k = [&](int t, int slot, const Row& of, const Codes& k) {
    const uint32_t exist = (uint32_t)(__ballot(of.paged && k0 + 64 * t + srow < k1) & 0xFFFFu);
    if constexpr (D == 128)
      *reinterpret_cast<uint4*>(s.k[slot] + srow * 64 + ((part ^ (srow >> 2 & 3)) << 4)) =
          make_uint4(k.w[0], k.w[1], k.w[2], k.w[3]);
    else
      *reinterpret_cast<uint2*>(s.k[slot] + srow * 32 + 8 * part) = make_uint2(k.w[0], k.w[1]);
    if (D == 128 || (part & 1) == 0)
      s.ks[slot][srow * (D / 32) + scale_of] = (uint8_t)(k.scale > 252 ? 255 : k.scale);
    if (lane == 0) s.exist[t & 3][wave] = exist;
  };
  // V in four (two) pieces; what stands in for its codes and scale where the row is not there, or stands for NaN and is
  // not seen by every row.
  bool v_none;
  float v_scale;
  auto store_v = [&](int t, const Row& of, const Codes& v, int i) __attribute__((always_inline)) {
    const int b = t & 1;
    if (i == 0) {
      const bool there = of.paged && k0 + 64 * t + srow < k1, partial = least < k1 && k0 + 64 * t + 64 > least;
      const unsigned long long special = __ballot(partial && there && v.scale > 252);
      v_none = !there || (partial && v.scale > 252);
      v_scale = mx4_scale(v_none ? 0 : v.scale);
      if (lane == 0) s.special[b][wave] = special;
    }
    char* to = reinterpret_cast<char*>(s.v[b]) + srow * ROWB + (((W * part + i) ^ swizzle(srow)) << 4);
    *reinterpret_cast<uint4*>(to) = mx4_unpack(v_none ? 0u : v.w[i], v_scale);
  };

  float run_max = -INFINITY, run_sum = 0.f, ref = -INFINITY;
  fa_f32x16 sc;  // scores of the present 32 keys
  fa_f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = fa_f32x16{};
  const uint32_t lds_v0 = paged_lds(s.v[0]);
  const int r = lane & 15, v_row = 4 * half + (r >> 2);
  const uint32_t lds_v =
      lds_v0 + v_row * ROWB + (((2 * (lane >> 4 & 1) + (r & 3) / 2) ^ swizzle(v_row)) << 4) + (r & 1) * 8;
  auto read_v = [&](uint32_t base, int kt, int d) {  // keys 16 kt .. of the tile
    const pa_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s16x4*)((base ^ (d << 6)) + kt * (16 * ROWB)));
    const pa_s16x4 hi =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s16x4*)((base ^ (32 | d << 6)) + kt * (16 * ROWB) + 8 * ROWB));
    const pa_s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(fa_bf16x8, both);
  };
  // Operands of the scores of keys 32 sub .. of the tile in slot `slot`, and the i-th of their 2 KS products.
  struct Keys {
    uint4 codes[KS];
    uint32_t scales;
  };
  auto read_keys = [&](int slot, int sub, Keys& to) __attribute__((always_inline)) {
    const int key = 32 * sub + col;
    if constexpr (D == 128) to.scales = *reinterpret_cast<const uint32_t*>(s.ks[slot] + 4 * key) >> (8 * half);
    else to.scales = s.ks[slot][2 * key + half];
#pragma unroll
    for (int st = 0; st < KS; ++st)
      to.codes[st] = D == 128 ? *reinterpret_cast<const uint4*>(s.k[slot] + key * 64 +
                                                                (((2 * st + half) ^ (key >> 2 & 3)) << 4))
                              : *reinterpret_cast<const uint4*>(s.k[slot] + key * 32 + 16 * half);
  };
  auto product = [&](int i, const Keys& k, const fa_f32x16& sum) __attribute__((always_inline)) {
    return i == 0   ? mx4_product<0, 1>(k.codes[0], k.scales, ql[0], q_scale[0], sum)
           : i == 1 ? mx4_product<0, 0>(k.codes[0], k.scales, qh[0], q_scale[0], sum)
           : i == 2 ? mx4_product<2, 1>(k.codes[KS - 1], k.scales, ql[KS - 1], q_scale[KS - 1], sum)
                    : mx4_product<2, 0>(k.codes[KS - 1], k.scales, qh[KS - 1], q_scale[KS - 1], sum);
  };
  // Whether every row sees every key of tile t: uniform, and told so.
  auto whole = [&](int t) {
    const uint32_t exist = s.exist[t & 3][0] & s.exist[t & 3][1] & s.exist[t & 3][2] & s.exist[t & 3][3];
    return __builtin_amdgcn_readfirstlane(exist == 0xFFFFu && k0 + 64 * t + 64 <= least) != 0;
  };
  // The scores of keys 32 sub .. of tile t that a row may not see, or that are of no page, leave.
  auto mask = [&](int t, int sub) {
    if (whole(t)) return;
    const int sees = limit - (k0 + 64 * t + 32 * sub + 4 * half);
    const uint32_t exist = (s.exist[t & 3][2 * sub] | s.exist[t & 3][2 * sub + 1] << 16) >> (4 * half);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int k = 8 * (e >> 2) + (e & 3);
      sc[e] = (exist >> k & 1) && k < sees ? sc[e] : -INFINITY;
    }
  };
  // Two of the weights of the present scores, rounded to what the matrix units take (the sum adds the rounded ones). A
  // row without a reference (-inf) gets infinities or NaN, which lead to one.
  auto pair = [&](int u) __attribute__((always_inline)) {
    return cvt_pk_bf16(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * u], c2, -ref)),
                       __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * u + 1], c2, -ref)));
  };
  // Scores sc of keys 32 sub .. of tile t: their weights go among the products of the scores behind them (operands in
  // `keys`), then their product with V; the keys of the step after it are read at the end. `beside(i)`: what else goes
  // among the products with V, i of 2 DT.
  Keys keys_next;
  auto step = [&](int t, int sub, int later_slot, int later_sub, auto beside) __attribute__((always_inline)) {
    const uint32_t v_base = lds_v + (t & 1) * TILEB;
    uint32_t w[8];
    fa_bf16x8 vf[3];
    fa_f32x16 next = fa_f32x16{};
#pragma unroll
    for (int i = 0; i < 2 * KS; ++i) {
      next = product(i, keys_next, next);
#pragma unroll
      for (int u = 0; u < 4 / KS; ++u) w[4 / KS * i + u] = pair(4 / KS * i + u);
      if (i == 2 * KS - 1) vf[0] = read_v(v_base, 2 * sub, 0), vf[1] = read_v(v_base, 2 * sub, 1);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) asm volatile("" : "+v"(w[u]));
    uint32_t most = w[0];
#pragma unroll
    for (int u = 1; u < 8; ++u) most = mx4_larger(most, w[u]);
    // The reference moves only where a weight is above 1, and then 2^8 ahead of the largest score; O and the sum
    // follow.
    if (__any((most & 0xFFFFu) > 0x3F80u || most > 0x3F80FFFFu)) {
      // a use on this way too: else the products move behind the branch, where the exponentials are not beside them
      asm volatile("" : "+v"(next));
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, sc[e]);
      top = xor32_max(top) * c2;
      const float moved = top > run_max ? top + 8.f : run_max;
      const float keep = moved == run_max || run_max == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(run_max - moved);
      run_max = moved;
      ref = moved == -INFINITY ? 0.f : moved;
      run_sum *= keep;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= keep;
#pragma unroll
      for (int u = 0; u < 8; ++u) w[u] = pair(u);
      ref = run_max;  // none yet: the next scores look for one
    }
#pragma unroll
    for (int m = 0; m < 2 * DT; ++m) {
      const int kt = m / DT, d = m % DT;
      if (m + 2 < 2 * DT) vf[(m + 2) % 3] = read_v(v_base, 2 * sub + (m + 2) / DT, (m + 2) % DT);
      else if (m + 2 == 2 * DT) read_keys(later_slot, later_sub, keys_next);
      const uint32_t x[4] = {w[4 * kt], w[4 * kt + 1], w[4 * kt + 2], w[4 * kt + 3]};
      o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[m % 3], __builtin_bit_cast(fa_bf16x8, x), o[d], 0, 0, 0);
#pragma unroll
      for (int u = 4 / DT * m; u < 4 / DT * (m + 1); ++u)
        run_sum = dot2_bf16(w[u], 0x3F803F80u, run_sum);  // the rounded weights' sum
      beside(m);
      __builtin_amdgcn_sched_barrier(0);
    }
    sc = next;
  };

  // At tile t: K of tiles t and t + 1 and V of tile t are in LDS, K of tile t + 2 and V of tile t + 1 in registers or
  // on their way; they go to LDS while the tile is worked on, and those behind them are asked for.
  Row row_k, row_v;
  Codes code_k, code_v;
  if (tiles > 0) {
    Row first;
    look(0);
    place(first);
    look(1);
    fetch(keys, key_scales, first, code_k);
    fetch(values, value_scales, first, code_v);
    place(row_v);
    look(2);
    store_k(0, 0, first, code_k);
#pragma unroll
    for (int i = 0; i < W; ++i) store_v(0, first, code_v, i);
    fetch(keys, key_scales, row_v, code_k);
    place(row_k);
    look(3);
    store_k(1, 1, row_v, code_k);
    fetch(keys, key_scales, row_k, code_k);
    fetch(values, value_scales, row_v, code_v);
    __syncthreads();
    if (active) {
      sc = fa_f32x16{};
      read_keys(0, 0, keys_next);
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i) sc = product(i, keys_next, sc);
      mask(0, 0);
      read_keys(0, 1, keys_next);
    }
  }
  int slot = 0;  // t mod 3
  auto after = [](int n) { return n == 2 ? 0 : n + 1; };
  // V's words of tile t + 1, K of tile t + 2, then what comes after them.
  auto stage = [&](int t, int i) __attribute__((always_inline)) {
    if (i < W) store_v(t + 1, row_v, code_v, i);
    if (i == W) store_k(t + 2, slot == 0 ? 2 : slot - 1, row_k, code_k);
    if (i == W + 1) {
      row_v = row_k;
      place(row_k);
      fetch(keys, key_scales, row_k, code_k);
      fetch(values, value_scales, row_v, code_v);
      look(t + 4);
    }
  };
  if (!active) {
    for (int t = 0; t < tiles; ++t, slot = after(slot)) {
#pragma unroll
      for (int i = 0; i < W + 2; ++i) stage(t, i);
      __syncthreads();
    }
    return;
  }
  for (int t = 0; t < tiles; ++t, slot = after(slot)) {
    step(t, 0, after(slot), 0, [&](int m) __attribute__((always_inline)) {
      if (D == 128) stage(t, m);
      else if (m < 2) stage(t, 2 * m), stage(t, 2 * m + 1);
    });
    mask(t, 1);
    step(t, 1, after(slot), 1, [](int) {});
    mask(t + 1, 0);
    if (!whole(t)) {
#pragma unroll 1
      for (int w = 0; w < 4; ++w) {
        unsigned long long special = s.special[t & 1][w];
        while (special) {
          const int from = __ffsll(special) - 1;
          special &= special - 1;
          const int k = k0 + 64 * t + 16 * w + (from & 15), of = (from >> 4) * (D / 4) / 32;
#pragma unroll
          for (int d = 0; d < DT; ++d)
            if (d == of && k < limit) o[d] += NAN;
        }
      }
    }
    __syncthreads();
  }
  const float sum = xor32_sum(run_sum);
  if (row >= live) return;
  const bool none = run_max == -INFINITY && sum == 0.f && k0 < limit;
  if (__builtin_expect(__any(none), 0))
    if (none && paged_sees(a, table, k0, limit)) run_max = kPagedNoWeight;
  if (unit.parts > 1) {
    float* rec = paged_record(a, unit.record + unit.part, kvh, row, D);
    if (half == 0) rec[0] = run_max, rec[1] = sum;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float2* at = reinterpret_cast<float2*>(rec + 2 + 32 * d + 8 * g + 4 * half);
        at[0] = make_float2(o[d][4 * g], o[d][4 * g + 1]);
        at[1] = make_float2(o[d][4 * g + 2], o[d][4 * g + 3]);
      }
  } else {
    const float inv = paged_inverse(run_max, sum);
    uint16_t* to = a.out + ((size_t)(unit.begin + token) * a.query_heads + kvh * group + head) * D + 4 * half;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<uint2*>(to + 32 * d + 8 * g) =
            make_uint2(cvt_pk_bf16(o[d][4 * g] * inv, o[d][4 * g + 1] * inv),
                       cvt_pk_bf16(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv));
  }
}

// ------------------------------------------------------------------------------------------------------- the blocks
template <int D, int NT>
__device__ void paged_mx4_attention_narrow(const PagedMx4AttentionArgs& a) {
  __shared__ __attribute__((aligned(16))) PagedNarrowShared<D, NT> s;
  const int kvh = blockIdx.x % a.base.kv_heads;
  PagedWalk<false> walk;
  if (!walk.start(a.base, blockIdx.x / a.base.kv_heads)) return;
  for (PagedUnit unit; walk.next(a.base, unit); __syncthreads()) {
    paged_note(a.base, unit, kvh);
    paged_mx4_narrow<D, NT>(a, unit, kvh, s);
  }
}

template <int D>
__device__ void paged_mx4_attention_mixed(const PagedMx4AttentionArgs& a) {
  __shared__ __attribute__((aligned(256))) union {  // the wide form's addresses are XORed within a row
    PagedNarrowShared<D, 1> narrow;
    PagedMx4WideShared<D> wide;
  } s;
  const int kvh = blockIdx.x % a.base.kv_heads;
  int u = blockIdx.x / a.base.kv_heads;
  if (u >= a.turn_from && u < a.turn_to) u = a.turn_from + a.turn_to - 1 - u;
  PagedWalk<true> walk;
  if (!walk.start(a.base, u)) return;
  for (PagedUnit unit; walk.next(a.base, unit); __syncthreads()) {
    paged_note(a.base, unit, kvh);
    if (unit.narrow) paged_mx4_narrow<D, 1>(a, unit, kvh, s.narrow);
    else paged_mx4_wide<D>(a, unit, kvh, s.wide);
  }
}

}  // namespace aoto

#define AOTO_PAGED_MX4_ATTENTION(D)                                                                                  \
  extern "C" __global__ __launch_bounds__(256, 3) void aoto_paged_attention_mx4_d##D##_n1(PagedMx4AttentionArgs a) { \
    aoto::paged_mx4_attention_narrow<D, 1>(a);                                                                       \
  }                                                                                                                  \
  extern "C" __global__ __launch_bounds__(256, 2) void aoto_paged_attention_mx4_d##D##_n2(PagedMx4AttentionArgs a) { \
    aoto::paged_mx4_attention_narrow<D, 2>(a);                                                                       \
  }                                                                                                                  \
  extern "C" __global__ __launch_bounds__(256, 2) void aoto_paged_attention_mx4_d##D##_w(PagedMx4AttentionArgs a) {  \
    aoto::paged_mx4_attention_mixed<D>(a);                                                                           \
  }
