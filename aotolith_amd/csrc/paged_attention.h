// Attention of requests' new tokens over their pages of a shared key/value cache.
//
//   out[t][h] = sum_j softmax_j(scale * q[t][h] . k_j) v_j
// over the keys j of token t's request r that it may see: with n_r = query_start[r + 1] - query_start[r] rows and
// kv_r keys, row i sees j < kv_r - n_r + i + 1 (causal) or j < kv_r, as far as the block table row goes and where its
// entry names a page of the cache; a row that sees none gives 0. Key j of head h / (Hq / Hkv) is row j % page of page
// block_tables[r][j / page]. Scores, maxima and sums in f32.
#pragma once

#include "common.h"
#include "paged_args.h"

namespace aoto {

// The request that owns token t (t < query_start[requests]): the last r with query_start[r] <= t, found 64 ways a
// step. All lanes of the wave call it with the same t.
AOTO_DEVICE int paged_request(const int* __restrict__ query_start, int requests, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = requests;  // the answer is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int at = lo + lane * step;
    const unsigned long long below = __ballot(at < hi && query_start[min(at, requests)] <= t);
    const int last = below ? 63 - __clzll((long long)below) : 0;
    lo += last * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

template <int D>
__device__ void paged_attention_simple(const PagedAttentionArgs& a) {
  constexpr int LPK = D / 8, KPI = 64 / LPK;
  const int t = blockIdx.x / a.query_heads, h = blockIdx.x % a.query_heads;
  const int lane = threadIdx.x, sub = lane % LPK, kin = lane / LPK;
  if (t >= a.query_start[a.requests]) return;
  const int r = paged_request(a.query_start, a.requests, t);
  const int begin = a.query_start[r], n = a.query_start[r + 1] - begin;
  int keys = a.kv_lens[r];
  if (a.causal) keys = min(keys, keys - n + (t - begin) + 1);
  keys = min(keys, (int)min((long long)a.max_blocks * a.page, 0x7FFFFFFFLL));
  const int kvh = h / (a.query_heads / a.kv_heads);
  const uint4 qc = *reinterpret_cast<const uint4*>(a.q + t * a.q_token_stride + h * a.q_head_stride + 8 * sub);
  float m = -INFINITY, l = 0.f, acc[8] = {};
  for (int j0 = 0; j0 < keys; j0 += KPI) {
    const int j = j0 + kin;
    const int page = j < keys ? a.block_tables[r * a.table_stride + j / a.page] : -1;
    const bool there = page >= 0 && page < a.pages;
    const long long at = there ? page * a.page_stride + kvh * a.head_stride + (j % a.page) * a.slot_stride : 0;
    const uint4 k = *reinterpret_cast<const uint4*>(a.keys + at + 8 * sub);
    const uint4 v = *reinterpret_cast<const uint4*>(a.values + at + 8 * sub);
    float dot = dot2_bf16(k.x, qc.x, 0.f);
    dot = dot2_bf16(k.y, qc.y, dot);
    dot = dot2_bf16(k.z, qc.z, dot);
    dot = dot2_bf16(k.w, qc.w, dot);
    const float score = there ? group_sum<LPK>(dot) * a.scale : -INFINITY;
    const float big = fmaxf(m, score);
    const float ref = big == -INFINITY ? 0.f : big;
    const float p = expf(score - ref), keep = expf(m - ref);
    m = big;
    l = l * keep + p;
    const uint32_t va[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc[2 * i] = acc[2 * i] * keep + (there ? p * bf16_lo(va[i]) : 0.f);
      acc[2 * i + 1] = acc[2 * i + 1] * keep + (there ? p * bf16_hi(va[i]) : 0.f);
    }
  }
  const float big = wave_max(m);
  const float f = m == -INFINITY ? 0.f : expf(m - big);
  const float sum = wave_sum(sub == 0 ? l * f : 0.f);
  float o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float v = acc[e] * f;
    for (int d = LPK; d < 64; d <<= 1) v += __shfl_xor(v, d);
    o[e] = sum > 0.f ? v / sum : 0.f;
  }
  if (kin == 0) {
    uint4 w = make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]),
                         pack_bf16x2(o[6], o[7]));
    *reinterpret_cast<uint4*>(a.out + ((size_t)t * a.query_heads + h) * D + 8 * sub) = w;
  }
}

}  // namespace aoto

extern "C" __global__ __launch_bounds__(64) void aoto_paged_attention_d64(PagedAttentionArgs a) {
  aoto::paged_attention_simple<64>(a);
}
extern "C" __global__ __launch_bounds__(64) void aoto_paged_attention_d128(PagedAttentionArgs a) {
  aoto::paged_attention_simple<128>(a);
}
