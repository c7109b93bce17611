// A paged key/value cache held in 4 bits: the format, its write and its values.
//
// A head's row of D dims is D / 32 groups of 32. A group has one scale byte b, 2^(b - 127), and 32 codes of 4 bits: a
// sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (E2M1; dim 2i in the low half of byte i). The matrix units and the
// conversion instructions of gfx950 take codes and scales as they are. A group is written with the smallest power of
// two of which its largest magnitude is at most 7 (b from 1 to 252) and each dim as the nearest code, ties to the even
// one; what lies above 6 becomes 6, so that nothing is off by more than half of the widest step. A group that holds an
// infinity or a NaN has b = 255 and stands for NaN; so do scale bytes from 253 on, whose 6 would be infinite.
#pragma once

#include "common.h"
#include "paged_args.h"

namespace aoto {

// The scale byte of a group whose largest magnitude has these bits. Up to 1.75 of a power of two 2^k the scale is
// 2^(k - 2), above it 2^(k - 1): a carry out of the mantissa.
AOTO_DEVICE uint32_t mx4_scale_byte(uint32_t bits) {
  return bits >= 0x7F800000u ? 255u : (uint32_t)min(max((int)((bits + 0x1FFFFFu) >> 23) - 2, 1), 252);
}
// A scale byte as the conversions take it: the exponent of a float.
AOTO_DEVICE float mx4_scale(uint32_t byte) { return __uint_as_float((byte > 252u ? 255u : byte) << 23); }

// Eight dims as codes (v_cvt_scalef32_pk_fp4_f32: nearest, ties to even, above 6 to 6; checked on gfx950).
AOTO_DEVICE uint32_t mx4_pack(const float (&x)[8], float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}

// Eight codes as bf16, exactly: the least of them but 0, 2^-127 / 2, is a subnormal number of bf16 (2^-133 and its
// multiples). NaN for a scale byte of 255.
AOTO_DEVICE uint4 mx4_unpack(uint32_t codes, float scale) {
  uint4 v;
  v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  return v;
}

}  // namespace aoto

// RoPE of a step's q and k rows, q to a dense [T][Hq][D], the rotated keys and the values to their cache slots in 4
// bits: k goes to its codes from f32, without a rounding to bf16 between. A thread takes 8 dims of a head's first half
// and their partners in the second, so that four neighbours hold a group of each half. 32 / 8 heads of 128: 32 tokens
// take 3.6 us, the way of a load and a store; 2048 take 11.3 us, 45 MB at 4.0 TB/s.
extern "C" __global__ __launch_bounds__(256) void aoto_paged_rope_append_mx4(PagedMx4AppendArgs a) {
  using namespace aoto;
  const int half = a.head_dim >> 1, lanes = half >> 3;
  const int heads = a.query_heads + 2 * a.kv_heads;
  const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
  const int per_token = heads * lanes;
  const long long t = item / per_token;
  if (t >= a.tokens) return;  // the four lanes of a group together
  const int within = (int)(item - t * per_token);
  const int h = within / lanes, d = 8 * (within - h * lanes);
  const long long slot = a.slots[t], position = a.positions[t];
  const bool stored = slot >= 0 && slot < a.slot_count;
  if (!stored || position < 0 || position >= a.table_rows) {
    if (a.error && slot != -1 && within == 0) atomicOr(a.error, stored ? AOTO_PAGED_BAD_POSITION : AOTO_PAGED_BAD_SLOT);
    return;
  }
  const uint16_t* src = a.qkv + t * a.row_stride + (size_t)h * a.head_dim + d;
  const uint4 lo = *reinterpret_cast<const uint4*>(src), hi = *reinterpret_cast<const uint4*>(src + half);
  const uint32_t la[4] = {lo.x, lo.y, lo.z, lo.w}, ha[4] = {hi.x, hi.y, hi.z, hi.w};
  float l[8], g[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    l[2 * i] = bf16_lo(la[i]), l[2 * i + 1] = bf16_hi(la[i]);
    g[2 * i] = bf16_lo(ha[i]), g[2 * i + 1] = bf16_hi(ha[i]);
  }
  if (h < a.query_heads + a.kv_heads) {
    const uint16_t* cos_row = a.cos_table + position * a.head_dim + d;
    const uint16_t* sin_row = a.sin_table + position * a.head_dim + d;
    const uint4 c0 = *reinterpret_cast<const uint4*>(cos_row), c1 = *reinterpret_cast<const uint4*>(cos_row + half);
    const uint4 s0 = *reinterpret_cast<const uint4*>(sin_row), s1 = *reinterpret_cast<const uint4*>(sin_row + half);
    const uint32_t ca[4] = {c0.x, c0.y, c0.z, c0.w}, cb[4] = {c1.x, c1.y, c1.z, c1.w};
    const uint32_t sa[4] = {s0.x, s0.y, s0.z, s0.w}, sb[4] = {s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float l0 = l[2 * i], l1 = l[2 * i + 1], g0 = g[2 * i], g1 = g[2 * i + 1];
      l[2 * i] = l0 * bf16_lo(ca[i]) - g0 * bf16_lo(sa[i]), l[2 * i + 1] = l1 * bf16_hi(ca[i]) - g1 * bf16_hi(sa[i]);
      g[2 * i] = g0 * bf16_lo(cb[i]) + l0 * bf16_lo(sb[i]), g[2 * i + 1] = g1 * bf16_hi(cb[i]) + l1 * bf16_hi(sb[i]);
    }
  }
  if (h < a.query_heads) {
    uint16_t* dst = a.q_out + (t * a.query_heads + h) * a.head_dim + d;
    *reinterpret_cast<uint4*>(dst) = make_uint4(cvt_pk_bf16(l[0], l[1]), cvt_pk_bf16(l[2], l[3]),
                                                cvt_pk_bf16(l[4], l[5]), cvt_pk_bf16(l[6], l[7]));
    *reinterpret_cast<uint4*>(dst + half) = make_uint4(cvt_pk_bf16(g[0], g[1]), cvt_pk_bf16(g[2], g[3]),
                                                       cvt_pk_bf16(g[4], g[5]), cvt_pk_bf16(g[6], g[7]));
    return;
  }
  // magnitudes as integers: an infinity or a NaN is above everything else
  uint32_t most_l = 0, most_g = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    most_l = max(most_l, __float_as_uint(l[i]) & 0x7FFFFFFFu);
    most_g = max(most_g, __float_as_uint(g[i]) & 0x7FFFFFFFu);
  }
  auto most_of_four = [](uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppXor1, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppXor2, 0xF, 0xF, false));
  };
  const uint32_t byte_l = mx4_scale_byte(most_of_four(most_l)), byte_g = mx4_scale_byte(most_of_four(most_g));
  const int kh = (h - a.query_heads) % a.kv_heads;
  const bool key = h < a.query_heads + a.kv_heads;
  const long long page = slot / a.page, row = slot - page * a.page;
  const PagedMx4Cache& c = a.cache;
  uint8_t* codes = (key ? c.keys : c.values) + page * c.page_stride + kh * c.head_stride + row * c.slot_stride;
  uint8_t* scales = (key ? c.key_scales : c.value_scales) + page * c.scale_page_stride + kh * c.scale_head_stride +
                    row * c.scale_slot_stride;
  *reinterpret_cast<uint32_t*>(codes + d / 2) = byte_l == 255u ? 0u : mx4_pack(l, mx4_scale(byte_l));
  *reinterpret_cast<uint32_t*>(codes + (half + d) / 2) = byte_g == 255u ? 0u : mx4_pack(g, mx4_scale(byte_g));
  if ((d & 31) == 0) {
    scales[d / 32] = (uint8_t)byte_l;
    scales[(half + d) / 32] = (uint8_t)byte_g;
  }
}

// The values of a whole cache, bf16 [pages][Hkv][page][D]: block x's page, 16 dims a thread. Bound by the write, four
// fifths of its bytes (4608 rows of 8 heads of 128: 24 MB in 7.0 us).
extern "C" __global__ __launch_bounds__(256) void aoto_paged_unpack_mx4(PagedMx4UnpackArgs a) {
  using namespace aoto;
  const int per_row = a.head_dim >> 4, rows = a.kv_heads * a.page;
  const int within = blockIdx.y * 256 + threadIdx.x;
  if (within >= rows * per_row) return;
  const int row = within / per_row, part = within - row * per_row;
  const int h = row / a.page, slot = row - h * a.page;
  const PagedMx4Cache& c = a.cache;
  const long long code = blockIdx.x * c.page_stride + h * c.head_stride + slot * c.slot_stride + 8 * part;
  const long long scale = blockIdx.x * c.scale_page_stride + h * c.scale_head_stride + slot * c.scale_slot_stride +
                          (part >> 1);
  const uint2 k = *reinterpret_cast<const uint2*>(c.keys + code), v = *reinterpret_cast<const uint2*>(c.values + code);
  const float ks = mx4_scale(c.key_scales[scale]), vs = mx4_scale(c.value_scales[scale]);
  const size_t to = ((size_t)blockIdx.x * rows + row) * a.head_dim + 16 * part;
  *reinterpret_cast<uint4*>(a.keys_out + to) = mx4_unpack(k.x, ks);
  *reinterpret_cast<uint4*>(a.keys_out + to + 8) = mx4_unpack(k.y, ks);
  *reinterpret_cast<uint4*>(a.values_out + to) = mx4_unpack(v.x, vs);
  *reinterpret_cast<uint4*>(a.values_out + to + 8) = mx4_unpack(v.y, vs);
}
