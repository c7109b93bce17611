// What is done to a request's logits before a token is chosen: penalties for tokens that its text holds, biases, and a
// mask of the tokens that may follow.
//
// With n_v whether token v is in the request's text (prompt and answer, and the drafts before a row) and g_v how often
// its answer holds it:
//   z' = (n_v ? (z > 0 ? z / repetition : z * repetition) : z) - (g_v ? frequency * g_v + presence : 0) + bias_v
// and -inf where the row's mask has no bit for v. f32, rounded once.
//
// A block takes 2048 tokens of the vocabulary, eight a thread, for all rows of a request. The text is counted by
// passing over it once in every block: counters of the block's own tokens in LDS, then in registers, where the drafts
// are added row by row. Nothing of the size of the vocabulary is kept between launches.
#pragma once

#include "common.h"
#include "paged_args.h"

namespace aoto {

template <bool F32>
__device__ void adjust_logits(const AdjustArgs& a) {
  constexpr int SIZE = F32 ? 4 : 2;
  constexpr uint32_t SEEN = 0x80000000u;
  __shared__ uint32_t s_text[kAdjustChunk];  // bit 31: in the text; below it: how often in the answer
  __shared__ int s_bias[kAdjustChunk];       // the last entry of the list that names the token, and one
  const int r = blockIdx.y, tid = threadIdx.x;
  const int first = a.query_start ? min(max(a.query_start[r], 0), a.rows) : min(r, a.rows);
  const int end = a.query_start ? min(max(a.query_start[r + 1], first), a.rows) : min(r + 1, a.rows);
  if (first >= end) return;
  const int v0 = blockIdx.x * kAdjustChunk, own = v0 + 8 * tid;
  uint32_t text[8] = {};
  float bias[8] = {};
  bool touched = false;
  if (a.history_len > 0 || a.biases > 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s_text[256 * i + tid] = 0, s_bias[256 * i + tid] = 0;
    __syncthreads();
    const int told = a.history_lens ? a.history_lens[r] : a.history_len;
    const int len = min(max(told, 0), a.history_len);
    const int prompt = a.prompt_lens ? a.prompt_lens[r] : 0;
    const long long* history = a.history + r * a.history_stride;
#pragma unroll 8
    for (int j = tid; j < len; j += 256) {
      const unsigned long long at = (unsigned long long)(history[j] - v0);
      if (at < kAdjustChunk) {
        atomicOr(&s_text[at], SEEN);
        if (j >= prompt) atomicAdd(&s_text[at], 1u);
      }
    }
    for (int j = tid; j < a.biases; j += 256) {
      const unsigned long long at = (unsigned long long)(a.bias_tokens[r * a.bias_stride + j] - v0);
      if (at < kAdjustChunk) atomicMax(&s_bias[at], j + 1);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      text[i] = s_text[8 * tid + i];
      const int entry = s_bias[8 * tid + i];
      if (entry) bias[i] = a.bias_values[r * a.value_stride + entry - 1];
      touched |= text[i] != 0 || entry != 0;
    }
  }
  if (own >= a.vocab) return;
  const int count = min(8, a.vocab - own);
  const float repetition = a.repetition ? a.repetition[r] : 1.f;
  const float presence = a.presence ? a.presence[r] : 0.f, frequency = a.frequency ? a.frequency[r] : 0.f;
  const char* in = static_cast<const char*>(a.logits) + ((long long)first * a.row_stride + own) * SIZE;
  char* out = static_cast<char*>(a.out) + ((long long)first * a.out_stride + own) * SIZE;
  const uint8_t* allowed = a.allowed ? a.allowed + first * a.allowed_stride + (own >> 3) : nullptr;
  for (int row = first; row < end; ++row) {
    const uint32_t mask = allowed ? *allowed : 0xFFu;
    float z[8];
    uint4 raw[F32 ? 2 : 1];
    const bool whole = count == 8 && ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    if (whole) {
#pragma unroll
      for (int i = 0; i < (F32 ? 2 : 1); ++i) raw[i] = reinterpret_cast<const uint4*>(in)[i];
      if constexpr (F32) {
        z[0] = __uint_as_float(raw[0].x), z[1] = __uint_as_float(raw[0].y);
        z[2] = __uint_as_float(raw[0].z), z[3] = __uint_as_float(raw[0].w);
        z[4] = __uint_as_float(raw[1].x), z[5] = __uint_as_float(raw[1].y);
        z[6] = __uint_as_float(raw[1].z), z[7] = __uint_as_float(raw[1].w);
      } else {
        z[0] = bf16_lo(raw[0].x), z[1] = bf16_hi(raw[0].x), z[2] = bf16_lo(raw[0].y), z[3] = bf16_hi(raw[0].y);
        z[4] = bf16_lo(raw[0].z), z[5] = bf16_hi(raw[0].z), z[6] = bf16_lo(raw[0].w), z[7] = bf16_hi(raw[0].w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < count)
          z[i] = F32 ? reinterpret_cast<const float*>(in)[i] : bf16_to_f32(reinterpret_cast<const uint16_t*>(in)[i]);
    }
    if (touched) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (text[i]) z[i] = z[i] > 0.f ? z[i] / repetition : z[i] * repetition;
        const uint32_t said = text[i] & ~SEEN;
        if (said) z[i] -= frequency * (float)said + presence;
        z[i] += bias[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(mask >> i & 1)) z[i] = -INFINITY;
    if (whole) {
      if constexpr (F32) {
        reinterpret_cast<float4*>(out)[0] = make_float4(z[0], z[1], z[2], z[3]);
        reinterpret_cast<float4*>(out)[1] = make_float4(z[4], z[5], z[6], z[7]);
      } else {
        *reinterpret_cast<uint4*>(out) = make_uint4(pack_bf16x2(z[0], z[1]), pack_bf16x2(z[2], z[3]),
                                                    pack_bf16x2(z[4], z[5]), pack_bf16x2(z[6], z[7]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < count) {
          if constexpr (F32) reinterpret_cast<float*>(out)[i] = z[i];
          else reinterpret_cast<uint16_t*>(out)[i] = (uint16_t)f32_to_bf16(z[i]);
        }
    }
    in += a.row_stride * SIZE, out += a.out_stride * SIZE;
    if (allowed) allowed += a.allowed_stride;
    // the draft that this row judges is in the text of the rows behind it
    const int i = row - first;
    if (i < a.drafts) {
      const unsigned long long at = (unsigned long long)(a.draft_tokens[r * a.draft_stride + i] - own);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (at == (unsigned long long)k) text[k] = (text[k] + 1) | SEEN, touched = true;
    }
  }
}

}  // namespace aoto

#define AOTO_ADJUST_INSTANCE(NAME, F32)                                                       \
  extern "C" __global__ __launch_bounds__(256) void aoto_adjust_logits_##NAME(AdjustArgs a) { \
    aoto::adjust_logits<F32>(a);                                                              \
  }
