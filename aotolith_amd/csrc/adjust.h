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
// are added row by row. Nothing of the size of the vocabulary is kept between launches. Four rows are on their way at a
// time, the first four while the text is counted. With out = logits, threads whose tokens nothing changes neither read
// nor write.
//
// The read and write of the logits bound it where there are rows enough: bf16, 203 rows of 64 requests over 128256
// tokens, with masks and texts of 2000, 108 MB in 27.3 us (3.9 TB/s). One request's four rows over 151936 with a text
// of 6000 take 10.2 us, 5.3 of them a launch and one row without a text. Blocks of 4096 tokens count a text half as
// often, but fewer of them share the rows: 30.9 and 10.4 us, and 11.3 instead of 11.0 for 16 requests' 4 rows each over
// 50257 in f32. Only texts as long as a quarter of the vocabulary gain (eight rows over 128256 with texts of 32000:
// 17.2 us, 12.2 with 4096, 10.8 with 8192). 16 tokens of a text at a time take registers, and with them waves: 30.5 us
// for the first.
#pragma once

#include "common.h"
#include "paged_args.h"

namespace aoto {

// Eight logits at an address of their type's alignment: global memory takes wide loads and stores at any.
template <bool F32>
struct __attribute__((packed, aligned(F32 ? 4 : 2))) AdjustEight {
  uint32_t w[F32 ? 8 : 4];
};

template <bool F32>
__device__ void adjust_logits(const AdjustArgs& a) {
  using Eight = AdjustEight<F32>;
  constexpr int SIZE = F32 ? 4 : 2, ROWS = 4;
  constexpr uint32_t SEEN = 0x80000000u;
  __shared__ uint32_t s_text[kAdjustChunk];  // bit 31: in the text; below it: how often in the answer
  __shared__ int s_bias[kAdjustChunk];       // the last entry of the list that names the token, and one
  const int r = blockIdx.y, tid = threadIdx.x;
  const int first = a.query_start ? min(max(a.query_start[r], 0), a.rows) : min(r, a.rows);
  const int end = a.query_start ? min(max(a.query_start[r + 1], first), a.rows) : min(r + 1, a.rows);
  if (first >= end) return;
  const int v0 = blockIdx.x * kAdjustChunk, own = v0 + 8 * tid;
  const int count = min(8, a.vocab - own);  // tokens of this thread, none where not above 0
  const bool same = a.logits == a.out;
  const char* in = static_cast<const char*>(a.logits) + ((long long)first * a.row_stride + own) * SIZE;
  char* out = static_cast<char*>(a.out) + ((long long)first * a.out_stride + own) * SIZE;
  const uint8_t* allowed = a.allowed ? a.allowed + first * a.allowed_stride + (own >> 3) : nullptr;
  Eight raw[ROWS];
  uint32_t mask[ROWS];
  // rows row .. row + 3, as far as there are; `all`: their logits too
  auto load = [&](int row, bool all) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      mask[i] = 0xFFu;
      if (row + i >= end || count <= 0) continue;
      if (allowed) mask[i] = allowed[(long long)(row + i - first) * a.allowed_stride];
      if (!all) continue;
      const char* at = in + (long long)(row + i - first) * a.row_stride * SIZE;
      if (count == 8) {
        raw[i] = *reinterpret_cast<const Eight*>(at);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if constexpr (F32) {
            raw[i].w[k] = k < count ? reinterpret_cast<const uint32_t*>(at)[k] : 0u;
          } else {
            const uint32_t half = k < count ? reinterpret_cast<const uint16_t*>(at)[k] : 0u;
            raw[i].w[k >> 1] = k & 1 ? raw[i].w[k >> 1] | half << 16 : half;
          }
        }
      }
    }
  };
  if (!same) load(first, true);
  const float repetition = a.repetition ? a.repetition[r] : 1.f;
  const float presence = a.presence ? a.presence[r] : 0.f, frequency = a.frequency ? a.frequency[r] : 0.f;
  uint32_t text[8] = {};
  float bias[8] = {};
  bool touched = false;
  if (a.history_len > 0 || a.biases > 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s_text[kAdjustThreads * i + tid] = 0, s_bias[kAdjustThreads * i + tid] = 0;
    const int told = a.history_lens ? a.history_lens[r] : a.history_len;
    const int len = min(max(told, 0), a.history_len);
    const int prompt = a.prompt_lens ? a.prompt_lens[r] : 0;
    const long long* history = a.history + r * a.history_stride;
    __syncthreads();
    constexpr int SOME = kAdjustSome;  // tokens of the text that a thread asks for at a time
    for (int base = 0; base < len; base += kAdjustThreads * SOME) {
      long long token[SOME];
#pragma unroll
      for (int i = 0; i < SOME; ++i) {
        const int j = base + kAdjustThreads * i + tid;
        token[i] = j < len ? history[j] : -1;
      }
#pragma unroll
      for (int i = 0; i < SOME; ++i) {
        const unsigned long long at = (unsigned long long)token[i] - v0;
        if (at < kAdjustChunk) {
          atomicOr(&s_text[at], SEEN);
          if (base + kAdjustThreads * i + tid >= prompt) atomicAdd(&s_text[at], 1u);
        }
      }
    }
    for (int j = tid; j < a.biases; j += kAdjustThreads) {
      const unsigned long long at = (unsigned long long)a.bias_tokens[r * a.bias_stride + j] - v0;
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
  if (count <= 0) return;
  for (int row = first; row < end; row += ROWS) {
    if (row > first || same) {
      // which of the next drafts are this thread's tokens is known before their rows are
      bool later = touched;
      for (int i = row - first; i < min(row - first + ROWS - 1, a.drafts); ++i)
        later |= (unsigned long long)a.draft_tokens[r * a.draft_stride + i] - own < 8;
      load(row, !same || later || allowed);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (row + i >= end) break;
      if (!same || touched || mask[i] != 0xFFu) {
        char* to = out + (long long)(row + i - first) * a.out_stride * SIZE;
        Eight made = raw[i];
        if (touched || mask[i] != 0xFFu) {
          float z[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            z[k] = F32 ? __uint_as_float(raw[i].w[k]) : k & 1 ? bf16_hi(raw[i].w[k >> 1]) : bf16_lo(raw[i].w[k >> 1]);
          if (touched) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              if (text[k]) z[k] = z[k] > 0.f ? z[k] / repetition : z[k] * repetition;
              const uint32_t said = text[k] & ~SEEN;
              if (said) z[k] -= frequency * (float)said + presence;
              z[k] += bias[k];
            }
          }
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (!(mask[i] >> k & 1)) z[k] = -INFINITY;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if constexpr (F32) made.w[k] = __float_as_uint(z[k]);
            else if (k & 1) made.w[k >> 1] = cvt_pk_bf16(z[k - 1], z[k]);
          }
        }
        if (count == 8) {
          *reinterpret_cast<Eight*>(to) = made;
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < count) {
              if constexpr (F32) reinterpret_cast<uint32_t*>(to)[k] = made.w[k];
              else reinterpret_cast<uint16_t*>(to)[k] = (uint16_t)(made.w[k >> 1] >> (16 * (k & 1)));
            }
        }
      }
      // the draft that this row judges is in the text of the rows behind it
      const int draft = row + i - first;
      if (draft < a.drafts) {
        const unsigned long long at = (unsigned long long)a.draft_tokens[r * a.draft_stride + draft] - own;
        if (at < 8) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (at == (unsigned long long)k) text[k] = (text[k] + 1) | SEEN;
          touched = true;
        }
      }
    }
  }
}

}  // namespace aoto

#define AOTO_ADJUST_INSTANCE(NAME, F32)                                                                  \
  extern "C" __global__ __launch_bounds__(kAdjustThreads) void aoto_adjust_logits_##NAME(AdjustArgs a) { \
    aoto::adjust_logits<F32>(a);                                                                         \
  }
