// What is done to a request's logits before a token is chosen: penalties for tokens that its text holds, biases, and a
// mask of the tokens that may follow.
//
// With n_v whether token v is in the request's text (prompt and answer, and the drafts before a row) and g_v how often
// its answer holds it:
//   z' = (n_v ? (z > 0 ? z / repetition : z * repetition) : z) - (g_v ? frequency * g_v + presence : 0) + bias_v
// and -inf where the row's mask has no bit for v. f32, rounded once.
//
// A block takes 1024 or 2048 tokens of the vocabulary, two to eight a thread, for all rows of a request. The text is
// counted by passing over it once in every block: counters of the block's own tokens in LDS, then in registers, where
// the drafts are added row by row. Nothing of the size of the vocabulary is kept between launches. Four rows are on
// their way at a time, the first four while the text is counted. With out = logits, threads whose tokens nothing
// changes neither read nor write.
//
// With few rows a wave's own instructions bound it (25 a token of the text and row), which fewer tokens a thread cut;
// with many the read and write of the logits, which want 16 bytes a lane, and as few passes over a text as there can be
// (tokens a thread x threads, us; "rows" are four a request, texts of 2000 tokens):
//                                             8 x 256   4 x 256   2 x 512
//   bf16, 4 rows x 151936, a text of 6000        10.1       8.0       6.4
//   bf16, 10 rows x 128256                        8.5       6.8       6.0
//   bf16, 47 rows x 50257                         9.5       8.2       8.3
//   bf16, 47 rows x 128256                       12.4      11.4      14.8
//   bf16, 72 rows x 128256                       15.4      15.6      22.4
//   bf16, 203 rows x 128256, masks               27.3      30.8      48.2
//   f32, 10 rows x 128256                         9.8       7.3       6.3
//   f32, 72 rows x 128256                        24.2      19.9      23.6
//   f32, 203 rows x 128256, masks                59.1      54.5
//   f32, 256 requests' one row, texts of 4000    91.3     100.0
// 108 MB of the sixth at 3.9 TB/s, of three times as many requests at 4.7. The rule goes by rows and vocabulary, which
// the host knows; history_len is only the room for texts, so the last line, whose time is its texts', loses by the rule.
// Blocks of 4096 and more tokens gain for texts as long as a quarter of the vocabulary only (bf16, 8 rows x 128256,
// texts of 32000: 17.2 us with 2048, 12.2 with 4096), 16 tokens of a text on their way instead of 8 for none (30.5 us
// for the sixth: registers, and with them waves).
#pragma once

#include "common.h"
#include "paged_args.h"

namespace aoto {

// A thread's logits of a row, at an address of their type's alignment: global memory takes wide loads and stores at
// any.
template <bool F32, int PER>
struct __attribute__((packed, aligned(F32 ? 4 : 2))) AdjustSome {
  uint32_t w[F32 ? PER : PER / 2];
};

template <bool F32, int PER, int THREADS>
__device__ void adjust_logits(const AdjustArgs& a) {
  using Some = AdjustSome<F32, PER>;
  constexpr int SIZE = F32 ? 4 : 2, ROWS = 4, CHUNK = PER * THREADS;
  constexpr uint32_t NONE = (1u << PER) - 1;  // masked
  constexpr uint32_t SEEN = 0x80000000u;
  __shared__ uint32_t s_text[CHUNK];  // bit 31: in the text; below it: how often in the answer
  __shared__ int s_bias[CHUNK];       // the last entry of the list that names the token, and one
  const int r = blockIdx.y, tid = threadIdx.x;
  const int first = a.query_start ? min(max(a.query_start[r], 0), a.rows) : min(r, a.rows);
  const int end = a.query_start ? min(max(a.query_start[r + 1], first), a.rows) : min(r + 1, a.rows);
  if (first >= end) return;
  const int v0 = blockIdx.x * CHUNK, own = v0 + PER * tid;
  const int count = min(PER, a.vocab - own);  // tokens of this thread, none where not above 0
  const bool same = a.logits == a.out;
  const char* in = static_cast<const char*>(a.logits) + ((long long)first * a.row_stride + own) * SIZE;
  char* out = static_cast<char*>(a.out) + ((long long)first * a.out_stride + own) * SIZE;
  const uint8_t* allowed = a.allowed ? a.allowed + first * a.allowed_stride + (own >> 3) : nullptr;
  Some raw[ROWS];
  uint32_t mask[ROWS];
  // rows row .. row + 3, as far as there are; `all`: their logits too
  auto load = [&](int row, bool all) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      mask[i] = NONE;
      if (row + i >= end || count <= 0) continue;
      if (allowed) mask[i] = allowed[(long long)(row + i - first) * a.allowed_stride] >> (own & 7) & NONE;
      if (!all) continue;
      const char* at = in + (long long)(row + i - first) * a.row_stride * SIZE;
      if (count == PER) {
        raw[i] = *reinterpret_cast<const Some*>(at);
      } else {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
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
  uint32_t text[PER] = {};
  float bias[PER] = {};
  bool touched = false;
  if (a.history_len > 0 || a.biases > 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) s_text[THREADS * i + tid] = 0, s_bias[THREADS * i + tid] = 0;
    const int told = a.history_lens ? a.history_lens[r] : a.history_len;
    const int len = min(max(told, 0), a.history_len);
    const int prompt = a.prompt_lens ? a.prompt_lens[r] : 0;
    const long long* history = a.history + r * a.history_stride;
    __syncthreads();
    constexpr int SOME = 8;  // tokens of the text that a thread asks for at a time
    for (int base = 0; base < len; base += THREADS * SOME) {
      long long token[SOME];
#pragma unroll
      for (int i = 0; i < SOME; ++i) {
        const int j = base + THREADS * i + tid;
        token[i] = j < len ? history[j] : -1;
      }
#pragma unroll
      for (int i = 0; i < SOME; ++i) {
        const unsigned long long at = (unsigned long long)token[i] - v0;
        if (at < CHUNK) {
          atomicOr(&s_text[at], SEEN);
          if (base + THREADS * i + tid >= prompt) atomicAdd(&s_text[at], 1u);
        }
      }
    }
    for (int j = tid; j < a.biases; j += THREADS) {
      const unsigned long long at = (unsigned long long)a.bias_tokens[r * a.bias_stride + j] - v0;
      if (at < CHUNK) atomicMax(&s_bias[at], j + 1);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      text[i] = s_text[PER * tid + i];
      const int entry = s_bias[PER * tid + i];
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
        later |= (unsigned long long)a.draft_tokens[r * a.draft_stride + i] - own < PER;
      load(row, !same || later || allowed);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (row + i >= end) break;
      if (!same || touched || mask[i] != NONE) {
        char* to = out + (long long)(row + i - first) * a.out_stride * SIZE;
        Some made = raw[i];
        if (touched || mask[i] != NONE) {
          float z[PER];
#pragma unroll
          for (int k = 0; k < PER; ++k)
            z[k] = F32 ? __uint_as_float(raw[i].w[k]) : k & 1 ? bf16_hi(raw[i].w[k >> 1]) : bf16_lo(raw[i].w[k >> 1]);
          if (touched) {
#pragma unroll
            for (int k = 0; k < PER; ++k) {
              if (text[k]) z[k] = z[k] > 0.f ? z[k] / repetition : z[k] * repetition;
              const uint32_t said = text[k] & ~SEEN;
              if (said) z[k] -= frequency * (float)said + presence;
              z[k] += bias[k];
            }
          }
#pragma unroll
          for (int k = 0; k < PER; ++k)
            if (!(mask[i] >> k & 1)) z[k] = -INFINITY;
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            if constexpr (F32) made.w[k] = __float_as_uint(z[k]);
            else if (k & 1) made.w[k >> 1] = cvt_pk_bf16(z[k - 1], z[k]);
          }
        }
        if (count == PER) {
          *reinterpret_cast<Some*>(to) = made;
        } else {
#pragma unroll
          for (int k = 0; k < PER; ++k)
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
        if (at < PER) {
#pragma unroll
          for (int k = 0; k < PER; ++k)
            if (at == (unsigned long long)k) text[k] = (text[k] + 1) | SEEN;
          touched = true;
        }
      }
    }
  }
}

}  // namespace aoto

#define AOTO_ADJUST_INSTANCE(NAME, F32, PER, THREADS)                                              \
  extern "C" __global__ __launch_bounds__(THREADS) void aoto_adjust_logits_##NAME(AdjustArgs a) { \
    aoto::adjust_logits<F32, PER, THREADS>(a);                                                     \
  }
