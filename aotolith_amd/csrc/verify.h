// Verification of drafted tokens against the target's logits, from given random numbers.
//
// Laws of a row of logits z at temperature T > 0: p_v = w_v / sum w, w_v = exp((z_v - max z) / T); a NaN counts as
// -inf, a row without a number above -inf has w = 0. Draft i of request r (drafted from q, a point mass where no draft
// logits are given) stands while u_i q(x_i) < p_i(x_i); at the first that does not, the token that follows is drawn
// from max(p_i - q_i, 0) (from p_i where that is 0 throughout), after all of them from the last row's p: the first v
// at which the running sum of weights passes u_last times their total. T <= 0: a draft stands where it is the row's
// first maximum, which is also the token that follows.
//
// All of it is held in 64 bits, the exponentials too: a token is where a sum over the vocabulary passes a random
// number, and the sums' noise in 32 bits (1e-7 of the total, against a typical weight of 1e-5 to 1e-6 of it) would
// move it in a percent of the calls.
//
// Three launches over chunks of kVerifyChunk tokens: every row's maximum, its place and sum of weights by chunk; the
// weights the following token is drawn from, summed by chunk; the token. Bound by the first one's read of the logits.
#pragma once

#include "common.h"
#include "paged_args.h"

namespace aoto {

// What the first launch leaves of a chunk of a row: the sum of exp((z - max) / T), the maximum and its first place.
struct VerifyChunk {
  double sum;
  float top;
  int place;
};
static_assert(sizeof(VerifyChunk) == kVerifyChunkBytes, "as the workspace is sized");

// 2^x for x <= 0 (and -inf): the power series of 2^f = e^(f ln 2) to the 13th term over |f| <= 1/2, whose remainder
// is below (ln 2 / 2)^14 / 14! = 4e-18, and the exponent's shift.
AOTO_DEVICE double exp2_below(double x) {
  x = fmax(x, -1100.0);
  const double n = rint(x), y = (x - n) * 0.6931471805599453094;
  double s = 1.0 / 6227020800.0;
  s = fma(s, y, 1.0 / 479001600.0);
  s = fma(s, y, 1.0 / 39916800.0);
  s = fma(s, y, 1.0 / 3628800.0);
  s = fma(s, y, 1.0 / 362880.0);
  s = fma(s, y, 1.0 / 40320.0);
  s = fma(s, y, 1.0 / 5040.0);
  s = fma(s, y, 1.0 / 720.0);
  s = fma(s, y, 1.0 / 120.0);
  s = fma(s, y, 1.0 / 24.0);
  s = fma(s, y, 1.0 / 6.0);
  s = fma(s, y, 0.5);
  s = fma(s, y, 1.0);
  s = fma(s, y, 1.0);
  return ldexp(s, (int)n);
}

// exp((z - top) / T) with heat = log2(e) / T; infinite values compare equal to an infinite top.
AOTO_DEVICE double verify_weight(float z, float top, double heat) {
  if (z == -INFINITY) return 0.0;
  return z == top ? 1.0 : exp2_below(((double)z - (double)top) * heat);
}

template <bool F32>
AOTO_DEVICE float verify_logit(const void* row, int v) {
  const float z = F32 ? static_cast<const float*>(row)[v] : bf16_to_f32(static_cast<const uint16_t*>(row)[v]);
  return z != z ? -INFINITY : z;
}

// log2(e) / T, or kVerifyGreedy.
constexpr double kVerifyGreedy = -1.0;
AOTO_DEVICE double verify_heat(const VerifyArgs& a, int r) {
  const float t = a.temperature ? a.temperature[r] : 0.f;
  return t > 0.f ? 1.4426950408889634074 / (double)t : kVerifyGreedy;
}

// Rows of request r: its first, and how many drafts of it there are.
AOTO_DEVICE void verify_rows(const VerifyArgs& a, int r, int& first, int& count) {
  first = min(max(a.query_start[r], 0), a.rows);
  const int end = min(max(a.query_start[r + 1], first), a.rows);
  count = min(end - first - 1, a.drafts);  // -1: the request has no row
}

AOTO_DEVICE double wave_sum_f64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// The whole row's maximum, its first place and the sum of weights below it, from its chunks.
AOTO_DEVICE VerifyChunk verify_join(const VerifyChunk* chunks, int count, double heat) {
  VerifyChunk all{0.0, -INFINITY, 0};
  for (int c = 0; c < count; ++c)
    if (chunks[c].top > all.top) all.top = chunks[c].top, all.place = chunks[c].place;
  for (int c = 0; c < count; ++c) all.sum += chunks[c].sum * verify_weight(chunks[c].top, all.top, heat);
  return all;
}

template <bool F32>
AOTO_DEVICE const void* verify_row(const void* base, long long at) {
  return F32 ? (const void*)(static_cast<const float*>(base) + at)
             : (const void*)(static_cast<const uint16_t*>(base) + at);
}

// Block (chunk, r * (2 drafts + 1) + i): target row i of request r (i <= drafts), or its draft row i - drafts - 1.
template <bool F32>
__device__ void verify_stats(const VerifyArgs& a) {
  __shared__ float s_top[4];
  __shared__ int s_place[4];
  __shared__ double s_sum[4];
  const int per = 2 * a.drafts + 1;
  const int r = blockIdx.y / per, i = blockIdx.y % per;
  int first, count;
  verify_rows(a, r, first, count);
  const bool draft = i > a.drafts;
  const double heat = verify_heat(a, r);
  if (draft ? (a.draft_logits == nullptr || i - a.drafts - 1 >= count || heat == kVerifyGreedy) : i > count) return;
  const void* row = draft ? verify_row<F32>(a.draft_logits, r * a.draft_request_stride +
                                                                (i - a.drafts - 1) * a.draft_row_stride)
                          : verify_row<F32>(a.logits, (first + i) * a.row_stride);
  const int begin = blockIdx.x * kVerifyChunk, end = min(a.vocab, begin + kVerifyChunk);
  float z[kVerifyChunk / 256], top = -INFINITY;
  int place = begin;
#pragma unroll
  for (int e = 0; e < kVerifyChunk / 256; ++e) {
    const int v = begin + 256 * e + threadIdx.x;
    z[e] = v < end ? verify_logit<F32>(row, v) : -INFINITY;
    if (z[e] > top) top = z[e], place = v;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const float t = __shfl_xor(top, d);
    const int p = __shfl_xor(place, d);
    if (t > top || (t == top && p < place)) top = t, place = p;
  }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) s_top[wave] = top, s_place[wave] = place;
  __syncthreads();
  top = s_top[0], place = s_place[0];
  for (int w = 1; w < 4; ++w)
    if (s_top[w] > top || (s_top[w] == top && s_place[w] < place)) top = s_top[w], place = s_place[w];
  double sum = 0.0;
  if (heat != kVerifyGreedy) {
#pragma unroll
    for (int e = 0; e < kVerifyChunk / 256; ++e) sum += verify_weight(z[e], top, heat);
    sum = wave_sum_f64(sum);
    if ((threadIdx.x & 63) == 0) s_sum[wave] = sum;
    __syncthreads();
    sum = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
  }
  if (threadIdx.x == 0) {
    VerifyChunk* out = static_cast<VerifyChunk*>(a.workspace) + (size_t)blockIdx.y * a.chunks + blockIdx.x;
    *out = VerifyChunk{sum, top, place};
  }
}

// How many drafts of request r stand, and the law that the following token is drawn from.
struct VerifyLaw {
  int accepted, place;     // place: the row's first maximum
  int removed;             // a drafted token of point mass that the law leaves out, or -1
  const void* row;
  const void* draft_row;   // null: nothing is subtracted
  float top, draft_top;
  double sum, draft_sum, heat;
};

// By one wave: lane i judges draft i (drafts <= 63), then the ballot finds the first that falls.
template <bool F32>
AOTO_DEVICE VerifyLaw verify_law(const VerifyArgs& a, int r) {
  int first, count;
  verify_rows(a, r, first, count);
  const int lane = threadIdx.x & 63;
  const double heat = verify_heat(a, r);
  const VerifyChunk* chunks = static_cast<const VerifyChunk*>(a.workspace) + (size_t)r * (2 * a.drafts + 1) * a.chunks;
  VerifyChunk p{0.0, -INFINITY, 0}, q{0.0, -INFINITY, 0};
  bool stands = false;
  const bool sampled = heat != kVerifyGreedy;
  if (lane <= count) p = verify_join(chunks + (size_t)lane * a.chunks, a.chunks, heat);
  if (lane < count) {
    const long long x = a.draft_tokens[(size_t)r * a.drafts + lane];
    if (a.draft_logits && sampled) q = verify_join(chunks + (size_t)(a.drafts + 1 + lane) * a.chunks, a.chunks, heat);
    if (x >= 0 && x < a.vocab) {
      if (sampled) {
        const double px = verify_weight(verify_logit<F32>(verify_row<F32>(a.logits, (first + lane) * a.row_stride), (int)x),
                                        p.top, heat);
        double qx = 1.0;
        if (a.draft_logits) {
          const float z = verify_logit<F32>(
              verify_row<F32>(a.draft_logits, r * a.draft_request_stride + lane * a.draft_row_stride), (int)x);
          qx = q.sum > 0.0 ? verify_weight(z, q.top, heat) / q.sum : 0.0;
        }
        stands = p.sum > 0.0 && (double)a.uniforms[(size_t)r * (a.drafts + 1) + lane] * qx < px / p.sum;
      } else {
        stands = p.top > -INFINITY && p.place == (int)x;
      }
    }
  }
  const unsigned long long falls = ~__ballot(stands);
  VerifyLaw law{};
  const int k = min(max(count, 0), __ffsll((long long)falls) - 1);
  law.accepted = k;
  law.heat = heat;
  law.place = __shfl(p.place, k);
  law.top = __shfl(p.top, k);
  law.sum = __shfl(p.sum, k);
  law.row = verify_row<F32>(a.logits, (long long)min(first + k, a.rows - 1) * a.row_stride);
  law.removed = -1;
  if (k < count && sampled) {
    if (a.draft_logits) {
      law.draft_row = verify_row<F32>(a.draft_logits, r * a.draft_request_stride + k * a.draft_row_stride);
      law.draft_top = __shfl(q.top, k);
      law.draft_sum = __shfl(q.sum, k);
    } else {
      const long long x = a.draft_tokens[(size_t)r * a.drafts + k];
      law.removed = x >= 0 && x < a.vocab ? (int)x : -1;
    }
  }
  return law;
}

// The weight of token v under the target's law and what is left of it.
template <bool F32>
AOTO_DEVICE void verify_left(const VerifyLaw& law, int v, double& whole, double& left) {
  whole = law.sum > 0.0 ? verify_weight(verify_logit<F32>(law.row, v), law.top, law.heat) / law.sum : 0.0;
  left = v == law.removed ? 0.0 : whole;
  if (law.draft_row && law.draft_sum > 0.0)
    left = fmax(whole - verify_weight(verify_logit<F32>(law.draft_row, v), law.draft_top, law.heat) / law.draft_sum, 0.0);
}

AOTO_DEVICE double* verify_masses(const VerifyArgs& a, int r) {
  const size_t chunks = (size_t)a.requests * (2 * a.drafts + 1) * a.chunks;
  return reinterpret_cast<double*>(static_cast<VerifyChunk*>(a.workspace) + chunks) + (size_t)r * 2 * a.chunks;
}

// Block (chunk, r): the chunk's sums of what is left and of the whole.
template <bool F32>
__device__ void verify_mass(const VerifyArgs& a) {
  __shared__ double s_sum[4][2];
  const int r = blockIdx.y;
  if (verify_heat(a, r) == kVerifyGreedy) return;
  const VerifyLaw law = verify_law<F32>(a, r);
  const int begin = blockIdx.x * kVerifyChunk, end = min(a.vocab, begin + kVerifyChunk);
  double sums[2] = {0.0, 0.0};
  for (int v = begin + threadIdx.x; v < end; v += 256) {
    double whole, left;
    verify_left<F32>(law, v, whole, left);
    sums[0] += left;
    sums[1] += whole;
  }
  for (int i = 0; i < 2; ++i) {
    sums[i] = wave_sum_f64(sums[i]);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6][i] = sums[i];
  }
  __syncthreads();
  if (threadIdx.x < 2)
    verify_masses(a, r)[threadIdx.x * a.chunks + blockIdx.x] =
        s_sum[0][threadIdx.x] + s_sum[1][threadIdx.x] + s_sum[2][threadIdx.x] + s_sum[3][threadIdx.x];
}

// Block r: the chunk in which the running sum passes, then the token in it.
template <bool F32>
__device__ void verify_pick(const VerifyArgs& a) {
  __shared__ double s_sum[256];
  __shared__ int s_last[256];
  const int r = blockIdx.x;
  const VerifyLaw law = verify_law<F32>(a, r);
  int first, count;
  verify_rows(a, r, first, count);
  long long token = law.place;
  if (count >= 0 && law.heat != kVerifyGreedy) {
    const double* masses = verify_masses(a, r);
    double total = 0.0;
    for (int c = 0; c < a.chunks; ++c) total += masses[c];
    const bool whole = !(total > 0.0);
    if (whole) {
      masses += a.chunks;
      total = 0.0;
      for (int c = 0; c < a.chunks; ++c) total += masses[c];
    }
    const double target = (double)a.uniforms[(size_t)r * (a.drafts + 1) + a.drafts] * total;
    // the chunk; past the total (a random number of 1, or the sums' last bits) the last one that has weight
    double before = 0.0, run = 0.0;
    int chunk = 0;
    for (int c = 0; c < a.chunks; ++c) {
      const double mass = masses[c];
      if (mass > 0.0) {
        chunk = c, before = run;
        if (run + mass > target) break;
      }
      run += mass;
    }
    // a thread sums its run of tokens, then walks it if the sum passes there
    const int begin = chunk * kVerifyChunk, end = min(a.vocab, begin + kVerifyChunk);
    const int mine = begin + threadIdx.x * (kVerifyChunk / 256), stop = min(end, mine + kVerifyChunk / 256);
    double sum = 0.0;
    int last = -1;
    for (int v = mine; v < stop; ++v) {
      double all, left;
      verify_left<F32>(law, v, all, left);
      const double w = whole ? all : left;
      sum += w;
      if (w > 0.0) last = v;
    }
    s_sum[threadIdx.x] = sum;
    s_last[threadIdx.x] = last;
    __syncthreads();
    double at = before;
    int owner = -1, final = -1;
    double from = 0.0;
    for (int i = 0; i < 256; ++i) {
      if (s_last[i] >= 0) {
        final = s_last[i];
        if (owner < 0 && at + s_sum[i] > target) owner = i, from = at;
      }
      at += s_sum[i];
    }
    token = final >= 0 ? final : law.place;
    if (owner >= 0) {
      token = s_last[owner];
      int v = begin + owner * (kVerifyChunk / 256);
      const int until = min(end, v + kVerifyChunk / 256);
      for (; v < until; ++v) {
        double all, left;
        verify_left<F32>(law, v, all, left);
        from += whole ? all : left;
        if (from > target) {
          token = v;
          break;
        }
      }
    }
  }
  for (int i = threadIdx.x; i <= a.drafts; i += 256) {
    long long out = -1;
    if (count >= 0 && i < law.accepted) out = a.draft_tokens[(size_t)r * a.drafts + i];
    if (count >= 0 && i == law.accepted) out = token;
    a.tokens_out[(size_t)r * (a.drafts + 1) + i] = out;
  }
  if (threadIdx.x == 0) a.accepted[r] = law.accepted;
}

}  // namespace aoto

#define AOTO_VERIFY_INSTANCE(NAME, F32)                                                               \
  extern "C" __global__ __launch_bounds__(256) void aoto_verify_stats_##NAME(VerifyArgs a) {          \
    aoto::verify_stats<F32>(a);                                                                       \
  }                                                                                                   \
  extern "C" __global__ __launch_bounds__(256) void aoto_verify_mass_##NAME(VerifyArgs a) {           \
    aoto::verify_mass<F32>(a);                                                                        \
  }                                                                                                   \
  extern "C" __global__ __launch_bounds__(256) void aoto_verify_pick_##NAME(VerifyArgs a) {           \
    aoto::verify_pick<F32>(a);                                                                        \
  }
