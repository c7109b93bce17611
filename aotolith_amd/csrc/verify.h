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
// Three launches over chunks of kVerifyChunk tokens: every row's maximum, its place and sum of weights by chunk; what
// stands, and the weights the following token is drawn from, summed by chunk; the token. Bound by the first one's read
// of the logits and, where they are sampled from, about as much by its 20 f64 operations a logit.
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

// 2^x for -2048 < x <= 0 (0 from 2^-1075 on): the series of 2^f = e^(f ln 2) over |f| <= 1/2 to the 12th power, whose
// remainder is below (ln 2 / 2)^13 / 13! = 1.7e-16, and the exponent's shift. x = d * heat is rounded to the nearest
// whole number by a sum with 1.5 * 2^52, whose low bits are that number; f = x - n in one rounding.
AOTO_DEVICE double exp2_of(double d, double heat) {
  constexpr double kRound = 6755399441055744.0;
  const double t = fma(d, heat, kRound);
  const double f = fma(d, heat, kRound - t);
  double s = 2.5678435993488206e-11;  // ln 2 ^ 12 / 12!, and on to the 0th
  s = fma(s, f, 4.4455382718708116e-10);
  s = fma(s, f, 7.054911620801123e-09);
  s = fma(s, f, 1.01780860092397e-07);
  s = fma(s, f, 1.321548679014431e-06);
  s = fma(s, f, 1.5252733804059841e-05);
  s = fma(s, f, 0.0001540353039338161);
  s = fma(s, f, 0.0013333558146428443);
  s = fma(s, f, 0.009618129107628477);
  s = fma(s, f, 0.05550410866482158);
  s = fma(s, f, 0.24022650695910072);
  s = fma(s, f, 0.6931471805599453);
  s = fma(s, f, 1.0);
  return ldexp(s, __double2loint(t));
}

// The weights exp((z - top) / T) of a row's tokens: heat = log2(e) / T. A NaN or -inf weighs 0; the logits equal to an
// infinite top weigh 1 and nothing else does.
struct VerifyScale {
  double top, heat;
  float floor;    // logits below it are taken as it, 2^-2000 of the top: 0
  bool plain;     // nothing is infinite, and the floor is where it should be after its rounding to 32 bits
  AOTO_DEVICE VerifyScale(float t, double h) : top(t), heat(h) {
    floor = (float)((double)t - 2000.0 / h);
    const double reach = (top - (double)floor) * h;
    plain = fabsf(t) < INFINITY && reach >= 1100.0 && reach <= 4000.0;
  }
  AOTO_DEVICE double operator()(float z) const {
    if (plain) return exp2_of((double)fmaxf(z, floor) - top, heat);  // fmaxf: a NaN gives the floor
    if (!(z > -INFINITY)) return 0.0;
    if ((double)z == top) return 1.0;
    return top == INFINITY ? 0.0 : exp2_of(fmax(((double)z - top) * heat, -2000.0), 1.0);
  }
};

AOTO_DEVICE double verify_weight(float z, float top, double heat) { return VerifyScale(top, heat)(z); }

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

template <bool F32>
AOTO_DEVICE const void* verify_row(const void* base, long long at) {
  return F32 ? (const void*)(static_cast<const float*>(base) + at)
             : (const void*)(static_cast<const uint16_t*>(base) + at);
}

// Tokens v .. v + 7 of a row (-inf past `end`), in 16-byte loads where the row allows it.
template <bool F32>
AOTO_DEVICE void verify_load(const void* row, int v, int end, float (&z)[8]) {
  if ((reinterpret_cast<uintptr_t>(row) & 15) == 0 && v + 8 <= end) {
    if constexpr (F32) {
      const float4* from = reinterpret_cast<const float4*>(static_cast<const float*>(row) + v);
      const float4 a = from[0], b = from[1];
      z[0] = a.x, z[1] = a.y, z[2] = a.z, z[3] = a.w, z[4] = b.x, z[5] = b.y, z[6] = b.z, z[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + v);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) z[2 * i] = bf16_lo(w[i]), z[2 * i + 1] = bf16_hi(w[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = fmaxf(z[i], -INFINITY);  // a NaN counts as -inf
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = v + i < end ? verify_logit<F32>(row, v + i) : -INFINITY;
  }
}

// Block (chunk, r * (2 drafts + 1) + i): target row i of request r (i <= drafts), or its draft row i - drafts - 1.
// A thread has 32 logits in registers and weighs them against its own maximum; the threads' sums are then brought to
// the block's. A greedy row's places are kept instead of weights.
template <bool F32>
__device__ void verify_stats(const VerifyArgs& a) {
  constexpr int GROUPS = kVerifyChunk / 2048;
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
  const int mine = begin + 8 * threadIdx.x;
  float z[GROUPS][8];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) verify_load<F32>(row, mine + 2048 * g, end, z[g]);
  float top = -INFINITY;
  int place = begin;
  double sum = 0.0;
  const int wave = threadIdx.x >> 6;
  if (heat == kVerifyGreedy) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (z[g][e] > top) top = z[g][e], place = mine + 2048 * g + e;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const float t = __shfl_xor(top, d);
      const int p = __shfl_xor(place, d);
      if (t > top || (t == top && p < place)) top = t, place = p;
    }
  } else {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, z[g][e]);
    const VerifyScale weight(top, heat);
    if (weight.plain) {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += exp2_of((double)fmaxf(z[g][e], weight.floor) - weight.top, heat);
    } else {
#pragma unroll 1
      for (int k = 0; k < 8 * GROUPS; ++k) {
        float x = -INFINITY;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
#pragma unroll
          for (int e = 0; e < 8; ++e) x = k == 8 * g + e ? z[g][e] : x;
        sum += weight(x);
      }
    }
    const float all = wave_max(top);
    sum = wave_sum_f64(sum == 0.0 ? 0.0 : sum * verify_weight(top, all, heat));
    top = all;
  }
  if ((threadIdx.x & 63) == 0) s_top[wave] = top, s_place[wave] = place, s_sum[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w)
      if (s_top[w] > top || (s_top[w] == top && s_place[w] < place)) top = s_top[w], place = s_place[w];
    sum = 0.0;
    if (heat != kVerifyGreedy)
      for (int w = 0; w < 4; ++w)
        if (s_sum[w] != 0.0) sum += s_sum[w] * verify_weight(s_top[w], top, heat);
    VerifyChunk* out = static_cast<VerifyChunk*>(a.workspace) + (size_t)blockIdx.y * a.chunks + blockIdx.x;
    *out = VerifyChunk{sum, top, place};
  }
}

// How many drafts of request r stand, and the law that the following token is drawn from.
struct VerifyLaw {
  int count, accepted;
  int place;               // the row's first maximum
  int removed;             // a drafted token of point mass that the law leaves out, or -1
  const void* row;
  const void* draft_row;   // null: nothing is subtracted
  float top, draft_top;
  double sum, draft_sum, heat;
};
static_assert(sizeof(VerifyLaw) <= kVerifyLawBytes, "as the workspace is sized");

// By the whole block: 16 lanes join the chunks of a row, then lane i of the first wave judges draft i and the ballot
// finds the first that falls.
template <bool F32, int THREADS>
AOTO_DEVICE VerifyLaw verify_law(const VerifyArgs& a, int r) {
  __shared__ float s_top[126];
  __shared__ double s_sum[126];
  __shared__ int s_place[126];
  __shared__ VerifyLaw s_law;
  int first, count;
  verify_rows(a, r, first, count);
  const int lane = threadIdx.x & 63, part = threadIdx.x & 15;
  const double heat = verify_heat(a, r);
  const bool sampled = heat != kVerifyGreedy, laws = a.draft_logits && sampled;
  const VerifyChunk* chunks = static_cast<const VerifyChunk*>(a.workspace) + (size_t)r * (2 * a.drafts + 1) * a.chunks;
  const int rows = count + 1 + (laws && count > 0 ? count : 0);
  for (int j0 = 0; j0 < rows; j0 += THREADS / 16) {
    const int j = j0 + (threadIdx.x >> 4);
    const bool live = j < rows;
    const VerifyChunk* from = chunks + (size_t)(j <= count ? j : a.drafts + j - count) * a.chunks;
    float top = -INFINITY;
    int place = 0;
    for (int c = part; live && c < a.chunks; c += 16)
      if (from[c].top > top) top = from[c].top, place = from[c].place;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      const float t = __shfl_xor(top, d);
      const int p = __shfl_xor(place, d);
      if (t > top || (t == top && p < place)) top = t, place = p;
    }
    double sum = 0.0;
    if (sampled) {
      for (int c = part; live && c < a.chunks; c += 16)
        if (from[c].sum != 0.0) sum += from[c].sum * verify_weight(from[c].top, top, heat);
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor(sum, d);
    }
    if (live && part == 0) s_top[j] = top, s_sum[j] = sum, s_place[j] = top > -INFINITY ? place : 0;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    bool stands = false;
    if (lane < count) {
      const long long x = a.draft_tokens[(size_t)r * a.drafts + lane];
      if (x >= 0 && x < a.vocab) {
        if (sampled) {
          const float z = verify_logit<F32>(verify_row<F32>(a.logits, (first + lane) * a.row_stride), (int)x);
          const double px = s_sum[lane] > 0.0 ? verify_weight(z, s_top[lane], heat) / s_sum[lane] : 0.0;
          double qx = 1.0;
          if (laws) {
            const float y = verify_logit<F32>(
                verify_row<F32>(a.draft_logits, r * a.draft_request_stride + lane * a.draft_row_stride), (int)x);
            const int j = count + 1 + lane;
            qx = s_sum[j] > 0.0 ? verify_weight(y, s_top[j], heat) / s_sum[j] : 0.0;
          }
          stands = (double)a.uniforms[(size_t)r * (a.drafts + 1) + lane] * qx < px;
        } else {
          stands = s_top[lane] > -INFINITY && s_place[lane] == (int)x;
        }
      }
    }
    const int k = min(max(count, 0), __ffsll(~__ballot(stands)) - 1);
    if (lane == 0) {
      VerifyLaw law{};
      law.count = count, law.accepted = k, law.heat = heat, law.removed = -1;
      law.row = verify_row<F32>(a.logits, (long long)min(first + k, a.rows - 1) * a.row_stride);
      if (count >= 0) law.place = s_place[k], law.top = s_top[k], law.sum = s_sum[k];
      if (k < count && sampled) {
        if (laws) {
          law.draft_row = verify_row<F32>(a.draft_logits, r * a.draft_request_stride + k * a.draft_row_stride);
          law.draft_top = s_top[count + 1 + k], law.draft_sum = s_sum[count + 1 + k];
        } else {
          const long long x = a.draft_tokens[(size_t)r * a.drafts + k];
          law.removed = x >= 0 && x < a.vocab ? (int)x : -1;
        }
      }
      s_law = law;
    }
  }
  __syncthreads();
  return s_law;
}

// The weights of tokens v .. v + 7 under the target's law and what is left of them.
template <bool F32>
AOTO_DEVICE void verify_left(const VerifyLaw& law, int v, int end, double (&whole)[8], double (&left)[8]) {
  float z[8];
  verify_load<F32>(law.row, v, end, z);
  const VerifyScale weight(law.top, law.heat);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    whole[i] = law.sum > 0.0 && v + i < end ? weight(z[i]) : 0.0;
    left[i] = v + i == law.removed ? 0.0 : whole[i];
  }
  if (law.draft_row && law.draft_sum > 0.0) {
    // p - q, times the target's sum
    const double ratio = law.sum / law.draft_sum;
    const VerifyScale other(law.draft_top, law.heat);
    verify_load<F32>(law.draft_row, v, end, z);
#pragma unroll
    for (int i = 0; i < 8; ++i) left[i] = v + i < end ? fmax(whole[i] - ratio * other(z[i]), 0.0) : 0.0;
  }
}

AOTO_DEVICE double* verify_masses(const VerifyArgs& a, int r) {
  const size_t chunks = (size_t)a.requests * (2 * a.drafts + 1) * a.chunks;
  return reinterpret_cast<double*>(static_cast<VerifyChunk*>(a.workspace) + chunks) + (size_t)r * 2 * a.chunks;
}
AOTO_DEVICE VerifyLaw* verify_laws(const VerifyArgs& a) {
  return reinterpret_cast<VerifyLaw*>(verify_masses(a, a.requests));
}

// Block (chunk, r): the chunk's sums of what is left and of the whole; the first one's law is kept.
template <bool F32>
__device__ void verify_mass(const VerifyArgs& a) {
  __shared__ double s_sum[4][2];
  const int r = blockIdx.y;
  const VerifyLaw law = verify_law<F32, 256>(a, r);
  if (blockIdx.x == 0 && threadIdx.x == 0) verify_laws(a)[r] = law;
  if (law.heat == kVerifyGreedy) return;
  const int begin = blockIdx.x * kVerifyChunk, end = min(a.vocab, begin + kVerifyChunk);
  double sums[2] = {0.0, 0.0};
#pragma unroll 1
  for (int v = begin + 8 * threadIdx.x; v < end; v += 2048) {
    double whole[8], left[8];
    verify_left<F32>(law, v, end, whole, left);
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[0] += left[i], sums[1] += whole[i];
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

// Running sums over a wave.
AOTO_DEVICE double wave_scan_f64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double up = __shfl_up(v, d);
    if ((int)(threadIdx.x & 63) >= d) v += up;
  }
  return v;
}

// Block r, 1024 threads: the chunk in which the running sum passes, then the token in it, eight a thread.
template <bool F32, bool KEPT>
__device__ void verify_pick(const VerifyArgs& a) {
  static_assert(kVerifyChunk == 8 * 1024, "a chunk is eight tokens a thread");
  __shared__ double s_sum[16], s_before;
  __shared__ int s_chunk, s_token, s_last;
  const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  VerifyLaw law;
  if constexpr (KEPT) law = verify_laws(a)[r];
  else law = verify_law<F32, 1024>(a, r);
  long long token = law.place;
  if (KEPT && law.count >= 0 && law.heat != kVerifyGreedy) {
    const float u = a.uniforms[(size_t)r * (a.drafts + 1) + a.drafts];
    const double* masses = verify_masses(a, r);
    double total = 0.0;
    for (int c = 0; c < a.chunks; c += 64) total += wave_sum_f64(c + lane < a.chunks ? masses[c + lane] : 0.0);
    const bool whole = !(total > 0.0);
    if (whole) {
      masses += a.chunks;
      total = 0.0;
      for (int c = 0; c < a.chunks; c += 64) total += wave_sum_f64(c + lane < a.chunks ? masses[c + lane] : 0.0);
    }
    const double target = (double)u * total;
    if (wave == 0) {
      // the chunk; past the total (a random number of 1, or the sums' last bits) the last one that has weight
      double run = 0.0, before = 0.0;
      int chunk = 0;
      for (int c = 0; c < a.chunks; c += 64) {
        const double mass = c + lane < a.chunks ? masses[c + lane] : 0.0;
        const double upto = run + wave_scan_f64(mass);
        const unsigned long long some = __ballot(mass > 0.0), past = __ballot(mass > 0.0 && upto > target);
        const int at = past ? __ffsll(past) - 1 : some ? 63 - __clzll((long long)some) : -1;
        if (at >= 0) chunk = c + at, before = __shfl(upto - mass, at);
        if (past) break;
        run = __shfl(upto, 63);
      }
      if (lane == 0) s_chunk = chunk, s_before = before;
    }
    if (threadIdx.x == 0) s_token = 0x7FFFFFFF, s_last = -1;
    __syncthreads();
    const int begin = s_chunk * kVerifyChunk, end = min(a.vocab, begin + kVerifyChunk);
    const int v = begin + 8 * threadIdx.x;
    double all[8], left[8];
    verify_left<F32>(law, v, end, all, left);
    double sum = 0.0;
    int last = -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (whole) left[i] = all[i];
      sum += left[i];
      if (left[i] > 0.0) last = v + i;
    }
    const double upto = wave_scan_f64(sum);
    if (lane == 63) s_sum[wave] = upto;
    __syncthreads();
    double run = s_before;
    for (int w = 0; w < wave; ++w) run += s_sum[w];
    run += upto - sum;
    int found = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      run += left[i];
      if (left[i] > 0.0 && run > target) found = min(found, v + i);
    }
    if (found != 0x7FFFFFFF) atomicMin(&s_token, found);
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    if (s_token != 0x7FFFFFFF) token = s_token;
    else if (s_last >= 0) token = s_last;
  }
  for (int i = threadIdx.x; i <= a.drafts; i += 1024) {
    long long out = -1;
    if (law.count >= 0 && i < law.accepted) out = a.draft_tokens[(size_t)r * a.drafts + i];
    if (law.count >= 0 && i == law.accepted) out = token;
    a.tokens_out[(size_t)r * (a.drafts + 1) + i] = out;
  }
  if (threadIdx.x == 0) a.accepted[r] = law.accepted;
}

}  // namespace aoto

#define AOTO_VERIFY_INSTANCE(NAME, F32)                                                                  \
  extern "C" __global__ __launch_bounds__(256) void aoto_verify_stats_##NAME(VerifyArgs a) {             \
    aoto::verify_stats<F32>(a);                                                                          \
  }                                                                                                      \
  extern "C" __global__ __launch_bounds__(256) void aoto_verify_mass_##NAME(VerifyArgs a) {              \
    aoto::verify_mass<F32>(a);                                                                           \
  }                                                                                                      \
  extern "C" __global__ __launch_bounds__(1024) void aoto_verify_pick_##NAME(VerifyArgs a) {             \
    aoto::verify_pick<F32, true>(a);                                                                     \
  }                                                                                                      \
  extern "C" __global__ __launch_bounds__(1024) void aoto_verify_greedy_##NAME(VerifyArgs a) {           \
    aoto::verify_pick<F32, false>(a);                                                                    \
  }
