// Verification of drafted tokens against the target's logits, from given random numbers.
//
// Laws of a row of logits z at temperature T > 0: p_v = w_v / sum w, w_v = exp((z_v - max z) / T); a NaN counts as
// -inf, a row without a number above -inf has w = 0. Draft i of request r (drafted from q, a point mass where no draft
// logits are given) stands while u_i q(x_i) < p_i(x_i); at the first that does not, the token that follows is drawn
// from max(p_i - q_i, 0) (from p_i where that is 0 throughout), after all of them from the last row's p: the first v
// at which the running sum of weights passes u_last times their total. T <= 0: a draft stands where it is the row's
// first maximum, which is also the token that follows.
//
// All of it is held in 64 bits, the exponentials too (right to 3e-15 of themselves, exp2.h): a token is where a sum
// over the vocabulary passes a random number, and the sums' noise in 32 bits (1e-7 of the total, against a typical
// weight of 1e-5 to 1e-6 of it) would move it in a percent of the calls.
//
// Launches over chunks of kVerifyChunk tokens: every row's maximum, its place and sum of weights by chunk; with a draft
// model's logits, what stands and the weights the following token is drawn from, summed by chunk; the token.
//
// The first is bound by its instructions, 20 a logit of which 11 in 64 bits (64 requests, up to five drafts with their
// logits, 128256 bf16 tokens: 33 us of 57), after it by the chain request -> statistics -> law -> chunk -> token, each
// a round trip to memory: 6 + 10 + 10 us there, 13 of 25 us without a draft model. Chunks of 2048 tokens deal the work
// out evenly (57 us; 4096: 63, 1024: 64 us) and leave the joins short. A loop over the chunk's loads, for less code,
// cost more than the instructions it fetched (1 to 2 us).
#pragma once

#include "common.h"
#include "exp2.h"
#include "paged_args.h"

namespace aoto {

constexpr int kVerifyPick = kVerifyChunk / 8;  // threads of the last launch: a chunk is eight tokens each

// What the first launch leaves of a chunk of a row: the sum of exp((z - max) / T), the maximum and its first place.
struct VerifyChunk {
  double sum;
  float top;
  int place;
};
static_assert(sizeof(VerifyChunk) == kVerifyChunkBytes, "as the workspace is sized");

// 2^(j / 32), in LDS: every kernel below fills it before its first weight. All 32 lie in banks of their own.
struct VerifyTable {
  double at[32];
};
AOTO_DEVICE void verify_table(VerifyTable& table) {
  if (threadIdx.x < 32) table.at[threadIdx.x] = exp2_32nds(threadIdx.x);
}

// A request's temperature: 32 log2(e) / T and its inverse; heat32 < 0: greedy.
struct VerifyHeat {
  double heat32, cool;
  AOTO_DEVICE bool greedy() const { return heat32 < 0.0; }
};
AOTO_DEVICE float verify_temperature(const VerifyArgs& a, int r) { return a.temperature ? a.temperature[r] : 0.f; }
AOTO_DEVICE VerifyHeat verify_heat(float t) {
  if (!(t > 0.f)) return {-1.0, 0.0};
  return {46.166241308446828384 / (double)t, (double)t * (1.0 / 46.166241308446828384)};
}

// The weights exp((z - top) / T) of a row's tokens. A NaN or -inf weighs 0; the logits equal to an infinite top weigh 1
// and nothing else does.
struct VerifyScale {
  double top, heat32;
  const VerifyTable& table;
  float floor;    // logits below it are taken as it: at 2^-2000 of the top, 0
  bool plain;     // nothing is infinite, and the floor is where it should be after its rounding to 32 bits
  // `below`: the powers of two under the top that the floor lies
  AOTO_DEVICE VerifyScale(float t, const VerifyHeat& h, const VerifyTable& tab, double below = 2000.0)
      : top(t), heat32(h.heat32), table(tab) {
    floor = (float)((double)t - 32.0 * below * h.cool);
    const double reach = (top - (double)floor) * heat32;
    plain = fabsf(t) < INFINITY && reach >= 0.95 * 32.0 * below && reach <= 1.02 * 32.0 * below;
  }
  AOTO_DEVICE double operator()(float z) const { return plain ? quick(z) : careful(z); }
  AOTO_DEVICE double quick(float z) const {
    return exp2_of((double)fmaxf(z, floor) - top, heat32, table.at);  // fmaxf: a NaN gives the floor
  }
  AOTO_DEVICE double careful(float z) const {
    if (!(z > -INFINITY)) return 0.0;
    if ((double)z == top) return 1.0;
    return top == INFINITY ? 0.0 : exp2_of(fmax(((double)z - top) * heat32, -64000.0), 1.0, table.at);
  }
};

template <bool F32>
AOTO_DEVICE float verify_logit(const void* row, int v) {
  const float z = F32 ? static_cast<const float*>(row)[v] : bf16_to_f32(static_cast<const uint16_t*>(row)[v]);
  return z != z ? -INFINITY : z;
}

// Rows of request r: its first, and how many drafts of it there are.
AOTO_DEVICE void verify_rows(const VerifyArgs& a, int r, int& first, int& count) {
  first = min(max(a.query_start[r], 0), a.rows);
  const int end = min(max(a.query_start[r + 1], first), a.rows);
  count = min(end - first - 1, a.drafts);  // -1: the request has no row
}

// A double moved across lanes as its two halves (0 where the move has no source or the row is left out).
template <int CTRL, int ROWS>
AOTO_DEVICE double dpp_f64(double v) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xF, true);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xF, true);
  return __hiloint2double(hi, lo);
}
// Running sums over a wave: within rows of 16 by shifts of 1, 2, 4 and 8, then the rows' last lanes on to the rows
// behind them.
AOTO_DEVICE double wave_scan_f64(double v) {
  v += dpp_f64<0x111, 0xF>(v);
  v += dpp_f64<0x112, 0xF>(v);
  v += dpp_f64<0x114, 0xF>(v);
  v += dpp_f64<0x118, 0xF>(v);
  v += dpp_f64<0x142, 0xA>(v);
  v += dpp_f64<0x143, 0xC>(v);
  return v;
}
AOTO_DEVICE double wave_last_f64(double v) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), 63),
                          __builtin_amdgcn_readlane(__double2loint(v), 63));
}
// The wave's total, in every lane.
AOTO_DEVICE double wave_sum_f64(double v) { return wave_last_f64(wave_scan_f64(v)); }

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

// The logits of a chunk that a lane of one wave holds: 16 bytes at a time, 1 KB a wave and load.
template <bool F32>
struct VerifyHeld {
  static constexpr int EACH = F32 ? 4 : 8, LOADS = kVerifyChunk / 64 / EACH;
  uint4 raw[LOADS];
  AOTO_DEVICE static int at(int load) { return (64 * load + (int)(threadIdx.x & 63)) * EACH; }
  AOTO_DEVICE void get(int load, float (&z)[EACH]) const {
    const uint32_t w[4] = {raw[load].x, raw[load].y, raw[load].z, raw[load].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (F32) z[i] = __uint_as_float(w[i]);
      else z[2 * i] = bf16_lo(w[i]), z[2 * i + 1] = bf16_hi(w[i]);
    }
  }
};

// Wave (chunk, r * judged + i): target row i of request r (i <= drafts), or its draft row i - drafts - 1. All of the
// chunk's loads go out at once and stay in registers: a lane's maximum, then its weights against that, then the lanes'
// sums brought to the wave's maximum. Nothing is shared between waves, so none waits for another. A greedy row's first
// place is kept instead of weights.
template <bool F32>
__device__ void verify_stats(const VerifyArgs& a) {
  using Held = VerifyHeld<F32>;
  __shared__ VerifyTable table;
  const int r = blockIdx.y / a.judged, i = blockIdx.y % a.judged;
  const int chunk = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int first, count;
  verify_rows(a, r, first, count);
  const bool draft = i > a.drafts;
  const float temperature = verify_temperature(a, r);
  if (draft ? (a.draft_logits == nullptr || i - a.drafts - 1 >= count || !(temperature > 0.f)) : i > count) return;
  const void* row = draft ? verify_row<F32>(a.draft_logits, r * a.draft_request_stride +
                                                                (i - a.drafts - 1) * a.draft_row_stride)
                          : verify_row<F32>(a.logits, (first + i) * a.row_stride);
  const int begin = chunk * kVerifyChunk, end = min(a.vocab, begin + kVerifyChunk);
  // loads past the row's end, and those of a row that is not 16-byte aligned, are put together from single logits
  const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
  const uint4* from = reinterpret_cast<const uint4*>(verify_row<F32>(row, begin));
  Held held;
#pragma unroll
  for (int l = 0; l < Held::LOADS; ++l) held.raw[l] = make_uint4(0, 0, 0, 0);
  if (aligned) {
#pragma unroll
    for (int l = 0; l < Held::LOADS; ++l)
      if (begin + Held::at(l) + Held::EACH <= end) held.raw[l] = from[Held::at(l) / Held::EACH];
  }
  if (!aligned || begin + kVerifyChunk > end) {
#pragma unroll
    for (int l = 0; l < Held::LOADS; ++l)
      if (!aligned || begin + Held::at(l) + Held::EACH > end) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int v = begin + Held::at(l) + (F32 ? k : 2 * k);
          const float lo = v < end ? verify_logit<F32>(row, v) : -INFINITY;
          const float hi = !F32 && v + 1 < end ? verify_logit<F32>(row, v + 1) : -INFINITY;
          w[k] = F32 ? __float_as_uint(lo) : __float_as_uint(lo) >> 16 | (__float_as_uint(hi) & 0xFFFF0000u);
        }
        held.raw[l] = make_uint4(w[0], w[1], w[2], w[3]);
      }
  }
  // while the loads are on their way
  const VerifyHeat heat = verify_heat(temperature);
  if (!heat.greedy()) {
    verify_table(table);
    __syncthreads();
  }
  if (chunk >= a.chunks) return;  // it held nothing
  float top = -INFINITY;
  int place = begin;
  double sum = 0.0;
  float z[Held::EACH];
  if (heat.greedy()) {
#pragma unroll
    for (int l = 0; l < Held::LOADS; ++l) {
      held.get(l, z);
#pragma unroll
      for (int e = 0; e < Held::EACH; ++e)
        if (z[e] > top) top = z[e], place = begin + Held::at(l) + e;  // a NaN is above nothing
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const float t = __shfl_xor(top, d);
      const int p = __shfl_xor(place, d);
      if (t > top || (t == top && p < place)) top = t, place = p;
    }
  } else {
#pragma unroll
    for (int l = 0; l < Held::LOADS; ++l) {
      held.get(l, z);
#pragma unroll
      for (int e = 0; e < Held::EACH; ++e) top = fmaxf(top, z[e]);  // past a NaN
    }
    const VerifyScale weight(top, heat, table, 980.0);  // what lies lower adds 2^-980 instead of less
    if (weight.plain) {
#pragma unroll
      for (int l = 0; l < Held::LOADS; ++l) {
        held.get(l, z);
#pragma unroll
        for (int e = 0; e < Held::EACH; ++e)
          sum = exp2_added((double)fmaxf(z[e], weight.floor) - weight.top, heat.heat32, table.at, sum);
      }
    } else if (top > -INFINITY) {
#pragma unroll
      for (int l = 0; l < Held::LOADS; ++l) {
        held.get(l, z);
#pragma unroll 1
        for (int e = 0; e < Held::EACH; ++e) {
          float x = z[0];
#pragma unroll
          for (int k = 1; k < Held::EACH; ++k) x = e == k ? z[k] : x;
          sum += weight(x);
        }
      }
    }
    const float all = wave_max(top);
    sum = wave_sum_f64(sum == 0.0 ? 0.0 : sum * VerifyScale(all, heat, table)(top));
    top = all;
  }
  if (lane == 0) {
    VerifyChunk* out = static_cast<VerifyChunk*>(a.workspace) +
                       ((size_t)r * (2 * a.drafts + 1) + i) * a.chunks + chunk;
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
  double sum, draft_sum;
  double fell;             // the removed token's weight
  VerifyHeat heat;
};
static_assert(sizeof(VerifyLaw) <= kVerifyLawBytes, "as the workspace is sized");

// By the whole block: 16 lanes join the chunks of a row, then lane i of the first wave judges draft i and the ballot
// finds the first that falls. Two round trips to memory: what is known of the request, then the chunks' statistics
// beside the drafted tokens' logits.
template <bool F32, int THREADS>
AOTO_DEVICE VerifyLaw verify_law(const VerifyArgs& a, int r, VerifyTable& table) {
  __shared__ float s_top[126];
  __shared__ double s_sum[126];
  __shared__ int s_place[126];
  __shared__ VerifyLaw s_law;
  const int lane = threadIdx.x & 63, part = threadIdx.x & 15;
  long long x = -1;
  float u = 0.f;
  if (threadIdx.x < a.drafts) {
    x = a.draft_tokens[(size_t)r * a.drafts + threadIdx.x];
    if (a.uniforms) u = a.uniforms[(size_t)r * (a.drafts + 1) + threadIdx.x];
  }
  int first, count;
  verify_rows(a, r, first, count);
  const VerifyHeat heat = verify_heat(verify_temperature(a, r));
  const bool sampled = !heat.greedy(), laws = a.draft_logits && sampled;
  const bool known = (int)threadIdx.x < count && x >= 0 && x < a.vocab;
  float zx = -INFINITY, yx = -INFINITY;
  if (known && sampled) {
    zx = verify_logit<F32>(verify_row<F32>(a.logits, (first + lane) * a.row_stride), (int)x);
    if (laws)
      yx = verify_logit<F32>(
          verify_row<F32>(a.draft_logits, r * a.draft_request_stride + lane * a.draft_row_stride), (int)x);
  }
  const VerifyChunk* chunks = static_cast<const VerifyChunk*>(a.workspace) + (size_t)r * (2 * a.drafts + 1) * a.chunks;
  const int rows = count + 1 + (laws && count > 0 ? count : 0);
  verify_table(table);
  __syncthreads();
  for (int j0 = 0; j0 < rows; j0 += THREADS / 16) {
    const int j = j0 + (threadIdx.x >> 4);
    const bool live = j < rows;
    const VerifyChunk* from = chunks + (size_t)(j <= count ? j : a.drafts + j - count) * a.chunks;
    constexpr int SOME = 5;  // a lane's chunks that are loaded at once: 163840 tokens
    VerifyChunk mine[SOME];
#pragma unroll
    for (int k = 0; k < SOME; ++k) {
      mine[k] = VerifyChunk{0.0, -INFINITY, 0};
      if (live && part + 16 * k < a.chunks) mine[k] = from[part + 16 * k];
    }
    float top = -INFINITY;
    int place = 0;
    auto better = [&](const VerifyChunk& one) {
      if (one.top > top) top = one.top, place = one.place;
    };
#pragma unroll
    for (int k = 0; k < SOME; ++k) better(mine[k]);
    for (int c = part + 16 * SOME; live && c < a.chunks; c += 16) better(from[c]);
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      const float t = __shfl_xor(top, d);
      const int p = __shfl_xor(place, d);
      if (t > top || (t == top && p < place)) top = t, place = p;
    }
    double sum = 0.0;
    if (sampled) {
      const VerifyScale weight(top, heat, table);
      auto add = [&](const VerifyChunk& one) {
        if (one.sum != 0.0) sum += one.sum * weight(one.top);
      };
#pragma unroll
      for (int k = 0; k < SOME; ++k) add(mine[k]);
      for (int c = part + 16 * SOME; live && c < a.chunks; c += 16) add(from[c]);
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor(sum, d);
    }
    if (live && part == 0) s_top[j] = top, s_sum[j] = sum, s_place[j] = top > -INFINITY ? place : 0;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    bool stands = false;
    double wx = 0.0;
    if (known) {
      if (sampled) {
        if (s_sum[lane] > 0.0) wx = VerifyScale(s_top[lane], heat, table)(zx);
        const double px = s_sum[lane] > 0.0 ? wx / s_sum[lane] : 0.0;
        const int j = count + 1 + lane;
        const double qx = !laws ? 1.0 : s_sum[j] > 0.0 ? VerifyScale(s_top[j], heat, table)(yx) / s_sum[j] : 0.0;
        stands = (double)u * qx < px;
      } else {
        stands = s_top[lane] > -INFINITY && s_place[lane] == (int)x;
      }
    }
    const int k = min(max(count, 0), __ffsll(~__ballot(stands)) - 1);
    const long long fell = __shfl(x, k);
    const double weighed = __shfl(wx, k);
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
          law.removed = fell >= 0 && fell < a.vocab ? (int)fell : -1;
          law.fell = weighed;
        }
      }
      s_law = law;
    }
  }
  __syncthreads();
  return s_law;
}

// The weights of eight logits, 0 from the `count`th on. (What is not plain is rare and kept out of the way.)
AOTO_DEVICE void verify_weights(const VerifyScale& weight, const float (&z)[8], int count, double (&w)[8]) {
  if (weight.plain) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = weight.quick(z[i]);
  } else {
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      float x = z[0];
#pragma unroll
      for (int k = 1; k < 8; ++k) x = i == k ? z[k] : x;
      const double one = weight.careful(x);
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = i == k ? one : w[k];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = i < count ? w[i] : 0.0;
}

// The weights of tokens v .. v + 7 under the target's law and what is left of them.
template <bool F32>
AOTO_DEVICE void verify_left(const VerifyLaw& law, const VerifyTable& table, int v, int end, double (&whole)[8],
                             double (&left)[8]) {
  const bool minus = law.draft_row && law.draft_sum > 0.0;
  float z[8], y[8];
  verify_load<F32>(law.row, v, end, z);
  if (minus) verify_load<F32>(law.draft_row, v, end, y);
  verify_weights(VerifyScale(law.top, law.heat, table), z, law.sum > 0.0 ? end - v : 0, whole);
#pragma unroll
  for (int i = 0; i < 8; ++i) left[i] = v + i == law.removed ? 0.0 : whole[i];
  if (minus) {
    // p - q, times the target's sum
    const double ratio = law.sum / law.draft_sum;
    double other[8];
    verify_weights(VerifyScale(law.draft_top, law.heat, table), y, end - v, other);
#pragma unroll
    for (int i = 0; i < 8; ++i) left[i] = fmax(whole[i] - ratio * other[i], 0.0);
  }
}

AOTO_DEVICE double* verify_masses(const VerifyArgs& a, int r) {
  const size_t chunks = (size_t)a.requests * (2 * a.drafts + 1) * a.chunks;
  return reinterpret_cast<double*>(static_cast<VerifyChunk*>(a.workspace) + chunks) + (size_t)r * a.chunks;
}
AOTO_DEVICE VerifyLaw* verify_laws(const VerifyArgs& a) {
  return reinterpret_cast<VerifyLaw*>(verify_masses(a, a.requests));
}

// Block r: the request's law, for the two launches behind it (every chunk's block finding it anew cost more: the sums
// of 64 requests took 21 us, against 5 for this launch and 10).
template <bool F32>
__device__ void verify_keep(const VerifyArgs& a) {
  __shared__ VerifyTable table;
  const VerifyLaw law = verify_law<F32, 256>(a, blockIdx.x, table);
  if (threadIdx.x == 0) verify_laws(a)[blockIdx.x] = law;
}

// Block (chunk, r): the chunk's sum of what a draft model's law leaves of the target's, where a draft fell. (Other
// requests' chunk sums are those of the statistics, less a removed token's weight.)
template <bool F32>
__device__ void verify_mass(const VerifyArgs& a) {
  static_assert(kVerifyChunk == 8 * 256, "a chunk is eight tokens a thread");
  __shared__ VerifyTable table;
  __shared__ double s_sum[4];
  const int r = blockIdx.y;
  const VerifyLaw law = verify_laws(a)[r];
  if (law.draft_row == nullptr) return;
  verify_table(table);
  __syncthreads();
  const int begin = blockIdx.x * kVerifyChunk, end = min(a.vocab, begin + kVerifyChunk);
  const int v = begin + 8 * threadIdx.x;
  double sum = 0.0;
  if (v < end) {
    double whole[8], left[8];
    verify_left<F32>(law, table, v, end, whole, left);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += left[i];
  }
  sum = wave_sum_f64(sum);
  if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) verify_masses(a, r)[blockIdx.x] = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
}

// Block r: the chunk in which the running sum passes, then the token in it, eight a thread. KEPT: the law
// and the sums of subtracted laws are there already.
template <bool F32, bool KEPT>
__device__ void verify_pick(const VerifyArgs& a) {
  static_assert(kVerifyChunk == 8 * kVerifyPick, "a chunk is eight tokens a thread");
  __shared__ double s_sum[kVerifyPick / 64], s_before, s_target;
  __shared__ int s_chunk, s_whole, s_token, s_last;
  const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __shared__ VerifyTable table;
  const float u = a.uniforms ? a.uniforms[(size_t)r * (a.drafts + 1) + a.drafts] : 0.f;
  VerifyLaw law;
  if constexpr (KEPT) {
    law = verify_laws(a)[r];
    verify_table(table);
    __syncthreads();
  } else {
    law = verify_law<F32, kVerifyPick>(a, r, table);
  }
  long long token = law.place;
  if (law.count >= 0 && !law.heat.greedy()) {
    if (wave == 0) {
      const VerifyChunk* chunks = static_cast<const VerifyChunk*>(a.workspace) +
                                  ((size_t)r * (2 * a.drafts + 1) + law.accepted) * a.chunks;
      const VerifyScale weight(law.top, law.heat, table);
      bool whole = false;
      // a chunk's weight: as a subtracted law left it, or of its statistics
      auto load = [&](int c) {
        const int at = min(c, a.chunks - 1);
        if (!whole && law.draft_row) return VerifyChunk{verify_masses(a, r)[at], law.top, 0};
        return chunks[at];
      };
      auto mass = [&](int c, const VerifyChunk& of) {
        if (c >= a.chunks || !(of.sum > 0.0)) return 0.0;
        if (!whole && law.draft_row) return of.sum;
        const double sum = of.sum * weight(of.top);
        if (whole || law.removed < 0 || law.removed / kVerifyChunk != c) return sum;
        // what a removed token leaves of its chunk; of the difference's rounding nothing
        const double left = sum - law.fell;
        return left > 0x1p-50 * sum ? left : 0.0;
      };
      constexpr int NEAR = 2;  // chunks a lane that are loaded once and stay in registers: 262144 tokens
      double near[NEAR];
      auto sum_up = [&] {
        VerifyChunk of[NEAR];
#pragma unroll
        for (int n = 0; n < NEAR; ++n) of[n] = load(64 * n + lane);
        double total = 0.0;
#pragma unroll
        for (int n = 0; n < NEAR; ++n) near[n] = mass(64 * n + lane, of[n]), total += near[n];
        for (int c = 64 * NEAR + lane; c < a.chunks; c += 64) total += mass(c, load(c));
        return wave_sum_f64(total);
      };
      double total = sum_up();
      if (!(total > 0.0)) whole = true, total = sum_up();
      const double target = (double)u * total;
      // the chunk; past the total (a random number of 1, or the sums' last bits) the last one that has weight
      double run = 0.0, before = 0.0;
      int chunk = 0;
      for (int c = 0; c < a.chunks; c += 64) {
        const double m = c == 0 ? near[0] : c == 64 ? near[1] : mass(c + lane, load(c + lane));
        const double upto = run + wave_scan_f64(m);
        const unsigned long long some = __ballot(m > 0.0), past = __ballot(m > 0.0 && upto > target);
        const int at = past ? __ffsll(past) - 1 : some ? 63 - __clzll((long long)some) : -1;
        if (at >= 0) chunk = c + at, before = __shfl(upto - m, at);
        if (past) break;
        run = wave_last_f64(upto);
      }
      if (lane == 0) s_chunk = chunk, s_before = before, s_whole = whole, s_target = target;
    }
    if (threadIdx.x == 0) s_token = 0x7FFFFFFF, s_last = -1;
    __syncthreads();
    const double target = s_target;
    const int begin = s_chunk * kVerifyChunk, end = min(a.vocab, begin + kVerifyChunk);
    const int v = begin + 8 * threadIdx.x;
    double all[8], left[8];
    verify_left<F32>(law, table, v, end, all, left);
    double sum = 0.0;
    int last = -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (s_whole) left[i] = all[i];
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
  for (int i = threadIdx.x; i <= a.drafts; i += kVerifyPick) {
    long long out = -1;
    if (law.count >= 0 && i < law.accepted) out = a.draft_tokens[(size_t)r * a.drafts + i];
    if (law.count >= 0 && i == law.accepted) out = token;
    a.tokens_out[(size_t)r * (a.drafts + 1) + i] = out;
  }
  if (threadIdx.x == 0) a.accepted[r] = law.accepted;
}

}  // namespace aoto

#define AOTO_VERIFY_INSTANCE(NAME, F32)                                                                    \
  extern "C" __global__ __launch_bounds__(256) void aoto_verify_stats_##NAME(VerifyArgs a) {               \
    aoto::verify_stats<F32>(a);                                                                            \
  }                                                                                                        \
  extern "C" __global__ __launch_bounds__(256) void aoto_verify_law_##NAME(VerifyArgs a) {                 \
    aoto::verify_keep<F32>(a);                                                                             \
  }                                                                                                        \
  extern "C" __global__ __launch_bounds__(256) void aoto_verify_mass_##NAME(VerifyArgs a) {                \
    aoto::verify_mass<F32>(a);                                                                             \
  }                                                                                                        \
  extern "C" __global__ __launch_bounds__(aoto::kVerifyPick) void aoto_verify_pick_##NAME(VerifyArgs a) {  \
    aoto::verify_pick<F32, true>(a);                                                                       \
  }                                                                                                        \
  extern "C" __global__ __launch_bounds__(aoto::kVerifyPick) void aoto_verify_follow_##NAME(VerifyArgs a) {\
    aoto::verify_pick<F32, false>(a);                                                                      \
  }
