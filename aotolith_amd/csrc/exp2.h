// Powers of two in 64 bits, for the verification of drafted tokens. (Follows common.h; nothing here but arithmetic, so
// that a host compiler can check it.)
//
// 2^x, x = d * heat32 / 32, for -2048 < x <= 0 (0 from 2^-1075 on): 32 x is rounded to a whole number k by a sum with
// 1.5 * 2^52, whose low bits are k; what is left, f = 32 x - k in one rounding, |f| <= 1/2, goes through the series of
// e^(f ln 2 / 32) to the 5th power, k mod 32 through a table, the rest of k to the exponent. Off by the series'
// remainder, below (ln 2 / 64)^6 / 6! = 2.3e-15 or 20 steps of 2^-53, and by 6 such steps of roundings.
#pragma once

namespace aoto {

// 2^(j / 32), 0 <= j < 32: the series of e^y, 0 <= y < ln 2, to the 20th power (remainder 1e-23).
AOTO_DEVICE double exp2_32nds(int j) {
  const double y = j * (0.6931471805599453094 / 32);
  double s = 1.0;
#pragma unroll
  for (int k = 20; k > 0; --k) s = fma(s, y * (1.0 / k), 1.0);
  return s;
}

struct Exp2Parts {
  double series;
  int k;
};
AOTO_DEVICE Exp2Parts exp2_parts(double d, double heat32) {
  constexpr double kRound = 6755399441055744.0;
  const double t = fma(d, heat32, kRound);
  const double f = fma(d, heat32, kRound - t);
  double s = 3.973709984549416e-11;  // (ln 2 / 32)^5 / 5!, and on to the 0th
  s = fma(s, f, 9.172562701824643e-09);
  s = fma(s, f, 1.693850972437182e-06);
  s = fma(s, f, 0.0002345961982022468);
  s = fma(s, f, 0.02166084939249829);
  return {fma(s, f, 1.0), __double2loint(t)};
}
// `table`: the 32 powers.
AOTO_DEVICE double exp2_of(double d, double heat32, const double* table) {
  const Exp2Parts p = exp2_parts(d, heat32);
  return ldexp(p.series * table[p.k & 31], p.k >> 5);
}
// sum + 2^x for x > -1000: the exponent goes into the table's number by whole-number arithmetic.
AOTO_DEVICE double exp2_added(double d, double heat32, const double* table, double sum) {
  const Exp2Parts p = exp2_parts(d, heat32);
  const double scale = table[p.k & 31];
  return fma(p.series, __hiloint2double(__double2hiint(scale) + ((p.k >> 5) << 20), __double2loint(scale)), sum);
}

}  // namespace aoto
