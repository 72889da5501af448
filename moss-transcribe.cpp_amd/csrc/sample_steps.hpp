// sample_steps.hpp - the steps of a flat row's histogram (sample.hip), and the logits that bound a run of them. Plain
// functions, so that the host tests run the very rules the kernels use.
#pragma once

#include <math.h>
#include <stdint.h>

#include "paged_kv.hpp"

#ifdef __HIPCC__
#define MTG_NOUNROLL _Pragma("nounroll")
#else
#define MTG_NOUNROLL
#endif

namespace mtg {
namespace sample {

constexpr int kSteps = 1024;      // of the histogram
constexpr double kPerNat = 32.0;  // of its steps

// t = 32 (top - x) / T of a logit x <= top, infinite where the weight is 0 whatever T. c: 32 / T.
MTG_HD double t_of(float x, float top, double c) {
  if (x == top) return 0.0;
  return top == INFINITY ? INFINITY : ((double)top - (double)x) * c;
}

// A t in 2^-24: adding 1.5 * 2^28 rounds to that, and the sum's lowest bits are the number. What is beyond the last step (and
// NaN) counts as its middle.
MTG_HD uint64_t fixed_of(double t) {
  return __builtin_bit_cast(uint64_t, fmin(t, kSteps - 0.5) + 0x1.8p28) & 0x3ffffffffull;
}
MTG_HD int step_of(double t) { return (int)(fixed_of(t) >> 24); }

// The next float below.
MTG_HD float below(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return __builtin_bit_cast(float, x > 0.0f ? b - 1 : x == 0.0f ? 0x80000001u : b + 1);
}
// The least logit in a step or before it, if it is found: t rounds up to the next step from step + 1 - 2^-25 on, and it is a float
// or two next to the logit of that t (but for logits so near 0 that t does not tell them apart).
MTG_HD bool least_of(float top, double c, int step, float* least) {
  auto in = [&](float x) { return x > -INFINITY && step_of(t_of(x, top, c)) <= step; };
  float x = fminf(fmaxf((float)((double)top - ((double)(step + 1) - 0x1p-25) / c), -3.4028235e38f), top);
  MTG_NOUNROLL for (int i = 0; i < 3 && !in(x); ++i) x = -below(-x);
  MTG_NOUNROLL for (int i = 0; i < 3 && in(below(x)); ++i) x = below(x);
  *least = x;
  return in(x) && !in(below(x));
}

// The lowest and the highest logit in steps from .. to, if they are found; both infinite where no float lies in them, which is
// where T / 32 is below the floats' distance (one that is above the other would bound the steps on both sides of the run).
MTG_HD bool bounds_of(float top, double c, int from, int to, float* low, float* high) {
  *low = -3.4028235e38f, *high = top;
  bool found = top != INFINITY && (to == kSteps - 1 || least_of(top, c, to, low));
  if (from > 0) found = least_of(top, c, from - 1, high) && found, *high = below(*high);
  if (*low > *high) *low = *high = INFINITY;
  return found;
}

}  // namespace sample
}  // namespace mtg
