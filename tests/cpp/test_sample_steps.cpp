// The steps of a flat row's histogram (csrc/sample_steps.hpp): two logits bound exactly the floats of a run of steps, also
// where no float lies in it because the temperature is small against the floats' distance.
#include "../../moss-transcribe.cpp_amd/csrc/sample_steps.hpp"

#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

using namespace mtg::sample;

static int failures = 0;
#define CHECK(x)                                                        \
  do {                                                                  \
    if (!(x)) {                                                         \
      if (++failures < 20) std::fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #x); \
    }                                                                   \
  } while (0)

// As the kernel takes an id: the median of the three is the logit.
static bool between(float x, float low, float high) {
  float v[3] = {x, low, high};
  std::sort(v, v + 3);
  return v[1] == x;
}

int main() {
  std::mt19937 rng(5);
  int empty = 0, found = 0;
  for (int turn = 0; turn < 4000; ++turn) {
    const float top = turn % 3 ? 32.0f + (float)(rng() % 1000) / 64 : -40.0f + (float)(rng() % 80000) / 1000;
    // from many floats a step to many steps between two floats
    const float T = std::ldexp(1.0f + (float)(rng() % 1000) / 1000, (int)(rng() % 24) - 22);
    const double c = kPerNat / (double)T;
    std::vector<float> x{top};
    while (x.size() < 400) x.push_back(below(x.back()));
    for (int step = 0; step < kSteps; step += 1 + rng() % 20) {  // and some around each step's ends
      float y = (float)((double)top - step / c);
      for (int i = 0; i < 3; ++i) y = -below(-y);
      for (int i = 0; i < 6; ++i, y = below(y))
        if (y <= top) x.push_back(y);
    }
    for (int i = 0; i < 40; ++i) {
      const int from = rng() % 200, to = from + (i % 2 ? 0 : rng() % 30);
      float low, high;
      if (!bounds_of(top, c, from, to, &low, &high)) continue;
      ++found;
      empty += low == INFINITY;
      for (float y : x) {
        const int step = step_of(t_of(y, top, c));
        CHECK(between(y, low, high) == (step >= from && step <= to));
      }
    }
  }
  CHECK(empty > 1000 && found - empty > 1000);

  // Ten ids at 32 and 8,000 at each of the four floats below: at T = 1e-5 step 22, in which min-p's border at half of the
  // largest weight lies, holds no float, so no id is one of that run's.
  std::vector<float> row(10, 32.0f);
  float y = 32.0f;
  for (int i = 0; i < 4; ++i) {
    y = below(y);
    row.insert(row.end(), 8000, y);
  }
  const double c = kPerNat / (double)1e-5f;
  const int mstep = step_of(-kPerNat * std::log(0.5));
  CHECK(mstep == 22);
  float low, high;
  CHECK(bounds_of(32.0f, c, mstep, mstep, &low, &high));
  CHECK(std::count_if(row.begin(), row.end(), [&](float x) { return between(x, low, high); }) == 0);
  CHECK(bounds_of(32.0f, c, 0, 0, &low, &high));
  CHECK(std::count_if(row.begin(), row.end(), [&](float x) { return between(x, low, high); }) == 10);
  std::printf("{\"record\": \"sampleSteps\", \"failures\": %d}\n", failures);
  return 0;
}
