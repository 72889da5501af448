// sample.hip - mtg_sample_dev: one id for each row of logits, by temperature, top-k, top-p and min-p from a given random
// number.
//
// With the ids in the order of their logits (the largest first, of equal ones the lowest id), every filter keeps a first
// part of that order, and the choice is the first id at which the running sum of the weights w = exp((x - max) / T) passes a
// target. No row is sorted: the part of the order that decides is found first, and only that is.
//
// k_sample_rows reads the logits once (HBM bounds it, and the 64-bit exponentials where they are summed up): the maximum of
// each unit of 128 ids goes to the workspace, and where the row's filters need the sum of all weights, that too.
// k_sample_pick, one workgroup to a row, has the answer for nearly all rows that a program samples: a threshold that at
// least `want` units' maxima reach is reached by at least that many ids, which lie in those units alone; they are gathered (a
// few hundred as a rule), put in order and summed up. With top-k that is k ids or somewhat more, else about 128. If the target lies beyond what was
// gathered (a flat row), the row is left to two more kernels, whose workgroups end at once for all other rows: k_sample_steps
// makes a histogram of its weights over 1,024 steps of 1/32 in (max - x) / T, by many workgroups, and k_sample_flat, one to a row,
// gathers only the steps in which a border or the choice may lie; if those hold too many ids as well (equal logits by the
// thousand), it narrows the borders down one by one, by the bits of the logits and then of the ids.
//
// For vocabularies of 150,000 one row takes 18 us, nearly all of it latency (four launches, a dozen barriers, instructions
// that no cache holds yet, for which reason code that runs once is kept short); 256 rows in f32 with top-k 200 55 us, of them 25 the reading
// at 6.2 TB/s; 61 flat rows in f16 89 to 95 us, of them 35 in k_sample_flat and 17 each in the first two. No workgroup waits for
// another one or has the last word: with marks between workgroups in one kernel 256 rows took 77 us, flat ones 461 instead of 140.
//
// Sums that decide are in 64 bits: an error of 2^-24 would move one choice in a few hundred rows, where it falls on a border.
#include "kernels.hpp"
#include "paged_dev.hpp"
#include "sample_steps.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

namespace mtg {
namespace {

using namespace paged;
using namespace sample;

constexpr int kThreads = 1024, kWaves = kThreads / 64;  // of a workgroup that decides
constexpr int kReadWaves = 8;                           // of one of k_sample_rows
constexpr int kPair = 256;       // ids that a wave reads at once: two units
constexpr int kUnit = 128;       // ids whose maximum is kept
constexpr int kUnits = 2048;     // most units of a row that a threshold is looked for in
constexpr int kFewUnits = 128;   // that many units' maxima are asked for without top-k
constexpr int kFew = 1024;        // most ids that k_sample_pick sorts
constexpr int kGather = 4096;    // and k_sample_flat
constexpr int kSlice = 32768;    // most ids of a workgroup (a step's count has 16 bits, its weights 48)

typedef f4 f4u __attribute__((aligned(4)));
typedef h4 h4u __attribute__((aligned(2)));

struct SampleArgs {
  mtg_sample a;
  int pairs, slices, per_slice;  // pairs of units of a row and of a workgroup
  float* tops;                   // [row][unit] maxima
  double* sums;                  // [row][slice][2]: a reference, the sum of exp((x - reference) / T)
  uint64_t* steps;               // [row][slice][step]: count << 48 | sum of 2^32 exp(-(t - step) / 32)
  float* left;                   // [row]: the largest logit where the row is left to k_sample_flat, else NaN
};

// A row's settings: ids kept by their number (0: all), by the share of the sum and by t = 32 (max - x) / T.
struct Settings {
  double c;      // 32 / T
  int k;
  double p;      // 1 or more: all
  double limit;  // of t; infinite: all
  double u;
};
__device__ __forceinline__ Settings settings_of(const mtg_sample& a, int row) {
  Settings s;
  const float T = a.settings[3 * row], p = a.settings[3 * row + 1], m = a.settings[3 * row + 2];
  const float u = a.uniform[row];
  s.k = a.top_k ? max(a.top_k[row], 0) : 0;
  s.c = kPerNat / (double)T;
  if (!(T > 0.0f) || p <= 0.0f || m > 1.0f) s.k = 1;
  if (!(T > 0.0f)) s.c = kPerNat;
  s.p = p < 1.0f && s.k != 1 ? (double)p : 2.0;
  s.limit = m > 0.0f && m <= 1.0f ? -kPerNat * log((double)m) : INFINITY;
  s.u = u > 0.0f ? fmin((double)u, 1.0 - 0x1p-24) : 0.0;
  return s;
}

// A logit that takes part, as bits in ascending order; 0 for NaN and -inf.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float((o >> 31) ? o & 0x7fffffffu : ~o); }

// 2^-y for y >= 0, to 2^-34: whole part and a polynomial (interpolated at the Chebyshev points of degree 7) for the rest;
// from y = 1,000 on 2^-1000. Adding 1.5 * 2^52 rounds to whole numbers, which then are the sum's lowest bits.
__device__ __forceinline__ double pow2_neg(double y) {
  y = fmin(y, 1000.0);
  const double n = y + 0x1.8p52, f = y - (n - 0x1.8p52);
  double p = -1.5303699258698893e-05;
  p = fma(p, f, 0.00015469729227549479);
  p = fma(p, f, -0.0013333478480007015);
  p = fma(p, f, 0.0096180256133226102);
  p = fma(p, f, -0.05550410906317723);
  p = fma(p, f, 0.2402265121349727);
  p = fma(p, f, -0.69314718055683522);
  p = fma(p, f, 0.99999999995956235);
  const uint64_t bits = __builtin_bit_cast(uint64_t, p) - (__builtin_bit_cast(uint64_t, n) << 52);
  return __builtin_bit_cast(double, bits);
}

// The largest of the values of lanes 0 to 31 and of the others, in all lanes. Rows of 16 lanes by shifts within them, the four
// rows by their last lanes.
__device__ __forceinline__ float2 max_halves(float x) {
  auto shifted = [](float x, auto by) {
    const int old = __float_as_int(x);
    return __int_as_float(__builtin_amdgcn_update_dpp(old, old, 0x110 + decltype(by)::value, 0xf, 0xf, false));  // row_shr
  };
  x = fmaxf(x, shifted(x, std::integral_constant<int, 1>{}));
  x = fmaxf(x, shifted(x, std::integral_constant<int, 2>{}));
  x = fmaxf(x, shifted(x, std::integral_constant<int, 4>{}));
  x = fmaxf(x, shifted(x, std::integral_constant<int, 8>{}));
  auto lane = [&](int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), i)); };
  return make_float2(fmaxf(lane(15), lane(31)), fmaxf(lane(47), lane(63)));
}
__device__ __forceinline__ float max_wave(float x) {
  const float2 m = max_halves(x);
  return fmaxf(m.x, m.y);
}

// The least of a wave's numbers, in all lanes.
__device__ __forceinline__ int min_wave(int x) {
  auto shifted = [](int x, auto by) { return __builtin_amdgcn_update_dpp(x, x, 0x110 + decltype(by)::value, 0xf, 0xf, false); };
  x = min(x, shifted(x, std::integral_constant<int, 1>{}));
  x = min(x, shifted(x, std::integral_constant<int, 2>{}));
  x = min(x, shifted(x, std::integral_constant<int, 4>{}));
  x = min(x, shifted(x, std::integral_constant<int, 8>{}));
  auto lane = [&](int i) { return __builtin_amdgcn_readlane(x, i); };
  return min(min(lane(15), lane(31)), min(lane(47), lane(63)));
}

// A lane's four ids 4 lane .. of a pair, -inf behind the row's end. All but the last one are whole: a branch of the wave.
__device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
  const f4u v = *(const f4u*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = v[i];
}
__device__ __forceinline__ void load4(const _Float16* p, float (&x)[4]) {
  const h4u v = *(const h4u*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = (float)v[i];
}
template <typename IO>
__device__ __forceinline__ void load_ids(const IO* row, int base, int end, int vocab, float (&x)[4]) {
  if (end <= vocab) {
    load4(row + base, x);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = base + i < vocab ? (float)row[base + i] : -INFINITY;
  }
}
template <typename IO>
__device__ __forceinline__ void load_pair(const IO* row, int pair, int vocab, float (&x)[4]) {
  load_ids(row, pair * kPair + 4 * (int)(threadIdx.x & 63), pair * kPair + kPair, vocab, x);
}

// ---- over a workgroup ----
template <int MOST>
struct Shared {
  static constexpr int kMost = MOST;
  uint64_t key[MOST];  // ~order << 32 | id: ascending in the order of the ids
  double sum[MOST];    // running sums of their weights
  float tops[kUnits];  // of the row's units, where there are so few
  uint16_t unit[kUnits];
  double red[kWaves];
  int redi[kWaves];
  int n, units, at[4];
  double z[4];
};

// Running sums of v[0 .. N-1] of thread 0, 1, ..: each becomes the sum up to and with it. Always in the same order.
template <int N, class T>
__device__ __forceinline__ void scan_block(T* red, T (&v)[N]) {
#pragma unroll
  for (int i = 1; i < N; ++i) v[i] += v[i - 1];
  T x = v[N - 1];
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const T y = __shfl_up(x, m);
    if (lane >= m) x += y;
  }
  __syncthreads();
  if (lane == 63) red[threadIdx.x >> 6] = x;
  const T left = __shfl_up(x, 1);
  __syncthreads();
  T before = 0;
#pragma nounroll
  for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) before += red[w];
  if (lane) before += left;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] += before;
}

// Puts the n keys in order. bucket(key): 0 .. n - 1, no less for a later key; few keys have the same one.
template <class S, class B>
__device__ __forceinline__ void sort_keys(S& s, int n, const B& bucket) {
  constexpr int N = S::kMost / kThreads;
  static_assert(S::kMost % kThreads == 0, "");
  if (n <= kThreads / 4) {  // few: each is held against all, by four threads
    const int i = threadIdx.x >> 2;
    const uint64_t key = i < n ? s.key[i] : 0;
    int before = 0;
#pragma unroll 4
    for (int k = threadIdx.x & 3; k < n; k += 4) before += s.key[k] < key;
    before += __shfl_xor(before, 1);
    before += __shfl_xor(before, 2);
    __syncthreads();
    if (i < n && (threadIdx.x & 3) == 0) s.key[before] = key;
    __syncthreads();
    return;
  }
  int* count = (int*)s.sum;  // of a bucket's keys, then where they begin
  uint64_t key[N];
  int at[N], place[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int k = i * kThreads + (int)threadIdx.x;
    if (k < n) key[i] = s.key[k], count[k] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i * kThreads + (int)threadIdx.x < n) at[i] = bucket(key[i]), place[i] = atomicAdd(&count[at[i]], 1);
  __syncthreads();
  int begin[N];
#pragma unroll
  for (int i = 0; i < N; ++i) begin[i] = (int)threadIdx.x * N + i < n ? count[threadIdx.x * N + i] : 0;
  int own[N];
#pragma unroll
  for (int i = 0; i < N; ++i) own[i] = begin[i];
  scan_block<N>(s.redi, begin);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if ((int)threadIdx.x * N + i < n) count[threadIdx.x * N + i] = begin[i] - own[i];
  if (threadIdx.x == 0) count[n] = n;  // (of 2 kMost)
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i * kThreads + (int)threadIdx.x < n) s.key[count[at[i]] + place[i]] = key[i];
  __syncthreads();
  // within its bucket a key's place is the number of those before it
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i * kThreads + (int)threadIdx.x >= n) continue;
    const int lo = count[at[i]], hi = count[at[i] + 1];
    place[i] = lo;
#pragma nounroll
    for (int k = lo; k < hi; ++k) place[i] += s.key[k] < key[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i * kThreads + (int)threadIdx.x < n) s.key[place[i]] = key[i];
  __syncthreads();
}

// The least i of any thread (INT_MAX: none). slot: one of s.at, set to INT_MAX before the last barrier.
template <class S>
__device__ __forceinline__ void offer(S& s, int slot, int i) {
  i = min_wave(i);
  if ((threadIdx.x & 63) == 0 && i != INT_MAX) atomicMin(&s.at[slot], i);
}
template <class S>
__device__ __forceinline__ int first_of(S& s, int slot, int i) {
  offer(s, slot, i);
  __syncthreads();
  return s.at[slot];
}

template <typename IO>
struct Line {  // a row
  const IO* x;
  int row, vocab, pairs, units;
  const float* tops;  // in memory
  float top;  // the largest logit that takes part
  Settings s;
};

// A unit's maximum: of a row of up to kUnits units from LDS.
template <class S, typename IO>
__device__ __forceinline__ float top_at(const S& s, const Line<IO>& r, int unit) {
  if (r.units <= kUnits) return s.tops[unit];
  return __builtin_nontemporal_load(r.tops + unit);  // (a plain load would be made one of either memory)
}

// A place in a list of n entries for each lane that says yes. All lanes of the wave.
__device__ __forceinline__ int place_in(int* n, bool yes) {
  const uint64_t all = __ballot(yes);
  int base = 0;
  if (all && (threadIdx.x & 63) == 0) base = atomicAdd(n, __builtin_popcountll(all));
  return __builtin_amdgcn_readfirstlane(base) + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
}

// Appends ids of units whose maximum passes `unit` and whose logit passes `id` to s.key; s.n counts them all.
template <class S, typename IO, class U, class I>
__device__ __forceinline__ void gather(S& s, const Line<IO>& r, const U& unit, const I& id) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = threadIdx.x >> 5 & 1, within = threadIdx.x & 31;
  __syncthreads();
  if (threadIdx.x == 0) s.n = 0;
#pragma nounroll
  for (int first = 0; first < r.units; first += kUnits) {  // (a row of more units: in parts)
    if (threadIdx.x == 0) s.units = 0;
    __syncthreads();
#pragma nounroll
    for (int i = threadIdx.x; i < kUnits; i += kThreads) {
      const bool yes = first + i < r.units && unit(top_at(s, r, first + i));
      const int at = place_in(&s.units, yes);
      if (yes) s.unit[at] = (uint16_t)i;
    }
    __syncthreads();
    const int units = s.units;
    constexpr int kTime = 8;  // loads under way, of a unit for each half of the wave
#pragma nounroll
    for (int u = 2 * wave; u < units; u += 2 * kWaves * kTime) {
      float x[kTime][4];
#pragma unroll
      for (int k = 0; k < kTime; ++k) {
        const int i = u + 2 * kWaves * k + half;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[k][j] = -INFINITY;
        if (i >= units) continue;
        const int base = (first + s.unit[i]) * kUnit;
        load_ids(r.x, base + 4 * within, base + kUnit, r.vocab, x[k]);
      }
      // one bit for an id; the few that are set one after the other, for what is unrolled 32 times had better be short (no
      // instruction of it is in the cache yet)
      uint32_t yes = 0;
#pragma unroll
      for (int k = 0; k < kTime; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) yes |= id(x[k][i]) ? 1u << (4 * k + i) : 0u;
#pragma nounroll
      while (__ballot(yes != 0)) {
        const int to = place_in(&s.n, yes != 0);
        if (yes) {
          const int bit = __builtin_ctz(yes);
          yes &= yes - 1;
          if (to < S::kMost) s.key[to] = (uint32_t)((first + s.unit[u + 2 * kWaves * (bit >> 2) + half]) * kUnit + 4 * within + (bit & 3));
        }
      }
    }
    __syncthreads();
  }
  const int n = min(s.n, S::kMost);
#pragma nounroll
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint32_t id = (uint32_t)s.key[i];
    s.key[i] = (uint64_t)~order_of((float)r.x[id]) << 32 | id;
  }
  __syncthreads();
}

// A first part of the order: logits whose distance from the largest, in 2,048 steps of `scale`, is at most `end`.
struct Reach {
  float scale;
  int end;  // -1: every logit that takes part
};
__device__ __forceinline__ int reach_of(float x, float top, float scale) {
  const float d = (top - x) * scale;
  return d < (float)kUnits ? (int)d : kUnits;
}
template <typename IO>
__device__ __forceinline__ bool within(const Line<IO>& r, const Reach& h, float x) {
  return x > -INFINITY && (h.end < 0 || x == r.top || reach_of(x, r.top, h.scale) <= h.end);
}

// The part of the order that at least `want` of the row's units' maxima lie in (all, if fewer have one), and not many more:
// from their histogram.
template <class S, typename IO>
__device__ __forceinline__ Reach reach_for(S& s, const Line<IO>& r, int want) {
  constexpr int N = kUnits / kThreads;
  int* count = (int*)s.sum;
  float low = INFINITY;
  int have = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int u = i * kThreads + (int)threadIdx.x;
    count[u] = 0;
    if (u < r.units && s.tops[u] > -INFINITY) low = fminf(low, s.tops[u]), ++have;
  }
  low = -max_wave(-low);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = low;
  if (threadIdx.x == 0) s.at[0] = INT_MAX, s.at[1] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) place_in(&s.at[1], have > i);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) low = fminf(low, (float)s.red[w]);
  const float wide = r.top - low;
  const float scale = wide > 0.0f ? (float)kUnits / wide : INFINITY;  // (0 of an infinite one: the largest alone, and all others)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int u = i * kThreads + (int)threadIdx.x;
    if (u < r.units && s.tops[u] > -INFINITY) atomicAdd(&count[s.tops[u] == r.top ? 0 : min(reach_of(s.tops[u], r.top, scale), kUnits - 1)], 1);
  }
  __syncthreads();
  const bool all = s.at[1] <= want;
  int c[N];
#pragma unroll
  for (int i = 0; i < N; ++i) c[i] = count[threadIdx.x * N + i];
  scan_block<N>(s.redi, c);
  int end = INT_MAX;
#pragma unroll
  for (int i = N - 1; i >= 0; --i)
    if (c[i] >= want) end = threadIdx.x * N + i;
  end = first_of(s, 0, end);
  // (the last step holds what rounding puts behind it too)
  return {scale, all || end >= kUnits - 1 ? -1 : end};
}

__device__ __forceinline__ float logit_of(uint64_t key) { return value_of(~(uint32_t)(key >> 32)); }
__device__ __forceinline__ double weight_of(double t) { return pow2_neg(t * (1.4426950408889634 / kPerNat)); }

// Sorts the n gathered ids (bucket: see sort_keys) and sums up their weights.
template <class S, typename IO, class B>
__device__ __forceinline__ void order_and_sum(S& s, const Line<IO>& r, int n, const B& bucket) {
  sort_keys(s, n, bucket);
  constexpr int N = S::kMost / kThreads;
  double w[N];
  const int per = n <= kThreads ? 1 : n <= 2 * kThreads ? 2 : N;  // neighbours of a thread
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (int)threadIdx.x * per + i;
    w[i] = i < per && at < n ? weight_of(t_of(logit_of(s.key[at]), r.top, r.s.c)) : 0.0;
  }
  scan_block<N>(s.red, w);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (int)threadIdx.x * per + i;
    if (i < per && at < n) s.sum[at] = w[i];
  }
  if (threadIdx.x < 4) s.at[threadIdx.x] = INT_MAX;
  __syncthreads();
}

template <typename IO>
__device__ __forceinline__ void answer(const SampleArgs& a, const Line<IO>& r, int id, double prob) {
  if (threadIdx.x) return;
  a.a.choice[r.row] = id;
  if (a.a.prob) a.a.prob[r.row] = (float)prob;
}

// The answer from the first n ids of the order, those in `reach`, if it lies among them. z: the sum of all weights.
template <class S, typename IO>
__device__ __forceinline__ bool decide_first(S& s, const SampleArgs& a, const Line<IO>& r, int n, const Reach& reach, double z) {
  const bool all = reach.end < 0;  // there are no others
  // buckets of the square of the distance from the largest logit: few are far up
  const float scale = reach.scale < INFINITY ? reach.scale / (float)(all ? kUnits : reach.end + 1) : 0.0f;
  order_and_sum(s, r, n, [&](uint64_t key) {
    const float d = fminf((r.top - logit_of(key)) * scale, 1.0f);
    return d > 0.0f ? min((int)(d * d * (float)n), n - 1) : 0;
  });
  if (all) z = s.sum[n - 1];
  const int beyond = INT_MAX;
  int cut = all ? n : beyond;
  double zk = z;
  if (r.s.k > 0 && r.s.k <= n) cut = r.s.k, zk = s.sum[r.s.k - 1];
  if (r.s.k > n && !all) return false;
  const int end = min(cut, n);
  const double target = r.s.p * zk;
  int reached = INT_MAX, under = INT_MAX;
#pragma nounroll
  for (int i = threadIdx.x; i < end; i += kThreads) {
    if (r.s.p < 1.0 && s.sum[i] >= target) reached = min(reached, i);
    if (t_of(logit_of(s.key[i]), r.top, r.s.c) > r.s.limit) under = min(under, i);
  }
  offer(s, 0, reached);
  under = first_of(s, 1, under);  // >= 1: the first id's t is 0
  reached = s.at[0];
  if (reached != INT_MAX) cut = min(cut, reached + 1);
  if (under != INT_MAX) cut = min(cut, under);
  if (cut == beyond && (r.s.p < 1.0 || r.s.limit < INFINITY)) return false;
  const double kept = cut == beyond ? z : s.sum[cut - 1];
  int chosen = INT_MAX;
#pragma nounroll
  for (int i = threadIdx.x; i < min(cut, n); i += kThreads)
    if (s.sum[i] > r.s.u * kept) chosen = min(chosen, i);
  chosen = first_of(s, 2, chosen);
  if (chosen == INT_MAX) {
    if (cut == beyond) return false;
    chosen = cut - 1;
  }
  const uint64_t key = s.key[chosen];
  answer(a, r, (int)(uint32_t)key, weight_of(t_of(logit_of(key), r.top, r.s.c)) / kept);
  return true;
}

// The largest logit that takes part; the units' maxima go to s.tops if there is room.
template <class S, typename IO>
__device__ __forceinline__ float top_of(const Line<IO>& r, S& s) {
  float m = -INFINITY;
#pragma nounroll
  for (int u = threadIdx.x; u < r.units; u += kThreads) {
    const float x = r.tops[u];
    if (u < kUnits) s.tops[u] = x;
    m = fmaxf(m, x);
  }
  m = max_wave(m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, (float)s.red[w]);
  __syncthreads();
  return m;
}

// The lowest id with the largest logit.
template <class S, typename IO>
__device__ __forceinline__ int first_top(const Line<IO>& r, S& s) {
  if (threadIdx.x == 0) s.at[0] = s.at[1] = INT_MAX;
  __syncthreads();
  int u = INT_MAX;
#pragma nounroll
  for (int i = threadIdx.x; i < r.units && u == INT_MAX; i += kThreads)
    if (top_at(s, r, i) == r.top) u = i;
  u = first_of(s, 0, u);
  int id = u * kUnit + (int)threadIdx.x;
  if (threadIdx.x >= kUnit || id >= r.vocab || (float)r.x[id] != r.top) id = INT_MAX;
  return first_of(s, 1, id);
}

template <typename IO>
__device__ __forceinline__ Line<IO> line_of(const SampleArgs& a, int row) {
  Line<IO> r;
  r.x = (const IO*)a.a.logits + (int64_t)row * a.a.stride;
  r.row = row, r.vocab = a.a.vocab, r.pairs = a.pairs, r.units = 2 * a.pairs;
  r.tops = a.tops + (int64_t)row * r.units;
  r.s = settings_of(a.a, row);
  return r;
}

// Whether the sum of all weights is asked for (where the answer is looked for among the first ids at all).
template <typename IO>
__device__ __forceinline__ bool needs_sum(const Line<IO>& r) {
  return r.s.k == 0 && r.vocab > kFew && r.units <= kUnits && (r.s.p < 1.0 || r.s.limit == INFINITY);
}

template <typename IO>
__global__ void __launch_bounds__(64 * kReadWaves) k_sample_rows(SampleArgs a) {
  __shared__ double sh_ref[kReadWaves], sh_sum[kReadWaves];
  const int slice = blockIdx.x, row = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  Line<IO> r = line_of<IO>(a, row);
  const bool with_sum = needs_sum(r);
  const int u0 = slice * a.per_slice, u1 = min(u0 + a.per_slice, r.pairs);

  float ref = -INFINITY;  // of the wave's sums
  double sum = 0.0;       // of the lane: exp((x - ref) / T)
  const double c2 = r.s.c * (1.4426950408889634 / kPerNat);
  constexpr int kTime = 4;
  for (int u = u0 + wave; u < u1; u += kReadWaves * kTime) {
    float x[kTime][4];
#pragma unroll
    for (int k = 0; k < kTime; ++k) {
      const int at = u + kReadWaves * k;
      if (at < u1) load_pair(r.x, at, r.vocab, x[k]);
    }
#pragma unroll
    for (int k = 0; k < kTime; ++k) {
      const int at = u + kReadWaves * k;
      if (at >= u1) continue;
      const float2 two = max_halves(fmaxf(fmaxf(fmaxf(x[k][0], x[k][1]), fmaxf(x[k][2], x[k][3])), -INFINITY));  // no NaN is the larger one
      if (lane == 0) *(float2*)(a.tops + (int64_t)row * r.units + 2 * at) = two;
      const float m = fmaxf(two.x, two.y);
      if (with_sum && m > -INFINITY) {
        if (m > ref) {
          sum = ref == -INFINITY || m == INFINITY ? 0.0 : sum * pow2_neg(((double)m - (double)ref) * c2);
          ref = m;
        }
        if (ref == INFINITY) {
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += x[k][i] == INFINITY ? 1.0 : 0.0;
        } else {  // (of -inf and NaN 2^-1000)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += pow2_neg(((double)ref - (double)x[k][i]) * c2);
        }
      }
    }
  }
  if (with_sum) {
#pragma unroll
    for (int b = 1; b < 64; b <<= 1) sum += __shfl_xor(sum, b);
    if (lane == 0) sh_sum[wave] = sum, sh_ref[wave] = ref;
    __syncthreads();
    if (threadIdx.x == 0) {
      double most = -INFINITY, all = 0.0;
#pragma nounroll
      for (int w = 0; w < kReadWaves; ++w) most = fmax(most, sh_ref[w]);
#pragma nounroll
      for (int w = 0; w < kReadWaves; ++w)
        if (sh_ref[w] > -INFINITY) all += sh_ref[w] == most ? sh_sum[w] : most == INFINITY ? 0.0 : sh_sum[w] * pow2_neg((most - sh_ref[w]) * c2);
      a.sums[2 * ((int64_t)row * a.slices + slice)] = most;
      a.sums[2 * ((int64_t)row * a.slices + slice) + 1] = all;
    }
  }
}

// One workgroup to a row: the answer, where it lies among the first ids of the order.
template <typename IO>
__global__ void __launch_bounds__(kThreads) k_sample_pick(SampleArgs a) {
  __shared__ Shared<kFew> s;
  const int row = blockIdx.x;
  Line<IO> r = line_of<IO>(a, row);
  r.top = top_of(r, s);
  bool done = true;
  if (r.top == -INFINITY) {
    answer(a, r, -1, 0.0);
  } else if (r.s.k == 1) {
    const int id = first_top(r, s);
    answer(a, r, id, 1.0);
  } else {
    double z = 0.0;
    if (needs_sum(r)) {
      const double c2 = r.s.c * (1.4426950408889634 / kPerNat);
#pragma nounroll
      for (int i = threadIdx.x; i < a.slices; i += kThreads) {
        const double m = a.sums[2 * ((int64_t)row * a.slices + i)], v = a.sums[2 * ((int64_t)row * a.slices + i) + 1];
        z += m == r.top ? v : r.top == INFINITY || m == -INFINITY ? 0.0 : v * pow2_neg(((double)r.top - m) * c2);
      }
      double one[1] = {z};
      scan_block<1>(s.red, one);
      if (threadIdx.x == kThreads - 1) s.z[0] = one[0];
      __syncthreads();
      z = s.z[0];
    }
    done = false;
    const bool whole = r.vocab <= kFew;
    if (whole || (r.units <= kUnits && r.s.k <= min(r.units, kFew))) {
      // (whole: buckets over 32 nats)
      const Reach reach = whole ? Reach{(float)fmin(2.0 * r.s.c, 1e30), -1} : reach_for(s, r, r.s.k ? r.s.k : min(kFewUnits, r.units));
      auto in = [&](float x) { return within(r, reach, x); };
      gather(s, r, in, in);
      done = s.n <= kFew && decide_first(s, a, r, s.n, reach, z);
    }
  }
  if (threadIdx.x == 0) a.left[row] = done ? NAN : r.top;
}

// ---- rows whose answer lies further down ----

// The weight of a t over that of its step's first one, exp(-(t - step) / 32), in 2^-32. With d = (t - step) / 32 below 1/32 it is
// 1 - d + d^2/2 - d^3/6 + d^4/24 to 2^-32.
__device__ __forceinline__ uint64_t share_of(uint64_t fixed) {
  const float d = (float)((uint32_t)fixed & 0xffffffu) * (float)(0x1p-24 / kPerNat);
  const float g = d * (1.0f - d * (0.5f - d * (1.0f / 6 - d * (1.0f / 24))));
  return 0x100000000ull - (uint32_t)(g * 0x1p32f + 0.5f);
}
// Of the last step, whose weights lie 2^-46 and more below the largest: by a float's exponential.
__device__ __forceinline__ uint64_t last_share_of(double t) {
  return (uint64_t)(__builtin_amdgcn_exp2f((float)(t - (kSteps - 1)) * (float)(-1.4426950408889634 / kPerNat)) * 0x1p32f);
}

// A border in the order of the ids, or the choice: what comes up to and with it.
struct Border {
  int count;
  double sum;
};

// By the bits of the logits, then of the ids: where a border lies among any number of ids.
struct Narrow {
  uint32_t key;  // ~order of the logits at the border
  int before, equal;
  double sum, one;  // of those before it; of each at it
};
// A weight in 2^-62: whole numbers, whose sums (their upper and lower 24 bits apart) no order changes.
template <typename IO>
__device__ __forceinline__ uint64_t fixed_weight(const Line<IO>& r, float x) { return (uint64_t)rint(weight_of(t_of(x, r.top, r.s.c)) * 0x1p62); }
__device__ __forceinline__ double whole_sum(uint64_t high, uint64_t low) { return (double)high * 0x1p-38 + (double)low * 0x1p-62; }

template <typename IO, class F>
__device__ __forceinline__ void each_logit(const Line<IO>& r, const F& f) {
  for (int u = threadIdx.x >> 6; u < r.pairs; u += kWaves) {
    float x[4];
    load_pair(r.x, u, r.vocab, x);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (x[i] > -INFINITY) f(x[i]);
  }
}

// past(count, sum): whether the border lies before or at an id up to and with which that is the count and the sum.
template <typename IO, class P>
__device__ __forceinline__ Narrow narrow(Shared<kGather>& s, const Line<IO>& r, const P& past) {
  constexpr int kBins = 2048, N = kBins / kThreads;
  uint64_t *high = s.key, *low = (uint64_t*)s.sum;
  int* counts = (int*)(s.key + kBins);
  Narrow b{0, 0, 0, 0, 0};
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, wide = level == 2 ? 10 : 11;  // bits of this level
    for (int i = threadIdx.x; i < kBins; i += kThreads) high[i] = low[i] = 0, counts[i] = 0;
    if (threadIdx.x == 0) s.at[0] = INT_MAX;
    __syncthreads();
    each_logit(r, [&](float x) {
      const uint32_t key = ~order_of(x);
      if (level && (key ^ b.key) >> (shift + wide)) return;
      const int bin = key >> shift & ((1 << wide) - 1);
      atomicAdd(&counts[bin], 1);
      const uint64_t w = fixed_weight(r, x);
      atomicAdd((unsigned long long*)&high[bin], (unsigned long long)(w >> 24));
      atomicAdd((unsigned long long*)&low[bin], (unsigned long long)(w & 0xffffffu));
    });
    __syncthreads();
    int c[N];
    double w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = counts[threadIdx.x * N + i], w[i] = whole_sum(high[threadIdx.x * N + i], low[threadIdx.x * N + i]);
    scan_block<N>(s.redi, c);
    scan_block<N>(s.red, w);
    int bin = INT_MAX, last = -1;
#pragma unroll
    for (int i = N - 1; i >= 0; --i) {
      if (counts[threadIdx.x * N + i] && past(b.before + c[i], b.sum + w[i])) bin = threadIdx.x * N + i;
      if (counts[threadIdx.x * N + i] && last < 0) last = threadIdx.x * N + i;
    }
    bin = first_of(s, 0, bin);
    if (bin == INT_MAX) {  // the border is the last id's (rounding alone comes here)
      __syncthreads();
      if (threadIdx.x == 0) s.at[0] = -1;
      __syncthreads();
      if (last >= 0) atomicMax(&s.at[0], last);
      __syncthreads();
      bin = s.at[0];
    }
    if ((int)threadIdx.x == bin / N) {
      const int i = bin % N;
      double sum = 0;
      int count = 0;
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (k == i) sum = w[k], count = c[k];
      s.at[1] = count - counts[bin];
      s.at[2] = counts[bin];
      s.z[0] = sum - whole_sum(high[bin], low[bin]);
    }
    __syncthreads();
    b.key |= (uint32_t)bin << shift;
    b.before += s.at[1];
    b.sum += s.z[0];
    b.equal = s.at[2];
    __syncthreads();
  }
  b.one = weight_of(t_of(value_of(~b.key), r.top, r.s.c));
  return b;
}

// The nth (from 1) lowest of the ids with that logit.
template <typename IO>
__device__ __forceinline__ int nth_id(Shared<kGather>& s, const Line<IO>& r, uint32_t key, int nth) {
  int before = 0;
  if (threadIdx.x == 0) s.at[0] = INT_MAX;
  __syncthreads();
  for (int base = 0; base < r.vocab; base += 4 * kThreads) {
    float x[4];
    const int at = base + 4 * (int)threadIdx.x;
    int c[4] = {0, 0, 0, 0};
    if (at < r.vocab) {
      load_pair(r.x, at / kPair, r.vocab, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = x[i] > -INFINITY && ~order_of(x[i]) == key;
    }
    scan_block<4>(s.redi, c);
    int id = INT_MAX;
#pragma unroll
    for (int i = 3; i >= 0; --i)
      if (before + c[i] >= nth) id = at + i;
    id = first_of(s, 0, id);
    if (id != INT_MAX) return id;
    if (threadIdx.x == kThreads - 1) s.at[1] = c[3];
    __syncthreads();
    before += s.at[1];
    __syncthreads();
  }
  return -1;
}

// The answer for any row of n ids, each border for itself. z: the sum of all weights.
template <typename IO>
__device__ __forceinline__ void decide_any(Shared<kGather>& s, const SampleArgs& a, const Line<IO>& r, int n, double z) {
  Border cut{n, z};
  auto at = [](const Narrow& b, int rank) { return Border{b.before + rank, b.sum + b.one * rank}; };
  // the first id, of those at a border, at which the sum passes (or reaches) the target
  auto rank_of = [](const Narrow& b, double target, bool beyond) {
    if (b.one == 0.0) return 1;
    const double x = (target - b.sum) / b.one;
    const double i = beyond ? floor(x) + 1 : ceil(x);
    return (int)fmin(fmax(i, 1.0), (double)b.equal);
  };
  if (r.s.k > 0 && r.s.k < n) {
    const int k = r.s.k;
    const Narrow b = narrow(s, r, [&](int count, double) { return count >= k; });
    cut = at(b, k - b.before);
  }
  const double zk = cut.sum;
  if (r.s.p < 1.0) {
    const double target = r.s.p * zk;
    const Narrow b = narrow(s, r, [&](int, double sum) { return sum >= target; });
    const Border x = at(b, rank_of(b, target, false));
    if (x.count < cut.count) cut = x;
  }
  if (r.s.limit < INFINITY) {
    int c[1] = {0};
    double w[1] = {0.0};
    each_logit(r, [&](float x) {
      const double t = t_of(x, r.top, r.s.c);
      if (t <= r.s.limit) c[0] += 1, w[0] += weight_of(t);
    });
    scan_block<1>(s.redi, c);
    scan_block<1>(s.red, w);
    if (threadIdx.x == kThreads - 1) s.at[1] = c[0], s.z[0] = w[0];
    __syncthreads();
    if (s.at[1] < cut.count) cut = {s.at[1], s.z[0]};
    __syncthreads();
  }
  const double target = r.s.u * cut.sum;
  const Narrow b = narrow(s, r, [&](int, double sum) { return sum > target; });
  const int rank = min(rank_of(b, target, true), max(1, cut.count - b.before));
  answer(a, r, nth_id(s, r, b.key, rank), b.one / cut.sum);
}

__device__ __forceinline__ float uniform(float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); }

__device__ __forceinline__ bool between(float x, float low, float high) { return __builtin_amdgcn_fmed3f(x, low, high) == x; }

struct Steps {
  double sum[kSteps];  // of all steps before it
  int count[kSteps];
  int own[kSteps];     // of its own
  int first[kSteps];   // of the gathered ids, the step's first; -1: none are gathered
  float low[4], high[4];  // logits that bound up to four runs of steps
};

template <typename IO>
__global__ void __launch_bounds__(64 * kReadWaves) k_sample_steps(SampleArgs a) {
  __shared__ uint64_t steps[kSteps];
  const int slice = blockIdx.x, row = blockIdx.y;
  const float top = a.left[row];
  if (top != top) return;
  Line<IO> r = line_of<IO>(a, row);
  r.top = top;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < kSteps; i += 64 * kReadWaves) steps[i] = 0;
  __syncthreads();
  const int u0 = slice * a.per_slice, u1 = min(u0 + a.per_slice, r.pairs);
  uint64_t rest = 0;  // of the last step
  constexpr int kTime = 4;
  for (int u = u0 + wave; u < u1; u += kReadWaves * kTime) {
    float x[kTime][4];
#pragma unroll
    for (int k = 0; k < kTime; ++k)
      if (u + kReadWaves * k < u1) load_pair(r.x, u + kReadWaves * k, r.vocab, x[k]);
#pragma unroll
    for (int k = 0; k < kTime; ++k) {
      if (u + kReadWaves * k >= u1) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!(x[k][i] > -INFINITY)) continue;
        const double t = t_of(x[k][i], r.top, r.s.c);
        const uint64_t fixed = fixed_of(t);
        const int step = (int)(fixed >> 24);
        if (step == kSteps - 1) rest += (1ull << 48) + last_share_of(t);
        else atomicAdd((unsigned long long*)&steps[step], (unsigned long long)((1ull << 48) + share_of(fixed)));
      }
    }
  }
#pragma unroll
  for (int b = 1; b < 64; b <<= 1) rest += __shfl_xor((unsigned long long)rest, b);
  if (lane == 0 && rest) atomicAdd((unsigned long long*)&steps[kSteps - 1], (unsigned long long)rest);
  __syncthreads();
  uint64_t* mine = a.steps + ((int64_t)row * a.slices + slice) * kSteps;
  for (int i = threadIdx.x; i < kSteps; i += 64 * kReadWaves) mine[i] = steps[i];
}

// One workgroup to a row.
template <typename IO>
__global__ void __launch_bounds__(kThreads) k_sample_flat(SampleArgs a) {
  __shared__ Shared<kGather> s;
  __shared__ Steps st;
  const int row = blockIdx.x;
  if (a.left[row] != a.left[row]) return;
  Line<IO> r = line_of<IO>(a, row);
  r.top = top_of(r, s);

  // the workgroups' steps summed up
  constexpr int N = kSteps / kThreads;
  int count[N], own[N];
  double sum[N], weight[N];
  {
    uint64_t c[N] = {}, w[N] = {};
    const uint64_t* from = a.steps + (int64_t)row * a.slices * kSteps + threadIdx.x * N;
    constexpr int kTime = 8;  // loads under way
    for (int i = 0; i < a.slices; i += kTime) {
      uint64_t v[kTime][N];
#pragma unroll
      for (int j = 0; j < kTime; ++j)
#pragma unroll
        for (int k = 0; k < N; ++k) v[j][k] = i + j < a.slices ? from[(int64_t)(i + j) * kSteps + k] : 0;
#pragma unroll
      for (int j = 0; j < kTime; ++j)
#pragma unroll
        for (int k = 0; k < N; ++k) c[k] += v[j][k] >> 48, w[k] += v[j][k] & 0xffffffffffffull;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      count[k] = own[k] = (int)c[k];
      sum[k] = weight[k] = (double)w[k] * 0x1p-32 * exp(-(double)(threadIdx.x * N + k) / kPerNat);
    }
  }
  scan_block<N>(s.redi, count);
  scan_block<N>(s.red, sum);
  if (threadIdx.x == kThreads - 1) s.n = count[N - 1], s.z[0] = sum[N - 1];
  if (threadIdx.x < 4) s.at[threadIdx.x] = INT_MAX;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    st.count[threadIdx.x * N + k] = count[k] - own[k];
    st.own[threadIdx.x * N + k] = own[k];
    st.sum[threadIdx.x * N + k] = sum[k] - weight[k];
  }
  __syncthreads();
  const int all = s.n;
  const double z = s.z[0];
  const double slack = 1e-7;  // of a bound, far above what rounding leaves the sums off by

  // the first step for which yes(count, sum up to and with it) holds, or the last one
  auto step_where = [&](int slot, auto&& yes) {
    int at = INT_MAX;
#pragma unroll
    for (int k = N - 1; k >= 0; --k)
      if (yes(count[k], sum[k])) at = threadIdx.x * N + k;
    return min(first_of(s, slot, at), kSteps - 1);
  };
  auto sum_before = [&](int step) { return st.sum[step]; };
  auto sum_with = [&](int step) { return step + 1 < kSteps ? st.sum[step + 1] : z; };
  // bounds of the kept ids' sum, and the last step that has some
  double low = z, high = z;
  int end = kSteps - 1, kstep = -1, p0 = -1, p1 = -1, mstep = -1;
  if (r.s.k > 0 && r.s.k < all) {
    kstep = step_where(0, [&](int c, double) { return c >= r.s.k; });
    low = sum_before(kstep), high = sum_with(kstep), end = kstep;
  }
  if (r.s.p < 1.0) {
    const double from = r.s.p * low * (1 - slack), to = r.s.p * high * (1 + slack);
    p0 = step_where(1, [&](int, double x) { return x >= from; });
    p1 = min(step_where(2, [&](int, double x) { return x >= to; }), end);
    p0 = min(p0, p1);
    low = fmin(low, sum_before(p0)), high = fmin(high, sum_with(p1)), end = min(end, p1);
  }
  if (r.s.limit < INFINITY && step_of(r.s.limit) <= end) {
    mstep = step_of(r.s.limit);
    low = fmin(low, sum_before(mstep)), high = fmin(high, sum_with(mstep));
    if (mstep < end) {
      end = mstep;
      // borders that lie behind the last kept id
      if (r.s.p >= 1.0) kstep = -1;
      if (mstep < p0) kstep = p0 = p1 = -1;
    }
  }
  __syncthreads();  // all have read them
  if (threadIdx.x < 4) s.at[threadIdx.x] = INT_MAX;
  __syncthreads();
  const double from = r.s.u * low * (1 - slack), to = r.s.u * high * (1 + slack);
  int c0 = step_where(0, [&](int, double x) { return x > from; });
  const int c1 = min(step_where(1, [&](int, double x) { return x > to; }), end);
  c0 = min(c0, c1);
  auto needed = [&](int i) { return i == kstep || (i >= p0 && i <= p1) || i == mstep || (i >= c0 && i <= c1); };
  int before[N], last = -1;
#pragma unroll
  for (int k = 0; k < N; ++k) before[k] = needed(threadIdx.x * N + k) ? own[k] : 0;
  scan_block<N>(s.redi, before);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = threadIdx.x * N + k;
    st.first[i] = needed(i) ? before[k] - own[k] : -1;
    if (needed(i)) last = i;
  }
  if (threadIdx.x == kThreads - 1) s.at[3] = before[N - 1];
  __syncthreads();  // all have read them
  if (threadIdx.x == 0) s.at[2] = 0, s.at[1] = INT_MAX;
  __syncthreads();
  int n = s.at[3];
  if (last >= 0) atomicMax(&s.at[2], last), atomicMin(&s.at[1], last);
  __syncthreads();
  last = s.at[2];
  // If the steps between them fit too, they are taken along: then two logits bound what is gathered.
  const int from_step = s.at[1];
  const int span = n > 0 ? st.count[last] + st.own[last] - st.count[from_step] : 0;
  const bool together = n > 0 && span <= kGather;
  __syncthreads();
  if (together) {
    n = span;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = threadIdx.x * N + k;
      st.first[i] = i >= from_step && i <= last ? st.count[i] - st.count[from_step] : -1;
    }
  }
  __syncthreads();

  bool done = false;
  if (n > 0 && n <= kGather) {
    auto unit = [&](float top) { return top > -INFINITY && step_of(t_of(top, r.top, r.s.c)) <= last; };
    // Its lowest and its highest float tell the ids of a run of steps, where they are found. A few runs cover what is needed.
    int bad = 0;
    if (threadIdx.x < 4) {
      const int run = threadIdx.x;
      int from = run == 0 ? c0 : run == 1 ? p0 : run == 2 ? kstep : mstep, to = run == 0 ? c1 : run == 1 ? p1 : run == 2 ? kstep : mstep;
      if (together) from = run ? -1 : from_step, to = last;
      float low = INFINITY, high = INFINITY;  // no run: no logit is that large where the bounds are used
      if (from >= 0) {
        bad = !bounds_of(r.top, r.s.c, from, to, &low, &high);
      }
      st.low[run] = low, st.high[run] = high;
    }
    if (!__syncthreads_or(bad)) {
      float low[4], high[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) low[i] = uniform(st.low[i]), high[i] = uniform(st.high[i]);
      const bool more = !together && (kstep >= 0 || mstep >= 0);
      gather(s, r, unit, [&](float x) {
        bool in = between(x, low[0], high[0]) | between(x, low[1], high[1]);
        if (more) in = in | between(x, low[2], high[2]) | between(x, low[3], high[3]);
        return in;
      });
    } else {
      gather(s, r, unit, [&](float x) { return x > -INFINITY && st.first[step_of(t_of(x, r.top, r.s.c))] >= 0; });
    }
    done = s.n == n;  // else bounds took in other steps' ids: each border is looked for by itself
  }
  if (done) {
    order_and_sum(s, r, n, [&](uint64_t key) {  // a step has as many buckets as ids
      const uint64_t fixed = fixed_of(t_of(logit_of(key), r.top, r.s.c));
      const int step = (int)(fixed >> 24), first = st.first[step];
      return first + (int)((fixed & 0xffffffu) * (uint32_t)st.own[step] >> 24);
    });
    auto t_at = [&](int i) { return t_of(logit_of(s.key[i]), r.top, r.s.c); };
    auto border = [&](int i) {  // up to and with gathered id i
      const int step = step_of(t_at(i)), first = st.first[step];
      return Border{st.count[step] + i - first + 1, st.sum[step] + s.sum[i] - (first ? s.sum[first - 1] : 0.0)};
    };
    // each thread's ids, looked at once a question
    auto first_where = [&](int slot, auto&& yes) {
      int found = INT_MAX;
      for (int i = threadIdx.x; i < n && found == INT_MAX; i += kThreads)
        if (yes(i)) found = i;
      return first_of(s, slot, found);
    };
    Border cut{all, z};
    if (kstep >= 0) cut = border(st.first[kstep] + r.s.k - st.count[kstep] - 1);
    const double zk = cut.sum;
    if (p0 >= 0) {
      const int i = first_where(0, [&](int i) { return border(i).sum >= r.s.p * zk; });
      if (i == INT_MAX) done = false;
      else if (border(i).count < cut.count) cut = border(i);
    }
    if (mstep >= 0) {
      const int i = first_where(1, [&](int i) { return t_at(i) > r.s.limit || step_of(t_at(i)) > mstep; });
      // the one before, or the end of the step before
      const int upto = i == INT_MAX ? n : i, first = st.first[mstep];
      const Border x = upto > first ? border(upto - 1) : Border{st.count[mstep], st.sum[mstep]};
      if (x.count < cut.count) cut = x;
    }
    const double target = r.s.u * cut.sum;
    const int i = first_where(2, [&](int i) { return border(i).sum > target; });
    if (i == INT_MAX || border(i).count > cut.count) done = false;
    if (done) {
      const uint64_t key = s.key[i];
      answer(a, r, (int)(uint32_t)key, weight_of(t_of(logit_of(key), r.top, r.s.c)) / cut.sum);
    }
  }
  if (!done) {
    __syncthreads();
    decide_any(s, a, r, all, z);
  }
}

// ---- host ----
int fail(int rc, const char* why) {
  set_call_error(std::string("sample: ") + why);
  return rc;
}

bool sizes_ok(const mtg_sample& a) { return a.rows >= 0 && a.rows <= 65535 && a.vocab > 0 && a.vocab <= (1 << 24); }

struct Plan {
  int pairs, per_slice, slices;
  size_t sums_at, steps_at, left_at, bytes;
};
// Workgroups of 4,096 ids or more, two a CU or more where there are so many, and of kSlice at most.
Plan plan_of(const mtg_sample& a) {
  Plan p;
  p.pairs = (a.vocab + kPair - 1) / kPair;
  const int want = a.rows ? (1024 + a.rows - 1) / a.rows : 1;
  p.per_slice = std::min(std::max((p.pairs + want - 1) / want, 4096 / kPair), kSlice / kPair);
  p.slices = (p.pairs + p.per_slice - 1) / p.per_slice;
  const size_t rows = a.rows, parts = rows * p.slices;
  auto up = [](size_t x) { return (x + 15) / 16 * 16; };
  p.sums_at = up(rows * p.pairs * 8);
  p.steps_at = p.sums_at + parts * 16;
  p.left_at = p.steps_at + parts * kSteps * 8;
  p.bytes = up(p.left_at + rows * 4);
  return p;
}

template <typename IO>
hipError_t run(const SampleArgs& a, hipStream_t s) {
  const dim3 grid(a.slices, a.a.rows);
  hipError_t e = launch(k_sample_rows<IO>, grid, dim3(64 * kReadWaves), 0, s, a);
  if (e == hipSuccess) e = launch(k_sample_pick<IO>, dim3(a.a.rows), dim3(kThreads), 0, s, a);
  if (e == hipSuccess && a.a.vocab > kFew) e = launch(k_sample_steps<IO>, grid, dim3(64 * kReadWaves), 0, s, a);  // (of fewer ids all rows are done)
  if (e == hipSuccess && a.a.vocab > kFew) e = launch(k_sample_flat<IO>, dim3(a.a.rows), dim3(kThreads), 0, s, a);
  return e;
}

}  // namespace
}  // namespace mtg

extern "C" size_t mtg_sample_workspace(const mtg_sample* a) {
  return a && mtg::sizes_ok(*a) && a->rows ? mtg::plan_of(*a).bytes : 0;
}

extern "C" int mtg_sample_dev(const mtg_sample* p, void* stream) {
  using namespace mtg;
  try {
    if (!p) return fail(MTG_ERR_INVALID, "no description");
    const mtg_sample& a = *p;
    if (!sizes_ok(a)) return fail(MTG_ERR_INVALID, "rows 0 to 65535, vocab 1 to 2^24");
    if (a.io_type != MTG_TYPE_F32 && a.io_type != MTG_TYPE_F16) return fail(MTG_ERR_UNSUPPORTED, "io_type is not f32 or f16");
    if (a.rows == 0) return MTG_OK;
    if (!a.logits || !a.settings || !a.uniform || !a.choice) return fail(MTG_ERR_INVALID, "logits, settings, uniform or choice is NULL");
    if (a.stride < a.vocab || a.stride > ((int64_t)1 << 40)) return fail(MTG_ERR_INVALID, "a row stride below vocab");
    const size_t eb = type_bytes(a.io_type), rows = (size_t)a.rows;
    if (!aligned(a.logits, eb) || !aligned(a.settings, 4) || !aligned(a.top_k, 4) || !aligned(a.uniform, 4) || !aligned(a.choice, 4) ||
        !aligned(a.prob, 4))
      return fail(MTG_ERR_INVALID, "an array not aligned to its elements");
    const Plan plan = plan_of(a);
    if (!a.workspace || !aligned(a.workspace, 16)) return fail(MTG_ERR_INVALID, "workspace NULL or unaligned");
    if (a.workspace_bytes < plan.bytes) return fail(MTG_ERR_CAPACITY, "workspace smaller than mtg_sample_workspace");
    // what one workgroup writes others may still read
    const Array read[] = {{a.logits, extent(a.rows, a.stride, a.vocab, eb)}, {a.settings, 12 * rows}, {a.top_k, 4 * rows}, {a.uniform, 4 * rows}};
    const Array written[] = {{a.choice, 4 * rows}, {a.prob, 4 * rows}, {a.workspace, plan.bytes}};
    for (const Array& w : written) {
      for (const Array& x : read)
        if (overlap(w.at, w.bytes, x.at, x.bytes)) return fail(MTG_ERR_INVALID, "choice, prob or workspace overlaps what is read");
      for (const Array& x : written)
        if (&x != &w && overlap(w.at, w.bytes, x.at, x.bytes)) return fail(MTG_ERR_INVALID, "choice, prob and workspace overlap");
    }
    char* work = (char*)a.workspace;
    const SampleArgs r{a, plan.pairs, plan.slices, plan.per_slice, (float*)work, (double*)(work + plan.sums_at),
                       (uint64_t*)(work + plan.steps_at), (float*)(work + plan.left_at)};
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = a.io_type == MTG_TYPE_F16 ? run<_Float16>(r, s) : run<float>(r, s);
    if (e != hipSuccess) return fail(MTG_ERR_DEVICE, hipGetErrorString(e));
    return MTG_OK;
  } catch (...) {
    return MTG_ERR_NOMEM;
  }
}
