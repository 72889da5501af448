// rope_dev.hpp - what the kernels that append rows to a paged cache do to a lane's 8 neighbouring elements of a head:
// the head's norm, and the cos and sin of its pairs.
#pragma once

#include "paged_dev.hpp"

namespace mtg {
namespace rope {

using paged::f4;
using paged::h8;

__device__ __forceinline__ void load8(const float* p, float* x) {
  const f4 a = *(const f4*)p, b = *(const f4*)(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
}
__device__ __forceinline__ void load8(const _Float16* p, float* x) {
  const h8 a = *(const h8*)p;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
}
__device__ __forceinline__ void store8(float* p, const float* x) {
  f4 a, b;
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = x[i], b[i] = x[4 + i];
  *(f4*)p = a;
  *(f4*)(p + 4) = b;
}
__device__ __forceinline__ void store8(_Float16* p, const float* x) {
  h8 a;
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = (_Float16)x[i];  // to nearest even: the one rounding of the value
  // a wave writes whole lines: past L2, whose lines the end of the kernel would wait for (f32 rows take two stores
  // a line, which that way reach memory as halves: 102 us instead of 76 for 8,192 rows of 40 heads)
  __builtin_nontemporal_store(a, (h8*)p);
}

// mscale (cos, sin) of the angle pos * freq. FINE: of the angle in 64 bits.
template <bool FINE = false>
__device__ __forceinline__ float2 cos_sin(int pos, double freq, float mscale) {
  const double turns = (double)pos * (freq * 0.15915494309189533577);
  if constexpr (FINE) {
    // The nearest quarter of a turn, and what is left of it, |r| <= pi/4, by the power series up to r^11 and r^10 (off by 2^-33).
    const double part = turns - rint(turns), quarter = rint(4.0 * part);
    const double r = fma(-0.25, quarter, part) * 6.28318530717958648, z = r * r;
    double s = fma(z, -1.0 / 39916800, 1.0 / 362880), c = fma(z, -1.0 / 3628800, 1.0 / 40320);
    s = fma(z, s, -1.0 / 5040), c = fma(z, c, -1.0 / 720);
    s = fma(z, s, 1.0 / 120), c = fma(z, c, 1.0 / 24);
    s = fma(z, s, -1.0 / 6), c = fma(z, c, -0.5);
    s = fma(z * r, s, r), c = fma(z, c, 1.0);
    const int k = (int)quarter;
    const float x = (k & 1) ? (float)s : (float)c, y = (k & 1) ? (float)c : (float)s;
    return make_float2(((k + 1) & 2) ? -x * mscale : x * mscale, (k & 2) ? -y * mscale : y * mscale);
  }
  // |part| <= 1/2; off by its rounding, 2^-26 turns, and by three of 64 bits, 2^-51 of all turns (2^-25 beside it from
  // positions of 2^28 on). A float's cos and sin of it are off by 4.6e-8 as a norm, of the angle in 64 bits by 3.8e-8.
  const float part = (float)(turns - rint(turns));
  float s, c;
  sincospif(2.0f * part, &s, &c);
  return make_float2(c * mscale, s * mscale);
}

// x *= gain / sqrt(mean(x^2) + eps), the mean over the D / 8 neighbouring lanes that hold the head; gain: of this lane's elements.
template <int D>
__device__ __forceinline__ void norm8(float (&x)[8], const float* gain, float eps) {
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
  for (int m = 1; m < D / 8; m <<= 1) ss += __shfl_xor(ss, m);
  const float scale = 1.0f / sqrtf(ss * (1.0f / D) + eps);
  float g[8];
  load8(gain, g);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = x[i] * scale * g[i];
}

}  // namespace rope
}  // namespace mtg
