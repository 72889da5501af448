// rope_append_f8.hip - mtg_rope_append_f8_dev: rotary positions of the new rows of a batch, their keys and values
// stored as e4m3 codes into the pages of a cache in 8 bits, one power of two to scale each block of 16 positions.
//
// A block's scale is the least 2^e with |x| <= 448 * 2^e over its new rows, and no less than it was where earlier rows lie
// in the block. So division by it is exact, and the codes of earlier rows follow a larger scale by another exponent alone (rounded once
// more only where they fall below 2^-6, the least number with all of its mantissa).
//
// A workgroup takes the rows of one block of 16 positions and some heads, one after the other: 16 or 8 lanes hold a row
// of a head, 8 neighbouring elements each, and all of the block's rows of a head, normed and turned, stand in the
// registers when its maximum is known. cos and sin, the only 64-bit work, are made once for the workgroup's heads.
#include "kernels.hpp"
#include "paged_dev.hpp"
#include "rope_checks.hpp"
#include "rope_dev.hpp"

#include <algorithm>

namespace mtg {
namespace {

using namespace paged;
using namespace rope;

struct RopeArgs {
  mtg_rope_append a;
  mtg_f8_scales scales;
  int shift, cap;  // of the page size; positions a table row names
  int heads;       // heads of a row taken: q, k and v, or those there are
  int q_heads, kv_heads;
  int rounds;      // of PASSES heads, for a workgroup
};

constexpr int kBlock = MTG_F8_BLOCK;

// Finite |x| as bits in ascending order, 0 for what is not finite.
__device__ __forceinline__ uint32_t size_bits(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0;
}

// 8 codes of x * factor, which is at most 448 in size where x is finite; what is not becomes the code NaN.
__device__ __forceinline__ u2 codes_of(const float (&x)[8], float factor) {
  u2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * factor, x[4 * i + 1] * factor, 0, false);
    w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * factor, x[4 * i + 3] * factor, c, true);
  }
  return w;
}
__device__ __forceinline__ void values_of(u2 w, float (&x)[8]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
    x[4 * i] = a[0], x[4 * i + 1] = a[1], x[4 * i + 2] = b[0], x[4 * i + 3] = b[1];
  }
}

// STEPS: a thread takes places slot, slot + 16 / STEPS .. of the block.
template <typename IO, int D, int STEPS, int PASSES>
__global__ void __launch_bounds__(16 / STEPS * D / 8) k_rope_append_f8(RopeArgs r) {
  constexpr int kLanes = D / 8, kSlots = kBlock / STEPS, kThreads = kSlots * kLanes, kWaves = kThreads / 64;
  const mtg_rope_append& a = r.a;
  __shared__ float rows[kThreads * 8];
  __shared__ float2 cs[kBlock][D / 2];
  __shared__ uint32_t tops[2][PASSES][kWaves];
  const int tile = blockIdx.x, tid = threadIdx.x, sub = tid % kLanes, slot = tid / kLanes, d0 = sub * 8;

  Rows seq;
  const int b = seq_of_rows(a.kv, [&](int start, int i) { return first_block(start, i, a.kv.n_tokens) <= tile; }, &seq);
  if (b < 0) return;
  const int64_t p0 = ((int64_t)(seq.pos0 >> 4) + (tile - first_block(seq.row0, b, a.kv.n_tokens))) * kBlock;
  // the block's new rows: places lo .. hi - 1; rows before them are the sequence's earlier ones
  const int lo = (int)max((int64_t)0, seq.pos0 - p0), hi = (int)min((int64_t)kBlock, (int64_t)seq.pos0 + seq.n - p0);
  if (hi <= lo) return;
  const int row0 = seq.row0 + (int)(p0 - seq.pos0);  // of place 0

  const int h0 = blockIdx.y * r.rounds * PASSES;
  float x[PASSES][STEPS][8];
  auto kind_of = [&](int h) { return h < r.q_heads ? 0 : h < r.q_heads + r.kv_heads ? 1 : h < r.heads ? 2 : 3; };
  auto load = [&](int first) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int h = first + p, kind = kind_of(h);
      if (kind == 3) continue;
      const int head = kind == 0 ? h : kind == 1 ? h - r.q_heads : h - r.q_heads - r.kv_heads;
      const IO* src = (const IO*)(kind == 0 ? a.q : kind == 1 ? a.k_new : a.v_new) + head * D + d0;
      const int64_t stride = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int pl = s * kSlots + slot;
        if (pl >= lo && pl < hi) {
          load8(src + (int64_t)(row0 + pl) * stride, x[p][s]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[p][s][i] = 0.0f;
        }
      }
    }
  };
  load(h0);

  int page = -1;
  if (r.kv_heads && p0 >= 0 && p0 < r.cap) page = page_of(a.kv.page_table + (int64_t)b * a.kv.table_stride, (int)p0, r.shift, r.cap, a.kv.n_pages);
  const int place = (int)p0 & (a.kv.page_size - 1);

  const int half = a.rot_dim >> 1;
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int pl = s * kSlots + slot;
    if (pl < lo || pl >= hi) continue;
    const int pos = a.positions ? a.positions[row0 + pl] : (int)p0 + pl;
    for (int i = sub; i < half; i += kLanes) cs[pl][i] = cos_sin(pos, a.freqs[i], a.mscale);
  }
  __syncthreads();

  for (int round = 0; round < r.rounds; ++round) {
    const int first = h0 + round * PASSES;
    if (first >= r.heads) break;
    if (round) load(first);
    uint8_t was[PASSES];
    uint32_t top[PASSES];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int h = first + p, kind = kind_of(h);
      top[p] = 0;
      was[p] = 0;
      if (kind == 3) continue;
      if (kind && page >= 0 && lo > 0) {
        const int head = kind == 1 ? h - r.q_heads : h - r.q_heads - r.kv_heads;
        was[p] = (kind == 1 ? r.scales.k : r.scales.v)[page * r.scales.page_stride + head * r.scales.head_stride + place / kBlock];
      }
      const float* gain = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int pl = s * kSlots + slot;
        if (pl < lo || pl >= hi) continue;  // lanes of one row take the same way
        if (gain) norm8<D>(x[p][s], gain + d0, a.eps);
        if (kind != 2 && d0 < a.rot_dim) rotate8(x[p][s], rows + slot * D, d0, a.rot_dim, a.interleaved, cs[pl]);
        if (kind == 0) {
          store8((IO*)a.q_out + (int64_t)(row0 + pl) * a.q_out_stride + h * D + d0, x[p][s]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) top[p] = max(top[p], size_bits(x[p][s][i]));
        }
      }
      if (kind) {
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) top[p] = max(top[p], (uint32_t)__shfl_xor((int)top[p], m));
        if (kWaves > 1 && (tid & 63) == 0) tops[round & 1][p][tid >> 6] = top[p];
      }
    }
    // (in turns of two: the next round's are written while slow waves still read these; all have read the scales)
    if (kWaves > 1) __syncthreads();
    if (page < 0) continue;
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int h = first + p, kind = kind_of(h);
      if (kind == 0 || kind == 3) continue;
      const int head = kind == 1 ? h - r.q_heads : h - r.q_heads - r.kv_heads;
#pragma unroll
      for (int w = 0; kWaves > 1 && w < kWaves; ++w) top[p] = max(top[p], tops[round & 1][p][w]);
      int e = scale_exponent(top[p]), grown = 0;
      if (lo > 0) {
        const int old = min((int)was[p], 254) - 127;
        e = max(e, old);
        grown = e - old;
      }
      const float factor = ldexpf(1.0f, -e);
      uint8_t* to = (uint8_t*)(kind == 1 ? a.kv.k : a.kv.v) + page * a.kv.page_stride + head * a.kv.head_stride + place * D + d0;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int pl = s * kSlots + slot;
        if (pl >= hi || (pl < lo && !grown)) continue;
        u2* at = (u2*)(to + pl * D);
        if (pl < lo) {
          float y[8];
          values_of(*at, y);
          *at = codes_of(y, ldexpf(1.0f, -grown));
        } else {
          *at = codes_of(x[p][s], factor);
        }
      }
      if (tid == 0)
        (kind == 1 ? r.scales.k : r.scales.v)[page * r.scales.page_stride + head * r.scales.head_stride + place / kBlock] = (uint8_t)(e + 127);
    }
  }
}

template <typename IO, int D>
hipError_t run(RopeArgs& r, hipStream_t s) {
  const mtg_paged_kv& kv = r.a.kv;
  const unsigned tiles = (unsigned)blocks_bound(kv.n_tokens, kv.n_seqs);
  r.rounds = 1;
  if (kv.n_tokens <= 4 * (int64_t)kv.n_seqs) return launch(k_rope_append_f8<IO, D, D / 32, 1>, dim3(tiles, r.heads), dim3(64), 0, s, r);
  return launch(k_rope_append_f8<IO, D, 1, 1>, dim3(tiles, r.heads), dim3(2 * D), 0, s, r);
}

int fail(int rc, const char* why) {
  set_call_error(std::string("rope_append_f8: ") + why);
  return rc;
}

}  // namespace
}  // namespace mtg

extern "C" int mtg_rope_append_f8_dev(const mtg_rope_append_f8* p, void* stream) {
  using namespace mtg;
  try {
    if (!p) return fail(MTG_ERR_INVALID, "no description");
    const mtg_rope_append& a = p->a;
    const mtg_paged_kv& kv = a.kv;
    int rc = 0;
    if (const char* why = refused(a, true, &rc, &p->scales)) return fail(rc, why);
    if (kv.n_seqs == 0 || kv.n_tokens == 0) return MTG_OK;
    RopeArgs r{a, p->scales, 0, 0, 0, a.q ? a.n_heads : 0, a.k_new ? kv.n_kv_heads : 0, 1};
    if (a.k_new) r.shift = log2_of(kv.page_size), r.cap = capacity(kv.table_stride, r.shift);
    r.heads = r.q_heads + 2 * r.kv_heads;
    hipStream_t s = (hipStream_t)stream;
    const bool f16 = a.io_type == MTG_TYPE_F16;
    const hipError_t e = kv.head_dim == 128 ? f16 ? run<_Float16, 128>(r, s) : run<float, 128>(r, s)
                                            : f16 ? run<_Float16, 64>(r, s) : run<float, 64>(r, s);
    if (e != hipSuccess) return fail(MTG_ERR_DEVICE, hipGetErrorString(e));
    return MTG_OK;
  } catch (...) {
    return MTG_ERR_NOMEM;
  }
}
