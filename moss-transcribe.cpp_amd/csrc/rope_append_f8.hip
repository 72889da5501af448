// rope_append_f8.hip - mtg_rope_append_f8_dev: rotary positions of the new rows of a batch, their keys and values
// stored as e4m3 codes into the pages of a cache in 8 bits, one power of two to scale each block of 16 positions.
//
// A block's scale is the least 2^e with |x| <= 448 * 2^e over its new rows, and no less than it was where earlier rows lie
// in the block. So division by it is exact, and the codes of earlier rows follow a larger scale by another exponent alone (rounded once
// more only where they fall below 2^-6, the least number with all of its mantissa).
//
// A workgroup takes the rows of one block of 16 positions and some heads, one after the other: 16 or 8 lanes hold a row
// of a head, 8 neighbouring elements each, and all of the block's rows of a head, normed and turned, stand in the
// registers when its maximum is known. cos and sin, the only 64-bit work, are made once for the workgroup's heads, and lie
// in a thread's registers as factors of its own elements.
//
// Bound by the bytes of q, k and v in and of q and the codes out, and by cos and sin where a workgroup has few heads to use them
// for: 16,384 rows of 16 + 8 + 8 heads of 128 (f16, 235 MB) in 70 us, 3.4 TB/s, where a copy of as much takes 49.
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
  int rounds;      // heads of a workgroup
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

// What turns a lane's elements d0 .. d0 + 7 of a row's heads: of element i and the other one of its pair, o, it makes x c + o s.
struct Turn {
  float c[8], s[8];
};
__device__ __forceinline__ void load_turn(const float2* cs, int d0, int rot_dim, bool interleaved, Turn& t) {
  const int half = rot_dim >> 1;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = d0 + i;
    const bool in = d < rot_dim, first = interleaved ? !(i & 1) : d < half;
    const float2 w = cs[!in ? 0 : interleaved ? d >> 1 : first ? d : d - half];
    t.c[i] = w.x;
    t.s[i] = first ? -w.y : w.y;
  }
}
// row: D floats of LDS that only the head's lanes touch, all of one wave. The sums are k_rope_append's, a product and its sum in
// one rounding.
__device__ __forceinline__ void turn8(float (&x)[8], float* row, int d0, int rot_dim, bool interleaved, const Turn& t) {
  const int half = rot_dim >> 1;
  float o[8];
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = x[i ^ 1];
  } else {
    store8(row + d0, x);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (half % 8 == 0) {  // the other halves of a lane's pairs are neighbours too
      load8(row + (d0 < half ? d0 + half : d0 - half), o);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = d0 + i;
        o[i] = row[d >= rot_dim ? 0 : d < half ? d + half : d - half];
      }
    }
    // the next head's rows must not be written before these reads
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = d0 + i < rot_dim ? fmaf(x[i], t.c[i], o[i] * t.s[i]) : x[i];
}

// STEPS: a thread takes places slot, slot + 16 / STEPS .. of the block. WAVES: a SIMD holds that many at least.
template <typename IO, int D, int STEPS, int WAVES>
__global__ void __launch_bounds__(16 / STEPS * D / 8) __attribute__((amdgpu_waves_per_eu(WAVES))) k_rope_append_f8(RopeArgs r) {
  constexpr int kLanes = D / 8, kSlots = kBlock / STEPS, kThreads = kSlots * kLanes, kWaves = kThreads / 64;
  const mtg_rope_append& a = r.a;
  __shared__ float rows[kThreads * 8];
  __shared__ float2 cs[kBlock][D / 2];
  __shared__ uint32_t tops[2][kWaves];
  const int tile = blockIdx.x, tid = threadIdx.x, sub = tid % kLanes, slot = tid / kLanes, d0 = sub * 8;

  Rows seq;
  const int b = seq_of_rows(a.kv, [&](int start, int i) { return first_block(start, i, a.kv.n_tokens) <= tile; }, &seq);
  if (b < 0) return;
  const int64_t p0 = ((int64_t)(seq.pos0 >> 4) + (tile - first_block(seq.row0, b, a.kv.n_tokens))) * kBlock;
  // the block's new rows: places lo .. hi - 1; rows before them are the sequence's earlier ones
  const int lo = (int)max((int64_t)0, seq.pos0 - p0), hi = (int)min((int64_t)kBlock, (int64_t)seq.pos0 + seq.n - p0);
  if (hi <= lo) return;
  const int row0 = seq.row0 + (int)(p0 - seq.pos0);  // of place 0

  const int h0 = blockIdx.y * r.rounds;
  float x[STEPS][8];
  auto kind_of = [&](int h) { return h < r.q_heads ? 0 : h < r.q_heads + r.kv_heads ? 1 : h < r.heads ? 2 : 3; };
  auto load = [&](int h) {
    const int kind = kind_of(h);
    if (kind == 3) return;
    const int head = kind == 0 ? h : kind == 1 ? h - r.q_heads : h - r.q_heads - r.kv_heads;
    const IO* src = (const IO*)(kind == 0 ? a.q : kind == 1 ? a.k_new : a.v_new) + head * D + d0;
    const int64_t stride = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int pl = s * kSlots + slot;
      if (pl >= lo && pl < hi) load8(src + (int64_t)(row0 + pl) * stride, x[s]);
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
    for (int i = sub; i < half; i += kLanes) cs[pl][i] = cos_sin<true>(pos, a.freqs[i], a.mscale);
  }
  __syncthreads();

  Turn turn;  // of the thread's row, if it has but one
  if (STEPS == 1 && d0 < a.rot_dim && slot >= lo && slot < hi) load_turn(cs[slot], d0, a.rot_dim, a.interleaved, turn);
  for (int round = 0; round < r.rounds; ++round) {
    const int h = h0 + round, kind = kind_of(h);
    if (kind == 3) break;
    const int head = kind == 0 ? h : kind == 1 ? h - r.q_heads : h - r.q_heads - r.kv_heads;
    if (round) load(h);
    uint8_t* scale = (kind == 1 ? r.scales.k : r.scales.v) + (page < 0 ? 0 : page * r.scales.page_stride + head * r.scales.head_stride + place / kBlock);
    const int was = kind && page >= 0 && lo > 0 ? *scale : 0;
    uint32_t top = 0;
    const float* gain = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int pl = s * kSlots + slot;
      if (pl < lo || pl >= hi) continue;  // lanes of one row take the same way
      if (gain) norm8<D>(x[s], gain + d0, a.eps);
      if (kind != 2 && d0 < a.rot_dim) {
        if (STEPS > 1) load_turn(cs[pl], d0, a.rot_dim, a.interleaved, turn);
        turn8(x[s], rows + slot * D, d0, a.rot_dim, a.interleaved, turn);
      }
      if (kind == 0) {
        store8((IO*)a.q_out + (int64_t)(row0 + pl) * a.q_out_stride + h * D + d0, x[s]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, size_bits(x[s][i]));
      }
    }
    if (kind == 0) continue;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
    if (kWaves > 1) {
      // (in turns of two: the next head's are written while slow waves still read these; all have read the scale)
      if ((tid & 63) == 0) tops[round & 1][tid >> 6] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = max(top, tops[round & 1][w]);
    }
    if (page < 0) continue;
    int e = scale_exponent(top), grown = 0;
    if (lo > 0) {
      const int old = min(was, 254) - 127;
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
        *at = codes_of(x[s], factor);
      }
    }
    if (tid == 0) *scale = (uint8_t)(e + 127);
  }
}

template <typename IO, int D>
hipError_t run(RopeArgs& r, hipStream_t s) {
  const mtg_paged_kv& kv = r.a.kv;
  const unsigned tiles = (unsigned)blocks_bound(kv.n_tokens, kv.n_seqs);
  r.rounds = 1;
  // A block that gets few rows: one wave takes it whole, so the rows that are not new cost no lanes.
  if (kv.n_tokens <= 4 * (int64_t)kv.n_seqs) return launch(k_rope_append_f8<IO, D, D / 32, 1>, dim3(tiles, r.heads), dim3(64), 0, s, r);
  // The more heads a workgroup takes, the rarer cos and sin, as long as about 1,024 workgroups stay for the 256 CUs. One
  // head against this rule's count: 16,384 rows 138 and 70 us (8 heads), 2,048 rows 19.3 and 14.8 (4), 48 x 13 rows
  // 11.5 and 10.5 (2); 512 rows, with one head a workgroup, 8.0 against 8.3 with two. 16 heads: 16,384 rows the same as 8, 24,000 113 and 100.
  r.rounds = (int)std::min<int64_t>(8, std::max<int64_t>(1, (int64_t)tiles * r.heads / 1024));
  const dim3 grid(tiles, (r.heads + r.rounds - 1) / r.rounds);
  // Eight waves a SIMD, for which a few registers go without, where all places are filled more than once (16,384 rows 69.8 us, with
  // seven waves 75.4; heads of 64 31.9 and 37.2), else seven (2,048 rows 14.7 and 15.6, 48 x 13 10.5 and 11.0).
  return r.rounds == 8 ? launch(k_rope_append_f8<IO, D, 1, 8>, grid, dim3(2 * D), 0, s, r)
                       : launch(k_rope_append_f8<IO, D, 1, 1>, grid, dim3(2 * D), 0, s, r);
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
