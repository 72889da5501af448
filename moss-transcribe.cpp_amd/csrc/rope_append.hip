// rope_append.hip - mtg_rope_append_dev: rotary positions of the new rows of a batch, their
// keys and values stored into the pages of the cache (reference for one sequence over a
// contiguous cache: src/qwen3.cpp:101-134).
//
// Every element is read once and written once, with about ten 32-bit operations, so HBM
// bounds it; a single row is bound by the launch and the chain sequence - page. A workgroup takes one
// row (token). A lane holds 8 neighbouring elements of a head (16 bytes of f16), 16 or 8 lanes a head:
// the norm's sum is a butterfly over those lanes, the other half of a half-layout pair comes from the
// wave's own LDS rows, interleaved pairs lie in one lane. The row's cos / sin, the only 64-bit work, are
// made once per workgroup while its heads' loads, issued first, are on the way (issued last, one pass of
// heads after the other: 86 us for 16,384 rows of 32 f16 heads of 128 with norms; now 59, 4.5 TB/s). One row
// takes 3.7 us.
#include "kernels.hpp"
#include "paged_dev.hpp"

#include <algorithm>
#include <cmath>

namespace mtg {
namespace {

using namespace paged;

struct RopeArgs {
  mtg_rope_append a;
  int shift, cap;  // of the page size; positions a table row names
  int heads;       // heads of a row taken: q, k and v, or those there are
  int q_heads, kv_heads;
};

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

constexpr int kThreads = 256;  // of a workgroup at most

template <typename IO, typename KV, int D, int PASSES>
__global__ void __launch_bounds__(kThreads) k_rope_append(RopeArgs r) {
  constexpr int kLanes = D / 8;               // of one head
  const int heads = blockDim.x / kLanes;      // of one pass
  const mtg_rope_append& a = r.a;
  __shared__ float rows[kThreads * 8];
  __shared__ float2 cs[D / 2];
  const int t = blockIdx.x, tid = threadIdx.x, sub = tid % kLanes, d0 = sub * 8;

  // the loads first: what they hold is needed last
  float x[PASSES][8];
  int kind[PASSES], head[PASSES];  // 0 q, 1 k, 2 v, 3 none
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int h = (blockIdx.y * PASSES + p) * heads + tid / kLanes;
    kind[p] = h < r.q_heads ? 0 : h < r.q_heads + r.kv_heads ? 1 : h < r.heads ? 2 : 3;
    head[p] = kind[p] == 0 ? h : kind[p] == 1 ? h - r.q_heads : h - r.q_heads - r.kv_heads;
    const IO* src = kind[p] == 0   ? (const IO*)a.q + (int64_t)t * a.q_stride
                    : kind[p] == 1 ? (const IO*)a.k_new + (int64_t)t * a.k_stride
                                   : (const IO*)a.v_new + (int64_t)t * a.v_stride;
    if (kind[p] < 3) load8(src + head[p] * D + d0, x[p]);
  }

  // the row's sequence; every wave finds it for itself
  Rows seq;
  const int b = seq_of_rows(a.kv, [&](int start, int) { return start <= t; }, &seq);
  if (b < 0 || t >= seq.row0 + seq.n) return;
  const int pos = seq.pos0 + (t - seq.row0);

  const int half = a.rot_dim >> 1;
  if (tid < half) {
    const double turns = (double)(a.positions ? a.positions[t] : pos) * (a.freqs[tid] * 0.15915494309189533577);
    // |part| <= 1/2; off by its rounding, 2^-26 turns, and by three of 64 bits, 2^-51 of all turns (2^-25 beside it from
    // positions of 2^28 on). A float's cos and sin of it are off by 4.6e-8 as a norm, of the angle in 64 bits by 3.8e-8.
    const float part = (float)(turns - rint(turns));
    float s, c;
    sincospif(2.0f * part, &s, &c);
    cs[tid] = make_float2(c * a.mscale, s * a.mscale);
  }
  // where k and v go
  int64_t place = -1;
  if (r.kv_heads) {
    const int page = page_of(a.kv.page_table + (int64_t)b * a.kv.table_stride, pos, r.shift, r.cap, a.kv.n_pages);
    if (page >= 0) place = (int64_t)page * a.kv.page_stride + (int64_t)(pos & (a.kv.page_size - 1)) * D;
  }
  __syncthreads();

#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    if (kind[p] == 3) continue;
    const float* gain = kind[p] == 0 ? a.q_norm : kind[p] == 1 ? a.k_norm : nullptr;
    // lanes of one head take the same way: whole heads differ, never lanes of a butterfly
    if (gain) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[p][i], x[p][i], ss);
#pragma unroll
      for (int m = 1; m < kLanes; m <<= 1) ss += __shfl_xor(ss, m);
      const float scale = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
      float g[8];
      load8(gain + d0, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[p][i] = x[p][i] * scale * g[i];
    }
    if (kind[p] != 2 && d0 < a.rot_dim) {
      float y[8];
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const bool in = d0 + i < a.rot_dim;
          const float2 w = cs[in ? (d0 + i) >> 1 : 0];
          y[i] = in ? x[p][i] * w.x - x[p][i + 1] * w.y : x[p][i];
          y[i + 1] = in ? x[p][i] * w.y + x[p][i + 1] * w.x : x[p][i + 1];
        }
      } else {
        float* row = rows + (tid / kLanes) * D;
        store8(row + d0, x[p]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (half % 8 == 0) {  // the other halves of a lane's pairs are neighbours too
          const bool low = d0 < half;
          const int first = low ? d0 : d0 - half;
          float other[8];
          load8(row + (low ? d0 + half : first), other);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 w = cs[first + i];
            y[i] = low ? x[p][i] * w.x - other[i] * w.y : other[i] * w.y + x[p][i] * w.x;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int d = d0 + i;
            const bool in = d < a.rot_dim, low = d < half;
            const float2 w = cs[!in ? 0 : low ? d : d - half];
            const float other = row[!in ? 0 : low ? d + half : d - half];
            y[i] = !in ? x[p][i] : low ? x[p][i] * w.x - other * w.y : other * w.y + x[p][i] * w.x;
          }
        }
        // the next pass's rows must not be written before these reads
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[p][i] = y[i];
    }
    if (kind[p] == 0)
      store8((IO*)a.q_out + (int64_t)t * a.q_out_stride + head[p] * D + d0, x[p]);
    else if (place >= 0)
      store8((KV*)(kind[p] == 1 ? a.kv.k : a.kv.v) + place + (int64_t)head[p] * a.kv.head_stride + d0, x[p]);
  }
}

template <typename IO, typename KV, int D>
hipError_t run(const RopeArgs& r, hipStream_t s) {
  // few heads: smaller workgroups, so that more of them fit a CU (16,384 rows of 4 heads of 64: 256 threads 18 us, 64 10.7)
  const int threads = std::min(kThreads, (r.heads * (D / 8) + 63) / 64 * 64), per = threads * 8 / D;
  const int passes = (r.heads + per - 1) / per;
  // enough rows to fill the chip: two heads a thread, both loads under way at once (16,384 rows of 32 heads, f16: one
  // head 69.3 us, two 60.5, four 67.4); below, more workgroups (512 rows: 4.9 us and 5.6)
  if (r.a.kv.n_tokens >= 1024 && passes > 1)
    return launch(k_rope_append<IO, KV, D, 2>, dim3(r.a.kv.n_tokens, (passes + 1) / 2), dim3(threads), 0, s, r);
  return launch(k_rope_append<IO, KV, D, 1>, dim3(r.a.kv.n_tokens, passes), dim3(threads), 0, s, r);
}
template <typename IO, typename KV>
hipError_t run(const RopeArgs& r, hipStream_t s) {
  return r.a.kv.head_dim == 128 ? run<IO, KV, 128>(r, s) : run<IO, KV, 64>(r, s);
}

int fail(int rc, const char* why) {
  set_call_error(std::string("rope_append: ") + why);
  return rc;
}

}  // namespace
}  // namespace mtg

extern "C" int mtg_rope_append_dev(const mtg_rope_append* p, void* stream) {
  using namespace mtg;
  try {
    if (!p) return fail(MTG_ERR_INVALID, "no description");
    const mtg_rope_append& a = *p;
    const mtg_paged_kv& kv = a.kv;
    const bool with_q = a.q || a.q_out, with_kv = a.k_new || a.v_new;
    int rc = 0;
    if (const char* why = check(kv, with_kv, &rc)) return fail(rc, why);
    if (!(a.io_type == MTG_TYPE_F32 && (!with_kv || kv.kv_type == MTG_TYPE_F32 || kv.kv_type == MTG_TYPE_F16)) &&
        !(a.io_type == MTG_TYPE_F16 && (!with_kv || kv.kv_type == MTG_TYPE_F16)))
      return fail(MTG_ERR_UNSUPPORTED, "types: f32 rows with an f32 or f16 cache, f16 rows with an f16 cache");
    if (a.rot_dim < 0 || a.rot_dim > kv.head_dim || a.rot_dim % 2) return fail(MTG_ERR_INVALID, "rot_dim");
    if (with_q && (a.n_heads <= 0 || a.n_heads > 1024)) return fail(MTG_ERR_INVALID, "n_heads");
    if ((a.q == nullptr) != (a.q_out == nullptr)) return fail(MTG_ERR_INVALID, "one of q and q_out is NULL");
    if ((a.k_new == nullptr) != (a.v_new == nullptr)) return fail(MTG_ERR_INVALID, "one of k_new and v_new is NULL");
    if (kv.n_seqs == 0 || kv.n_tokens == 0) return MTG_OK;
    if (!with_q && !with_kv) return fail(MTG_ERR_INVALID, "neither q nor k and v");
    if (a.rot_dim && !a.freqs) return fail(MTG_ERR_INVALID, "freqs is NULL");
    if (!aligned(a.freqs, 8) || !aligned(a.positions, 4)) return fail(MTG_ERR_INVALID, "unaligned freqs or positions");
    if (!aligned(a.q_norm, 16) || !aligned(a.k_norm, 16))
      return fail(MTG_ERR_UNSUPPORTED, "norms not aligned to 16 bytes");
    const int64_t unit = 16 / (int64_t)type_bytes(a.io_type);
    const int64_t qw = with_q ? (int64_t)a.n_heads * kv.head_dim : 0, kw = with_kv ? (int64_t)kv.n_kv_heads * kv.head_dim : 0;
    const struct {
      const void* at;
      int64_t stride, width;
    } in[] = {{a.q, a.q_stride, qw}, {a.k_new, a.k_stride, kw}, {a.v_new, a.v_stride, kw}, {a.q_out, a.q_out_stride, qw}};
    for (const auto& x : in) {
      if (!x.at) continue;
      if (x.stride < x.width || x.stride > ((int64_t)1 << 40) || !reaches(kv.n_tokens, x.stride))
        return fail(MTG_ERR_INVALID, "a row stride below the row's width, or rows behind 2^46 elements");
      if (!aligned(x.at, 16) || x.stride % unit) return fail(MTG_ERR_UNSUPPORTED, "rows not aligned to 16 bytes");
    }
    const size_t eb = type_bytes(a.io_type), out_bytes = extent(kv.n_tokens, a.q_out_stride, qw, eb);
    // rows that interleave with another operand's (slices of one wide product) share no element
    // only if the strides are one and the columns apart; that is what in place means here
    auto apart = [&](const void* x, int64_t stride, int64_t width) {
      if (!overlap(a.q_out, out_bytes, x, extent(kv.n_tokens, stride, width, eb))) return true;
      if (stride != a.q_out_stride) return false;
      const int64_t row = stride * (int64_t)eb;
      const int64_t gap = (((int64_t)((uintptr_t)x - (uintptr_t)a.q_out)) % row + row) % row;
      return gap >= qw * (int64_t)eb && gap + width * (int64_t)eb <= row;
    };
    if (with_q) {
      if (!(a.q == a.q_out && a.q_stride == a.q_out_stride) && !apart(a.q, a.q_stride, qw))
        return fail(MTG_ERR_INVALID, "q_out overlaps q");
      if (with_kv && (!apart(a.k_new, a.k_stride, kw) || !apart(a.v_new, a.v_stride, kw)))
        return fail(MTG_ERR_INVALID, "q_out overlaps k_new or v_new");
    }
    // the other arrays that are read; what one workgroup writes others may still read
    auto shared = [&](const void* p, size_t n) {
      return meets(p, n, {{a.positions, 4 * (size_t)kv.n_tokens}, {a.freqs, 4 * (size_t)a.rot_dim},
                          {a.q_norm, with_q ? 4 * (size_t)kv.head_dim : 0}, {a.k_norm, with_kv ? 4 * (size_t)kv.head_dim : 0},
                          {kv.page_table, with_kv ? 4 * (size_t)kv.n_seqs * kv.table_stride : 0},
                          {kv.kv_len, 4 * (size_t)kv.n_seqs}, {kv.q_start, 4 * (size_t)kv.n_seqs + 4}});
    };
    if (with_q && shared(a.q_out, out_bytes)) return fail(MTG_ERR_INVALID, "q_out overlaps an index array, the frequencies or a norm");
    if (with_kv) {
      const size_t pool = pool_extent(kv);
      if (!k_and_v_apart(kv)) return fail(MTG_ERR_INVALID, "k and v share elements of one pool");
      for (const void* pages : {kv.k, kv.v}) {
        if (overlap(pages, pool, a.q_out, out_bytes)) return fail(MTG_ERR_INVALID, "q_out lies in the pages");
        if (meets(pages, pool, {{a.q, extent(kv.n_tokens, a.q_stride, qw, eb)}, {a.k_new, extent(kv.n_tokens, a.k_stride, kw, eb)},
                                {a.v_new, extent(kv.n_tokens, a.v_stride, kw, eb)}}))
          return fail(MTG_ERR_INVALID, "q, k_new or v_new lies in the pages");
        if (shared(pages, pool)) return fail(MTG_ERR_INVALID, "an index array, the frequencies or a norm lies in the pages");
      }
    }
    RopeArgs r{a, 0, 0, 0, with_q ? a.n_heads : 0, with_kv ? kv.n_kv_heads : 0};
    if (with_kv) r.shift = log2_of(kv.page_size), r.cap = capacity(kv.table_stride, r.shift);
    r.heads = r.q_heads + 2 * r.kv_heads;
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = a.io_type == MTG_TYPE_F16          ? run<_Float16, _Float16>(r, s)
                         : kv.kv_type == MTG_TYPE_F16 && with_kv ? run<float, _Float16>(r, s)
                                                            : run<float, float>(r, s);
    if (e != hipSuccess) return fail(MTG_ERR_DEVICE, hipGetErrorString(e));
    return MTG_OK;
  } catch (...) {
    return MTG_ERR_NOMEM;
  }
}

extern "C" int mtg_rope_freqs(int32_t kind, int32_t rot_dim, double base, double factor, double orig_ctx, double beta_fast,
                              double beta_slow, double* freqs, float* mscale) {
  using namespace mtg;
  try {
    const bool yarn = kind == MTG_ROPE_YARN;
    if (kind < MTG_ROPE_PLAIN || kind > MTG_ROPE_YARN || rot_dim <= 0 || rot_dim % 2 || !freqs || !mscale ||
        !(base > 1.0) || !std::isfinite(base) || !(factor >= 1.0) || !std::isfinite(factor) ||
        (kind == MTG_ROPE_NTK && rot_dim == 2))
      return fail(MTG_ERR_INVALID, "frequencies: kind, rot_dim, base > 1 or factor >= 1");
    if (yarn && (!(orig_ctx > 0) || !std::isfinite(orig_ctx) || !(beta_slow > 0) || !(beta_fast > beta_slow) || !std::isfinite(beta_fast)))
      return fail(MTG_ERR_INVALID, "frequencies: orig_ctx > 0, beta_fast > beta_slow > 0");
    const double pi = 3.14159265358979323846;
    if (kind == MTG_ROPE_NTK) base *= std::pow(factor, (double)rot_dim / (rot_dim - 2));
    // the pair that turns `turns` times within orig_ctx: base^(-2i/rot_dim) orig_ctx = 2 pi turns
    auto pair_of = [&](double turns) { return rot_dim * std::log(orig_ctx / (turns * 2 * pi)) / (2 * std::log(base)); };
    const double low = yarn ? std::fmax(std::floor(pair_of(beta_fast)), 0.0) : 0.0;
    const double high = yarn ? std::fmin(std::ceil(pair_of(beta_slow)), rot_dim - 1.0) : 0.0;
    for (int i = 0; i < rot_dim / 2; ++i) {
      const double f = std::pow(base, -2.0 * i / rot_dim);
      // (high first: at or below 0, where even the fastest pair turns fewer than beta_slow times, all are divided)
      const double slow = yarn ? i >= high ? 1.0 : i <= low ? 0.0 : (i - low) / (high - low) : kind == MTG_ROPE_LINEAR ? 1.0 : 0.0;
      freqs[i] = f / factor * slow + f * (1.0 - slow);
    }
    *mscale = yarn ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return MTG_OK;
  } catch (...) {
    return MTG_ERR_NOMEM;
  }
}
