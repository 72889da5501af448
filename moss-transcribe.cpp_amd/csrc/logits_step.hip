// logits_step.hip - mtg_logits_step_dev: penalties for repeated ids, biases and grammar masks on
// rows of logits, and the first-max choice of what remains (reference: the repetition penalty and
// the strict > of cpu_greedy_choice, src/cpu_speculative.cpp:39-50).
//
// Every logit is read once and written at most once, so HBM bounds it; a row or two are bound by
// the launches. A workgroup takes 4,096 ids of a row, 16 a thread. The row's lists (ids in no
// order, any number of times) are first spread over a dense table of those ids in LDS - counts by
// integer adds, the last bias entry by an integer maximum, so no order of arrival shows - while
// the logits' loads are on the way; a thread then looks at its 16 entries and only ids that a
// list names take the divisions. The choice is a maximum of 64-bit keys, the value's bits in
// ascending order above the inverted id: first of the workgroup, then of the row's workgroups in
// a second small kernel (a row of 4,096 ids or fewer needs none).
#include "kernels.hpp"
#include "paged_dev.hpp"

namespace mtg {
namespace {

using namespace paged;

constexpr int kThreads = 256, kPer = 16, kSlice = kThreads * kPer;

// Rows begin where the caller's stride puts them: vectors aligned to their elements only.
typedef f4 f4u __attribute__((aligned(4)));
typedef h8 h8u __attribute__((aligned(2)));

struct LogitsArgs {
  mtg_logits_step a;
  int slices;
};

__device__ __forceinline__ void load(const float* p, float* x) {
  const f4u v = *(const f4u*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = v[i];
}
__device__ __forceinline__ void load(const _Float16* p, float* x) {
  const h8u v = *(const h8u*)p;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
}
__device__ __forceinline__ void store(float* p, const float* x) {
  f4u v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = x[i];
  *(f4u*)p = v;
}
__device__ __forceinline__ void store(_Float16* p, const float* x) {
  h8u v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (_Float16)x[i];  // exact: x was rounded before
  *(h8u*)p = v;
}

// Larger for a larger value, for equal values (both zeros are) the lower id; 0 is none.
__device__ __forceinline__ uint64_t key_of(float y, int id) {
  const uint32_t b = __float_as_uint(y + 0.0f);
  return (uint64_t)((b >> 31) ? ~b : b | 0x80000000u) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ uint64_t max_wave(uint64_t k) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)k, m);
    k = o > k ? o : k;
  }
  return k;
}
__device__ __forceinline__ int id_of(uint64_t key) { return key ? (int)~(uint32_t)key : -1; }

// Entries lo .. hi - 1 of a list of n, whatever the range array holds.
__device__ __forceinline__ void range_of(const int32_t* range, int row, int n, int* lo, int* hi) {
  *lo = *hi = 0;
  if (!range) return;
  *lo = cut(range[2 * row], 0, n);
  *hi = cut(range[2 * row + 1], *lo, n);
}

template <typename IO>
__global__ void __launch_bounds__(kThreads) k_logits_step(LogitsArgs r) {
  constexpr int V = 16 / sizeof(IO), N = kPer / V;
  const mtg_logits_step& a = r.a;
  __shared__ uint32_t count[kSlice], entry[kSlice];
  __shared__ uint64_t best[kThreads / 64];
  const int slice = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, base = slice * kSlice;
  const IO* src = (const IO*)a.logits + (int64_t)row * a.stride;

  // the thread's ids: N vectors of V, kThreads vectors apart
  float x[N][V];
  uint32_t allowed[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int id = base + (k * kThreads + tid) * V;
    allowed[k] = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) x[k][i] = 0.0f;
    if (id + V <= a.vocab) {
      load(src + id, x[k]);
      allowed[k] = (1u << V) - 1;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (id + i < a.vocab) x[k][i] = (float)src[id + i], allowed[k] |= 1u << i;
    }
    // V divides 32: one word holds the vector's bits
    if (a.mask && id < a.vocab) allowed[k] &= a.mask[(int64_t)row * a.mask_stride + (id >> 5)] >> (id & 31);
  }

  int h0, h1, b0, b1;
  range_of(a.hist_range, row, a.n_history, &h0, &h1);
  range_of(a.bias_range, row, a.n_bias, &b0, &b1);
  float rep = 1.0f, freq = 0.0f, pres = 0.0f;
  if (h0 < h1) rep = a.penalties[3 * row], freq = a.penalties[3 * row + 1], pres = a.penalties[3 * row + 2];
  if (h0 < h1 || b0 < b1) {
    for (int i = tid * 4; i < kSlice; i += kThreads * 4) {
      *(u4*)&count[i] = u4{0, 0, 0, 0};
      *(u4*)&entry[i] = u4{0, 0, 0, 0};
    }
    __syncthreads();
    for (int i = h0 + tid; i < h1; i += kThreads) {
      const int id = a.history[i];
      if (id >= base && id - base < kSlice && id < a.vocab) atomicAdd(&count[id - base], 1u);
    }
    for (int i = b0 + tid; i < b1; i += kThreads) {
      const int id = a.bias_ids[i];
      if (id >= base && id - base < kSlice && id < a.vocab) atomicMax(&entry[id - base], (uint32_t)(i - b0) + 1);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        const int at = (k * kThreads + tid) * V + q;
        const u4 c = *(const u4*)&count[at], e = *(const u4*)&entry[at];
        if ((c[0] | c[1] | c[2] | c[3] | e[0] | e[1] | e[2] | e[3]) == 0) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y = x[k][q + i];
          if (c[i]) {
            if (rep > 1.0f) y = y > 0.0f ? y / rep : y * rep;
            y = y - (freq * (float)c[i] + pres);
          }
          if (e[i]) y = y + a.bias[b0 + (int)e[i] - 1];
          x[k][q + i] = y;
        }
      }
  }

  uint64_t top = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int id = base + (k * kThreads + tid) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float y = (float)(IO)x[k][i];  // the rounding of the result: the choice is made on what is stored
      const bool on = allowed[k] >> i & 1;
      x[k][i] = on ? y : -INFINITY;
      if (on && y == y) {
        const uint64_t key = key_of(y, id + i);
        top = key > top ? key : top;
      }
    }
    if (a.out) {
      IO* dst = (IO*)a.out + (int64_t)row * a.out_stride + id;
      if (id + V <= a.vocab) {
        store(dst, x[k]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (id + i < a.vocab) dst[i] = (IO)x[k][i];
      }
    }
  }
  if (!a.choice) return;
  top = max_wave(top);
  if ((tid & 63) == 0) best[tid >> 6] = top;
  __syncthreads();
  if (tid) return;
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) top = best[w] > top ? best[w] : top;
  if (r.slices == 1)
    a.choice[row] = id_of(top);
  else
    ((uint64_t*)a.workspace)[(int64_t)row * r.slices + slice] = top;
}

__global__ void __launch_bounds__(64) k_logits_choice(LogitsArgs r) {
  const uint64_t* keys = (const uint64_t*)r.a.workspace + (int64_t)blockIdx.x * r.slices;
  uint64_t top = 0;
  for (int i = threadIdx.x; i < r.slices; i += 64) top = keys[i] > top ? keys[i] : top;
  top = max_wave(top);
  if (threadIdx.x == 0) r.a.choice[blockIdx.x] = id_of(top);
}

int fail(int rc, const char* why) {
  set_call_error(std::string("logits_step: ") + why);
  return rc;
}

int slices_of(const mtg_logits_step& a) { return a.vocab / kSlice + (a.vocab % kSlice != 0); }
bool sizes_ok(const mtg_logits_step& a) {
  return a.rows >= 0 && a.rows <= 65535 && a.vocab > 0 && a.vocab <= (1 << 24) && a.n_history >= 0 && a.n_bias >= 0;
}
size_t workspace_of(const mtg_logits_step& a) {
  const int n = slices_of(a);
  return a.choice && n > 1 ? ((size_t)a.rows * n * 8 + 15) / 16 * 16 : 0;
}

}  // namespace
}  // namespace mtg

extern "C" size_t mtg_logits_step_workspace(const mtg_logits_step* a) {
  return a && mtg::sizes_ok(*a) ? mtg::workspace_of(*a) : 0;
}

extern "C" int mtg_logits_step_dev(const mtg_logits_step* p, void* stream) {
  using namespace mtg;
  try {
    if (!p) return fail(MTG_ERR_INVALID, "no description");
    const mtg_logits_step& a = *p;
    if (!sizes_ok(a)) return fail(MTG_ERR_INVALID, "rows 0 to 65535, vocab 1 to 2^24, lists of 0 or more");
    if (a.io_type != MTG_TYPE_F32 && a.io_type != MTG_TYPE_F16) return fail(MTG_ERR_UNSUPPORTED, "io_type is not f32 or f16");
    if (a.rows == 0) return MTG_OK;
    if (!a.logits || (!a.out && !a.choice)) return fail(MTG_ERR_INVALID, "logits is NULL, or both out and choice are");
    const int64_t most = (int64_t)1 << 40;
    if (a.stride < a.vocab || a.stride > most || (a.out && (a.out_stride < a.vocab || a.out_stride > most)))
      return fail(MTG_ERR_INVALID, "a row stride below vocab");
    if (a.history && (!a.hist_range || !a.penalties)) return fail(MTG_ERR_INVALID, "history without hist_range or penalties");
    if (a.bias && (!a.bias_ids || !a.bias_range)) return fail(MTG_ERR_INVALID, "bias without bias_ids or bias_range");
    const int64_t words = ((int64_t)a.vocab + 31) / 32;
    if (a.mask && a.mask_stride != 0 && (a.mask_stride < words || a.mask_stride > most))
      return fail(MTG_ERR_INVALID, "mask_stride");
    const size_t eb = type_bytes(a.io_type);
    if (!aligned(a.logits, eb) || !aligned(a.out, eb) || !aligned(a.history, 4) || !aligned(a.hist_range, 4) ||
        !aligned(a.penalties, 4) || !aligned(a.bias_ids, 4) || !aligned(a.bias, 4) || !aligned(a.bias_range, 4) ||
        !aligned(a.mask, 4) || !aligned(a.choice, 4))
      return fail(MTG_ERR_INVALID, "an array not aligned to its elements");
    const size_t in = extent(a.rows, a.stride, a.vocab, eb), out = a.out ? extent(a.rows, a.out_stride, a.vocab, eb) : 0;
    if (overlap(a.logits, in, a.out, out) && !(a.logits == a.out && a.stride == a.out_stride))
      return fail(MTG_ERR_INVALID, "out overlaps logits");
    const size_t need = workspace_of(a);
    if (need) {
      if (!a.workspace || !aligned(a.workspace, 16)) return fail(MTG_ERR_INVALID, "workspace NULL or unaligned");
      if (a.workspace_bytes < need) return fail(MTG_ERR_CAPACITY, "workspace smaller than mtg_logits_step_workspace");
      if (overlap(a.workspace, need, a.logits, in) || overlap(a.workspace, need, a.out, out))
        return fail(MTG_ERR_INVALID, "workspace overlaps logits or out");
    }
    LogitsArgs r{a, slices_of(a)};
    if (!a.history) r.a.hist_range = nullptr;
    if (!a.bias) r.a.bias_range = nullptr;
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid(r.slices, a.rows);
    hipError_t e = a.io_type == MTG_TYPE_F16 ? launch(k_logits_step<_Float16>, grid, dim3(kThreads), 0, s, r)
                                             : launch(k_logits_step<float>, grid, dim3(kThreads), 0, s, r);
    if (e == hipSuccess && need) e = launch(k_logits_choice, dim3(a.rows), dim3(64), 0, s, r);
    if (e != hipSuccess) return fail(MTG_ERR_DEVICE, hipGetErrorString(e));
    return MTG_OK;
  } catch (...) {
    return MTG_ERR_NOMEM;
  }
}
