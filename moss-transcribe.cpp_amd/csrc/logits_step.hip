// logits_step.hip - mtg_logits_step_dev: penalties for repeated ids, biases and grammar masks on
// rows of logits, and the first-max choice of what remains (reference: the repetition penalty and
// the strict > of cpu_greedy_choice, src/cpu_speculative.cpp:39-50).
//
// Every logit is read once and written at most once, so HBM bounds it; a row or two are bound by
// the launch and the chain range - ids - logits (one row of 151,936 under a mask 5.8 us). A workgroup
// takes 4,096 ids of a row. The row's lists (ids in no order, any number of times) are first spread over a dense table
// of those ids in LDS - counts by integer adds, the last bias entry by an integer maximum, so no order
// of arrival shows - while the logits' loads are on the way; a thread then looks at its entries and
// only ids that a list names take the divisions. The choice is a maximum of 64-bit keys, the value's
// bits in ascending order above the inverted id: first of the workgroup, then of the row's workgroups
// (in a second small kernel where there are many).
//
// Every workgroup reads its row's lists, 4 entries a thread at once and ahead of its logits: 256 rows of
// 151,936 f32 under a mask, 1,000 ids and 300 biases 69.5 us (4.6 TB/s), 61 rows of f16 with 2,000 ids 18.5 (12.3
// without lists and mask). Fewer and larger workgroups read them less often, but hold up more: with 8,192
// or 16,384 ids 80.7 and 81.4 us (then 72.5), with 32 ids a thread 90.9. The tables hold 16 bits an id (as 32, 16 KB
// each, half as many workgroups fit a CU: 108 us); a row with a list of more than 65,535 entries goes over them
// twice, with 32 bits for half of the ids.
#include "kernels.hpp"
#include "paged_dev.hpp"

namespace mtg {
namespace {

using namespace paged;

constexpr int kSlice = 4096;  // ids of a workgroup
constexpr int kFew = 1024;    // workgroups of 512 threads that the chip takes at once

// Rows begin where the caller's stride puts them: vectors aligned to their elements only.
typedef f4 f4u __attribute__((aligned(4)));
typedef h8 h8u __attribute__((aligned(2)));

struct LogitsArgs {
  mtg_logits_step a;
  int slices;     // workgroups of a row
  uint64_t mark;  // of this call, where they join the row themselves
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
// Past L2, whose lines the end of the kernel would wait for: 72.8 -> 69.7 us for 256 rows.
__device__ __forceinline__ void store(float* p, const float* x) {
  f4u v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = x[i];
  __builtin_nontemporal_store(v, (f4u*)p);
}
__device__ __forceinline__ void store(_Float16* p, const float* x) {
  h8u v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (_Float16)x[i];  // exact: x was rounded before
  __builtin_nontemporal_store(v, (h8u*)p);
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

// Values that all lanes read, through the scalar cache: they are there before the vector loads queue up.
typedef const __attribute__((address_space(4))) int32_t* Ints;
typedef const __attribute__((address_space(4))) float* Floats;

// Entries lo .. hi - 1 of a list of n, whatever the range array holds.
__device__ __forceinline__ void range_of(const int32_t* range, int row, int n, int* lo, int* hi) {
  *lo = *hi = 0;
  if (!range) return;
  *lo = cut(((Ints)range)[2 * row], 0, n);
  *hi = cut(((Ints)range)[2 * row + 1], *lo, n);
}

// The larger of 16 bits of a word and v, the other 16 as they are.
__device__ __forceinline__ void max16(uint32_t* w, int shift, uint32_t v) {
  uint32_t old = *w;
  while ((old >> shift & 0xffffu) < v) {
    const uint32_t seen = old;
    old = atomicCAS(w, seen, (seen & ~(0xffffu << shift)) | v << shift);
    if (old == seen) return;
  }
}

// Of 512 threads for up to kFew workgroups, which then join their rows themselves; else of 256.
template <typename IO, int kThreads>
__global__ void __launch_bounds__(kThreads) k_logits_step(LogitsArgs r) {
  constexpr bool kFewRows = kThreads == 512;
  constexpr int V = 16 / sizeof(IO), N = kSlice / kThreads / V;
  const mtg_logits_step& a = r.a;
  __shared__ __attribute__((aligned(16))) uint32_t count[kSlice / 2], entry[kSlice / 2];
  __shared__ uint64_t best[kThreads / 64];
  const int slice = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, base = slice * kSlice;
  const IO* src = (const IO*)a.logits + (int64_t)row * a.stride;

  int h0, h1, b0, b1;
  range_of(a.hist_range, row, a.n_history, &h0, &h1);
  range_of(a.bias_range, row, a.n_bias, &b0, &b1);
  float rep = 1.0f, freq = 0.0f, pres = 0.0f;
  if (a.hist_range) rep = ((Floats)a.penalties)[3 * row], freq = ((Floats)a.penalties)[3 * row + 1], pres = ((Floats)a.penalties)[3 * row + 2];
  // the lists' first entries, ahead of the logits in the queue: the tables wait for them, not for the logits
  constexpr int kTime = 4;  // of a list a thread
  auto ids_at = [&](const int32_t* list, int i, int hi, int (&id)[kTime]) {
#pragma unroll
    for (int k = 0; k < kTime; ++k) id[k] = i + k * kThreads < hi ? list[i + k * kThreads] : -1;
  };
  int hist_ids[kTime], bias_ids[kTime];
  ids_at(a.history, h0 + tid, h1, hist_ids);
  ids_at(a.bias_ids, b0 + tid, b1, bias_ids);

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

  const bool hist = h0 < h1, bias = b0 < b1;
  if (hist || bias) {
    auto clear = [&]() {
      for (int i = tid * 4; i < kSlice / 2; i += kThreads * 4) {
        if (hist) *(u4*)&count[i] = u4{0, 0, 0, 0};
        if (bias) *(u4*)&entry[i] = u4{0, 0, 0, 0};
      }
    };
    auto change = [&](float* y, uint32_t c, uint32_t e) {
      if (c) {
        if (rep > 1.0f) *y = *y > 0.0f ? *y / rep : *y * rep;
        *y = *y - (freq * (float)c + pres);
      }
      if (e) *y = *y + a.bias[b0 + (int)e - 1];
    };
    // ids first .. first + size - 1 that the lists name
    auto spread = [&](int first, int size, auto&& counted, auto&& listed) {
      const int end = first + size < a.vocab ? first + size : a.vocab;
      for (int i = h0 + tid; i < h1; i += kTime * kThreads) {
        int id[kTime];
#pragma unroll
        for (int k = 0; k < kTime; ++k) id[k] = hist_ids[k];
        if (i != h0 + tid) ids_at(a.history, i, h1, id);
#pragma unroll
        for (int k = 0; k < kTime; ++k)
          if (id[k] >= first && id[k] < end) counted(id[k] - first);
      }
      for (int i = b0 + tid; i < b1; i += kTime * kThreads) {
        int id[kTime];
#pragma unroll
        for (int k = 0; k < kTime; ++k) id[k] = bias_ids[k];
        if (i != b0 + tid) ids_at(a.bias_ids, i, b1, id);
#pragma unroll
        for (int k = 0; k < kTime; ++k)
          if (id[k] >= first && id[k] < end) listed(id[k] - first, (uint32_t)(i + k * kThreads - b0) + 1);
      }
    };
    if (h1 - h0 <= 65535 && b1 - b0 <= 65535) {
      clear();
      __syncthreads();
      spread(base, kSlice, [&](int at) { atomicAdd(&count[at >> 1], 1u << (at & 1) * 16); },
             [&](int at, uint32_t v) { max16(&entry[at >> 1], (at & 1) * 16, v); });
      __syncthreads();
#pragma unroll
      for (int k = 0; k < N; ++k)
#pragma unroll
        for (int q = 0; q < V; q += 4) {
          const int at = ((k * kThreads + tid) * V + q) >> 1;
          const u2 c = hist ? *(const u2*)&count[at] : u2{0, 0}, e = bias ? *(const u2*)&entry[at] : u2{0, 0};
          if ((c[0] | c[1] | e[0] | e[1]) == 0) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) change(&x[k][q + i], c[i >> 1] >> (i & 1) * 16 & 0xffffu, e[i >> 1] >> (i & 1) * 16 & 0xffffu);
        }
    } else {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (half) __syncthreads();
        clear();
        __syncthreads();
        spread(base + half * (kSlice / 2), kSlice / 2, [&](int at) { atomicAdd(&count[at], 1u); },
               [&](int at, uint32_t v) { atomicMax(&entry[at], v); });
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int at = (k * kThreads + tid) * V - half * (kSlice / 2);
          if (at < 0 || at >= kSlice / 2) continue;
#pragma unroll
          for (int i = 0; i < V; ++i) change(&x[k][i], hist ? count[at + i] : 0, bias ? entry[at + i] : 0);
        }
      }
    }
  }

  // the first id with the largest value above -inf, in the order of the thread's ids
  float most = -INFINITY;
  int at = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int id = base + (k * kThreads + tid) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float y = (float)(IO)x[k][i];  // the rounding of the result: the choice is made on what is stored
      x[k][i] = allowed[k] & (1u << i) ? y : -INFINITY;
      if (x[k][i] > most) most = x[k][i], at = id + i;  // no NaN is
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
  uint64_t top = most > -INFINITY ? key_of(most, at) : 0;
  if (top == 0) {  // an allowed -inf is a value too
#pragma unroll
    for (int k = N - 1; k >= 0; --k)
#pragma unroll
      for (int i = V - 1; i >= 0; --i)
        if ((allowed[k] & (1u << i)) && x[k][i] == -INFINITY) top = key_of(-INFINITY, base + (k * kThreads + tid) * V + i);
  }
  top = max_wave(top);
  if ((tid & 63) == 0) best[tid >> 6] = top;
  __syncthreads();
  if (tid >= 64) return;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) top = best[w] > top ? best[w] : top;
  if (r.slices == 1) {
    if (tid == 0) a.choice[row] = id_of(top);
    return;
  }
  uint64_t* keys = (uint64_t*)a.workspace + (int64_t)row * r.slices * (kFewRows ? 2 : 1);
  if constexpr (!kFewRows) {
    if (tid == 0) keys[slice] = top;
  } else {
    // Joined here: each half of a key goes out under half of the call's mark, and who then finds all of the row's halves
    // marked has them (the last one does; should two, both write the same). They are cleared, so a replayed call finds
    // none of its own: no half of a mark is 0. Stores and loads are the device's (past the caches of an XCD).
    auto put = [&](int i, uint64_t v) { __hip_atomic_store(keys + i, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto take = [&](int i) { return __hip_atomic_load(keys + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    const uint64_t high = r.mark >> 32 << 32, low = r.mark << 32;
    if (tid == 0) {
      put(2 * slice, high | top >> 32);
      put(2 * slice + 1, low | (uint32_t)top);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    bool all = true;
    top = 0;
    for (int i = tid; i < r.slices; i += 64) {
      const uint64_t x = take(2 * i) ^ high, y = take(2 * i + 1) ^ low, key = x << 32 | (uint32_t)y;
      all = all && (x >> 32 | y >> 32) == 0;
      top = key > top ? key : top;
    }
    if (!__all(all)) return;
    for (int i = tid; i < 2 * r.slices; i += 64) put(i, 0);
    top = max_wave(top);
    if (tid == 0) a.choice[row] = id_of(top);
  }
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

int slices_of(const mtg_logits_step& a) { return (a.vocab + kSlice - 1) / kSlice; }
bool sizes_ok(const mtg_logits_step& a) {
  // lists of at most 2^30: the steps through them stay within 31 bits
  return a.rows >= 0 && a.rows <= 65535 && a.vocab > 0 && a.vocab <= (1 << 24) && a.n_history >= 0 && a.n_history <= (1 << 30) &&
         a.n_bias >= 0 && a.n_bias <= (1 << 30);
}
bool few(const mtg_logits_step& a) { return (int64_t)a.rows * slices_of(a) <= kFew; }
size_t workspace_of(const mtg_logits_step& a) {
  const int n = slices_of(a);
  return a.choice && n > 1 ? ((size_t)a.rows * n * (few(a) ? 16 : 8) + 15) / 16 * 16 : 0;
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
    if (!sizes_ok(a)) return fail(MTG_ERR_INVALID, "rows 0 to 65535, vocab 1 to 2^24, lists of 0 to 2^30");
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
    }
    // what one workgroup writes others may still read: no array that is written shares a byte with another one
    const size_t rows = (size_t)a.rows, picks = a.choice ? 4 * rows : 0;
    const size_t listed = a.history ? 4 * (size_t)a.n_history : 0, biased = a.bias ? 4 * (size_t)a.n_bias : 0;
    const Array hist_range{a.hist_range, a.history ? 8 * rows : 0}, penalties{a.penalties, a.history ? 12 * rows : 0};
    const Array bias_range{a.bias_range, a.bias ? 8 * rows : 0}, mask{a.mask, extent(a.rows, a.mask_stride, words, 4)};
    auto shared = [&](const void* p, size_t n) {
      return meets(p, n, {{a.history, listed}, hist_range, penalties, {a.bias_ids, biased}, {a.bias, biased}, bias_range, mask});
    };
    if (shared(a.out, out)) return fail(MTG_ERR_INVALID, "out overlaps a list, its ranges, the penalties or the mask");
    if (shared(a.choice, picks) || meets(a.choice, picks, {{a.logits, in}, {a.out, out}}))
      return fail(MTG_ERR_INVALID, "choice overlaps another array");
    if (shared(a.workspace, need) || meets(a.workspace, need, {{a.logits, in}, {a.out, out}, {a.choice, picks}}))
      return fail(MTG_ERR_INVALID, "workspace overlaps another array");
    LogitsArgs r{a, slices_of(a), few(a) ? next_mark() : 0};
    if (!a.history) r.a.hist_range = nullptr;
    if (!a.bias) r.a.bias_range = nullptr;
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid(r.slices, a.rows);
    // few workgroups: more threads each, which are through sooner (f32, 1,000 ids a row: 20 rows 9.3 us and 10.3; 256 rows
    // 76.8 and 69.8), and no second launch (one row 5.8 us and 6.2, two 5.9 and 7.5, 50 of 32,000 ids 6.2 and 7.5)
    const bool f16 = a.io_type == MTG_TYPE_F16;
    hipError_t e = few(a) ? f16 ? launch(k_logits_step<_Float16, 512>, grid, dim3(512), 0, s, r)
                                : launch(k_logits_step<float, 512>, grid, dim3(512), 0, s, r)
                   : f16  ? launch(k_logits_step<_Float16, 256>, grid, dim3(256), 0, s, r)
                          : launch(k_logits_step<float, 256>, grid, dim3(256), 0, s, r);
    if (e == hipSuccess && need && !few(a)) e = launch(k_logits_choice, dim3(a.rows), dim3(64), 0, s, r);
    if (e != hipSuccess) return fail(MTG_ERR_DEVICE, hipGetErrorString(e));
    return MTG_OK;
  } catch (...) {
    return MTG_ERR_NOMEM;
  }
}
