// paged_dev.hpp - device helpers of the operators over paged caches.
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <atomic>
#include <random>
#include <string>

#include "paged_kv.hpp"

namespace mtg {
namespace paged {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// last_of over the lanes of a wave, pred(i) by i: for up to 64 sequences the search is one load per lane instead
// of a chain of dependent ones.
template <class P>
__device__ __forceinline__ int last_true(int n, const P& pred) {
  const int lane = threadIdx.x & 63;
  return __builtin_amdgcn_readfirstlane(last_of(n, [&](int lo, int step, int count) {
    const int off = lane * step;
    return (uint64_t)__ballot(off < count && pred(lo + off));
  }));
}

// The sequence at or before which `before(start, b)` last holds, and its rows: up to 64 sequences in one
// round trip to memory (what a short step waits for), more by a search first.
template <class P>
__device__ __forceinline__ int seq_of_rows(const mtg_paged_kv& c, const P& before, Rows* rows) {
  const int lane = threadIdx.x & 63;
  int at = 0, start = 0, end = 0, len = 0;
  if (c.n_seqs > 64) {
    at = last_true(c.n_seqs, [&](int i) { return before(c.q_start[i], i); });
    if (at < 0) return -1;
    start = c.q_start[at], end = c.q_start[at + 1], len = c.kv_len[at];
  } else {
    if (lane < c.n_seqs) start = c.q_start[lane], end = c.q_start[lane + 1], len = c.kv_len[lane];
    const uint64_t yes = __ballot(lane < c.n_seqs && before(start, lane));
    if (yes == 0) return -1;
    at = 63 - __builtin_clzll(yes);
    start = __builtin_amdgcn_readlane(start, at), end = __builtin_amdgcn_readlane(end, at), len = __builtin_amdgcn_readlane(len, at);
  }
  *rows = rows_of(start, end, len, c.n_tokens);
  return at;
}

// The mark of a call.
inline uint64_t next_mark() {
  static std::atomic<uint64_t> calls{((uint64_t)std::random_device{}() << 32) ^ std::random_device{}()};
  return next_mark(calls);
}

// Launch by hipLaunchKernel's own status: an error that an earlier call of the program left
// behind is not taken for this one's, and a refused launch leaves none.
template <class... A>
inline hipError_t launch(void (*kernel)(A...), dim3 grid, dim3 block, size_t lds, hipStream_t s, A... args) {
  void* list[] = {(void*)&args...};
  const hipError_t e = hipLaunchKernel((const void*)kernel, grid, block, list, lds, s);
  if (e != hipSuccess) (void)hipGetLastError();
  return e;
}

}  // namespace paged
}  // namespace mtg
