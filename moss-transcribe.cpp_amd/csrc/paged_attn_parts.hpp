// paged_attn_parts.hpp - what the attention kernels over paged caches have in common (paged_attn.hip: caches of f32 and
// f16; paged_attn_f8.hip: in 8 bits): operands in parts, tiles of rows, the running softmax, the join of splits, the
// choice of kernel and splits. What the operands' layouts are for is told at the head of paged_attn.hip.
#pragma once

#include "paged_dev.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

namespace mtg {
namespace attn {

using namespace paged;

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

struct Eight {
  float x[8];
};

struct AttnArgs {
  mtg_paged_attn a;
  int shift, cap;           // of the page size; positions a table row names
  int group;                // query heads of a kv head
  int split_keys, n_split;  // keys of a split (a multiple of 64, of 128 for k_paged_rows), most splits of a tile
  int tiles;                // of rows, at most
  float* part_o;            // [split][row][head_dim] of rows (token, head): sums, by the maximum of the split
  float* part_ml;           // [split][row][2]: that maximum, the weights' sum
  uint64_t* arrived;        // [tile][kv head][split]: `mark` once the split's part is written, 0 when joined
  uint64_t mark;            // of this call; 0: the join is a launch of its own
  float log2_scale;         // scale * log2(e)
  int sink;                 // first positions that stay visible beside a window
};

constexpr int kChunkRows = 128, kTileKeys = 64;  // of a workgroup of k_paged_chunk, and of its steps
constexpr float kSlack = 8.0f;  // a score above the maximum by more than 2^8 moves it

__device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mma(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// A lane's elements (or keys) 8 g .. 8 g + 7, one of each group g to a product.
__device__ __forceinline__ f4 mma(const Eight& a, const Eight& b, f4 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x[j], b.x[j], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ f16v mma32(h8 a, h8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// The product of a value in NA parts with one in NB, small terms first.
template <class MV, int NA, int NB>
__device__ __forceinline__ f4 product(const MV (&a)[NA], const MV (&b)[NB], f4 c) {
  constexpr int n = NA > NB ? NA : NB;
#pragma unroll
  for (int sum = n - 1; sum >= 0; --sum)
#pragma unroll
    for (int i = 0; i <= sum; ++i)
      if (i < NA && sum - i < NB) c = mma(a[i], b[sum - i], c);
  return c;
}

__device__ __forceinline__ void parts(const float* x, Eight (&p)[1]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) p[0].x[j] = x[j];
}
__device__ __forceinline__ void parts(const float* x, h8 (&p)[1]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) p[0][j] = (_Float16)x[j];
}
__device__ __forceinline__ void parts(const float* x, h8 (&p)[2]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    p[0][j] = (_Float16)x[j];
    p[1][j] = (_Float16)(x[j] - (float)p[0][j]);
  }
}
// Exact: 24 bits of a float are three times 8, each part the upper 16 bits of what is left.
__device__ __forceinline__ void parts(const float* x, b8 (&p)[3]) {
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = x[j];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    u4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = __float_as_uint(r[2 * j]), hi = __float_as_uint(r[2 * j + 1]);
      w[j] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
      if (k < 2) {
        r[2 * j] -= __uint_as_float(lo & 0xffff0000u);
        r[2 * j + 1] -= __uint_as_float(hi & 0xffff0000u);
      }
    }
    p[k] = __builtin_bit_cast(b8, w);
  }
}

// N neighbouring elements as they lie in memory, two f16 or one f32 to a word.
template <class T, int N>
struct Raw {
  uint32_t w[N * sizeof(T) / 4];
};
template <class T, int N>
__device__ __forceinline__ Raw<T, N> load_raw(const T* p) {
  constexpr int words = N * sizeof(T) / 4;
  Raw<T, N> r;
  if constexpr (words == 1) {
    r.w[0] = *(const uint32_t*)p;
  } else if constexpr (words == 2) {
    const u2 x = *(const u2*)p;
    r.w[0] = x[0], r.w[1] = x[1];
  } else {
    static_assert(words % 4 == 0, "");
#pragma unroll
    for (int i = 0; i < words; i += 4) {
      const u4 x = *(const u4*)((const uint32_t*)p + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) r.w[i + k] = x[k];
    }
  }
  return r;
}
__device__ __forceinline__ float value(const Raw<_Float16, 8>& r, int j) {
  return (float)__builtin_bit_cast(h2, r.w[j >> 1])[j & 1];
}
__device__ __forceinline__ float value(const Raw<float, 8>& r, int j) { return __uint_as_float(r.w[j]); }

__device__ __forceinline__ void store4(float* p, f4 x) { *(f4*)p = x; }
__device__ __forceinline__ void store4(_Float16* p, f4 x) {
  *(h4*)p = h4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
}

template <int ROWS>
__device__ __forceinline__ float max_row(float x) {  // over the lanes that hold one row
  if constexpr (ROWS == 16) x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}

// One kv head of one sequence's cache.
template <class KV>
struct Cache {
  const KV *k, *v;
  const int32_t* table;
  int64_t page_stride;
  int shift, mask, cap, n_pages;
  __device__ __forceinline__ int page(int key, int hi) const { return key < hi ? page_of(table, key, shift, cap, n_pages) : -1; }
};
template <class KV>
__device__ __forceinline__ Cache<KV> cache_of(const AttnArgs& r, int b, int kvh) {
  const mtg_paged_kv& c = r.a.kv;
  return {(const KV*)c.k + (int64_t)kvh * c.head_stride, (const KV*)c.v + (int64_t)kvh * c.head_stride,
          c.page_table + (int64_t)b * c.table_stride, c.page_stride, r.shift, c.page_size - 1, r.cap, c.n_pages};
}

// The rows of one tile: 16 per row tile, row lane % 16 of it in a lane.
struct Tile {
  Rows seq;
  int b, kvh;
  int first, count;  // rows of the sequence's (token, head) pairs
  Keys keys;         // of all its rows
  int gap;           // keys that no row sees between the sinks and the window (see axis_of)
  int min_hi, max_lo;  // keys that every row sees: max_lo .. min_hi - 1
  int oldest;          // the oldest key that some row sees, but for the sinks
};
template <bool SINK = false>
__device__ __forceinline__ bool tile_of(const AttnArgs& r, int tile, int kvh, int rows, Tile* t) {
  const mtg_paged_kv& c = r.a.kv;
  t->b = seq_of_rows(c, [&](int start, int i) { return first_tile(start, i, c.n_tokens, r.group, rows) <= tile; }, &t->seq);
  if (t->b < 0) return false;
  t->kvh = kvh;
  t->first = (tile - first_tile(t->seq.row0, t->b, c.n_tokens, r.group, rows)) * rows;
  t->count = t->seq.n * r.group - t->first;
  if (t->count <= 0) return false;
  if (t->count > rows) t->count = rows;
  const int head = t->first / r.group, tail = (t->first + t->count - 1) / r.group;
  t->keys = keys_of(t->seq, head, tail, r.a.window, r.cap);
  if constexpr (SINK) t->keys = axis_of(t->keys, r.sink, &t->gap);
  t->min_hi = cut(t->seq.pos0 + head + 1, 0, r.cap);
  t->max_lo = oldest_of(t->seq.pos0 + tail, r.a.window);
  t->oldest = oldest_of(t->seq.pos0 + head, r.a.window);
  return true;
}

// Row lane % 16 of a row tile: where it is and which keys it sees.
struct Row {
  int token, head;  // of the batch, of all heads
  int lo, hi;       // keys lo .. hi - 1
  bool real;
};
__device__ __forceinline__ Row row_of(const AttnArgs& r, const Tile& t, int i) {
  Row x;
  x.real = i < t.count;
  const int at = t.first + (x.real ? i : 0), tok = at / r.group;
  x.token = t.seq.row0 + tok;
  x.head = t.kvh * r.group + (at - tok * r.group);
  const int pos = t.seq.pos0 + tok;
  x.lo = oldest_of(pos, r.a.window);
  x.hi = !x.real || pos < 0 ? 0 : pos >= r.cap ? r.cap : pos + 1;
  return x;
}

// The row's elements place(c') + 8 g .. of all c', g of G / 8 lanes that share the row, as the score product's second
// operand; *factor turns a score into a power of two's exponent.
template <class F, int D, int G, class P>
__device__ __forceinline__ void load_row(const AttnArgs& r, const Row& x, typename F::MV (&q)[D / G][F::NQ], float* factor, const P& place) {
  const int g = (threadIdx.x & 63) / (512 / G);
  const typename F::IO* src = (const typename F::IO*)r.a.q + (int64_t)x.token * r.a.q_stride + x.head * D + 8 * g;
  float v[D / G][8];
  float top = 0.0f;
#pragma unroll
  for (int c = 0; c < D / G; ++c) {
    const Raw<typename F::IO, 8> w = load_raw<typename F::IO, 8>(src + place(c));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[c][j] = x.real ? value(w, j) : 0.0f;
      top = fmaxf(top, fabsf(v[c][j]));
    }
  }
  // a negative scale turns the row, so that larger products are larger scores; scale 0 is a row of zeros
  float s = r.log2_scale < 0.0f ? -1.0f : r.log2_scale == 0.0f ? 0.0f : 1.0f, back = 1.0f;
  if constexpr (F::NQ == 2) {  // to a maximum of 2^10 .. 2^11: a power of two, exact both ways
    const int e = (int)(__float_as_uint(max_row<512 / G>(top)) >> 23);
    if (e != 0 && e != 255) {
      const int se = cut(264 - e, 1, 250);
      s *= __uint_as_float((uint32_t)se << 23);
      back = __uint_as_float((uint32_t)(254 - se) << 23);
    }
  }
#pragma unroll
  for (int c = 0; c < D / G; ++c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[c][j] *= s;
    parts(v[c], q[c]);
  }
  // never 0: -inf marks what a row does not see
  *factor = fmaxf((r.log2_scale == 0.0f ? 1.0f : fabsf(r.log2_scale)) * back, 1.17549435e-38f);
}

template <class F, int D, int G>
__device__ __forceinline__ void load_row(const AttnArgs& r, const Row& x, typename F::MV (&q)[D / G][F::NQ], float* factor) {
  load_row<F, D, G>(r, x, q, factor, [](int c) { return G * c; });
}

// Where a lane of the two kernels has a key's weight, a row and an element of its sums: of a block of 32
// keys, group(key) of the lanes that hold the row has the weight of `key` as its weight(key)-th.
struct Direct {  // products of 16 rows, operands straight from memory
  static constexpr int kRows = 16, kWeights = 8;
  template <int D>
  static __device__ __forceinline__ int dim(int at, int g) { return (D / 16) * (4 * g + (at & 3)) + (at >> 2); }
  static __device__ __forceinline__ int group(int key) { return key >> 3; }
  static __device__ __forceinline__ int weight(int key) { return key & 7; }
};
struct Staged {  // products of 32 rows, operands from LDS
  static constexpr int kRows = 32, kWeights = 16;
  template <int D>
  static __device__ __forceinline__ int dim(int at, int g) { return 8 * (at >> 2) + 4 * g + (at & 3); }
  static __device__ __forceinline__ int group(int key) { return (key >> 2) & 1; }
  static __device__ __forceinline__ int weight(int key) { return 4 * (key >> 3) + (key & 3); }
};

// The running softmax of a row tile over one block of 32 keys: s (the lane's 8 products, -inf where
// the row does not see the key) becomes the 8 weights; the sums o and l are brought to the new
// maximum where that moves.
template <int DL>
__device__ __forceinline__ void weights(float* s, float factor, float lift, float* m, float* l, f4* o) {
  float top = s[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) top = fmaxf(top, s[j]);
  top *= factor;
  if (__any(top > *m + kSlack)) {  // from the first key on: m is -inf
    const float now = fmaxf(*m, max_row<16>(top));
    const float f = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(*m - now);
    *m = now;
    *l *= f;
#pragma unroll
    for (int t = 0; t < DL; ++t) o[t] *= f;
  }
  const float base = *m == -INFINITY ? 0.0f : lift - *m;
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = __builtin_amdgcn_exp2f(fmaf(s[j], factor, base));
  *l += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

// The order of the workgroups of a kv head: tile by tile. The chip seems to deal workgroups out to its engines in turn, so long and
// short (or empty) ones in a pattern that repeats, as a tile's last split is, would load them unevenly; the splits are
// therefore turned by another step in each tile (64 sequences of up to 5,000 keys 142 us, in plain order 168).
__device__ __forceinline__ void turn_of(const AttnArgs& r, int i, int* split, int* tile) {
  *tile = i / r.n_split;
  // the fractions of the multiples of the golden ratio, as even as steps can be
  const int at = i - *tile * r.n_split + (int)(((uint32_t)*tile * 0x9e3779b9u >> 16) * (uint32_t)r.n_split >> 16);
  *split = at < r.n_split ? at : at - r.n_split;
}

// ---- operands in LDS (k_paged_chunk and its like) ----
template <int D>
__device__ __forceinline__ int exchange(int row) {  // of 16-byte pieces of V's row in LDS
  return D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1);
}

template <class MV>
__device__ __forceinline__ MV read_piece(uint32_t lds) {
  return *(__attribute__((address_space(3))) const MV*)(uintptr_t)lds;
}

__device__ __forceinline__ h8 read_turned(uint32_t lds, int more) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s4 l4;
  const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((l4*)(uintptr_t)lds));
  const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((l4*)(uintptr_t)(lds + more)));
  return __builtin_bit_cast(h8, u4{a[0], a[1], b[0], b[1]});
}

// ---- splits of one tile's keys ----
//
// Each writes its sums to the workspace; a second launch joins them (k_paged_join). In a grid that the
// chip takes at once that launch is dear, so there (r.mark) each split also writes a mark, and whichever
// finds all marks set joins them. Stores and loads are then the device's (past the caches of an XCD); a
// mark is stored when its part is known to have arrived and looked for after that, so the last one finds
// all. Should two find all, both write the same bits. The marks are cleared then, so a replayed call
// finds none of its own; a mark is different in each call, and 64 bits long: what a fresh workspace holds
// is none. One row of 613 keys 9.0 us, with the second launch 10.8; 4 x 1,000 9.4 and 12.1; 8 x 1,600 14.0
// and 16.4 (f16 cache, 16 / 8 heads of 128). In larger grids the marks' round trips hold up workgroups that wait
// for a CU: 24 sequences of up to 8,000 keys 99 us, then 96 with the second launch (now 92).
__device__ __forceinline__ void put(float* p, float a, float b) {
  const uint64_t v = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
  __hip_atomic_store((uint64_t*)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void take(const float* p, float* a, float* b) {
  const uint64_t v = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  *a = __uint_as_float((uint32_t)v);
  *b = __uint_as_float((uint32_t)(v >> 32));
}

// All threads, after their part's stores: whether this workgroup joins the tile.
__device__ __forceinline__ bool all_arrived(const AttnArgs& r, int tile, int kvh, int split, int splits) {
  __shared__ int yes;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x < 64) {
    uint64_t* at = r.arrived + ((int64_t)tile * r.a.kv.n_kv_heads + kvh) * r.n_split;
    if (threadIdx.x == 0) __hip_atomic_store(at + split, r.mark, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    bool all = true;
    for (int s = threadIdx.x; s < splits; s += 64)
      all = all && __hip_atomic_load(at + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == r.mark;
    all = __all(all);
    if (all)
      for (int s = threadIdx.x; s < splits; s += 64) __hip_atomic_store(at + s, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (threadIdx.x == 0) yes = all;
  }
  __syncthreads();
  return yes;
}

// Elements d0 .. d0 + N - 1 of a row in T splits' parts; FAR: written by this launch.
template <int D, int N, bool FAR>
struct Parts {
  static constexpr int T = N == 8 ? 4 : 8;
  float m[T], l[T], o[T][N];
  // of splits s .. s + T - 1, the last one again for those beyond `end`
  __device__ __forceinline__ void load(const AttnArgs& r, int64_t at, int d0, int s, int end) {
    const int64_t all = (int64_t)r.a.kv.n_tokens * r.a.n_heads;
#pragma unroll
    for (int k = 0; k < T; ++k) {
      const int64_t slot = (s + k < end ? s + k : end - 1) * all + at;
      const float *ml = r.part_ml + 2 * slot, *po = r.part_o + slot * D + d0;
      if constexpr (FAR) {
        take(ml, &m[k], &l[k]);
#pragma unroll
        for (int d = 0; d < N; d += 2) take(po + d, &o[k][d], &o[k][d + 1]);
      } else {
        m[k] = ml[0], l[k] = ml[1];
#pragma unroll
        for (int d = 0; d < N; ++d) o[k][d] = po[d];
      }
    }
  }
};

// Some parts of a row, brought to the largest maximum.
template <int N>
struct Joined {
  float m = -INFINITY, l = 0.0f, o[N] = {};
  template <int T>
  __device__ __forceinline__ void add(int count, const float (&pm)[T], const float (&pl)[T], const float (&po)[T][N]) {
    float now = m;
#pragma unroll
    for (int k = 0; k < T; ++k)
      if (k < count) now = fmaxf(now, pm[k]);
    const float f = m == now ? 1.0f : __builtin_amdgcn_exp2f(m - now);  // both -inf: no key so far (or NaN alone)
    l *= f;
#pragma unroll
    for (int d = 0; d < N; ++d) o[d] *= f;
    m = now;
#pragma unroll
    for (int k = 0; k < T; ++k) {
      if (k >= count) break;
      const float w = pm[k] == now ? 1.0f : __builtin_amdgcn_exp2f(pm[k] - now);
      l = fmaf(pl[k], w, l);
#pragma unroll
      for (int d = 0; d < N; ++d) o[d] = fmaf(po[k][d], w, o[d]);
    }
  }
};

// Row `at` from its splits' parts, by `teams` teams of threads: team i takes parts i T .. i T + T - 1 (which p holds), then
// every teams T further on. The teams meet in LDS (sh: N + 2 floats for each of the block's n threads; `peer` threads lie
// between one team's thread and the next one's); all threads of the block come here with the same `teams`. One team
// reads many parts in a chain: one row, 130,000 keys 181 us, with 16 teams 104 (5.1 TB/s); 16,000 keys (8 teams) 21.5, 19.0.
template <typename IO, int D, int N, bool FAR>
__device__ __forceinline__ void join_row(const AttnArgs& r, bool row, int64_t at, IO* out, int d0, int splits, int team, int teams, int peer,
                                         int n, float* sh, Parts<D, N, FAR>& p) {
  constexpr int T = Parts<D, N, FAR>::T;
  Joined<N> j;
  if (row)
    for (int s = team * T; s < splits; s += teams * T) {
      if (s != team * T) p.load(r, at, d0, s, splits);
      j.add(splits - s, p.m, p.l, p.o);
    }
  if (teams > 1) {
    const int me = threadIdx.x;
    sh[me] = j.m;
    sh[n + me] = j.l;
#pragma unroll
    for (int d = 0; d < N; ++d) sh[(2 + d) * n + me] = j.o[d];
    __syncthreads();
    if (team) return;
    for (int i = 1; i < teams; ++i) {
      const int from = me + i * peer;
      float m[1] = {sh[from]}, l[1] = {sh[n + from]}, o[1][N];
#pragma unroll
      for (int d = 0; d < N; ++d) o[0][d] = sh[(2 + d) * n + from];
      j.add(1, m, l, o);
    }
  }
  if (!row) return;
  const float inv = j.l == 0.0f ? 0.0f : 1.0f / j.l;
#pragma unroll
  for (int d = 0; d < N; ++d) out[d0 + d] = (IO)(j.o[d] * inv);
}

// ---- the end of a workgroup of NW waves that took the keys of RT row tiles of 16 in turns ----
//
// o[i][d]: row lane % 16 of tile i, elements (D / 16) (4 (lane / 16) + k) + d; m, l: its maximum and the lane's part of the sum.
constexpr int kPadOf(int D) { return D + 4; }
template <class F, int D, int RT, int NW>
__device__ __forceinline__ void finish_rows(const AttnArgs& r, const Tile& t, int tile, int split, int splits, float (&m)[RT], float (&l)[RT],
                                            f4 (&o)[RT][D / 16], float (&sh_o)[NW][16][kPadOf(D)], float (&sh_ml)[NW][16 * RT][2]) {
  constexpr int DL = D / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, kvh = t.kvh;
  // the waves' sums, brought to one maximum, meet in LDS
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    l[i] += __shfl_xor(l[i], 16);
    l[i] += __shfl_xor(l[i], 32);
    if (g == 0) {
      sh_ml[wave][16 * i + col][0] = m[i];
      sh_ml[wave][16 * i + col][1] = l[i];
    }
  }
  __syncthreads();
  const int64_t all = (int64_t)r.a.kv.n_tokens * r.a.n_heads;
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, sh_ml[w][16 * i + col][0]);
    const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[i] - top);
    if (i) __syncthreads();
    if (16 * i + col < t.count) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int d = 0; d < DL; ++d) sh_o[wave][col][DL * (4 * g + k) + d] = o[i][d][k] * f;
    }
    __syncthreads();
    constexpr int per = 16 * D / (64 * NW);  // elements of a row a thread writes
    const int orow = threadIdx.x / (D / per), at = threadIdx.x % (D / per) * per;
    if (16 * i + orow < t.count) {
      top = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) top = fmaxf(top, sh_ml[w][16 * i + orow][0]);
#pragma unroll
      for (int w = 0; w < NW; ++w)
        sum += top == -INFINITY ? 0.0f : sh_ml[w][16 * i + orow][1] * __builtin_amdgcn_exp2f(sh_ml[w][16 * i + orow][0] - top);
      float x[per];
#pragma unroll
      for (int d = 0; d < per; ++d) {
        x[d] = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w += 4)
          x[d] += (sh_o[w][orow][at + d] + sh_o[w + 1][orow][at + d]) + (sh_o[w + 2][orow][at + d] + sh_o[w + 3][orow][at + d]);
      }
      const int pair = t.first + 16 * i + orow, tok = pair / r.group;
      const int token = t.seq.row0 + tok, head = kvh * r.group + (pair - tok * r.group);
      if (splits == 1) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        typename F::IO* out = (typename F::IO*)r.a.out + (int64_t)token * r.a.out_stride + head * D + at;
#pragma unroll
        for (int d = 0; d < per; ++d) out[d] = (typename F::IO)(x[d] * inv);
      } else {
        const int64_t slot = (int64_t)split * all + (int64_t)token * r.a.n_heads + head;
        if (r.mark) {
#pragma unroll
          for (int d = 0; d < per; d += 2) put(r.part_o + slot * D + at + d, x[d], x[d + 1]);
          if (at == 0) put(r.part_ml + 2 * slot, top, sum);
        } else {
#pragma unroll
          for (int d = 0; d < per; ++d) r.part_o[slot * D + at + d] = x[d];
          if (at == 0) {
            r.part_ml[2 * slot] = top;
            r.part_ml[2 * slot + 1] = sum;
          }
        }
      }
    }
  }
  if (splits > 1 && r.mark && all_arrived(r, tile, kvh, split, splits)) {
    constexpr int kLanes = D / 8, kTeams = 64 * NW / kLanes;
    static_assert(sizeof sh_o >= (8 + 2) * 64 * NW * 4, "LDS of join_row");
    const int who = threadIdx.x / kLanes, d0 = (int)threadIdx.x % kLanes * 8;
    auto join = [&](bool row, int i, int team, int teams) {
      const Row x = row_of(r, t, i);
      const int64_t at = (int64_t)x.token * r.a.n_heads + x.head;
      Parts<D, 8, true> p;
      p.load(r, at, d0, p.T * team, splits);
      join_row(r, row, at, (typename F::IO*)r.a.out + (int64_t)x.token * r.a.out_stride + x.head * D, d0, splits, team, teams,
               64 * NW / teams, 64 * NW, &sh_o[0][0][0], p);
    };
    // with many splits several teams to a row, if there are so few rows
    int log = 0;
    if (splits > 8)
      while ((t.count << (log + 1)) <= kTeams && (4 << log) < splits) ++log;
    if (log) {
      const int rows = kTeams >> log, i = who & (rows - 1);
      join(i < t.count, i < t.count ? i : 0, who / rows, 1 << log);
    } else {
      for (int i = who; i < t.count; i += kTeams) join(true, i, 0, 1);
    }
  }
}

// The joins as a launch of their own: four rows to a workgroup, a wave each, or a row to a workgroup of TEAMS waves.
template <typename IO, int D, int TEAMS, bool SINK>
__device__ __forceinline__ void join_of(const AttnArgs& r, int tile_rows) {
  __shared__ float sh[TEAMS > 1 ? (2 + D / 64) * 64 * TEAMS : 1];
  const mtg_paged_kv& c = r.a.kv;
  const int wave = threadIdx.x >> 6, team = TEAMS > 1 ? wave : 0;
  const int64_t all = (int64_t)c.n_tokens * r.a.n_heads, at = TEAMS > 1 ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  if (at >= all) return;
  const int token = (int)(at / r.a.n_heads), head = (int)(at % r.a.n_heads), d0 = (threadIdx.x & 63) * (D / 64);
  // read before it is known how many there are: what is not one is memory of the workspace all the same
  Parts<D, D / 64, false> p;
  p.load(r, at, d0, team * p.T, r.n_split);
  Rows seq;
  if (seq_of_rows(c, [&](int start, int) { return start <= token; }, &seq) < 0) return;
  if (token >= seq.row0 + seq.n) return;
  const int pair = (token - seq.row0) * r.group + head % r.group;
  const int first = pair / tile_rows * tile_rows, last = min(first + tile_rows, seq.n * r.group) - 1;
  Keys keys = keys_of(seq, first / r.group, last / r.group, r.a.window, r.cap);
  int gap;
  if constexpr (SINK) keys = axis_of(keys, r.sink, &gap);
  const int splits = splits_of(keys, r.split_keys, r.n_split);
  if (splits > 1)  // else its only split wrote it
    join_row(r, true, at, (IO*)r.a.out + (int64_t)token * r.a.out_stride + head * D, d0, splits, team, TEAMS, 64, 64 * TEAMS, sh, p);
}
template <typename IO, int D, int TEAMS>
__global__ void __launch_bounds__(TEAMS > 4 ? 64 * TEAMS : 256) k_paged_join(AttnArgs r, int tile_rows) {
  join_of<IO, D, TEAMS, false>(r, tile_rows);
}
template <typename IO, int D, int TEAMS>  // with first positions beside a window
__global__ void __launch_bounds__(TEAMS > 4 ? 64 * TEAMS : 256) k_paged_join_sink(AttnArgs r, int tile_rows) {
  join_of<IO, D, TEAMS, true>(r, tile_rows);
}

// ---- host ----
struct Plan {
  bool staged;      // k_paged_chunk
  bool eight;       // k_paged_rows of eight waves
  bool wide;        // k_paged_chunk_f8 of eight waves
  bool one_launch;  // the splits' join included
  bool apart;       // k_paged_rows_f8: no more than two workgroups a CU
  int tile_rows;
  int64_t tiles;
  int n_split, split_keys;
  size_t bytes, ml_at, arrived_at;
};

inline Plan plan_of(const mtg_paged_attn& a, int sink = 0) {
  const mtg_paged_kv& kv = a.kv;
  const int group = a.n_heads / kv.n_kv_heads;
  Plan p{};
  const int64_t per_seq = ((int64_t)kv.n_tokens * group + kv.n_seqs - 1) / kv.n_seqs;
  const bool codes = kv.kv_type == MTG_TYPE_F8_E4M3;
  p.staged = kv.kv_type != MTG_TYPE_F32 && per_seq > 64;
  // Codes: eight waves where a sequence fills some tiles of 256 rows (f16, 16 heads over 8: 1 x 512 rows 50.0 us with four waves, 48.5
  // with eight, 1 x 1,009 f32 163 and 155, 2 x 2,048 of 32 heads 1,046 and 963; but 4 x 300 rows 60 and 66, 32 x 60 38 and 55).
  p.wide = p.staged && codes && per_seq >= 1024;
  p.tile_rows = p.wide ? 2 * kChunkRows : p.staged ? kChunkRows : per_seq <= 16 ? 16 : 32;
  p.tiles = tiles_bound(kv.n_tokens, kv.n_seqs, group, p.tile_rows);
  const int64_t cap = (int64_t)kv.table_stride * kv.page_size;
  int64_t keys = a.max_kv > 0 && a.max_kv < cap ? a.max_kv : cap;
  if (a.window > 0) keys = std::min<int64_t>(keys, (int64_t)a.window + p.tile_rows + 32 + (sink + 31) / 32 * 32);
  // the workgroups of one split each, as if all sequences had the same number of rows
  const int64_t work = kv.n_seqs * ((per_seq + p.tile_rows - 1) / p.tile_rows) * kv.n_kv_heads;
  int64_t per;
  auto grid = [&](int64_t per) { return work * ((keys + per - 1) / per); };
  if (p.staged) {
    // Two workgroups a CU have work, if that leaves each 512 keys or more, else one, of 256 or more, for the parts cost more
    // to write and join than the second brings (60 rows each, group 2: 32 sequences of 500 keys 39.9 us unsplit, 61 in two
    // parts; two of 8,000: 29.2 in parts of 512, 32.5 of 256; but one tile of rows over 1,600: 21 of 256, 31 of 512).
    const int64_t want = std::max<int64_t>(1, (p.wide ? 256 : 512) / work);
    per = (keys + want - 1) / want;
    if (per < 512) per = std::max<int64_t>(256, (keys * work + 255) / 256);
  } else {
    // 512 keys, or so that there are 2,048 workgroups, whichever is more: one row each of 24 sequences of up to 8,000 keys
    // 94.5 us with 896 keys, 99.5 with 512, 124 with 1,664. In small grids fewer, down to 128, up to 128 workgroups (one
    // row, 1,600 keys: 128 keys 10.3 us, 512 12.5; 8,000 keys: 256 17.2, 512 15.9).
    per = 512;
    // (Of codes, half the bytes, up to 256: 8,000 keys 14.6 and 13.7 us, with heads of 64 11.1 and 10.2.)
    for (int64_t x : {256, 128})
      if (grid(x) <= (codes ? 256 : 128)) per = x;
    if (grid(512) > 2048) per = std::max<int64_t>(512, (keys * work + 2047) / 2048);
    // Even splits of 512 or more, and none of fewer than 1,024 where there is a workgroup a CU without (one row, f16: 64
    // sequences of up to 512 keys 17.1 us, with a second split of one key 28.8; of up to 800 28.9 and 40.7; f32, 40 of up
    // to 1,600: 83.5 in three, 104 in four).
    if (per >= 512) {
      const int64_t n = keys < 2 * per && work >= 256 ? 1 : std::max<int64_t>(1, (keys + per / 2) / per);
      per = std::max<int64_t>(128, (keys + n - 1) / n);
    }
    // Codes: no third workgroup on half of the CUs or fewer, if there is a number of splits that makes two on nearly all of them
    // (8 x 8 rows, group 2, 5,000 keys: ten splits 25.0 us, eight 22.4; heads of 64 19.1 and 17.4; 16 x 8 rows, 3,000
    // keys, six splits, three workgroups a CU, 24.7, four splits 25.1).
    if (codes && p.tile_rows == 16 && grid(per) > 512 && grid(per) <= 640 && 512 / work * work >= 448) per = (keys * work + 511) / 512;
    // Half as many workgroups as the chip takes: of eight waves, without splits, up to some 1,000 keys (one row each: 32
    // sequences of up to 1,000 keys 17.6 us, with four waves 23.6, of 2,000 37.5 and 40.6; 16 of 1,000 16.6 and 18.7, of
    // 1,500 22.0 and 18.8; f32, 32 x 2 rows, 1,000 keys 45.6 and 58.8; 24 x 4, 1,500 keys 60.5 and 52.8).
    if (p.tile_rows == 16 && work >= 128 && work <= 256 && keys > 256 && keys <= 512 + 4 * work) p.eight = true, per = keys;
    // (with few rows to join also for 512 workgroups: one row each of 16 sequences of 2,000 keys 19.9 us, else 21.5)
    // (Of codes with up to 8 rows to a head for 1,024: one row each of 32 sequences of 2,000 keys 21.8, else 22.9; 64 in a window
    // of 2,048, heads of 64, 8 to a kv head: 23.0 and 24.4; but 8 x 8 rows, group 2, 5,000 keys 28.4 and 25.0.)
    const bool few = per_seq <= (codes ? 8 : 4) && keys <= 32 * per;
    p.one_launch = grid(per) <= (few ? codes ? 1024 : 512 : 256);
    p.apart = grid(per) <= 512;
  }
  per = std::min(per, std::max<int64_t>(keys, 128));  // a share of what there is
  const int64_t step = p.staged ? 64 : 128;
  p.split_keys = (int)((per + step - 1) / step * step);
  p.n_split = (int)((keys + p.split_keys - 1) / p.split_keys);
  if (p.n_split < 1) p.n_split = 1;
  if (p.n_split > 1) {
    const size_t rows = (size_t)p.n_split * kv.n_tokens * a.n_heads;
    p.ml_at = rows * kv.head_dim * 4;
    p.arrived_at = p.ml_at + rows * 8;
    p.bytes = (p.arrived_at + (size_t)p.tiles * kv.n_kv_heads * p.n_split * 8 + 15) / 16 * 16;
  }
  return p;
}

inline float log2_scale(const mtg_paged_attn& a) { return a.scale * 1.44269504088896340736f; }

// Everything but the workspace; *rc MTG_OK where the call may run (or has nothing to do).
inline const char* refused(const mtg_paged_attn& a, bool f8, int* rc) {
  const mtg_paged_kv& kv = a.kv;
  if (const char* why = check(kv, true, rc, f8)) return why;
  *rc = MTG_ERR_UNSUPPORTED;
  if (f8 && a.io_type != MTG_TYPE_F32 && a.io_type != MTG_TYPE_F16) return "types: rows are f32 or f16";
  if (!f8 && !(a.io_type == MTG_TYPE_F32 || (a.io_type == MTG_TYPE_F16 && kv.kv_type == MTG_TYPE_F16)))
    return "types: f32 rows with an f32 or f16 cache, f16 rows with an f16 cache";
  *rc = MTG_ERR_INVALID;
  if (a.n_heads <= 0 || a.n_heads > 1024 || a.n_heads % kv.n_kv_heads) return "n_heads";
  if (a.max_kv < 0 || a.window < 0) return "max_kv or window";
  if (!std::isfinite(log2_scale(a))) return "scale";  // as the kernels take it
  if ((int64_t)kv.n_tokens * a.n_heads >= ((int64_t)1 << 30)) {
    *rc = MTG_ERR_UNSUPPORTED;
    return "2^30 or more rows of heads";
  }
  *rc = MTG_OK;
  return nullptr;
}

// The arrays of a call that refused() lets pass. scales (of a cache in 8 bits) may be NULL.
inline const char* refused_arrays(const mtg_paged_attn& a, const Plan& plan, int* rc, const mtg_f8_scales* scales = nullptr) {
  const mtg_paged_kv& kv = a.kv;
  auto no = [&](int status, const char* why) {
    *rc = status;
    return why;
  };
  if (!a.q || !a.out) return no(MTG_ERR_INVALID, "q or out is NULL");
  const size_t eb = type_bytes(a.io_type);
  const int64_t unit = 16 / (int64_t)eb, width = (int64_t)a.n_heads * kv.head_dim;
  const int64_t most = (int64_t)1 << 40;
  if (a.q_stride < width || a.out_stride < width || a.q_stride > most || a.out_stride > most ||
      !reaches(kv.n_tokens, a.q_stride) || !reaches(kv.n_tokens, a.out_stride))
    return no(MTG_ERR_INVALID, "a row stride below the row's width, or rows behind 2^46 elements");
  if (!aligned(a.q, 16) || !aligned(a.out, 16) || a.q_stride % unit || a.out_stride % unit)
    return no(MTG_ERR_UNSUPPORTED, "rows not aligned to 16 bytes");
  const size_t qn = extent(kv.n_tokens, a.q_stride, width, eb), on = extent(kv.n_tokens, a.out_stride, width, eb);
  if (overlap(a.q, qn, a.out, on) && !(a.q == a.out && a.q_stride == a.out_stride))
    return no(MTG_ERR_INVALID, "out overlaps q");
  const size_t pool = pool_extent(kv);
  if (overlap(kv.k, pool, a.out, on) || overlap(kv.v, pool, a.out, on)) return no(MTG_ERR_INVALID, "out lies in the pages");
  auto index = [&](const void* p, size_t n) {
    return meets(p, n, {{kv.page_table, 4 * (size_t)kv.n_seqs * kv.table_stride}, {kv.kv_len, 4 * (size_t)kv.n_seqs},
                        {kv.q_start, 4 * (size_t)kv.n_seqs + 4}});
  };
  if (index(a.out, on)) return no(MTG_ERR_INVALID, "out overlaps an index array");
  if (plan.tiles * kv.n_kv_heads * plan.n_split >= ((int64_t)1 << 24))
    return no(MTG_ERR_UNSUPPORTED, "more than 2^24 workgroups");
  if (plan.bytes) {
    if (!a.workspace || !aligned(a.workspace, 16)) return no(MTG_ERR_INVALID, "workspace NULL or unaligned");
    if (a.workspace_bytes < plan.bytes) return no(MTG_ERR_CAPACITY, "workspace smaller than mtg_paged_attn_workspace");
    if (meets(a.workspace, plan.bytes, {{a.out, on}, {a.q, qn}, {kv.k, pool}, {kv.v, pool}}) || index(a.workspace, plan.bytes))
      return no(MTG_ERR_INVALID, "workspace overlaps q, out, the pages or an index array");
  }
  if (scales) {
    if (const char* why = check_scales(kv, *scales, false)) return no(MTG_ERR_INVALID, why);
    const size_t n = scale_extent(kv, *scales);
    for (const uint8_t* x : {scales->k, scales->v})
      if (meets(x, n, {{a.out, on}, {a.workspace, plan.bytes}})) return no(MTG_ERR_INVALID, "scales overlap out or workspace");
  }
  return nullptr;
}

inline AttnArgs args_of(const mtg_paged_attn& a, const Plan& plan) {
  const mtg_paged_kv& kv = a.kv;
  AttnArgs r{};
  r.a = a;
  r.shift = log2_of(kv.page_size);
  r.cap = capacity(kv.table_stride, r.shift);
  r.group = a.n_heads / kv.n_kv_heads;
  r.split_keys = plan.split_keys;
  r.n_split = plan.n_split;
  r.tiles = (int)plan.tiles;
  r.part_o = (float*)a.workspace;
  r.part_ml = (float*)((char*)a.workspace + plan.ml_at);
  r.arrived = (uint64_t*)((char*)a.workspace + plan.arrived_at);
  r.mark = plan.bytes && plan.one_launch ? next_mark() : 0;
  r.log2_scale = log2_scale(a);
  return r;
}

template <typename IO, int D, bool SINK = false>
hipError_t run_join(const AttnArgs& r, const Plan& p, hipStream_t s) {
  const int64_t rows = (int64_t)r.a.kv.n_tokens * r.a.n_heads;
  auto join = [&](auto teams, int64_t grid) {
    constexpr int T = decltype(teams)::value;
    if constexpr (SINK) return launch(k_paged_join_sink<IO, D, T>, dim3((unsigned)grid), dim3(T > 4 ? 64 * T : 256), 0, s, r, p.tile_rows);
    else return launch(k_paged_join<IO, D, T>, dim3((unsigned)grid), dim3(T > 4 ? 64 * T : 256), 0, s, r, p.tile_rows);
  };
  return p.n_split <= 8    ? join(std::integral_constant<int, 1>{}, (rows + 3) / 4)
         : p.n_split <= 32 ? join(std::integral_constant<int, 4>{}, rows)
                           : join(std::integral_constant<int, 16>{}, rows);
}

}  // namespace attn
}  // namespace mtg
