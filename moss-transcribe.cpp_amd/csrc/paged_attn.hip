// paged_attn.hip - mtg_paged_attn_dev: causal attention of the new rows of a batch over a cache
// in pages (reference for one sequence over a contiguous cache: src/qwen3.cpp:150-186).
//
// Rows here are (token, head of the kv head's group) pairs, so that all query heads of a kv
// head share the reads of its keys. Scores and weighted sums run on matrix instructions of 16
// rows: the score product takes 16 keys x 32 elements as its first operand and the rows as its
// second, so a lane ends up with the scores of ONE row (lane % 16) and of 8 keys, which are,
// with the keys of two products laid out 8 (m / 4) + 4 tile + m % 4, neighbouring keys
// 8 (lane / 16) ..+7: exactly what the second product needs from that lane as its operand.
// The weights never leave their lane; the running maximum and sum are one register each.
// The second product's first operand is V with keys along k; product t holds dimensions
// (D / 16) m + t, so a lane's part of all of them is D / 16 neighbouring elements of 8 keys.
//
// The maximum that the weights refer to is moved only when a score exceeds it by 2^8
// (one comparison per score and a ballot; the exponential has room, f16 weights are kept at
// 2^15 or less, the largest at 2^7 or more, by a constant factor that the division takes out again).
//
// Formats. f16 rows and cache: one f16 product for the scores, two for the weights in two f16 parts (in
// one where the products bind, k_paged_chunk: 11 bits). f32 rows, f16 cache: the row is scaled to a
// maximum of 2^10..11 and split into two f16 parts, and so are the weights: two products each. Two parts
// keep 22 bits, or what f16's smallest step of 2^-24 leaves of small values: an element of a row 2^-35 of the row's
// largest, a weight 2^-32 of the largest. f32 cache, 16 rows or fewer: products of f32 (33 cycles for 4 elements, no splitting: with
// three bf16 parts 57 us for 8 sequences of 8 rows and up to 4,000 keys, with these 52). f32 cache, more rows: values split exactly into three bf16
// parts of 8 bits, the six products above 2^-24 (6 x 18 cycles for 32 elements against 8 x 33) are taken.
// The sums are f32 throughout.
#include "kernels.hpp"
#include "paged_dev.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

namespace mtg {
namespace {

using namespace paged;

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

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
};

constexpr int kChunkRows = 128, kTileKeys = 64;  // of a workgroup of k_paged_chunk, and of its steps
constexpr float kSlack = 8.0f;  // a score above the maximum by more than 2^8 moves it

struct F16 {  // rows and cache f16 (two parts of the weights are free in k_paged_rows: 24 rows of up to 8,000 keys 92.4 us, with one 92.1)
  using IO = _Float16;
  using KV = _Float16;
  using MV = h8;
  static constexpr int NA = 1, NQ = 1, NW = 2;  // parts of a cached value, of a row's, of a weight
  static constexpr float kLift = 7.0f;          // log2 of the weights' constant factor
};
struct F32F16 {  // rows f32, cache f16
  using IO = float;
  using KV = _Float16;
  using MV = h8;
  static constexpr int NA = 1, NQ = 2, NW = 2;
  static constexpr float kLift = 7.0f;
};
struct F8 {
  float x[8];
};
struct F32Few {  // rows and cache f32, 16 rows or fewer: products of f32, 4 elements each
  using IO = float;
  using KV = float;
  using MV = F8;
  static constexpr int NA = 1, NQ = 1, NW = 1;
  static constexpr float kLift = 0.0f;
};
struct F32 {  // rows and cache f32, more rows
  using IO = float;
  using KV = float;
  using MV = b8;
  static constexpr int NA = 3, NQ = 3, NW = 3;
  static constexpr float kLift = 0.0f;
};

__device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mma(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// A lane's elements (or keys) 8 g .. 8 g + 7, one of each group g to a product.
__device__ __forceinline__ f4 mma(const F8& a, const F8& b, f4 c) {
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

__device__ __forceinline__ void parts(const float* x, F8 (&p)[1]) {
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
  if constexpr (words == 2) {
    const u2 x = *(const u2*)p;
    r.w[0] = x[0], r.w[1] = x[1];
  } else {
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

// The first operands: 8 neighbouring elements of a key, or element d of 8 keys.
__device__ __forceinline__ void operand(const Raw<_Float16, 8>& r, h8 (&p)[1]) {
  p[0] = __builtin_bit_cast(h8, u4{r.w[0], r.w[1], r.w[2], r.w[3]});
}
__device__ __forceinline__ void operand(const Raw<float, 8>& r, b8 (&p)[3]) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(r.w[j]);
  parts(x, p);
}
template <int N>
__device__ __forceinline__ void operand(const Raw<_Float16, N> (&r)[8], int d, h8 (&p)[1]) {
  u4 w;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    w[j] = __builtin_amdgcn_perm(r[2 * j + 1].w[d >> 1], r[2 * j].w[d >> 1], d & 1 ? 0x07060302u : 0x05040100u);
  p[0] = __builtin_bit_cast(h8, w);
}
__device__ __forceinline__ void operand(const Raw<float, 8>& r, F8 (&p)[1]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) p[0].x[j] = __uint_as_float(r.w[j]);
}
template <int N>
__device__ __forceinline__ void operand(const Raw<float, N> (&r)[8], int d, F8 (&p)[1]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) p[0].x[j] = __uint_as_float(r[j].w[d]);
}
template <int N>
__device__ __forceinline__ void operand(const Raw<float, N> (&r)[8], int d, b8 (&p)[3]) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(r[j].w[d]);
  parts(x, p);
}

// Words with infinities or NaN, in integers (a compare would hold a lane mask per element): the
// exponent's bits plus one carry into the sign's place.
template <class T>
__device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
  return sizeof(T) == 4 ? ((w & 0x7f800000u) + 0x00800000u) & 0x80000000u : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}
template <class T>
__device__ __forceinline__ uint32_t without_odd(uint32_t w) {
  const uint32_t b = odd_bits<T>(w);
  return sizeof(T) == 4 ? w & ~(uint32_t)((int32_t)b >> 31) : w & ~((b >> 15) * 0xffffu);
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ bool finite(_Float16 x) {
  return (__builtin_bit_cast(uint16_t, x) & 0x7c00u) != 0x7c00u;
}

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
  int min_hi, max_lo;  // keys that every row sees: max_lo .. min_hi - 1
};
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
  t->min_hi = cut(t->seq.pos0 + head + 1, 0, r.cap);
  t->max_lo = oldest_of(t->seq.pos0 + tail, r.a.window);
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

// The row's elements G c' + 8 g .. of all c', as the score product's second operand (G / 8 lanes share
// the row); *factor turns a score into a power of two's exponent.
template <class F, int D, int G>
__device__ __forceinline__ void load_row(const AttnArgs& r, const Row& x, typename F::MV (&q)[D / G][F::NQ], float* factor) {
  const int g = (threadIdx.x & 63) / (512 / G);
  const typename F::IO* src = (const typename F::IO*)r.a.q + (int64_t)x.token * r.a.q_stride + x.head * D + 8 * g;
  float v[D / G][8];
  float top = 0.0f;
#pragma unroll
  for (int c = 0; c < D / G; ++c) {
    const Raw<typename F::IO, 8> w = load_raw<typename F::IO, 8>(src + G * c);
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

// What non-finite elements of V add to the rows that see them: the product took them as zero,
// since in a block that some rows do not see whole, 0 * NaN would reach those rows. o: the lane's sums.
template <class F, int D, class L>
__device__ __forceinline__ void add_non_finite(const Cache<typename F::KV>& c, const float* p, int kb, int hi, int row_lo,
                                               int row_hi, float* o) {
  const int lane = threadIdx.x & 63, row = lane % L::kRows, g = lane / L::kRows;
  for (int k = 0; k < 32; ++k) {
    float w = 0.0f;
#pragma unroll
    for (int j = 0; j < L::kWeights; ++j)
      if (L::weight(k) == j) w = p[j];
    w = __shfl(w, L::group(k) * L::kRows + row);
    const int key = kb + k, page = c.page(key, hi);
    if (page < 0 || key < row_lo || key >= row_hi) continue;
    const typename F::KV* v = c.v + page * c.page_stride + (int64_t)(key & c.mask) * D;
#pragma unroll
    for (int at = 0; at < D * L::kRows / 64; at += 4) {
      typename F::KV x[4];
      bool all = true;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = v[L::template dim<D>(at + i, g)];
        all &= finite(x[i]);
      }
      if (all) continue;  // four at a time, so that few are held at once
#pragma unroll
      for (int i = 0; i < 4; ++i) o[at + i] += finite(x[i]) ? 0.0f : w * (float)x[i];
    }
  }
}

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

// ---- few rows: 16 or 32 rows of one kv head, four waves (eight without splits) each with its own blocks of 32 keys ----
//
// HBM bounds it, and for short contexts the chain of dependent reads (sequence, page, keys). K and V go
// from memory straight into the operands' registers (no LDS, no barrier until the end): a lane reads 16
// bytes of a key for the score product and D / 16 elements of 8 keys for the second one. The loads of the
// next block's K are issued when the products with K are done, those of its V when the sums are; with two
// sets of registers and all of them issued a block ahead no faster (96.7 against 94.5 us for 24 sequences
// of up to 8,000 keys), with 8 waves slower (104).
template <class F, int D, int RT, int WAVES, int NW = 4>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(WAVES, WAVES))) k_paged_rows(AttnArgs r) {
  using KV = typename F::KV;
  using MV = typename F::MV;
  constexpr int NC = D / 32, DL = D / 16, kRows = 16 * RT, kPad = D + 4, kWords = DL * sizeof(KV) / 4, kStep = 32 * NW;
  __shared__ float sh_o[NW][16][kPad];
  __shared__ float sh_ml[NW][kRows][2];
  const int kvh = blockIdx.x % r.a.kv.n_kv_heads, rest = blockIdx.x / r.a.kv.n_kv_heads;
  int split, tile;
  turn_of(r, rest, &split, &tile);
  Tile t;
  if (!tile_of(r, tile, kvh, kRows, &t)) return;
  const int splits = NW == 4 ? splits_of(t.keys, r.split_keys, r.n_split) : 1;
  if (split >= splits) return;
  const Keys mine = split_keys_of(t.keys, split, r.split_keys, splits);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const Cache<KV> c = cache_of<KV>(r, t.b, kvh);
  // this lane's key of score product `tile`: 8 (col / 4) + 4 tile + col % 4; its V keys: 8 g + j
  const int kgroup = 8 * (col >> 2), krow = kgroup + (col & 3);
  Raw<KV, 8> kr[2][NC];
  Raw<KV, DL> vr[8];
  int kpage = -1, vpage = -1;  // of the block that is loaded next
  int at_page = -1;            // of the V that is held
  auto pages = [&](int kb) {
    kpage = c.page(kb + kgroup, mine.hi);
    vpage = c.page(kb + 8 * g, mine.hi);
  };
  auto load_k = [&](int kb) {
    const KV* k = c.k + (kpage < 0 ? 0 : kpage * c.page_stride + (int64_t)((kb + krow) & c.mask) * D) + 8 * g;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int i = 0; i < NC; ++i) kr[a][i] = load_raw<KV, 8>(k + a * 4 * D + 32 * i);
  };
  auto load_v = [&](int kb) {
    const KV* v = c.v + (vpage < 0 ? 0 : vpage * c.page_stride + (int64_t)((kb + 8 * g) & c.mask) * D) + DL * col;
#pragma unroll
    for (int j = 0; j < 8; ++j) vr[j] = load_raw<KV, DL>(v + j * D);
    at_page = vpage;
  };
  int kb = mine.lo + 32 * wave;
  if (kb < mine.hi) {
    pages(kb);
    load_k(kb);
    load_v(kb);
    pages(kb + kStep);
  }
  Row row[RT];
  MV q[RT][NC][F::NQ];
  float factor[RT], m[RT], l[RT];
  f4 o[RT][DL];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    row[i] = row_of(r, t, 16 * i + col);
    load_row<F, D, 32>(r, row[i], q[i], &factor[i]);
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int d = 0; d < DL; ++d) o[i][d] = f4{0, 0, 0, 0};
  }

  for (; kb < mine.hi; kb += kStep) {
    const bool more = kb + kStep < mine.hi;
    float s[RT][8];
    {
      f4 acc[RT][2];
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[i][0] = acc[i][1] = f4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          MV p[F::NA];
          operand(kr[a][k], p);
#pragma unroll
          for (int i = 0; i < RT; ++i) acc[i][a] = product(p, q[i][k], acc[i][a]);
        }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] = acc[i][j >> 2][j & 3];
    }
    if (more) load_k(kb + kStep);
    bool bad = false;
    if (!(kb >= t.max_lo && kb + 32 <= t.min_hi && kb + 32 <= mine.hi && __all(at_page >= 0))) {
      asm volatile("");  // a branch
      uint32_t odd = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = kb + 8 * g + j;
        const bool there = at_page >= 0 && key < mine.hi;
#pragma unroll
        for (int i = 0; i < RT; ++i)
          if (!there || key < row[i].lo || key >= row[i].hi) s[i][j] = -INFINITY;
        const uint32_t keep = there ? ~0u : 0u;
#pragma unroll
        for (int d = 0; d < kWords; ++d) {
          vr[j].w[d] &= keep;
          odd |= odd_bits<KV>(vr[j].w[d]);
        }
      }
      bad = __any(odd != 0);
      if (bad) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int d = 0; d < kWords; ++d) {
            asm volatile("" : "+v"(vr[j].w[d]));  // the bits above are not kept in registers for this
            vr[j].w[d] = without_odd<KV>(vr[j].w[d]);
          }
      }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) weights<DL>(s[i], factor[i], F::kLift, &m[i], &l[i], o[i]);
    MV w[RT][F::NW];
#pragma unroll
    for (int i = 0; i < RT; ++i) parts(s[i], w[i]);
#pragma unroll
    for (int d = 0; d < DL; ++d) {
      MV p[F::NA];
      operand(vr, d, p);
#pragma unroll
      for (int i = 0; i < RT; ++i) o[i][d] = product(p, w[i], o[i][d]);
    }
    if (bad) {
      asm volatile("");
#pragma unroll
      for (int i = 0; i < RT; ++i) add_non_finite<F, D, Direct>(c, s[i], kb, mine.hi, row[i].lo, row[i].hi, (float*)o[i]);
    }
    if (more) {
      load_v(kb + kStep);
      pages(kb + 2 * kStep);
    }
  }

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

// ---- many rows: 128 rows of one kv head, 32 a wave's, keys in tiles of 64 ----
//
// The matrix instructions bound it, with the exponentials beside them, and the card's power: at 2 x 2,048
// rows x 32 heads over 16,384 positions (f16, head_dim 128) 864 TFLOP/s, where the library's largest f16
// products reach 1,137, at 2.0 GHz of 2.4. So every step that is not needed costs clock even where it
// costs no cycles.
// Products of 32 x 32 x 16: half the instructions of 16 x 16 x 32, one row's statistics to a lane. K and
// V of a tile go from memory to LDS without passing registers, one tile ahead of their use; the only
// wait is at the end of a tile. A wave brings 16 neighbouring keys, which lie in one page.
//   K: in pieces [16 keys][32 elements][lane][16 bytes] as the operand wants it: no bank conflicts
//   V: rows as they are; a transposing read takes 4 neighbouring keys x 16 dimensions for 16 lanes.
//      4 rows x 64 bytes meet in one pass of LDS: the 16-byte pieces of a row are exchanged by its
//      number so that they fall on different banks.
// A lane has the products of row lane % 32 with keys 8 a + 4 (lane / 32) .. +3; the second product of
// 16 keys takes 8 of a lane's weights, so V's keys are read in that order. The products of the next 32
// keys stand beside this block's exponentials in one straight piece of code, so that both run at once
// (with the maximum taken first, scores and sums one after the other: 1,124 us; now 897). Whether the
// maximum has to move shows in the weights' sum, which is needed anyway.
// Two workgroups a CU: 64 KB of LDS and up to 256 registers a lane each. With 48 or 64 rows a wave a
// SIMD's second wave or the registers are lost (1,177 and 2,042 us when it took 1,124).

// 16 bytes per lane from base + off to LDS at lds + 16 lane, counted in vmcnt; base and lds are the
// wave's. m0 is named so that no value of the compiler's is taken to outlive the statement.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void fill16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop

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

template <class F, int D>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(F::NQ == 1 && D == 64 ? 3 : 2, F::NQ == 1 && D == 64 ? 3 : 2))) k_paged_chunk(AttnArgs r) {
  using KV = typename F::KV;
  using MV = typename F::MV;
  constexpr int NC = D / 16, ND = D / 32, kRowBytes = 2 * D, kBuf = kTileKeys * kRowBytes;
  constexpr int kFills = kRowBytes / 64;  // of 1 KB, for 16 rows
  // Parts of a weight. f16 rows: one, 11 bits, for the products bound this kernel: with two, 2 x 2,048 rows x 32 heads
  // over 16,384 positions take 1,198 us instead of 897 (2 x 1,000 x 16 heads of 64 over 8,000: 159, 120). It costs the f16
  // output at most 2^-11 of the weighted mean of |v|; there, as a norm, 2.8e-4 of the output where rounding alone is 2.1e-4.
  constexpr int kParts = F::NQ == 1 ? 1 : F::NW;
  __shared__ __attribute__((aligned(1024))) uint8_t sh[4 * kBuf];  // K, K, V, V
  __shared__ int sh_odd;                                           // V of the tile is not finite
  const int kvh = blockIdx.x % r.a.kv.n_kv_heads, rest = blockIdx.x / r.a.kv.n_kv_heads;
  int split, tile;
  turn_of(r, rest, &split, &tile);
  // later rows see more keys: the longest tiles first
  tile = r.tiles - 1 - tile;
  Tile t;
  if (!tile_of(r, tile, kvh, kChunkRows, &t)) return;
  const int splits = splits_of(t.keys, r.split_keys, r.n_split);
  if (split >= splits) return;
  const Keys mine = split_keys_of(t.keys, split, r.split_keys, splits);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, g = lane >> 5;
  const Cache<KV> c = cache_of<KV>(r, t.b, kvh);
  int row_lo;  // row lane % 32 sees keys row_lo .. row_lo + row_span - 1 of this split
  uint32_t row_span;
  MV q[NC][F::NQ];
  float factor, m = -INFINITY, l = 0.0f;
  {
    const Row row = row_of(r, t, 32 * wave + col);
    load_row<F, D, 16>(r, row, q, &factor);
    row_lo = row.lo;
    row_span = (uint32_t)max(0, min(row.hi, mine.hi) - row.lo);
  }
  if (row_span == 0) m = 0.0f;  // sees nothing here: its weights are 0 whatever the maximum
  bool fresh = true;            // a row of the wave may be without a maximum
  f16v o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)sh;
  const uint32_t koff = (lane & 15) * kRowBytes + (lane >> 4) * 16;
  uint32_t voff[2];  // fills 0 and 1; fill i + 2 is 2 KB further on in memory and in LDS
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int unit = 64 * i + lane, at = unit / (kRowBytes / 16);  // 16-byte piece and row of LDS
    voff[i] = at * kRowBytes + ((unit % (kRowBytes / 16)) ^ exchange<D>(at)) * 16;
  }
  // The pages of a tile's keys 16 x .. +15 in lanes x = 0 .. 3; a wave brings 16 keys. For a key
  // without a page (or behind the last) any memory is read: it takes no part.
  auto pages_of = [&](int kt) { return c.page(kt + 16 * (lane & 3), mine.hi); };
  auto place = [&](int key, int page) { return page < 0 ? 0 : page * c.page_stride + (int64_t)(key & c.mask) * D; };
  auto fill_k = [&](int key, int page, uint32_t to) {
    const KV* from = c.k + place(key, page);
#pragma unroll
    for (int k = 0; k < D / 32; ++k) fill16(from + 32 * k, koff, to + 1024 * k);
  };
  auto fill_v = [&](int key, int page, uint32_t to) {
    const KV* from = c.v + place(key, page);
#pragma unroll
    for (int i = 0; i < kFills; ++i) fill16(from + (i & ~1) * 512, voff[i & 1], to + 1024 * i);
  };
  // keys lane % 32 of a block, elements 8 g of 16: in the piece of 16 keys x 32 elements
  const uint32_t krow = lds + ((lane >> 4) & 1) * (D / 32) * 1024 + (g * 16 + (lane & 15)) * 16;
  // this lane's place in a transposing read: row 4 g + (lane % 16) / 4, 8 bytes of dimensions 16 ((lane / 16) % 2) + 4 (lane % 4)
  const int trow = 4 * g + ((lane & 15) >> 2);
  const uint32_t vrow = lds + 2 * kBuf + trow * kRowBytes + (lane & 1) * 8;
  const uint32_t vx = exchange<D>(trow) ^ (2 * ((lane >> 4) & 1) + ((lane & 3) >> 1));

  auto products = [&](uint32_t at, float (&s)[16]) {
    f16v acc;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const MV p = read_piece<MV>(at + (k >> 1) * 1024 + (k & 1) * 512);
#pragma unroll
      for (int e = F::NQ - 1; e >= 0; --e) acc = mma32(p, q[k][e], acc);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = acc[i];
  };
  MV w[2][kParts];
  auto weigh = [&](const float (&s)[16]) {
    const float base = m == -INFINITY ? 0.0f : F::kLift - m;
    float sum = 0.0f;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(s[8 * b + j], factor, base));
      sum += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      parts(p, w[b]);
    }
    return sum;
  };
  auto top_of = [&](const float (&s)[16]) {
    float top = s[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) top = fmaxf(top, s[j]);
    return max_row<32>(top * factor);
  };
  // A block of 32 keys from kb: their weights and what they add to the sums; beside it the products of
  // the next block, whose K lies at kat (behind the last: of what is there, unused). V lies at vat.
  // pages: bit x clear where keys 16 x of the block have no page; -1: every row sees every key.
  auto block = [&](int kb, uint32_t kat, uint32_t vat, int pages, bool odd, float (&s)[16], float (&next)[16]) {
    if (pages >= 0) {
      const int first = kb + 4 * g - row_lo;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const uint32_t at = first + 8 * (j >> 2) + (j & 3);
        s[j] = at < (pages >> (j >> 3) & 1 ? row_span : 0u) ? s[j] : -INFINITY;
      }
    }
    if (fresh) {
      const float top = top_of(s);
      if (m == -INFINITY) m = top;
      fresh = __any(m == -INFINITY);
    }
    products(kat, next);
    MV v[2][ND];
    auto read_v = [&](int b, int d) { v[b][d] = read_turned(vat + 16 * b * kRowBytes + ((4 * d) ^ vx) * 16, 8 * kRowBytes); };
    if constexpr (F::NQ == 1) {  // read here, no product waits for them (f32 rows leave no registers for that)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int d = 0; d < ND; ++d) read_v(b, d);
    }
    float sum = weigh(s);
    // a weight beyond 2^15 (f16 holds 2^16), or many near it: the maximum moves
    if (__any(sum > 32768.0f)) {
      asm volatile("");  // a branch: the compiler would rather compute both
      const float now = fmaxf(m, top_of(s));
      const float f = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - now);  // a row that saw no key yet stays at 0
      m = now;
      l *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= f;
      sum = weigh(s);
    }
    l += sum;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        if constexpr (F::NQ > 1) read_v(b, d);
#pragma unroll
        for (int e = kParts - 1; e >= 0; --e) o[d] = mma32(v[b][d], w[b][e], o[d]);
      }
    if (odd) {
      asm volatile("");  // as above
      float p[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        p[j] = (float)w[j >> 3][0][j & 7];
        if constexpr (kParts > 1) p[j] += (float)w[j >> 3][1][j & 7];
      }
      add_non_finite<F, D, Staged>(c, p, kb, mine.hi, row_lo, row_lo + (int)row_span, (float*)o);
    }
  };

  // Step i: the 64 keys from kt. V of tile i is used, and K of the keys 32 further on (the products run
  // one block ahead); V of tile i + 1 and its K are brought meanwhile.
  const int n = (mine.hi - mine.lo + kTileKeys - 1) / kTileKeys;
  const uint32_t wto = wave * 16 * kRowBytes;
  float s0[16], s1[16];
  int pages0 = 0, pages1 = 0, pages2 = 0;  // of tiles i, i + 1, i + 2
  auto fill = [&](int kt, int pv, int pk, uint32_t buf) {
    fill_v(kt + 16 * wave, __builtin_amdgcn_readlane(pv, wave), lds + 2 * kBuf + buf + wto);
    fill_k(kt + 32 + 16 * wave, wave < 2 ? __builtin_amdgcn_readlane(pv, wave + 2) : __builtin_amdgcn_readlane(pk, wave - 2),
           lds + buf + wto);
  };
  if (n > 0) {
    pages0 = pages_of(mine.lo);
    pages1 = pages_of(mine.lo + kTileKeys);
    pages2 = pages_of(mine.lo + 2 * kTileKeys);
    fill(mine.lo, pages0, pages1, 0);
    if (wave < 2) fill_k(mine.lo + 16 * wave, __builtin_amdgcn_readlane(pages0, wave), lds + kBuf + wto);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    products(krow + kBuf, s0);
  }
  uint32_t buf = 0;
  for (int i = 0, kt = mine.lo; i < n; ++i, kt += kTileKeys, buf ^= kBuf) {
    // this wave's fills and reads are done; behind the barrier everyone's are
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const uint64_t bad = __ballot(pages0 < 0 && lane < 4);
    if (i + 1 < n) fill(kt + kTileKeys, pages1, pages2, buf ^ kBuf);
    pages0 = pages1;
    pages1 = pages2;
    pages2 = pages_of(kt + 3 * kTileKeys);
    int pages = -1;
    bool odd = false;
    if (bad || kt < t.max_lo || kt + kTileKeys > t.min_hi) {
      // some row does not see some key: what V holds there must be finite
      pages = 15 & ~(int)bad;
      if (threadIdx.x == 0) sh_odd = 0;
      __syncthreads();
      for (int x = threadIdx.x; x < kBuf / 16; x += 256) {
        u4* p = (u4*)(sh + 2 * kBuf + buf + 16 * x);
        u4 v = *p;
        const int at = x / (kRowBytes / 16);
        const uint32_t keep = kt + at < mine.hi && (pages >> (at >> 4) & 1) ? ~0u : 0u;
        uint32_t bits = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[k] &= keep;
          bits |= odd_bits<KV>(v[k]);
          v[k] = without_odd<KV>(v[k]);
        }
        if (bits) sh_odd = 1;
        if (bits || !keep) *p = v;
      }
      __syncthreads();
      odd = __builtin_amdgcn_readfirstlane(sh_odd);
    }
    block(kt, krow + buf, vrow + buf, pages, odd, s0, s1);
    block(kt + 32, krow + buf + kBuf / 2, vrow + buf + kBuf / 2, pages < 0 ? -1 : pages >> 2, odd, s1, s0);
  }
  // no fill outlives the workgroup: the last step issues none and waited for all

  const int64_t all = (int64_t)r.a.kv.n_tokens * r.a.n_heads;
  l += __shfl_xor(l, 32);
  const Row row = row_of(r, t, 32 * wave + col);
  if (!row.real) return;
  if (splits == 1) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    typename F::IO* out = (typename F::IO*)r.a.out + (int64_t)row.token * r.a.out_stride + row.head * D + 4 * g;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store4(out + 32 * d + 8 * i, f4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * inv);
  } else {
    const int64_t at = (int64_t)split * all + (int64_t)row.token * r.a.n_heads + row.head;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store4(r.part_o + at * D + 32 * d + 8 * i + 4 * g, f4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]});
    if (g == 0) {
      r.part_ml[2 * at] = m;
      r.part_ml[2 * at + 1] = l;
    }
  }
}

// The joins as a launch of their own: four rows to a workgroup, a wave each, or a row to a workgroup of TEAMS waves.
template <typename IO, int D, int TEAMS>
__global__ void __launch_bounds__(TEAMS > 4 ? 64 * TEAMS : 256) k_paged_join(AttnArgs r, int tile_rows) {
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
  const Keys keys = keys_of(seq, first / r.group, last / r.group, r.a.window, r.cap);
  const int splits = splits_of(keys, r.split_keys, r.n_split);
  if (splits > 1)  // else its only split wrote it
    join_row(r, true, at, (IO*)r.a.out + (int64_t)token * r.a.out_stride + head * D, d0, splits, team, TEAMS, 64, 64 * TEAMS, sh, p);
}

// ---- host ----
struct Plan {
  bool staged;      // k_paged_chunk
  bool eight;       // k_paged_rows of eight waves
  bool one_launch;  // the splits' join included
  int tile_rows;
  int64_t tiles;
  int n_split, split_keys;
  size_t bytes, ml_at, arrived_at;
};

Plan plan_of(const mtg_paged_attn& a) {
  const mtg_paged_kv& kv = a.kv;
  const int group = a.n_heads / kv.n_kv_heads;
  Plan p{};
  const int64_t per_seq = ((int64_t)kv.n_tokens * group + kv.n_seqs - 1) / kv.n_seqs;
  p.staged = kv.kv_type == MTG_TYPE_F16 && per_seq > 64;
  p.tile_rows = p.staged ? kChunkRows : per_seq <= 16 ? 16 : 32;
  p.tiles = tiles_bound(kv.n_tokens, kv.n_seqs, group, p.tile_rows);
  const int64_t cap = (int64_t)kv.table_stride * kv.page_size;
  int64_t keys = a.max_kv > 0 && a.max_kv < cap ? a.max_kv : cap;
  if (a.window > 0) keys = std::min<int64_t>(keys, (int64_t)a.window + p.tile_rows + 32);
  // the workgroups of one split each, as if all sequences had the same number of rows
  const int64_t work = kv.n_seqs * ((per_seq + p.tile_rows - 1) / p.tile_rows) * kv.n_kv_heads;
  int64_t per;
  auto grid = [&](int64_t per) { return work * ((keys + per - 1) / per); };
  if (p.staged) {
    // Two workgroups a CU have work, if that leaves each 512 keys or more, else one, of 256 or more, for the parts cost more
    // to write and join than the second brings (60 rows each, group 2: 32 sequences of 500 keys 39.9 us unsplit, 61 in two
    // parts; two of 8,000: 29.2 in parts of 512, 32.5 of 256; but one tile of rows over 1,600: 21 of 256, 31 of 512).
    const int64_t want = std::max<int64_t>(1, 512 / work);
    per = (keys + want - 1) / want;
    if (per < 512) per = std::max<int64_t>(256, (keys * work + 255) / 256);
  } else {
    // 512 keys, or so that there are 2,048 workgroups, whichever is more: one row each of 24 sequences of up to 8,000 keys
    // 94.5 us with 896 keys, 99.5 with 512, 124 with 1,664. In small grids fewer, down to 128, up to 128 workgroups (one
    // row, 1,600 keys: 128 keys 10.3 us, 512 12.5; 8,000 keys: 256 17.2, 512 15.9).
    per = 512;
    for (int64_t x : {256, 128})
      if (grid(x) <= 128) per = x;
    if (grid(512) > 2048) per = std::max<int64_t>(512, (keys * work + 2047) / 2048);
    // Even splits of 512 or more, and none of fewer than 1,024 where there is a workgroup a CU without (one row, f16: 64
    // sequences of up to 512 keys 17.1 us, with a second split of one key 28.8; of up to 800 28.9 and 40.7; f32, 40 of up
    // to 1,600: 83.5 in three, 104 in four).
    if (per >= 512) {
      const int64_t n = keys < 2 * per && work >= 256 ? 1 : std::max<int64_t>(1, (keys + per / 2) / per);
      per = std::max<int64_t>(128, (keys + n - 1) / n);
    }
    // Half as many workgroups as the chip takes: of eight waves, without splits, up to some 1,000 keys (one row each: 32
    // sequences of up to 1,000 keys 17.6 us, with four waves 23.6, of 2,000 37.5 and 40.6; 16 of 1,000 16.6 and 18.7, of
    // 1,500 22.0 and 18.8; f32, 32 x 2 rows, 1,000 keys 45.6 and 58.8; 24 x 4, 1,500 keys 60.5 and 52.8).
    if (p.tile_rows == 16 && work >= 128 && work <= 256 && keys > 256 && keys <= 512 + 4 * work) p.eight = true, per = keys;
    // (with few rows to join also for 512 workgroups: one row each of 16 sequences of 2,000 keys 19.9 us, else 21.5)
    p.one_launch = grid(per) <= (per_seq <= 4 && keys <= 32 * per ? 512 : 256);
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

int fail(int rc, const char* why) {
  set_call_error(std::string("paged_attn: ") + why);
  return rc;
}

float log2_scale(const mtg_paged_attn& a) { return a.scale * 1.44269504088896340736f; }

// Everything but the workspace; *rc MTG_OK where the call may run (or has nothing to do).
const char* refused(const mtg_paged_attn& a, int* rc) {
  const mtg_paged_kv& kv = a.kv;
  if (const char* why = check(kv, true, rc)) return why;
  *rc = MTG_ERR_UNSUPPORTED;
  if (!(a.io_type == MTG_TYPE_F32 || (a.io_type == MTG_TYPE_F16 && kv.kv_type == MTG_TYPE_F16)))
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

template <class F, int D>
hipError_t run(const AttnArgs& r, const Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.tiles * r.a.kv.n_kv_heads * p.n_split));
  hipError_t e = hipSuccess;
  if constexpr (F::NA == 1) {
    if (p.staged) e = launch(k_paged_chunk<F, D>, grid, dim3(256), 0, s, r);
  }
  using Few = std::conditional_t<F::NA == 3, F32Few, F>;
  if (!p.staged) e = p.eight             ? launch(k_paged_rows<Few, D, 1, 2, 8>, grid, dim3(512), 0, s, r)
                     : p.tile_rows == 16 ? launch(k_paged_rows<Few, D, 1, 2>, grid, dim3(256), 0, s, r)
                                         : launch(k_paged_rows<F, D, 2, F::NA == 1 ? 2 : 1>, grid, dim3(256), 0, s, r);
  if (e == hipSuccess && p.n_split > 1 && !p.one_launch) {
    const int64_t rows = (int64_t)r.a.kv.n_tokens * r.a.n_heads;
    if (p.n_split <= 8)
      e = launch(k_paged_join<typename F::IO, D, 1>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, r, p.tile_rows);
    else if (p.n_split <= 32)
      e = launch(k_paged_join<typename F::IO, D, 4>, dim3((unsigned)rows), dim3(256), 0, s, r, p.tile_rows);
    else
      e = launch(k_paged_join<typename F::IO, D, 16>, dim3((unsigned)rows), dim3(1024), 0, s, r, p.tile_rows);
  }
  return e;
}
template <class F>
hipError_t run(const AttnArgs& r, const Plan& p, hipStream_t s) {
  return r.a.kv.head_dim == 128 ? run<F, 128>(r, p, s) : run<F, 64>(r, p, s);
}

}  // namespace
}  // namespace mtg

extern "C" size_t mtg_paged_attn_workspace(const mtg_paged_attn* a) {
  using namespace mtg;
  if (!a) return 0;
  mtg_paged_attn x = *a;  // sizes only: the pointers may not be there yet
  alignas(16) static const int32_t some[4] = {};
  x.kv.k = x.kv.v = (void*)some;
  x.kv.page_table = x.kv.kv_len = x.kv.q_start = some;
  int rc = 0;
  if (refused(x, &rc) || x.kv.n_seqs == 0 || x.kv.n_tokens == 0) return 0;
  return plan_of(x).bytes;
}

extern "C" int mtg_paged_attn_dev(const mtg_paged_attn* p, void* stream) {
  using namespace mtg;
  try {
    if (!p) return fail(MTG_ERR_INVALID, "no description");
    const mtg_paged_attn& a = *p;
    const mtg_paged_kv& kv = a.kv;
    int rc = 0;
    if (const char* why = refused(a, &rc)) return fail(rc, why);
    if (kv.n_seqs == 0 || kv.n_tokens == 0) return MTG_OK;
    if (!a.q || !a.out) return fail(MTG_ERR_INVALID, "q or out is NULL");
    const size_t eb = type_bytes(a.io_type);
    const int64_t unit = 16 / (int64_t)eb, width = (int64_t)a.n_heads * kv.head_dim;
    const int64_t most = (int64_t)1 << 40;
    if (a.q_stride < width || a.out_stride < width || a.q_stride > most || a.out_stride > most ||
        !reaches(kv.n_tokens, a.q_stride) || !reaches(kv.n_tokens, a.out_stride))
      return fail(MTG_ERR_INVALID, "a row stride below the row's width, or rows behind 2^46 elements");
    if (!aligned(a.q, 16) || !aligned(a.out, 16) || a.q_stride % unit || a.out_stride % unit)
      return fail(MTG_ERR_UNSUPPORTED, "rows not aligned to 16 bytes");
    const size_t qn = extent(kv.n_tokens, a.q_stride, width, eb), on = extent(kv.n_tokens, a.out_stride, width, eb);
    if (overlap(a.q, qn, a.out, on) && !(a.q == a.out && a.q_stride == a.out_stride))
      return fail(MTG_ERR_INVALID, "out overlaps q");
    const size_t pool = pool_extent(kv);
    if (overlap(kv.k, pool, a.out, on) || overlap(kv.v, pool, a.out, on)) return fail(MTG_ERR_INVALID, "out lies in the pages");
    auto index = [&](const void* p, size_t n) {
      return meets(p, n, {{kv.page_table, 4 * (size_t)kv.n_seqs * kv.table_stride}, {kv.kv_len, 4 * (size_t)kv.n_seqs},
                          {kv.q_start, 4 * (size_t)kv.n_seqs + 4}});
    };
    if (index(a.out, on)) return fail(MTG_ERR_INVALID, "out overlaps an index array");
    const Plan plan = plan_of(a);
    if (plan.tiles * kv.n_kv_heads * plan.n_split >= ((int64_t)1 << 24))
      return fail(MTG_ERR_UNSUPPORTED, "more than 2^24 workgroups");
    if (plan.bytes) {
      if (!a.workspace || !aligned(a.workspace, 16)) return fail(MTG_ERR_INVALID, "workspace NULL or unaligned");
      if (a.workspace_bytes < plan.bytes) return fail(MTG_ERR_CAPACITY, "workspace smaller than mtg_paged_attn_workspace");
      if (meets(a.workspace, plan.bytes, {{a.out, on}, {a.q, qn}, {kv.k, pool}, {kv.v, pool}}) || index(a.workspace, plan.bytes))
        return fail(MTG_ERR_INVALID, "workspace overlaps q, out, the pages or an index array");
    }
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
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = a.io_type == MTG_TYPE_F16      ? run<F16>(r, plan, s)
                         : kv.kv_type == MTG_TYPE_F16 ? run<F32F16>(r, plan, s)
                                                        : run<F32>(r, plan, s);
    if (e != hipSuccess) return fail(MTG_ERR_DEVICE, hipGetErrorString(e));
    return MTG_OK;
  } catch (...) {
    return MTG_ERR_NOMEM;
  }
}
