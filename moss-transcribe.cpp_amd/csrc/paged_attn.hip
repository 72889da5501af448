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
// 2^-15 .. 2^15 by a constant factor that the division takes out again).
//
// Formats. f16 rows and cache: one f16 product. f32 rows, f16 cache: the row is scaled to a
// maximum of 2^10..11 and split into two f16 parts (22 bits), and so are the weights: two
// products. f32 cache: values split exactly into three bf16 parts of 8 bits, the six products
// above 2^-24 are taken. The sums are f32 throughout.
#include "kernels.hpp"
#include "paged_dev.hpp"

#include <algorithm>
#include <climits>
#include <cmath>

namespace mtg {
namespace {

using namespace paged;

typedef __bf16 b8 __attribute__((ext_vector_type(8)));

struct AttnArgs {
  mtg_paged_attn a;
  int shift, cap;           // of the page size; positions a table row names
  int group;                // query heads of a kv head
  int split_keys, n_split;  // keys of a split (a multiple of 128), most splits of a tile
  float* part_o;            // [split][row][head_dim] of rows (token, head)
  float* part_ml;           // [split][row][2]
  float log2_scale;         // scale * log2(e)
};

constexpr float kSlack = 8.0f;  // a score above the maximum by more than 2^8 moves it

struct F16 {  // rows and cache f16
  using IO = _Float16;
  using KV = _Float16;
  using MV = h8;
  static constexpr int NA = 1, NB = 1;
  static constexpr float kLift = 7.0f;  // log2 of the weights' constant factor
};
struct F32F16 {  // rows f32, cache f16
  using IO = float;
  using KV = _Float16;
  using MV = h8;
  static constexpr int NA = 1, NB = 2;
  static constexpr float kLift = 7.0f;
};
struct F32 {
  using IO = float;
  using KV = float;
  using MV = b8;
  static constexpr int NA = 3, NB = 3;
  static constexpr float kLift = 0.0f;
};

__device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mma(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// The product of a value in NA parts with one in NB, small terms first.
template <class F>
__device__ __forceinline__ f4 product(const typename F::MV* a, const typename F::MV* b, f4 c) {
  constexpr int n = F::NA > F::NB ? F::NA : F::NB;
#pragma unroll
  for (int sum = n - 1; sum >= 0; --sum)
#pragma unroll
    for (int i = 0; i <= sum; ++i)
      if (i < F::NA && sum - i < F::NB) c = mma(a[i], b[sum - i], c);
  return c;
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

__device__ __forceinline__ float max16(float x) {  // over the four lanes that hold one row
  x = fmaxf(x, __shfl_xor(x, 16));
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
  const int32_t* starts = c.q_start;
  t->b = last_true(c.n_seqs, [&](int i) { return first_tile(starts[i], i, c.n_tokens, r.group, rows) <= tile; });
  if (t->b < 0) return false;
  t->kvh = kvh;
  t->seq = rows_of(starts[t->b], starts[t->b + 1], c.kv_len[t->b], c.n_tokens);
  t->first = (tile - first_tile(starts[t->b], t->b, c.n_tokens, r.group, rows)) * rows;
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

// The row's elements 32 c + 8 g .. of all c, as the score product's second operand; *factor
// turns a score into a power of two's exponent.
template <class F, int D>
__device__ __forceinline__ void load_row(const AttnArgs& r, const Row& x, typename F::MV (&q)[D / 32][F::NB], float* factor) {
  const int g = (threadIdx.x & 63) >> 4;
  const typename F::IO* src = (const typename F::IO*)r.a.q + (int64_t)x.token * r.a.q_stride + x.head * D + 8 * g;
  float v[D / 32][8];
  float top = 0.0f;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    const Raw<typename F::IO, 8> w = load_raw<typename F::IO, 8>(src + 32 * c);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[c][j] = x.real ? value(w, j) : 0.0f;
      top = fmaxf(top, fabsf(v[c][j]));
    }
  }
  // a negative scale turns the row, so that larger products are larger scores; scale 0 is a row of zeros
  float s = r.log2_scale < 0.0f ? -1.0f : r.log2_scale == 0.0f ? 0.0f : 1.0f, back = 1.0f;
  if constexpr (F::NB == 2) {  // to a maximum of 2^10 .. 2^11: a power of two, exact both ways
    const int e = (int)(__float_as_uint(max16(top)) >> 23);
    if (e != 0 && e != 255) {
      const int se = cut(264 - e, 1, 250);
      s *= __uint_as_float((uint32_t)se << 23);
      back = __uint_as_float((uint32_t)(254 - se) << 23);
    }
  }
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[c][j] *= s;
    parts(v[c], q[c]);
  }
  // never 0: -inf marks what a row does not see
  *factor = fmaxf((r.log2_scale == 0.0f ? 1.0f : fabsf(r.log2_scale)) * back, 1.17549435e-38f);
}

// Which of a block's 32 keys weight j of a lane in group g belongs to, and which dimension element i
// of product t, in the layouts of the two kernels.
struct Direct {  // operands straight from memory
  template <int D>
  static __device__ __forceinline__ int dim(int t, int g, int i) { return (D / 16) * (4 * g + i) + t; }
  static __device__ __forceinline__ int group(int key) { return key >> 3; }
  static __device__ __forceinline__ int weight(int key) { return key & 7; }
};
struct Staged {  // operands from LDS, tiles of 16 neighbouring keys
  template <int D>
  static __device__ __forceinline__ int dim(int t, int g, int i) { return 16 * t + 4 * g + i; }
  static __device__ __forceinline__ int group(int key) { return (key >> 2) & 3; }
  static __device__ __forceinline__ int weight(int key) { return (key & 3) + ((key >> 4) << 2); }
};

// What non-finite elements of V add to the rows that see them: the product took them as zero,
// since in a block that some rows do not see whole, 0 * NaN would reach those rows.
template <class F, int D, class Layout>
__device__ __forceinline__ void add_non_finite(const Cache<typename F::KV>& c, const float* p, int kb, int hi, int row_lo,
                                               int row_hi, f4* o) {
  const int lane = threadIdx.x & 63, row = lane & 15, g = lane >> 4;
  for (int k = 0; k < 32; ++k) {
    float w = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (Layout::weight(k) == j) w = p[j];
    w = __shfl(w, Layout::group(k) * 16 + row);
    const int key = kb + k, page = c.page(key, hi);
    if (page < 0 || key < row_lo || key >= row_hi) continue;
    const typename F::KV* v = c.v + page * c.page_stride + (int64_t)(key & c.mask) * D;
#pragma unroll
    for (int t = 0; t < D / 16; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const typename F::KV x = v[Layout::template dim<D>(t, g, i)];
        if (!finite(x)) o[t][i] += w * (float)x;
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
    const float now = fmaxf(*m, max16(top));
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

// ---- few rows: 16 or 32 rows of one kv head, four waves each with its own blocks of 32 keys ----
//
// HBM bounds it. K and V go from memory straight into the operands' registers (no LDS, no
// barrier until the end): a lane reads 16 bytes of a key for the score product and D / 16
// elements of 8 keys for the second one. The loads of the next block's K are issued when the
// scores are done, those of its V when the sums are.
template <class F, int D, int RT>
__global__ void __launch_bounds__(256) k_paged_rows(AttnArgs r) {
  using KV = typename F::KV;
  using MV = typename F::MV;
  constexpr int NC = D / 32, DL = D / 16, kRows = 16 * RT, kPad = D + 4, kWords = DL * sizeof(KV) / 4;
  __shared__ float sh_o[4][16][kPad];
  __shared__ float sh_ml[4][kRows][2];
  const int kvh = blockIdx.x % r.a.kv.n_kv_heads, rest = blockIdx.x / r.a.kv.n_kv_heads;
  const int split = rest % r.n_split, tile = rest / r.n_split;
  Tile t;
  if (!tile_of(r, tile, kvh, kRows, &t)) return;
  const int splits = splits_of(t.keys, r.split_keys, r.n_split);
  if (split >= splits) return;
  const Keys mine = split_keys_of(t.keys, split, r.split_keys, splits);

  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const Cache<KV> c = cache_of<KV>(r, t.b, kvh);
  Row row[RT];
  MV q[RT][NC][F::NB];
  float factor[RT], m[RT], l[RT];
  f4 o[RT][DL];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    row[i] = row_of(r, t, 16 * i + col);
    load_row<F, D>(r, row[i], q[i], &factor[i]);
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int d = 0; d < DL; ++d) o[i][d] = f4{0, 0, 0, 0};
  }

  // this lane's key of score product `tile`: 8 (col / 4) + 4 tile + col % 4; its V keys: 8 g + j
  const int kgroup = 8 * (col >> 2), krow = kgroup + (col & 3);
  Raw<KV, 8> kr[2][NC];
  Raw<KV, DL> vr[8];
  auto load_k = [&](int kb, int page) {
    const KV* p = c.k + (page < 0 ? 0 : page * c.page_stride + (int64_t)((kb + krow) & c.mask) * D) + 8 * g;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int k = 0; k < NC; ++k) kr[a][k] = load_raw<KV, 8>(p + a * 4 * D + 32 * k);
  };
  auto load_v = [&](int kb, int page) {
    const KV* p = c.v + (page < 0 ? 0 : page * c.page_stride + (int64_t)((kb + 8 * g) & c.mask) * D) + DL * col;
#pragma unroll
    for (int j = 0; j < 8; ++j) vr[j] = load_raw<KV, DL>(p + j * D);
  };
  int kb = mine.lo + 32 * wave;
  int vpage = -1;
  if (kb < mine.hi) {
    vpage = c.page(kb + 8 * g, mine.hi);
    load_k(kb, c.page(kb + kgroup, mine.hi));
    load_v(kb, vpage);
  }
  for (; kb < mine.hi; kb += 128) {
    const int next = kb + 128;
    const int kpage_next = c.page(next + kgroup, mine.hi), vpage_next = c.page(next + 8 * g, mine.hi);
    float s[RT][8];
    {
      f4 acc[RT][2];
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[i][0] = acc[i][1] = f4{0, 0, 0, 0};
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          MV p[F::NA];
          operand(kr[a][k], p);
#pragma unroll
          for (int i = 0; i < RT; ++i) acc[i][a] = product<F>(p, q[i][k], acc[i][a]);
        }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] = acc[i][j >> 2][j & 3];
    }
    if (next < mine.hi) load_k(next, kpage_next);

    bool bad = false;
    const bool whole = kb >= t.max_lo && kb + 32 <= t.min_hi && kb + 32 <= mine.hi && __all(vpage >= 0);
    if (!whole) {
      uint32_t odd = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = kb + 8 * g + j;
        const bool there = vpage >= 0 && key < mine.hi;
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
          for (int d = 0; d < kWords; ++d) vr[j].w[d] = without_odd<KV>(vr[j].w[d]);
      }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) weights<DL>(s[i], factor[i], F::kLift, &m[i], &l[i], o[i]);
    MV w[RT][F::NB];
#pragma unroll
    for (int i = 0; i < RT; ++i) parts(s[i], w[i]);
#pragma unroll
    for (int d = 0; d < DL; ++d) {
      MV p[F::NA];
      operand(vr, d, p);
#pragma unroll
      for (int i = 0; i < RT; ++i) o[i][d] = product<F>(p, w[i], o[i][d]);
    }
    if (bad) {
#pragma unroll
      for (int i = 0; i < RT; ++i) add_non_finite<F, D, Direct>(c, s[i], kb, mine.hi, row[i].lo, row[i].hi, o[i]);
    }
    vpage = vpage_next;
    if (next < mine.hi) load_v(next, vpage);
  }

  // the four waves' sums, brought to one maximum, meet in LDS
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
    for (int w = 0; w < 4; ++w) top = fmaxf(top, sh_ml[w][16 * i + col][0]);
    const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[i] - top);
    if (i) __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int d = 0; d < DL; ++d) sh_o[wave][col][DL * (4 * g + k) + d] = o[i][d][k] * f;
    __syncthreads();
    const int orow = threadIdx.x >> 4, at = (threadIdx.x & 15) * DL;
    if (16 * i + orow < t.count) {
      top = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, sh_ml[w][16 * i + orow][0]);
#pragma unroll
      for (int w = 0; w < 4; ++w)
        sum += top == -INFINITY ? 0.0f : sh_ml[w][16 * i + orow][1] * __builtin_amdgcn_exp2f(sh_ml[w][16 * i + orow][0] - top);
      float x[DL];
#pragma unroll
      for (int d = 0; d < DL; ++d) x[d] = (sh_o[0][orow][at + d] + sh_o[1][orow][at + d]) + (sh_o[2][orow][at + d] + sh_o[3][orow][at + d]);
      const int pair = t.first + 16 * i + orow, tok = pair / r.group;
      const int token = t.seq.row0 + tok, head = kvh * r.group + (pair - tok * r.group);
      if (splits == 1) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        typename F::IO* out = (typename F::IO*)r.a.out + (int64_t)token * r.a.out_stride + head * D + at;
#pragma unroll
        for (int d = 0; d < DL; ++d) out[d] = (typename F::IO)(x[d] * inv);
      } else {
        const int64_t slot = (int64_t)split * all + (int64_t)token * r.a.n_heads + head;
#pragma unroll
        for (int d = 0; d < DL; ++d) r.part_o[slot * D + at + d] = x[d];
        if ((threadIdx.x & 15) == 0) {
          r.part_ml[2 * slot] = top;
          r.part_ml[2 * slot + 1] = sum;
        }
      }
    }
  }
}

// ---- many rows: 64 RT rows of one kv head, 16 RT of them a wave's, keys in tiles of 64 ----
//
// The matrix instructions bound it, with the exponentials beside them (a unit of 16 rows x 32 keys
// x 128 elements is 16 products of 18 cycles and about 200 cycles of vector work). K and V of a
// tile go from memory to LDS without passing registers, one tile ahead of their use; the only
// wait is at the end of a tile. Wave w brings keys 16 w .. +15, which lie in one page.
//   K: as the first operand takes it, [16 keys][32 elements][lane][16 bytes]: reads without bank conflicts
//   V: rows as they are; a transposing read takes 4 neighbouring keys x 16 dimensions for 16 lanes.
//      16 rows meet in one read: the 16-byte pieces of a row are exchanged by its number so that
//      they fall on different banks.
// With keys in their order a lane's weights are those of keys 4 g .. +3 of two tiles of 16: the
// transposing reads take the same keys.
constexpr int kTileKeys = 64;
constexpr int kChunkTiles = 2;  // 16 RT rows a wave; 3 and 4 spill or lose the second wave of a SIMD

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
  return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3);
}

__device__ __forceinline__ h8 read_turned(uint32_t lds, int more) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s4 l4;
  const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((l4*)(uintptr_t)lds));
  const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((l4*)(uintptr_t)(lds + more)));
  return __builtin_bit_cast(h8, u4{a[0], a[1], b[0], b[1]});
}

template <class F, int D, int RT>
__global__ void __launch_bounds__(256, 2) k_paged_chunk(AttnArgs r) {
  using KV = typename F::KV;
  using MV = typename F::MV;
  constexpr int NC = D / 32, ND = D / 16, kRows = 64 * RT, kRowBytes = 2 * D, kBuf = kTileKeys * kRowBytes;
  constexpr int kFills = kRowBytes / 64;  // of 1 KB: 16 rows
  __shared__ __attribute__((aligned(1024))) uint8_t sh[4 * kBuf];  // K, K, V, V
  __shared__ int sh_flag[3];                                       // tile i, slot i % 3: 1 bad page, 2 non-finite V
  const int kvh = blockIdx.x % r.a.kv.n_kv_heads, rest = blockIdx.x / r.a.kv.n_kv_heads;
  const int split = rest % r.n_split;
  // later rows see more keys: the longest tiles first
  const int tile = (int)(gridDim.x / (r.a.kv.n_kv_heads * r.n_split)) - 1 - rest / r.n_split;
  Tile t;
  if (!tile_of(r, tile, kvh, kRows, &t)) return;
  const int splits = splits_of(t.keys, r.split_keys, r.n_split);
  if (split >= splits) return;
  const Keys mine = split_keys_of(t.keys, split, r.split_keys, splits);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const Cache<KV> c = cache_of<KV>(r, t.b, kvh);
  Row row[RT];
  MV q[RT][NC][F::NB];
  float factor[RT], m[RT], l[RT];
  f4 o[RT][ND];
  int wave_lo = INT_MAX, wave_hi = 0, wave_min_hi = INT_MAX, wave_max_lo = 0;  // keys any, and every, row of the wave sees
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    row[i] = row_of(r, t, 16 * (RT * wave + i) + col);
    load_row<F, D>(r, row[i], q[i], &factor[i]);
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[i][d] = f4{0, 0, 0, 0};
  }
  {
    const int first = 16 * RT * wave, last = min(first + 16 * RT, t.count) - 1;
    if (first < t.count) {
      const int head = t.seq.pos0 + (t.first + first) / r.group, tail = t.seq.pos0 + (t.first + last) / r.group;
      wave_lo = oldest_of(head, r.a.window);
      wave_hi = cut(tail + 1, 0, r.cap);
      wave_max_lo = oldest_of(tail, r.a.window);
      wave_min_hi = cut(head + 1, 0, r.cap);
    }
  }

  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)sh;
  uint32_t koff[NC], voff[kFills];
#pragma unroll
  for (int k = 0; k < NC; ++k) koff[k] = col * kRowBytes + k * 64 + g * 16;
#pragma unroll
  for (int i = 0; i < kFills; ++i) {
    const int unit = 64 * i + lane, at = unit / (kRowBytes / 16);  // 16-byte piece and row of LDS
    voff[i] = at * kRowBytes + ((unit % (kRowBytes / 16)) ^ exchange<D>(at)) * 16;
  }
  // the page of this wave's 16 keys of the tile at kt; a bad one is flagged and any memory read instead
  auto page_at = [&](int kt) { return c.page(kt + 16 * wave, mine.hi); };
  auto fill = [&](int kt, int page, int buf, int slot) {
    const int key = kt + 16 * wave;
    if (page < 0 && key < mine.hi && lane == 0) atomicOr(&sh_flag[slot], 1);
    const int64_t at = page < 0 ? 0 : page * c.page_stride + (int64_t)(key & c.mask) * D;
    const uint64_t kp = (uint64_t)(c.k + at), vp = (uint64_t)(c.v + at);
    const uint32_t to = lds + buf * kBuf + wave * 16 * kRowBytes;
#pragma unroll
    for (int k = 0; k < NC; ++k) fill16((const void*)kp, koff[k], to + 1024 * k);
#pragma unroll
    for (int i = 0; i < kFills; ++i) fill16((const void*)vp, voff[i], to + 2 * kBuf + 1024 * i);
  };

  if (threadIdx.x < 3) sh_flag[threadIdx.x] = 0;
  __syncthreads();
  int page = __builtin_amdgcn_readfirstlane(page_at(mine.lo));
  if (mine.lo < mine.hi) fill(mine.lo, page, 0, 0);
  page = __builtin_amdgcn_readfirstlane(page_at(mine.lo + kTileKeys));
  // this lane's place in a transposing read: row 4 g + (lane % 16) / 4 of 16, piece lane % 4 of 8 bytes
  const int trow = 4 * g + (col >> 2);
  const uint32_t vrow = lds + 2 * kBuf + trow * kRowBytes + (col & 1) * 8, vx = exchange<D>(trow), vpiece = (col & 3) >> 1;

  int slot = 0;
  for (int kt = mine.lo, buf = 0; kt < mine.hi; kt += kTileKeys, buf ^= 1) {
    const int next_slot = slot == 2 ? 0 : slot + 1, old_slot = next_slot == 2 ? 0 : next_slot + 1;
    // this wave's fills and reads are done; behind the barrier everyone's are
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int flag = __builtin_amdgcn_readfirstlane(*(volatile int*)&sh_flag[slot]);
    if (threadIdx.x == 0) sh_flag[old_slot] = 0;
    if (kt + kTileKeys < mine.hi) {
      fill(kt + kTileKeys, page, buf ^ 1, next_slot);
      page = page_at(kt + 2 * kTileKeys);
    }
    int odd = 0;
    if ((flag & 1) || kt < t.max_lo || kt + kTileKeys > t.min_hi || kt + kTileKeys > mine.hi) {
      // some row does not see some key: what V holds there must be finite
      for (int i = threadIdx.x; i < kBuf / 16; i += 256) {
        const int at = i / (kRowBytes / 16), key = kt + at;
        u4* p = (u4*)(sh + (2 + buf) * kBuf + 16 * i);
        u4 w = *p;
        const uint32_t keep = c.page(key, mine.hi) >= 0 ? ~0u : 0u;
        uint32_t bits = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          w[k] &= keep;
          bits |= odd_bits<KV>(w[k]);
          w[k] = without_odd<KV>(w[k]);
        }
        if (bits) atomicOr(&sh_flag[slot], 2);
        if (bits || !keep) *p = w;
      }
      __syncthreads();
      odd = __builtin_amdgcn_readfirstlane(*(volatile int*)&sh_flag[slot]) & 2;
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int kb = kt + 32 * half;
      if (kb >= wave_hi || kb + 32 <= wave_lo || kb >= mine.hi) continue;
      float s[RT][8];
      {
        f4 acc[RT][2];
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[i][0] = acc[i][1] = f4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const MV p[1] = {*(const MV*)(sh + buf * kBuf + ((2 * half + a) * NC + k) * 1024 + 16 * lane)};
#pragma unroll
            for (int i = 0; i < RT; ++i) acc[i][a] = product<F>(p, q[i][k], acc[i][a]);
          }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) s[i][j] = acc[i][j >> 2][j & 3];
      }
      if ((flag & 1) || kb < wave_max_lo || kb + 32 > wave_min_hi || kb + 32 > mine.hi) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = kb + 4 * g + (j & 3) + ((j >> 2) << 4);
          const bool there = c.page(key, mine.hi) >= 0;
#pragma unroll
          for (int i = 0; i < RT; ++i)
            if (!there || key < row[i].lo || key >= row[i].hi) s[i][j] = -INFINITY;
        }
      }
      MV w[RT][F::NB];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        weights<ND>(s[i], factor[i], F::kLift, &m[i], &l[i], o[i]);
        parts(s[i], w[i]);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const MV p[1] = {read_turned(vrow + buf * kBuf + 32 * half * kRowBytes + (((2 * d + vpiece) ^ vx) * 16), 16 * kRowBytes)};
#pragma unroll
        for (int i = 0; i < RT; ++i) o[i][d] = product<F>(p, w[i], o[i][d]);
      }
      if (odd) {
#pragma unroll
        for (int i = 0; i < RT; ++i) add_non_finite<F, D, Staged>(c, s[i], kb, mine.hi, row[i].lo, row[i].hi, o[i]);
      }
    }
    page = __builtin_amdgcn_readfirstlane(page);
    slot = next_slot;
  }
  // a fill never outlives the workgroup: the last tile's were waited for, and none follows it

  const int64_t all = (int64_t)r.a.kv.n_tokens * r.a.n_heads;
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    l[i] += __shfl_xor(l[i], 16);
    l[i] += __shfl_xor(l[i], 32);
    if (!row[i].real) continue;
    if (splits == 1) {
      const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
      typename F::IO* out = (typename F::IO*)r.a.out + (int64_t)row[i].token * r.a.out_stride + row[i].head * D + 4 * g;
#pragma unroll
      for (int d = 0; d < ND; ++d) store4(out + 16 * d, o[i][d] * inv);
    } else {
      const int64_t at = (int64_t)split * all + (int64_t)row[i].token * r.a.n_heads + row[i].head;
#pragma unroll
      for (int d = 0; d < ND; ++d) store4(r.part_o + at * D + 16 * d + 4 * g, o[i][d]);
      if (g == 0) {
        r.part_ml[2 * at] = m[i];
        r.part_ml[2 * at + 1] = l[i];
      }
    }
  }
}

// The splits of each row joined, a wave to a row: sums brought to the largest maximum.
template <typename IO, int D>
__global__ void __launch_bounds__(256) k_paged_join(AttnArgs r, int tile_rows) {
  const mtg_paged_kv& c = r.a.kv;
  const int64_t all = (int64_t)c.n_tokens * r.a.n_heads, at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= all) return;
  const int token = (int)(at / r.a.n_heads), head = (int)(at % r.a.n_heads), lane = threadIdx.x & 63;
  const int32_t* starts = c.q_start;
  const int b = last_true(c.n_seqs, [&](int i) { return starts[i] <= token; });
  if (b < 0) return;
  const Rows seq = rows_of(starts[b], starts[b + 1], c.kv_len[b], c.n_tokens);
  if (token >= seq.row0 + seq.n) return;
  const int pair = (token - seq.row0) * r.group + head % r.group;
  const int first = pair / tile_rows * tile_rows, last = min(first + tile_rows, seq.n * r.group) - 1;
  const Keys keys = keys_of(seq, first / r.group, last / r.group, r.a.window, r.cap);
  const int splits = splits_of(keys, r.split_keys, r.n_split);
  if (splits == 1) return;  // written by its only split
  float top = -INFINITY;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, r.part_ml[2 * (s * all + at)]);
  float sum = 0.0f, x[D / 64];
#pragma unroll
  for (int d = 0; d < D / 64; ++d) x[d] = 0.0f;
  if (top != -INFINITY)
    for (int s = 0; s < splits; ++s) {
      const int64_t slot = s * all + at;
      const float f = __builtin_amdgcn_exp2f(r.part_ml[2 * slot] - top);
      sum = fmaf(r.part_ml[2 * slot + 1], f, sum);
#pragma unroll
      for (int d = 0; d < D / 64; ++d) x[d] = fmaf(r.part_o[slot * D + lane * (D / 64) + d], f, x[d]);
    }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  IO* out = (IO*)r.a.out + (int64_t)token * r.a.out_stride + head * D + lane * (D / 64);
#pragma unroll
  for (int d = 0; d < D / 64; ++d) out[d] = (IO)(x[d] * inv);
}

// ---- host ----
struct Plan {
  bool staged;    // k_paged_chunk
  int tile_rows;
  int64_t tiles;
  int n_split, split_keys;
  size_t bytes, ml_at;
};

Plan plan_of(const mtg_paged_attn& a) {
  const mtg_paged_kv& kv = a.kv;
  const int group = a.n_heads / kv.n_kv_heads;
  Plan p{};
  const int64_t per_seq = ((int64_t)kv.n_tokens * group + kv.n_seqs - 1) / kv.n_seqs;
  p.staged = kv.kv_type == MTG_TYPE_F16 && per_seq > 64;
  p.tile_rows = p.staged ? 64 * kChunkTiles : per_seq <= 16 ? 16 : 32;
  p.tiles = tiles_bound(kv.n_tokens, kv.n_seqs, group, p.tile_rows);
  const int64_t cap = (int64_t)kv.table_stride * kv.page_size;
  int64_t keys = a.max_kv > 0 && a.max_kv < cap ? a.max_kv : cap;
  if (a.window > 0) keys = std::min<int64_t>(keys, (int64_t)a.window + p.tile_rows + 32);
  // splits so that about 1,024 workgroups (four for each CU; many rows: two) have work, of 256 keys or more (512)
  const int64_t work = std::max<int64_t>(1, std::min<int64_t>(p.tiles, (int64_t)kv.n_tokens * group / p.tile_rows + 1)) * kv.n_kv_heads;
  const int64_t want = std::max<int64_t>(1, (p.staged ? 512 : 1024) / work);
  const int64_t per = std::max<int64_t>(p.staged ? 512 : 256, (keys + want - 1) / want);
  p.split_keys = (int)((per + 127) / 128 * 128);
  p.n_split = (int)((keys + p.split_keys - 1) / p.split_keys);
  if (p.n_split < 1) p.n_split = 1;
  if (p.n_split > 1) {
    const size_t rows = (size_t)p.n_split * kv.n_tokens * a.n_heads;
    p.ml_at = rows * kv.head_dim * 4;
    p.bytes = p.ml_at + (rows * 8 + 15) / 16 * 16;
  }
  return p;
}

int fail(int rc, const char* why) {
  set_call_error(std::string("paged_attn: ") + why);
  return rc;
}

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
  if (!std::isfinite(a.scale)) return "scale";
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
    if (p.staged) e = launch(k_paged_chunk<F, D, kChunkTiles>, grid, dim3(256), 0, s, r);
  }
  if (!p.staged) e = p.tile_rows == 16 ? launch(k_paged_rows<F, D, 1>, grid, dim3(256), 0, s, r)
                                   : launch(k_paged_rows<F, D, 2>, grid, dim3(256), 0, s, r);
  if (e == hipSuccess && p.n_split > 1) {
    const int64_t rows = (int64_t)r.a.kv.n_tokens * r.a.n_heads;
    e = launch(k_paged_join<typename F::IO, D>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, r, p.tile_rows);
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
    if (a.q_stride < width || a.out_stride < width || a.q_stride > most || a.out_stride > most)
      return fail(MTG_ERR_INVALID, "a row stride below the row's width");
    if (!aligned(a.q, 16) || !aligned(a.out, 16) || a.q_stride % unit || a.out_stride % unit)
      return fail(MTG_ERR_UNSUPPORTED, "rows not aligned to 16 bytes");
    const size_t qn = extent(kv.n_tokens, a.q_stride, width, eb), on = extent(kv.n_tokens, a.out_stride, width, eb);
    if (overlap(a.q, qn, a.out, on) && !(a.q == a.out && a.q_stride == a.out_stride))
      return fail(MTG_ERR_INVALID, "out overlaps q");
    const size_t pool = pool_extent(kv);
    if (overlap(kv.k, pool, a.out, on) || overlap(kv.v, pool, a.out, on)) return fail(MTG_ERR_INVALID, "out lies in the pages");
    const Plan plan = plan_of(a);
    if (plan.tiles * kv.n_kv_heads * plan.n_split >= ((int64_t)1 << 24))
      return fail(MTG_ERR_UNSUPPORTED, "more than 2^24 workgroups");
    if (plan.bytes) {
      if (!a.workspace || !aligned(a.workspace, 16)) return fail(MTG_ERR_INVALID, "workspace NULL or unaligned");
      if (a.workspace_bytes < plan.bytes) return fail(MTG_ERR_CAPACITY, "workspace smaller than mtg_paged_attn_workspace");
      if (overlap(a.workspace, plan.bytes, a.out, on) || overlap(a.workspace, plan.bytes, a.q, qn) ||
          overlap(a.workspace, plan.bytes, kv.k, pool) || overlap(a.workspace, plan.bytes, kv.v, pool))
        return fail(MTG_ERR_INVALID, "workspace overlaps q, out or the pages");
    }
    AttnArgs r{};
    r.a = a;
    r.shift = log2_of(kv.page_size);
    r.cap = capacity(kv.table_stride, r.shift);
    r.group = a.n_heads / kv.n_kv_heads;
    r.split_keys = plan.split_keys;
    r.n_split = plan.n_split;
    r.part_o = (float*)a.workspace;
    r.part_ml = (float*)((char*)a.workspace + plan.ml_at);
    r.log2_scale = a.scale * 1.44269504088896340736f;
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
