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
#include "paged_attn_parts.hpp"

namespace mtg {
namespace {

using namespace paged;
using namespace attn;

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
struct F32Few {  // rows and cache f32, 16 rows or fewer: products of f32, 4 elements each
  using IO = float;
  using KV = float;
  using MV = Eight;
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
__device__ __forceinline__ void operand(const Raw<float, 8>& r, Eight (&p)[1]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) p[0].x[j] = __uint_as_float(r.w[j]);
}
template <int N>
__device__ __forceinline__ void operand(const Raw<float, N> (&r)[8], int d, Eight (&p)[1]) {
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
  constexpr int NC = D / 32, DL = D / 16, kRows = 16 * RT, kWords = DL * sizeof(KV) / 4, kStep = 32 * NW;
  __shared__ float sh_o[NW][16][kPadOf(D)];
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


  finish_rows<F, D, RT, NW>(r, t, tile, split, splits, m, l, o, sh_o, sh_ml);
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

int fail(int rc, const char* why) {
  set_call_error(std::string("paged_attn: ") + why);
  return rc;
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
  if (e == hipSuccess && p.n_split > 1 && !p.one_launch) e = run_join<typename F::IO, D>(r, p, s);
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
  if (refused(x, false, &rc) || x.kv.n_seqs == 0 || x.kv.n_tokens == 0) return 0;
  return plan_of(x).bytes;
}

extern "C" int mtg_paged_attn_dev(const mtg_paged_attn* p, void* stream) {
  using namespace mtg;
  try {
    if (!p) return fail(MTG_ERR_INVALID, "no description");
    const mtg_paged_attn& a = *p;
    const mtg_paged_kv& kv = a.kv;
    int rc = 0;
    if (const char* why = refused(a, false, &rc)) return fail(rc, why);
    if (kv.n_seqs == 0 || kv.n_tokens == 0) return MTG_OK;
    const Plan plan = plan_of(a);
    if (const char* why = refused_arrays(a, plan, &rc)) return fail(rc, why);
    AttnArgs r = args_of(a, plan);
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
