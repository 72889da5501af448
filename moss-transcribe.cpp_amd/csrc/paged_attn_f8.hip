// paged_attn_f8.hip - mtg_paged_attn_f8_dev: causal attention of the new rows of a batch over a cache in pages of e4m3
// codes with one power of two for 16 positions of a kv head; in a window, the first positions beside it.
//
// The tiles, layouts and running softmax are those of paged_attn.hip over an f16 cache: an e4m3 number is an f16
// number. A block's scale of K goes into the factor of its scores. Its scale of V goes into its codes, for the instruction that turns
// two codes into two f16 numbers multiplies them by a power of two on the way: against the largest scale of the keys that the
// workgroup goes over (a look at all of them, a byte for 16 keys, comes first), as far as every code stays exact, 2^22 below it. The
// largest scale goes into the sums at the end, and what is left of a block's scale further below, its rest, into the weights
// before they become f16 numbers, over the largest rest among the blocks that the row has seen so far, its level. So no row's
// result depends on the scales of keys that it does not see, of later rows or of those in other rows' windows alone.
// Codes are exact; a weight keeps what f16's smallest step leaves of it, 2^-32 of the largest weight, times the codes
// of its key in the row's largest scale where there is a rest.
//
// With a window, a tile's keys are an axis without the gap between the first positions and the window (axis_of); blocks
// of 32 keys lie on one side of it.
#include "kernels.hpp"
#include "paged_attn_parts.hpp"

namespace mtg {
namespace {

using namespace paged;
using namespace attn;

struct Args : AttnArgs {
  mtg_f8_scales scales;
};

struct RowsF16 {
  using IO = _Float16;
  using MV = h8;
  static constexpr int NQ = 1, NW = 2;  // parts of a row's, of a weight
  static constexpr float kLift = 7.0f;          // log2 of the weights' constant factor
};
struct RowsF32 {
  using IO = float;
  using MV = h8;
  static constexpr int NQ = 2, NW = 2;
  static constexpr float kLift = 7.0f;
};

// One kv head of one sequence's cache, on the axis of a tile.
struct Codes : Cache<uint8_t> {
  const uint8_t *ks, *vs;
  int64_t scale_stride;
  int sink, gap, oldest;
  __device__ __forceinline__ int key(int at) const { return key_at(at, sink, gap); }
  // The page of a key that is the same in all lanes, through the scalar cache: what comes by vector loads the compiler would
  // wait for where it is loaded, with all loads before it, to have it in a scalar register.
  __device__ __forceinline__ int wave_page(int key) const {
    if (key < 0 || key >= cap) return -1;
    const int id = ((const __attribute__((address_space(4))) int32_t*)table)[key >> shift];
    return id >= 0 && id < n_pages ? id : -1;
  }
  // Where the scale of a key in a page lies.
  __device__ __forceinline__ int64_t scale_at(int page, int key) const { return page * scale_stride + ((key & mask) / MTG_F8_BLOCK); }
};
__device__ __forceinline__ Codes codes_of(const Args& r, const Tile& t) {
  Codes c;
  static_cast<Cache<uint8_t>&>(c) = cache_of<uint8_t>(r, t.b, t.kvh);
  c.ks = r.scales.k + t.kvh * r.scales.head_stride;
  c.vs = r.scales.v + t.kvh * r.scales.head_stride;
  c.scale_stride = r.scales.page_stride;
  c.sink = r.sink, c.gap = t.gap, c.oldest = t.oldest;
  return c;
}

__device__ __forceinline__ int scale_byte(uint8_t b) { return b < 254 ? b : 254; }

// Scale bytes of k (if asked for) and v.
struct Sizes {
  int k, v;            // the largest
  int kleast, vleast;  // the least that the lane met
  // all within what codes of both can hold
  __device__ __forceinline__ bool lane_near() const { return kleast >= k - kCodeSpan && vleast >= v - kCodeSpan; }
};
// Those of the blocks of keys lo .. hi - 1 (lo a multiple of 16) that rows of the tile see, of those that wave `mine` of `waves`
// looks at, 64 UNROLL blocks at once.
template <int UNROLL, bool K>
__device__ __forceinline__ Sizes sizes_of(const Codes& c, const Keys& x, int mine, int waves) {
  int k = 0, v = 0, kleast = 254, vleast = 254;
  for (int b = x.lo + MTG_F8_BLOCK * 64 * UNROLL * mine; b < x.hi; b += MTG_F8_BLOCK * 64 * UNROLL * waves) {
    int key[UNROLL], page[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const int at = b + MTG_F8_BLOCK * (64 * i + (int)(threadIdx.x & 63));
      key[i] = c.key(at);
      page[i] = at < x.hi && block_seen(key[i], c.oldest, c.sink) ? c.page(key[i], INT_MAX) : -1;
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      if (page[i] < 0) continue;
      const int of_v = scale_byte(c.vs[c.scale_at(page[i], key[i])]);
      v = max(v, of_v), vleast = min(vleast, of_v);
      if constexpr (K) {
        const int of_k = scale_byte(c.ks[c.scale_at(page[i], key[i])]);
        k = max(k, of_k), kleast = min(kleast, of_k);
      }
    }
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    if constexpr (K) k = max(k, __shfl_xor(k, m));
    v = max(v, __shfl_xor(v, m));
  }
  return {__builtin_amdgcn_readfirstlane(k), __builtin_amdgcn_readfirstlane(v), kleast, vleast};
}

// What codes in scale byte b are multiplied by (a block without a page has no byte, b < 0: none of its codes takes part).
__device__ __forceinline__ float scale_of(int b, int most) { return __uint_as_float((uint32_t)(127 + code_exponent(b, most)) << 23); }

// The factor of scores times 2^e: never 0, for -inf marks what a row does not see, nor infinite.
__device__ __forceinline__ float times2(float factor, int e) { return fminf(fmaxf(ldexpf(factor, e), 1.17549435e-38f), 3.0e38f); }

constexpr int kNoLevel = -1000;  // of a row that has seen no key
// A block's share of its row's level, 2^-60 at least: below, every weight, 2^15 at most, is 0 as an f16 number, while the sum of
// the weights, which is taken from what they are with it, keeps those down to 2^-66.
constexpr int kLeastShare = -60;

// Two codes of a word, lower or upper half, times a power of two.
template <int HALF>
__device__ __forceinline__ h2 two(uint32_t w, float scale) {
  return __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HALF));
}
__device__ __forceinline__ uint32_t bits(h2 x) { return __builtin_bit_cast(uint32_t, x); }
// 8 neighbouring codes of a key.
__device__ __forceinline__ h8 eight(uint32_t a, uint32_t b, float scale) {
  return __builtin_bit_cast(h8, u4{bits(two<0>(a, scale)), bits(two<1>(a, scale)), bits(two<0>(b, scale)), bits(two<1>(b, scale))});
}

// Bytes that are the code NaN, as their uppermost bit.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t without_nan(uint32_t w) { return w & ~((nan_codes(w) >> 7) * 0xffu); }

// The running softmax of a row tile over one block of 32 keys, as `weights` of paged_attn_parts.hpp has it, where the lane's 8
// keys' scale of V has a rest: of the row's level, the largest rest that it has seen, go 2^(rest - level) into the weights that s
// becomes. Their sum is that of the whole weights.
template <int DL>
__device__ __forceinline__ void weights(float* s, float factor, float lift, int rest, int* level, float* m, float* l, f4* o) {
  float top = s[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) top = fmaxf(top, s[j]);
  int high = top > -INFINITY ? max(*level, rest) : *level;
  top *= factor;
  if (__any(top > *m + kSlack || high != *level)) {  // from the first key on: m is -inf
    const float now = fmaxf(*m, max_row<16>(top));
    float f = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(*m - now);
    *m = now;
    *l *= f;
    high = max(high, __shfl_xor(high, 16));
    high = max(high, __shfl_xor(high, 32));
    f *= ldexpf(1.0f, *level - high);
    *level = high;
#pragma unroll
    for (int t = 0; t < DL; ++t) o[t] *= f;
  }
  const int share = cut(rest - *level, kLeastShare, 0);
  const float base = (*m == -INFINITY ? 0.0f : lift - *m) + (float)share;
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = __builtin_amdgcn_exp2f(fmaf(s[j], factor, base));
  *l += ldexpf(((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7])), -share);
}

// What codes NaN of V add to the rows that see them: the product took them as zero, since in a block that some rows do not
// see whole they would reach those rows. o: the lane's sums; at: the block's place on the axis.
template <int D, class L>
__device__ __forceinline__ void add_nan(const Codes& c, int at, int hi, int row_lo, int row_hi, float* o) {
  const int lane = threadIdx.x & 63, g = lane / L::kRows;
  for (int k = 0; k < 32 && at + k < hi; ++k) {
    const int key = c.key(at + k), page = c.page(key, row_hi);
    if (page < 0 || (key < row_lo && key >= c.sink)) continue;
    const uint8_t* v = c.v + page * c.page_stride + (int64_t)(key & c.mask) * D;
#pragma unroll
    for (int i = 0; i < D * L::kRows / 64; i += 4) {
      uint32_t x = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) x |= (uint32_t)v[L::template dim<D>(i + k, g)] << 8 * k;
      x = nan_codes(x);
      if (!x) continue;  // four at a time, so that few are held at once
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (x >> (8 * k + 7) & 1) o[i + k] = NAN;
    }
  }
}

// ---- few rows: 16 or 32 rows of one kv head, four waves (eight without splits) each with its own blocks of 32 keys ----
//
// HBM bounds it, and for short contexts the chain of dependent reads (sequence, page, keys). As in k_paged_rows K and V go from
// memory into the operands' registers; a lane reads 16 codes of a key, which are its parts of two score products (of the elements
// 64 c + 16 g .. each product takes 8), and D / 16 codes of 8 keys.
//
// As many waves a SIMD as their registers allow, three or four where k_paged_rows has two: what a block of keys waits for is
// less than half as many bytes (one row each of 32 sequences of up to 12,000 keys 101 us, with two waves 112; four of 20,000 29.2 and 37.1;
// heads of 64 in a window of 2,048 24.4 and 31.6). Scales that lie far apart cost nothing here: what is left of a block's scale is looked
// at in every step (8 x 8 rows over 5,000 keys 22.9 us, with scales in the codes alone 22.6; a second loop for far scales, or
// a branch, 24.2, for the registers of both).
constexpr int rows_waves(int d, int rt) { return rt == 1 ? d == 64 ? 4 : 3 : d == 64 ? 3 : 2; }
template <class F, int D, int RT, int NW = 4>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(rows_waves(D, RT), rows_waves(D, RT)))) k_paged_rows_f8(Args r) {
  using MV = typename F::MV;
  constexpr int NC = D / 32, DL = D / 16, kRows = 16 * RT, kWords = DL / 4, kStep = 32 * NW;
  __shared__ float sh_o[NW][16][kPadOf(D)];
  __shared__ float sh_ml[NW][kRows][2];
  const int kvh = blockIdx.x % r.a.kv.n_kv_heads, rest = blockIdx.x / r.a.kv.n_kv_heads;
  int split, tile;
  turn_of(r, rest, &split, &tile);
  Tile t;
  if (!tile_of<true>(r, tile, kvh, kRows, &t)) return;
  const int splits = NW == 4 ? splits_of(t.keys, r.split_keys, r.n_split) : 1;
  if (split >= splits) return;
  const Keys mine = split_keys_of(t.keys, split, r.split_keys, splits);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const Codes c = codes_of(r, t);
  // this lane's key of score product `tile`: 8 (col / 4) + 4 tile + col % 4; its V keys: 8 g + j
  const int kgroup = 8 * (col >> 2), krow = kgroup + (col & 3);
  u4 kr[2][D / 64];
  Raw<uint8_t, DL> vr[8];
  int kscale = 127, vscale = 127;  // bytes, both of the lane's V keys, which are those that its scores are of
  int kpage = -1, vpage = -1;      // of the block that is loaded next
  int at_page = -1;                // of the V that is held
  auto pages = [&](int at) {
    const int kb = c.key(at);
    kpage = c.page(kb + kgroup, kb + (mine.hi - at));
    vpage = c.page(kb + 8 * g, kb + (mine.hi - at));
  };
  auto load_k = [&](int at) {
    const int key = c.key(at) + krow;
    const uint8_t* k = c.k + (kpage < 0 ? 0 : kpage * c.page_stride + (int64_t)(key & c.mask) * D) + 16 * g;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int i = 0; i < D / 64; ++i) kr[a][i] = *(const u4*)(k + a * 4 * D + 64 * i);
    kscale = vpage < 0 ? -1 : c.ks[c.scale_at(vpage, c.key(at) + 8 * g)];
  };
  auto load_v = [&](int at) {
    const int key = c.key(at) + 8 * g;
    const uint8_t* v = c.v + (vpage < 0 ? 0 : vpage * c.page_stride + (int64_t)(key & c.mask) * D) + DL * col;
#pragma unroll
    for (int j = 0; j < 8; ++j) vr[j] = load_raw<uint8_t, DL>(v + j * D);
    vscale = vpage < 0 ? -1 : c.vs[c.scale_at(vpage, key)];
    at_page = vpage;
  };
  int at = mine.lo + 32 * wave;
  if (at < mine.hi) {
    pages(at);
    load_k(at);
    load_v(at);
    pages(at + kStep);
  }
  const int vmost = sizes_of<2, false>(c, mine, 0, 1).v;
  Row row[RT];
  MV q[RT][NC][F::NQ];
  float factor[RT], m[RT], l[RT];
  int level[RT];
  f4 o[RT][DL];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    row[i] = row_of(r, t, 16 * i + col);
    load_row<F, D, 32>(r, row[i], q[i], &factor[i], [&](int k) { return 64 * (k >> 1) + 8 * (k & 1) + 8 * g; });
    level[i] = kNoLevel;
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int d = 0; d < DL; ++d) o[i][d] = f4{0, 0, 0, 0};
  }

  for (; at < mine.hi; at += kStep) {
    const bool more = at + kStep < mine.hi;
    float s[RT][8];
    {
      f4 acc[RT][2];
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[i][0] = acc[i][1] = f4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const MV p[1] = {eight(kr[a][k >> 1][2 * (k & 1)], kr[a][k >> 1][2 * (k & 1) + 1], 1.0f)};
#pragma unroll
          for (int i = 0; i < RT; ++i) acc[i][a] = product(p, q[i][k], acc[i][a]);
        }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] = acc[i][j >> 2][j & 3];
    }
    const int k2 = min(kscale, 254) - 127;
    if (more) load_k(at + kStep);
    bool bad = false;
    const int kb = c.key(at);
    if (!((kb >= t.max_lo || kb + 32 <= c.sink) && kb + 32 <= t.min_hi && at + 32 <= mine.hi && __all(at_page >= 0))) {
      asm volatile("");  // a branch
      uint32_t odd = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = kb + 8 * g + j;
        const bool there = at_page >= 0 && at + 8 * g + j < mine.hi;
#pragma unroll
        for (int i = 0; i < RT; ++i)
          if (!there || (key < row[i].lo && key >= c.sink) || key >= row[i].hi) s[i][j] = -INFINITY;
        const uint32_t keep = there ? ~0u : 0u;
#pragma unroll
        for (int d = 0; d < kWords; ++d) {
          vr[j].w[d] &= keep;
          odd |= nan_codes(vr[j].w[d]);
        }
      }
      bad = __any(odd != 0);
      if (bad) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int d = 0; d < kWords; ++d) {
            asm volatile("" : "+v"(vr[j].w[d]));  // the bits above are not kept in registers for this
            vr[j].w[d] = without_nan(vr[j].w[d]);
          }
      }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) weights<DL>(s[i], times2(factor[i], k2), F::kLift, scale_rest(vscale, vmost), &level[i], &m[i], &l[i], o[i]);
    MV w[RT][F::NW];
#pragma unroll
    for (int i = 0; i < RT; ++i) parts(s[i], w[i]);
    const float vs = scale_of(vscale, vmost);
    auto pair = [&](const h2 (&x)[8], int d) {  // elements d, d + 1 of 8 keys
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = __builtin_amdgcn_perm(bits(x[2 * j + 1]), bits(x[2 * j]), h ? 0x07060302u : 0x05040100u);
        const MV p[1] = {__builtin_bit_cast(MV, y)};
#pragma unroll
        for (int i = 0; i < RT; ++i) o[i][d + h] = product(p, w[i], o[i][d + h]);
      }
    };
#pragma unroll
    for (int d = 0; d < DL; d += 4) {
      h2 x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = two<0>(vr[j].w[d / 4], vs);
      pair(x, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = two<1>(vr[j].w[d / 4], vs);
      pair(x, d + 2);
    }
    if (bad) {
      asm volatile("");
#pragma unroll
      for (int i = 0; i < RT; ++i) add_nan<D, Direct>(c, at, mine.hi, row[i].lo, row[i].hi, (float*)o[i]);
    }
    if (more) {
      load_v(at + kStep);
      pages(at + 2 * kStep);
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const float back = ldexpf(1.0f, vmost - 127 - kCodeLift + level[i]);
#pragma unroll
    for (int d = 0; d < DL; ++d) o[i][d] *= back;
  }
  finish_rows<F, D, RT, NW>(r, t, tile, split, splits, m, l, o, sh_o, sh_ml);
}

// ---- many rows: 128 or 256 rows of one kv head, 32 a wave's, keys in tiles of 64 ----
//
// As k_paged_chunk over an f16 cache, whose operands' places in LDS, products and softmax these are; what binds there binds
// here. The tile's codes come into registers during the step before the one that puts them into LDS as f16 numbers, so
// that no wave turns a code that another one turns: four waves bring 16 keys of K and of V each, eight 16 of either. Each
// instruction beside the products and the exponentials shows in the time (2 x 2,048 rows x 32 heads over 16,384 positions: 1,046 us with
// four waves, 963 with eight, 931 with the pages through the scalar cache; 1,063 before the places in LDS were kept in registers).
//
// So the scales of K go into its codes too, as those of V do, and where all of both lie within 2^22 of the largest (NEAR), which is
// nearly always, no rest is looked at. The other loop, of the same steps, has the factors of scores and shares of weights for
// each 16 keys: 937 us become 1,112 where half of the blocks are 2^40 larger, 1 x 1,009 f32 rows 154 and 170.
template <class F, int D, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(NW == 4 && F::NQ == 1 && D == 64 ? 3 : 2, NW == 4 && F::NQ == 1 && D == 64 ? 3 : 2))) k_paged_chunk_f8(Args r) {
  using MV = typename F::MV;
  constexpr int NC = D / 16, ND = D / 32, kRowBytes = 2 * D, kBuf = kTileKeys * kRowBytes, M = D / 64;
  constexpr int kParts = F::NQ == 1 ? 1 : F::NW;  // of a weight: as in k_paged_chunk
  __shared__ __attribute__((aligned(1024))) uint8_t sh[4 * kBuf];  // K, K, V, V
  __shared__ __attribute__((aligned(16))) int sh_said[2][4];       // of each wave's keys of V
  __shared__ __attribute__((aligned(16))) int sh_scale[2][2][4];   // bytes of V's and K's 16 keys, where they are asked for
  __shared__ int sh_sizes[NW][4];
  const int kvh = blockIdx.x % r.a.kv.n_kv_heads, rest = blockIdx.x / r.a.kv.n_kv_heads;
  int split, tile;
  turn_of(r, rest, &split, &tile);
  tile = r.tiles - 1 - tile;  // later rows see more keys: the longest tiles first
  Tile t;
  if (!tile_of<true>(r, tile, kvh, 32 * NW, &t)) return;
  const int splits = splits_of(t.keys, r.split_keys, r.n_split);
  if (split >= splits) return;
  const Keys mine = split_keys_of(t.keys, split, r.split_keys, splits);

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, g = lane >> 5;
  const Codes c = codes_of(r, t);
  Sizes sizes = sizes_of<4, true>(c, mine, wave, NW);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    sizes.kleast = min(sizes.kleast, __shfl_xor(sizes.kleast, x));
    sizes.vleast = min(sizes.vleast, __shfl_xor(sizes.vleast, x));
  }
  if (lane == 0) sh_sizes[wave][0] = sizes.k, sh_sizes[wave][1] = sizes.v, sh_sizes[wave][2] = sizes.kleast, sh_sizes[wave][3] = sizes.vleast;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    sizes.k = max(sizes.k, sh_sizes[w][0]), sizes.v = max(sizes.v, sh_sizes[w][1]);
    sizes.kleast = min(sizes.kleast, sh_sizes[w][2]), sizes.vleast = min(sizes.vleast, sh_sizes[w][3]);
  }
  const int kmost = __builtin_amdgcn_readfirstlane(sizes.k), vmost = __builtin_amdgcn_readfirstlane(sizes.v);
  const bool near = __builtin_amdgcn_readfirstlane((int)sizes.lane_near());

  int row_lo, sink_end;  // row lane % 32 sees keys row_lo .. row_lo + row_span - 1 and those before sink_end
  uint32_t row_span;
  MV q[NC][F::NQ];
  float factor, m = -INFINITY, l = 0.0f;
  {
    const Row row = row_of(r, t, 32 * wave + col);
    load_row<F, D, 16>(r, row, q, &factor);
    if (near) factor = times2(factor, kmost - 127 - kCodeLift);
    row_lo = row.lo;
    row_span = (uint32_t)max(0, row.hi - row.lo);
    sink_end = min(c.sink, row.hi);
  }
  if (row_span == 0 && sink_end == 0) m = 0.0f;  // sees nothing: its weights are 0 whatever the maximum
  bool fresh = true;                             // a row of the wave may be without a maximum
  int level = near ? 0 : kNoLevel;
  f16v o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)sh;
  // Waves bring 16 keys of V, at 16 part of a tile, or of K, 32 keys further on.
  constexpr int P = 8 / NW;  // of these, for a wave
  const int part = wave & 3;
  auto is_v = [&](int p) { return NW == 8 ? wave < 4 : p == 0; };
  u4 codes[P][M];  // V: keys lane / 4, codes 16 (lane % 4 + 4 m) ..; K: keys lane % 16, codes 16 (lane / 16 + 4 m) ..
  int byte[P];     // their scale
  int there[P];    // how many of the 16 there are
  int page[P];     // of the tile that is loaded next
  auto pages = [&](int kt) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int at = kt + 16 * part + (is_v(p) ? 0 : 32);
      page[p] = at >= 0 && at < mine.hi ? c.wave_page(c.key(at)) : -1;
    }
  };
  auto load = [&](int kt) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int at = kt + 16 * part + (is_v(p) ? 0 : 32), key = c.key(at);
      const uint8_t* x = (is_v(p) ? c.v : c.k) + (page[p] < 0 ? 0 : page[p] * c.page_stride + (int64_t)((key & c.mask) * D)) +
                         (is_v(p) ? (lane >> 2) * D + (lane & 3) * 16 : (lane & 15) * D + (lane >> 4) * 16);
#pragma unroll
      for (int i = 0; i < M; ++i) codes[p][i] = *(const u4*)(x + 64 * i);
      byte[p] = page[p] < 0 ? -1 : (is_v(p) ? c.vs : c.ks)[c.scale_at(page[p], key)];
      there[p] = page[p] < 0 ? 0 : cut(mine.hi - at, 0, 16);
    }
  };
  auto write = [&](uint32_t to, const u4& w, float scale, uint32_t second) {  // 8 of 16 codes, the others `second` bytes on
    typedef __attribute__((address_space(3))) h8 l8;
    *(l8*)(uintptr_t)to = eight(w[0], w[1], scale);
    *(l8*)(uintptr_t)(to + second) = eight(w[2], w[3], scale);
  };
  // K: pieces of [16 keys][32 elements]; the second half of 16 codes lies 256 bytes further on. V: rows, pieces exchanged; the
  // second half lies in the next piece, for exchanges are multiples of 2
  const uint32_t kto = lds + part * 16 * kRowBytes + (lane >> 5) * 1024 + ((lane >> 4) & 1) * 512 + (lane & 15) * 16;
  uint32_t vto[M];
#pragma unroll
  for (int i = 0; i < M; ++i)
    vto[i] = lds + 2 * kBuf + (16 * part + (lane >> 2)) * kRowBytes + ((2 * (lane & 3) + 8 * i) ^ exchange<D>(lane >> 2)) * 16;
  // (the scale bytes of the half tile before the first lie in the other buffer too)
  auto store_k = [&](auto is_near, int p, uint32_t buf) {
    if (!decltype(is_near)::value && lane == 0) sh_scale[buf != 0][1][part] = byte[p];
    const float scale = scale_of(byte[p], kmost);
#pragma unroll
    for (int i = 0; i < M; ++i) write(kto + buf + 2048 * i, codes[p][i], scale, 256);
  };
  // some: not every row sees every key of the tile, so what V holds there must be finite
  auto store_v = [&](auto is_near, int p, uint32_t buf, bool some) {
    if (!decltype(is_near)::value && lane == 0) sh_scale[buf != 0][0][part] = byte[p];
    int said = there[p] > 0;  // that the keys have a page, and whether there were codes NaN
    if (some || there[p] < 16) {
      asm volatile("");  // a branch
      uint32_t odd = 0;
#pragma unroll
      for (int i = 0; i < M; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          codes[p][i][k] = (lane >> 2) < there[p] ? codes[p][i][k] : 0;
          odd |= nan_codes(codes[p][i][k]);
          codes[p][i][k] = without_nan(codes[p][i][k]);
        }
      if (__any(odd != 0)) said |= 2;
    }
    if (lane == 0) sh_said[buf != 0][part] = said;
    const float scale = scale_of(byte[p], vmost);
#pragma unroll
    for (int i = 0; i < M; ++i) write(vto[i] + buf, codes[p][i], scale, 16);
  };
  auto store = [&](auto is_near, uint32_t buf, bool some) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (is_v(p)) store_v(is_near, p, buf, some);
      else store_k(is_near, p, buf);
    }
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
  // ke, rest (not NEAR): what is left of the scales of K, beside the factor, and of V, of a block's first and last 16 keys
  auto weigh = [&](auto is_near, const float (&s)[16], const int (&ke)[2], const int (&rest)[2]) {
    constexpr bool NEAR = decltype(is_near)::value;
    const float base = m == -INFINITY ? 0.0f : F::kLift - m;
    float sum = 0.0f;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      float p[8];
      const int share = NEAR ? 0 : cut(rest[b] - level, kLeastShare, 0);
      const float f = NEAR ? factor : times2(factor, ke[b]), from = NEAR ? base : base + (float)share;
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(s[8 * b + j], f, from));
      const float part = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      sum += NEAR ? part : ldexpf(part, -share);
      parts(p, w[b]);
    }
    return sum;
  };
  auto top8 = [&](const float* s) {
    float top = s[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, s[j]);
    return top;
  };
  auto top_of = [&](auto is_near, const float (&s)[16], const int (&ke)[2]) {
    if constexpr (decltype(is_near)::value) {
      float top = s[0];
#pragma unroll
      for (int j = 1; j < 16; ++j) top = fmaxf(top, s[j]);
      return max_row<32>(top * factor);
    }
    return max_row<32>(fmaxf(top8(s) * times2(factor, ke[0]), top8(s + 8) * times2(factor, ke[1])));
  };
  // A block of 32 keys at `at` of the axis: their weights and what they add to the sums; beside it the products of
  // the next block, whose K lies at kat (behind the last: of what is there, unused). V lies at vat.
  // pages: bit x clear where keys 16 x of the block have no page; -1: every row sees every key. kbyte, vbyte: scales (not NEAR).
  auto block = [&](auto is_near, int at, uint32_t kat, uint32_t vat, int pages, bool odd, const int (&kbyte)[2], const int (&vbyte)[2],
                   float (&s)[16], float (&next)[16]) {
    constexpr bool NEAR = decltype(is_near)::value;
    if (pages >= 0) {
      const int kb = c.key(at) + 4 * g, end = c.key(at) + (mine.hi - at);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int key = kb + 8 * (j >> 2) + (j & 3);
        const bool sees = (uint32_t)(key - row_lo) < row_span || key < sink_end;
        s[j] = sees && key < end && (pages >> (j >> 3) & 1) ? s[j] : -INFINITY;
      }
    }
    int ke[2] = {0, 0}, rest[2] = {0, 0};
    float back = 1.0f;  // what the level's rise takes off the sums
    if constexpr (!NEAR) {
      int now = level;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ke[h] = kmost - 127 - kCodeLift + scale_rest(kbyte[h], kmost);
        rest[h] = scale_rest(vbyte[h], vmost);
        if (top8(s + 8 * h) > -INFINITY) now = max(now, rest[h]);
      }
      now = max(now, __shfl_xor(now, 32));
      back = ldexpf(1.0f, level - now);
      level = now;
    }
    if (fresh) {
      const float top = top_of(is_near, s, ke);
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
    float sum = weigh(is_near, s, ke, rest);
    // a weight beyond 2^15 (f16 holds 2^16), or many near it: the maximum moves
    if (__any(sum > 32768.0f || back != 1.0f)) {
      asm volatile("");  // a branch: the compiler would rather compute both
      const float now = fmaxf(m, top_of(is_near, s, ke));
      float by = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - now);  // a row that saw no key yet stays at 0
      m = now;
      l *= by;
      by *= back;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= by;
      sum = weigh(is_near, s, ke, rest);
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
      add_nan<D, Staged>(c, at, mine.hi, row_lo, row_lo + (int)row_span, (float*)o);
    }
  };
  // whether some row does not see some key of the 64 from `at` on, wherever they lie
  auto some_of = [&](int at) {
    bool all = true;
#pragma unroll
    for (int i = 0; i < 64; i += 32) {
      const int kb = c.key(at + i);
      all = all && (kb >= t.max_lo || kb + 32 <= c.sink) && kb + 32 <= t.min_hi;
    }
    return !all;
  };

  // Step i: the 64 keys from kt. V of tile i is used, and K of the keys 32 further on (the products run
  // one block ahead); V of tile i + 1 and its K go to LDS, those of tile i + 2 into the registers.
  auto go = [&](auto is_near) {
    constexpr bool NEAR = decltype(is_near)::value;
    const int n = (mine.hi - mine.lo + kTileKeys - 1) / kTileKeys;
    float s0[16], s1[16];
    int kb[2] = {0, 0};  // K's scale bytes of the scores in s0
    if (n > 0) {
      // the first 32 keys of K, in the other buffer: as if of a tile before
      pages(mine.lo - kTileKeys);
      load(mine.lo - kTileKeys);
      pages(mine.lo);
      if (!is_v(P - 1) && part >= 2) store_k(is_near, P - 1, kBuf - 32 * kRowBytes);
      load(mine.lo);
      pages(mine.lo + kTileKeys);
      store(is_near, 0, some_of(mine.lo));
      load(mine.lo + kTileKeys);
      pages(mine.lo + 2 * kTileKeys);
      __syncthreads();
      if constexpr (!NEAR) kb[0] = __builtin_amdgcn_readfirstlane(sh_scale[1][1][2]), kb[1] = __builtin_amdgcn_readfirstlane(sh_scale[1][1][3]);
      products(krow + kBuf, s0);
    }
    uint32_t buf = 0;
    for (int i = 0, kt = mine.lo; i < n; ++i, kt += kTileKeys, buf ^= kBuf) {
      // what tile i needs is in LDS, and all waves are done with tile i - 1
      __syncthreads();
      const u4 said = *(const u4*)sh_said[buf != 0];
      u4 vb = {0, 0, 0, 0}, kn = {0, 0, 0, 0};
      if constexpr (!NEAR) {
        vb = *(const u4*)sh_scale[buf != 0][0], kn = *(const u4*)sh_scale[buf != 0][1];
#pragma unroll
        for (int x = 0; x < 4; ++x) vb[x] = __builtin_amdgcn_readfirstlane(vb[x]), kn[x] = __builtin_amdgcn_readfirstlane(kn[x]);
      }
      if (i + 1 < n) {
        store(is_near, buf ^ kBuf, some_of(kt + kTileKeys));
        if (i + 2 < n) {
          load(kt + 2 * kTileKeys);
          pages(kt + 3 * kTileKeys);
        }
      }
      const int here = __builtin_amdgcn_readfirstlane((int)((said[0] & 1) | (said[1] & 1) << 1 | (said[2] & 1) << 2 | (said[3] & 1) << 3));
      const bool odd = __builtin_amdgcn_readfirstlane((int)((said[0] | said[1] | said[2] | said[3]) & 2)) != 0;
      const int pages = here != 15 || some_of(kt) ? here : -1;
      block(is_near, kt, krow + buf, vrow + buf, pages, odd, kb, {(int)vb[0], (int)vb[1]}, s0, s1);
      block(is_near, kt + 32, krow + buf + kBuf / 2, vrow + buf + kBuf / 2, pages < 0 ? -1 : pages >> 2, odd, {(int)kn[0], (int)kn[1]},
            {(int)vb[2], (int)vb[3]}, s1, s0);
      kb[0] = (int)kn[2], kb[1] = (int)kn[3];
    }
  };
  if (near) go(std::true_type{});
  else go(std::false_type{});

  const int64_t all = (int64_t)r.a.kv.n_tokens * r.a.n_heads;
  l += __shfl_xor(l, 32);
  const Row row = row_of(r, t, 32 * wave + col);
  if (!row.real) return;
  const float back = ldexpf(1.0f, vmost - 127 - kCodeLift + level);
  if (splits == 1) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    typename F::IO* out = (typename F::IO*)r.a.out + (int64_t)row.token * r.a.out_stride + row.head * D + 4 * g;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store4(out + 32 * d + 8 * i, f4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * inv * back);
  } else {
    const int64_t at = (int64_t)split * all + (int64_t)row.token * r.a.n_heads + row.head;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store4(r.part_o + at * D + 32 * d + 8 * i + 4 * g, f4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * back);
    if (g == 0) {
      r.part_ml[2 * at] = l == 0.0f ? -INFINITY : m;  // without a key: no maximum that the other splits' would fall behind
      r.part_ml[2 * at + 1] = l;
    }
  }
}

int fail(int rc, const char* why) {
  set_call_error(std::string("paged_attn_f8: ") + why);
  return rc;
}

template <class F, int D>
hipError_t run(const Args& r, const Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.tiles * r.a.kv.n_kv_heads * p.n_split));
  // Where there are no more than two workgroups for a CU, none takes a third: so much LDS is asked for that no more fit (one row
  // each of 64 sequences of up to 500 keys 14.9 us, without 16.4).
  const size_t lds = p.apart && !p.staged && p.tile_rows == 16 ? D == 64 ? 37 * 1024 : 21 * 1024 : 0;
  hipError_t e = p.staged            ? p.tile_rows == kChunkRows ? launch(k_paged_chunk_f8<F, D, 4>, grid, dim3(256), 0, s, r)
                                                             : launch(k_paged_chunk_f8<F, D, 8>, grid, dim3(512), 0, s, r)
                 : p.eight           ? launch(k_paged_rows_f8<F, D, 1, 8>, grid, dim3(512), 0, s, r)
                 : p.tile_rows == 16 ? launch(k_paged_rows_f8<F, D, 1>, grid, dim3(256), lds, s, r)
                                     : launch(k_paged_rows_f8<F, D, 2>, grid, dim3(256), 0, s, r);
  if (e == hipSuccess && p.n_split > 1 && !p.one_launch) e = run_join<typename F::IO, D, true>(r, p, s);
  return e;
}
template <class F>
hipError_t run(const Args& r, const Plan& p, hipStream_t s) {
  return r.a.kv.head_dim == 128 ? run<F, 128>(r, p, s) : run<F, 64>(r, p, s);
}

const char* refused(const mtg_paged_attn_f8& x, int* rc) {
  if (const char* why = attn::refused(x.a, true, rc)) return why;
  if (x.sink < 0 || x.sink > (1 << 30)) {
    *rc = MTG_ERR_INVALID;
    return "sink";
  }
  return nullptr;
}

// Without a window all positions are seen.
int sink_of(const mtg_paged_attn_f8& x) { return x.a.window > 0 ? x.sink : 0; }

}  // namespace
}  // namespace mtg

extern "C" size_t mtg_paged_attn_f8_workspace(const mtg_paged_attn_f8* a) {
  using namespace mtg;
  if (!a) return 0;
  mtg_paged_attn_f8 x = *a;  // sizes only: the pointers may not be there yet
  alignas(16) static const int32_t some[4] = {};
  x.a.kv.k = x.a.kv.v = (void*)some;
  x.a.kv.page_table = x.a.kv.kv_len = x.a.kv.q_start = some;
  int rc = 0;
  if (refused(x, &rc) || x.a.kv.n_seqs == 0 || x.a.kv.n_tokens == 0) return 0;
  return plan_of(x.a, sink_of(x)).bytes;
}

extern "C" int mtg_paged_attn_f8_dev(const mtg_paged_attn_f8* p, void* stream) {
  using namespace mtg;
  try {
    if (!p) return fail(MTG_ERR_INVALID, "no description");
    const mtg_paged_attn& a = p->a;
    const mtg_paged_kv& kv = a.kv;
    int rc = 0;
    if (const char* why = refused(*p, &rc)) return fail(rc, why);
    if (kv.n_seqs == 0 || kv.n_tokens == 0) return MTG_OK;
    const Plan plan = plan_of(a, sink_of(*p));
    if (const char* why = refused_arrays(a, plan, &rc, &p->scales)) return fail(rc, why);
    Args r;
    static_cast<AttnArgs&>(r) = args_of(a, plan);
    r.scales = p->scales;
    r.sink = sink_of(*p);
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = a.io_type == MTG_TYPE_F16 ? run<RowsF16>(r, plan, s) : run<RowsF32>(r, plan, s);
    if (e != hipSuccess) return fail(MTG_ERR_DEVICE, hipGetErrorString(e));
    return MTG_OK;
  } catch (...) {
    return MTG_ERR_NOMEM;
  }
}
