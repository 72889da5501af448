// paged_attn_f8.hip - mtg_paged_attn_f8_dev: causal attention of the new rows of a batch over a cache in pages of e4m3
// codes with one power of two for 16 positions of a kv head; in a window, the first positions beside it.
//
// The tiles, layouts and running softmax are those of paged_attn.hip over an f16 cache: an e4m3 number is an f16
// number, and the instruction that turns two codes into two f16 numbers multiplies them by a power of two on the way. That
// power is the block's scale over the largest scale of the keys that the workgroup goes over (a look at all of their
// scales, a byte for 16 keys, comes first), so that what it takes off small blocks is far below the large ones'
// own steps: a code stays exact down to a scale of 2^-15 of the largest, and what is lost is 2^-25 of that at most. The
// largest scale itself goes into the factor of the scores and, at the end, of the sums.
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
  int sink, gap;
  __device__ __forceinline__ int key(int at) const { return key_at(at, sink, gap); }
  // Where the scale of a key in a page lies.
  __device__ __forceinline__ int64_t scale_at(int page, int key) const { return page * scale_stride + ((key & mask) / MTG_F8_BLOCK); }
};
__device__ __forceinline__ Codes codes_of(const Args& r, const Tile& t) {
  Codes c;
  static_cast<Cache<uint8_t>&>(c) = cache_of<uint8_t>(r, t.b, t.kvh);
  c.ks = r.scales.k + t.kvh * r.scales.head_stride;
  c.vs = r.scales.v + t.kvh * r.scales.head_stride;
  c.scale_stride = r.scales.page_stride;
  c.sink = r.sink, c.gap = t.gap;
  return c;
}

__device__ __forceinline__ int scale_byte(uint8_t b) { return b < 254 ? b : 254; }

// The largest scale bytes of k and v in the blocks of keys lo .. hi - 1 (lo a multiple of 16), by the lanes of a wave.
__device__ __forceinline__ void largest_scales(const Codes& c, const Keys& x, int* k, int* v) {
  int ek = 0, ev = 0;
  for (int at = x.lo + MTG_F8_BLOCK * (int)(threadIdx.x & 63); at < x.hi; at += MTG_F8_BLOCK * 64) {
    const int key = c.key(at), page = c.page(key, INT_MAX);
    if (page < 0) continue;
    ek = max(ek, scale_byte(c.ks[c.scale_at(page, key)]));
    ev = max(ev, scale_byte(c.vs[c.scale_at(page, key)]));
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    ek = max(ek, __shfl_xor(ek, m));
    ev = max(ev, __shfl_xor(ev, m));
  }
  *k = __builtin_amdgcn_readfirstlane(ek);
  *v = __builtin_amdgcn_readfirstlane(ev);
}

// The power of two of scale byte b over that of byte `most`; what lies 2^-40 below turns every code to 0.
__device__ __forceinline__ float over(int b, int most) { return __uint_as_float((uint32_t)(127 + cut(b - most, -40, 0)) << 23); }

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
    for (int i = 0; i < D * L::kRows / 64; ++i)
      if ((v[L::template dim<D>(i, g)] & 127) == 127) o[i] = NAN;
  }
}

// ---- few rows: 16 or 32 rows of one kv head, four waves (eight without splits) each with its own blocks of 32 keys ----
//
// HBM bounds it, and for short contexts the chain of dependent reads (sequence, page, keys). As in k_paged_rows K and V go from
// memory into the operands' registers; a lane reads 16 codes of a key, which are its parts of two score products (of the elements
// 64 c + 16 g .. each product takes 8), and D / 16 codes of 8 keys.
template <class F, int D, int RT, int NW = 4>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 2))) k_paged_rows_f8(Args r) {
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
  int kscale = 127, vscale = 127;  // bytes of what is held
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
    kscale = kpage < 0 ? -1 : c.ks[c.scale_at(kpage, key)];
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
  int kmost, vmost;
  largest_scales(c, mine, &kmost, &vmost);
  // (a block without a page: any scale, none of its codes takes part)
  auto scale_of = [](int b, int most) { return b < 0 ? 1.0f : over(min(b, 254), most); };
  Row row[RT];
  MV q[RT][NC][F::NQ];
  float factor[RT], m[RT], l[RT];
  f4 o[RT][DL];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    row[i] = row_of(r, t, 16 * i + col);
    load_row<F, D, 32>(r, row[i], q[i], &factor[i], [&](int k) { return 64 * (k >> 1) + 8 * (k & 1) + 8 * g; });
    factor[i] = fminf(fmaxf(ldexpf(factor[i], kmost - 127), 1.17549435e-38f), 3.0e38f);
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
      const float ks = scale_of(kscale, kmost);
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const MV p[1] = {eight(kr[a][k >> 1][2 * (k & 1)], kr[a][k >> 1][2 * (k & 1) + 1], ks)};
#pragma unroll
          for (int i = 0; i < RT; ++i) acc[i][a] = product(p, q[i][k], acc[i][a]);
        }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] = acc[i][j >> 2][j & 3];
    }
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
    for (int i = 0; i < RT; ++i) weights<DL>(s[i], factor[i], F::kLift, &m[i], &l[i], o[i]);
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
  const float back = ldexpf(1.0f, vmost - 127);
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int d = 0; d < DL; ++d) o[i][d] *= back;
  finish_rows<F, D, RT, NW>(r, t, tile, split, splits, m, l, o, sh_o, sh_ml);
}

int fail(int rc, const char* why) {
  set_call_error(std::string("paged_attn_f8: ") + why);
  return rc;
}

template <class F, int D>
hipError_t run(const Args& r, const Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.tiles * r.a.kv.n_kv_heads * p.n_split));
  hipError_t e = p.eight             ? launch(k_paged_rows_f8<F, D, 1, 8>, grid, dim3(512), 0, s, r)
                 : p.tile_rows == 16 ? launch(k_paged_rows_f8<F, D, 1>, grid, dim3(256), 0, s, r)
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
