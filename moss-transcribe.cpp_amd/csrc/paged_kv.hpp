// paged_kv.hpp - where a new row's positions and a cached key lie in a pool of pages
// (mtg_paged_kv): the index rules of the rotary append and the paged attention, and the
// checks of a description. Plain functions, so that the host tests run the very rules the
// kernels use; every index that a kernel forms from an array's contents is cut here to what
// the description allows, so that no content of those arrays can lead out of the buffers.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>

#include "../../include/mtg_verify.h"

#ifdef __HIPCC__
#define MTG_HD __host__ __device__ __forceinline__
#else
#define MTG_HD inline
#endif

namespace mtg {
namespace paged {

// New rows row0 .. row0 + n - 1 of a sequence; row i has position pos0 + i (below 0: no place).
struct Rows {
  int row0, n, pos0;
};

MTG_HD int cut(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

MTG_HD Rows rows_of(int start, int end, int kv_len, int n_tokens) {
  Rows r;
  r.row0 = cut(start, 0, n_tokens);
  r.n = cut(end, r.row0, n_tokens) - r.row0;
  // a length below -2^30 has no meaning and would overflow the subtraction
  r.pos0 = (kv_len < -(1 << 30) ? -(1 << 30) : kv_len) - r.n;
  return r;
}

// Positions a table row can name. table_stride << shift fits 31 bits (checked on the host).
MTG_HD int capacity(int table_stride, int shift) { return table_stride << shift; }

// The page of a position, or -1: outside the table's row, or an id that is no page.
MTG_HD int page_of(const int32_t* table_row, int pos, int shift, int cap, int n_pages) {
  if (pos < 0 || pos >= cap) return -1;
  const int id = table_row[pos >> shift];
  return id >= 0 && id < n_pages ? id : -1;
}

// The keys of rows first .. last (positions pos0 + first .. pos0 + last): [lo, hi), lo down to
// a multiple of 32 so that the blocks of 32 keys that the kernels take never straddle a page
// in a group of 8.
struct Keys {
  int lo, hi;
};
// The oldest position that a row at `pos` sees (a window of 0 leaves nothing out).
MTG_HD int oldest_of(int pos, int window) { return window > 0 && pos >= window ? pos - window + 1 : 0; }
MTG_HD Keys keys_of(const Rows& r, int first, int last, int window, int cap) {
  Keys k;
  const int top = r.pos0 + last;
  k.hi = top < 0 ? 0 : top >= cap ? cap : top + 1;
  const int oldest = oldest_of(r.pos0 + first, window);
  k.lo = (oldest < k.hi ? oldest : k.hi) & ~31;
  return k;
}

// The axis of those keys where a row sees the first `sink` positions too: from key 0, without the *gap keys that lie between
// the sinks (up to a multiple of 32, as k.lo is one) and k.lo.
MTG_HD Keys axis_of(const Keys& k, int sink, int* gap) {
  const int s = (sink + 31) & ~31;
  *gap = k.lo > s ? k.lo - s : 0;
  return {0, k.hi - *gap};
}
// The key at a place of that axis.
MTG_HD int key_at(int at, int sink, int gap) { return at < ((sink + 31) & ~31) ? at : at + gap; }
// Whether some row of a tile sees one of the keys key .. key + MTG_F8_BLOCK - 1 (key a multiple of that, below the tile's
// last key): its rows see all keys from `oldest`, the first row's oldest, on, and those before `sink`. An axis' ends at multiples
// of 32 hold blocks that none sees, of pages that may be another sequence's by now.
MTG_HD bool block_seen(int key, int oldest, int sink) { return key + MTG_F8_BLOCK > oldest || key < sink; }

// The codes of a block as f16 numbers, code * 2^code_exponent: against the largest scale byte of the keys that a workgroup goes
// over, `most`, as far as an f16 number holds every code exactly (448 * 2^7 < 2^16, the least, 2^-9 * 2^(7 - 22), is 2^-24).
// code * 2^(byte - 127) = that number * 2^(scale_rest + most - 127 - kCodeLift); the rest is 0 in all blocks that lie no more
// than 22 below `most`. (Bytes above it, and -1, are of blocks that take no part.)
constexpr int kCodeLift = 7, kCodeSpan = 22;
MTG_HD int code_exponent(int byte, int most) { return kCodeLift + cut(byte - most, -kCodeSpan, 0); }
MTG_HD int scale_rest(int byte, int most) { return cut(byte - most + kCodeSpan, -255, 0); }

// Splits of a tile's keys: as many as its length fills, split_keys each, the last of at most
// n_split taking the rest.
MTG_HD int splits_of(const Keys& k, int split_keys, int n_split) {
  const int n = k.hi - k.lo;
  const int s = n / split_keys + (n % split_keys != 0);
  return cut(s, 1, n_split);
}
MTG_HD Keys split_keys_of(const Keys& k, int split, int split_keys, int splits) {
  Keys s;
  s.lo = k.lo + split * split_keys;
  s.hi = split + 1 < splits ? s.lo + split_keys : k.hi;
  return s;
}

// The first tile of sequence b where tiles of `tile` (row, head) pairs are counted over the
// whole batch: at least ceil(n * group / tile) tiles lie before the next sequence's first.
MTG_HD int first_tile(int start, int b, int n_tokens, int group, int tile) {
  return cut(start, 0, n_tokens) * group / tile + b;
}
inline int64_t tiles_bound(int n_tokens, int n_seqs, int group, int tile) {
  return (int64_t)n_tokens * group / tile + n_seqs;
}

// The largest i < n for which a condition holds that is true up to some i and false from there on (-1: nowhere). Each
// round looks at 64 candidates: bit x of ballot(lo, step, count) says that x step < count and that it holds at
// lo + x step.
template <class B>
MTG_HD int last_of(int n, const B& ballot) {
  int lo = 0, count = n;
  while (true) {
    const int step = (count + 63) >> 6;
    const uint64_t yes = ballot(lo, step, count);
    if (yes == 0) return -1;
    const int k = 63 - __builtin_clzll(yes);
    lo += k * step;
    count = count - k * step < step ? count - k * step : step;
    if (step == 1) return lo;
  }
}

// The last sequence whose first tile is at or before `tile`, by halving (what the kernels' search has to find).
inline int seq_of(const int32_t* q_start, int n_seqs, int n_tokens, int group, int rows, int tile) {
  int lo = 0, n = n_seqs;
  while (n > 1) {
    const int half = n / 2;
    if (first_tile(q_start[lo + half], lo + half, n_tokens, group, rows) <= tile) lo += half, n -= half;
    else n = half;
  }
  return lo;
}

// A number of 64 bits that no other call of the process has, and no workspace holds but by chance: 2^-64, or 2^-32
// where its halves are looked for in words of their own. Neither half is 0, which is what a joined call leaves behind.
inline uint64_t next_mark(std::atomic<uint64_t>& calls) {
  while (true) {
    uint64_t x = calls.fetch_add(1, std::memory_order_relaxed) + 0x9e3779b97f4a7c15ull;  // splitmix64: one to one
    x = (x ^ (x >> 30)) * 0xbf58476d1ce4e5b9ull;
    x = (x ^ (x >> 27)) * 0x94d049bb133111ebull;
    x ^= x >> 31;
    if (x >> 32 && (uint32_t)x) return x;
  }
}

// ---- checks of a description (host) ----
inline bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
inline int log2_of(int x) {
  int s = 0;
  while ((1 << s) < x) ++s;
  return s;
}
inline size_t type_bytes(int type) { return type == MTG_TYPE_F32 ? 4 : type == MTG_TYPE_F8_E4M3 ? 1 : 2; }

// Whether n steps of `stride` elements, the last one's start, stay within 2^46 elements (256 TB of f32): what no
// address space holds is refused, so that no extent below passes 63 bits.
inline bool reaches(int64_t n, int64_t stride) { return n <= 1 || stride <= ((int64_t)1 << 46) / (n - 1); }

// Whether blocks of `one` elements, one for each page and kv head, never reach into another.
inline bool apart_by(const mtg_paged_kv& kv, int64_t page_stride, int64_t head_stride, int64_t one) {
  const bool heads_inside = (kv.n_kv_heads == 1 || head_stride >= one) &&
                            (kv.n_pages == 1 || page_stride >= head_stride * (kv.n_kv_heads - 1) + one);
  const bool pages_inside = (kv.n_pages == 1 || page_stride >= one) &&
                            (kv.n_kv_heads == 1 || head_stride >= page_stride * (kv.n_pages - 1) + one);
  return heads_inside || pages_inside;
}

// Why the cache description cannot be used, or nullptr; *rc gets the status. with_cache: k and
// v are read or written (else only the rows and positions are). f8: a cache in 8 bits, else one of f32 or f16.
inline const char* check(const mtg_paged_kv& kv, bool with_cache, int* rc, bool f8 = false) {
  *rc = MTG_ERR_INVALID;
  if (kv.n_seqs < 0 || kv.n_tokens < 0) return "negative size";
  if (kv.n_kv_heads <= 0 || kv.n_kv_heads > 1024) return "n_kv_heads";
  if (kv.head_dim != 64 && kv.head_dim != 128) {
    *rc = MTG_ERR_UNSUPPORTED;
    return "head_dim is not 64 or 128";
  }
  if (kv.n_seqs > (1 << 20) || kv.n_tokens > (1 << 22)) {
    *rc = MTG_ERR_UNSUPPORTED;
    return "more than 2^20 sequences or 2^22 rows";
  }
  if (kv.n_seqs == 0 || kv.n_tokens == 0) return nullptr;  // nothing to do
  if (!kv.kv_len || !kv.q_start) return "kv_len or q_start is NULL";
  if (!aligned(kv.kv_len, 4) || !aligned(kv.q_start, 4)) return "unaligned index array";
  if (!with_cache) return nullptr;
  if (f8 ? kv.kv_type != MTG_TYPE_F8_E4M3 : kv.kv_type != MTG_TYPE_F32 && kv.kv_type != MTG_TYPE_F16) {
    *rc = MTG_ERR_UNSUPPORTED;
    return "cache type";
  }
  if (!kv.k || !kv.v || !kv.page_table) return "k, v or page_table is NULL";
  if (!aligned(kv.page_table, 4)) return "unaligned index array";
  if (kv.n_pages <= 0 || kv.table_stride <= 0) return "n_pages or table_stride";
  if (kv.page_size < 16 || kv.page_size > 65536 || (kv.page_size & (kv.page_size - 1))) {
    *rc = MTG_ERR_UNSUPPORTED;
    return "page_size is not a power of two, 16 to 65536";
  }
  if ((int64_t)kv.table_stride * kv.page_size > (1 << 30)) {
    *rc = MTG_ERR_UNSUPPORTED;
    return "a table row names more than 2^30 positions";
  }
  const int64_t unit = 16 / (int64_t)type_bytes(kv.kv_type), one = (int64_t)kv.page_size * kv.head_dim;
  if (!aligned(kv.k, 16) || !aligned(kv.v, 16) || kv.page_stride % unit || kv.head_stride % unit) {
    *rc = MTG_ERR_UNSUPPORTED;
    return "pages not aligned to 16 bytes";
  }
  if (kv.page_stride < 0 || kv.head_stride < 0 || kv.page_stride > ((int64_t)1 << 40) || kv.head_stride > ((int64_t)1 << 40) ||
      !reaches(kv.n_pages, kv.page_stride) || !reaches(kv.n_kv_heads, kv.head_stride))
    return "page_stride or head_stride";
  if (!apart_by(kv, kv.page_stride, kv.head_stride, one)) return "strides that make pages overlap";
  return nullptr;
}

// Bytes from the first to behind the last element of `rows` rows.
inline size_t extent(int64_t rows, int64_t stride, int64_t width, size_t bytes) {
  return rows <= 0 ? 0 : (size_t)((rows - 1) * stride + width) * bytes;
}
// Bytes from k (or v) to behind its last element.
inline size_t pool_extent(const mtg_paged_kv& kv) {
  return (size_t)(kv.page_stride * (kv.n_pages - 1) + kv.head_stride * (kv.n_kv_heads - 1) +
                  (int64_t)kv.page_size * kv.head_dim) * type_bytes(kv.kv_type);
}
inline bool overlap(const void* a, size_t an, const void* b, size_t bn) {
  return a && b && an && bn && (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an;
}

// Arrays of a call (nullptr: not there), and whether one of them shares a byte with n bytes at p.
struct Array {
  const void* at;
  size_t bytes;
};
inline bool meets(const void* p, size_t n, std::initializer_list<Array> others) {
  for (const Array& x : others)
    if (overlap(p, n, x.at, x.bytes)) return true;
  return false;
}

// Whether no block at k (`one` elements of eb bytes for each page and kv head) shares a byte with one at v: two pools,
// or one that holds both side by side, per page, per head, or per (page, head) block.
inline bool blocks_apart(const mtg_paged_kv& kv, const void* k, const void* v, int64_t page_stride, int64_t head_stride, int64_t one, int64_t eb) {
  const size_t pool = (size_t)(page_stride * (kv.n_pages - 1) + head_stride * (kv.n_kv_heads - 1) + one) * eb;
  if (!overlap(k, pool, v, pool)) return true;
  one *= eb;
  const int64_t gap = (int64_t)((uintptr_t)v - (uintptr_t)k);
  const bool heads_inside = head_stride <= page_stride;
  const int64_t in = (heads_inside ? head_stride : page_stride) * eb, out = (heads_inside ? page_stride : head_stride) * eb;
  const int64_t n = heads_inside ? kv.n_kv_heads : kv.n_pages;
  auto between = [&](int64_t stride, int64_t width) {
    if (stride <= 0) return false;
    const int64_t at = (gap % stride + stride) % stride;
    return at >= width && at + width <= stride;
  };
  return between(out, in * (n - 1) + one) || (in > 0 && out % in == 0 && between(in, one));
}
inline bool k_and_v_apart(const mtg_paged_kv& kv) {
  return blocks_apart(kv, kv.k, kv.v, kv.page_stride, kv.head_stride, (int64_t)kv.page_size * kv.head_dim, (int64_t)type_bytes(kv.kv_type));
}

// ---- the scales of a cache in 8 bits ----
inline size_t scale_extent(const mtg_paged_kv& kv, const mtg_f8_scales& s) {
  return (size_t)(s.page_stride * (kv.n_pages - 1) + s.head_stride * (kv.n_kv_heads - 1) + kv.page_size / MTG_F8_BLOCK);
}
// Why they cannot be used, or nullptr (of a cache that check() found right). written: by this call.
inline const char* check_scales(const mtg_paged_kv& kv, const mtg_f8_scales& s, bool written) {
  const int64_t one = kv.page_size / MTG_F8_BLOCK;
  if (!s.k || !s.v) return "scales are NULL";
  if (s.page_stride < 0 || s.head_stride < 0 || s.page_stride > ((int64_t)1 << 40) || s.head_stride > ((int64_t)1 << 40) ||
      !reaches(kv.n_pages, s.page_stride) || !reaches(kv.n_kv_heads, s.head_stride))
    return "page_stride or head_stride of the scales";
  if (!apart_by(kv, s.page_stride, s.head_stride, one)) return "strides that make scales overlap";
  const size_t pool = pool_extent(kv), n = scale_extent(kv, s);
  for (const uint8_t* x : {s.k, s.v})
    if (meets(x, n, {{kv.k, pool}, {kv.v, pool}})) return "scales lie in the pages";
  if (written && !blocks_apart(kv, s.k, s.v, s.page_stride, s.head_stride, one, 1)) return "scales of k and v share bytes";
  return nullptr;
}

// The first tile of sequence b where the blocks of positions that new rows lie in are counted over the whole batch: n rows
// touch (n + 14) / 16 + 1 blocks at most, and at least n / 16 + 2 tiles lie before the next sequence's first.
MTG_HD int first_block(int start, int b, int n_tokens) { return cut(start, 0, n_tokens) / MTG_F8_BLOCK + 2 * b; }
inline int64_t blocks_bound(int n_tokens, int n_seqs) { return (int64_t)n_tokens / MTG_F8_BLOCK + 2 * (int64_t)n_seqs; }

// The exponent of a block's scale by the bits of its largest finite |x| (0: none): the least e >= -100 with |x| <= 448 * 2^e.
MTG_HD int scale_exponent(uint32_t bits) {
  const int e = (int)(bits >> 23) - 135 + ((bits & 0x7fffffu) > 0x600000u);  // 448 = 1.75 * 2^8; bits of a subnormal say less than -100 too
  return e < -100 ? -100 : e;
}

}  // namespace paged
}  // namespace mtg
