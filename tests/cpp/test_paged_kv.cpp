// The index rules of the paged operators (csrc/paged_kv.hpp) on the CPU: every page id, length and
// start that an array may hold leads to a place inside the buffers or to none, and the splits of a
// tile's keys cover what its rows see, once.
#include <climits>
#include <cstdio>
#include <random>
#include <vector>

#include "../../moss-transcribe.cpp_amd/csrc/paged_kv.hpp"

using namespace mtg::paged;

static int failures = 0;
static void expect(bool ok, const char* what, long a = 0, long b = 0) {
  if (ok) return;
  ++failures;
  std::fprintf(stderr, "FAILED: %s (%ld, %ld)\n", what, a, b);
}

static void pages() {
  const int32_t row[4] = {2, -1, 3, INT_MIN};
  const int shift = 4, n_pages = 3, cap = capacity(4, shift);
  expect(cap == 64, "capacity");
  expect(page_of(row, 0, shift, cap, n_pages) == 2 && page_of(row, 15, shift, cap, n_pages) == 2, "a page");
  const int none[] = {-1, INT_MIN, 16, 31, 32, 47, 48, 63, 64, INT_MAX};
  for (int p : none) expect(page_of(row, p, shift, cap, n_pages) == -1, "no page", p);
  const int32_t last[1] = {INT_MAX};
  expect(page_of(last, 3, 4, 16, n_pages) == -1, "an id far outside");
}

static void rows() {
  const int values[] = {INT_MIN, -5, 0, 3, 7, 9, INT_MAX};
  for (int s : values)
    for (int e : values)
      for (int len : values) {
        const Rows r = rows_of(s, e, len, 8);
        expect(r.row0 >= 0 && r.n >= 0 && r.row0 + r.n <= 8, "rows inside", s, e);
        for (int window : {0, 1, 5, INT_MAX})
          for (int first = 0; first < r.n; ++first) {
            const Keys k = keys_of(r, first, r.n - 1, window, 64);
            expect(k.lo >= 0 && k.lo <= k.hi && k.hi <= 64 && k.lo % 32 == 0, "keys inside", k.lo, k.hi);
            expect(oldest_of(r.pos0 + first, window) >= 0, "oldest", len, window);
          }
      }
}

// Tiles of a batch: every (token, head) pair of every sequence in exactly one tile.
static void tiles(std::mt19937& rng) {
  for (int round = 0; round < 300; ++round) {
    const int n_seqs = 1 + (int)(rng() % 9), group = 1 + (int)(rng() % 9), tile = rng() % 2 ? 16 : 128;
    std::vector<int32_t> start(1, (int)(rng() % 3));
    for (int b = 0; b < n_seqs; ++b) start.push_back(start.back() + (rng() % 3 ? (int)(rng() % 70) : 0));
    const int n_tokens = start.back() + (int)(rng() % 3);
    std::vector<int> seen((size_t)n_tokens * group, 0);
    const int64_t bound = tiles_bound(n_tokens, n_seqs, group, tile);
    for (int t = 0; t < bound; ++t) {
      const int b = seq_of(start.data(), n_seqs, n_tokens, group, tile, t);
      const Rows r = rows_of(start[b], start[b + 1], 100, n_tokens);
      const int first = (t - first_tile(start[b], b, n_tokens, group, tile)) * tile;
      if (first < 0) continue;  // before the first sequence
      for (int i = first; i < first + tile && i < r.n * group; ++i) ++seen[(size_t)r.row0 * group + i];
    }
    for (int i = 0; i < n_tokens * group; ++i)
      expect(seen[i] == (i >= start[0] * group && i < start.back() * group), "a pair's tiles", i, seen[i]);
  }
}

static void splits(std::mt19937& rng) {
  for (int round = 0; round < 2000; ++round) {
    const int n = 1 + (int)(rng() % 40), len = (int)(rng() % 5000), window = rng() % 2 ? (int)(rng() % 600) : 0;
    const int cap = 16 << (rng() % 9), per = 128 * (1 + (int)(rng() % 8)), most = 1 + (int)(rng() % 9);
    const Rows r = rows_of(0, n, len, 64);
    const int first = (int)(rng() % n), last = first + (int)(rng() % (n - first));
    const Keys k = keys_of(r, first, last, window, cap);
    const int s = splits_of(k, per, most);
    int at = k.lo;
    for (int i = 0; i < s; ++i) {
      const Keys x = split_keys_of(k, i, per, s);
      expect(x.lo == at && x.hi >= x.lo && x.lo % 32 == 0, "splits in a row", x.lo, at);
      at = x.hi;
    }
    expect(at == k.hi, "splits cover", at, k.hi);
    for (int i = first; i <= last; ++i) {
      const int pos = r.pos0 + i;
      if (pos < 0) continue;
      expect(k.lo <= oldest_of(pos, window) || oldest_of(pos, window) >= k.hi, "oldest key of a row", pos, k.lo);
      expect(k.hi >= (pos < cap ? pos + 1 : cap), "newest key of a row", pos, k.hi);
    }
  }
}

static void strides() {
  alignas(16) static char mem[1];
  mtg_paged_kv kv{};
  kv.k = mem;
  kv.v = mem + (1 << 20);
  kv.page_table = kv.kv_len = kv.q_start = (const int32_t*)mem;
  kv.kv_type = MTG_TYPE_F16;
  kv.n_pages = 6, kv.page_size = 16, kv.table_stride = 3, kv.n_seqs = 1, kv.n_tokens = 1, kv.n_kv_heads = 4, kv.head_dim = 64;
  const int64_t one = 16 * 64;
  int rc = 0;
  const struct {
    int64_t page, head;
    bool ok;
  } cases[] = {{4 * one, one, true}, {one, 6 * one, true}, {4 * one + 8, one, true}, {8 * one, 2 * one, true},
               {4 * one - 8, one, false}, {one, one, false}, {one, 5 * one, false}, {0, one, false},
               {4 * one, one - 8, false}, {-4 * one, one, false}, {(int64_t)1 << 41, one, false}, {INT64_MAX - 7, INT64_MAX - 7, false}};
  for (const auto& c : cases) {
    kv.page_stride = c.page, kv.head_stride = c.head;
    expect((check(kv, true, &rc) == nullptr) == c.ok, "strides", (long)c.page, (long)c.head);
  }
  // k and v side by side in one pool
  auto apart = [&](int64_t page, int64_t head, int64_t gap) {
    kv.page_stride = page, kv.head_stride = head;
    kv.v = (char*)kv.k + 2 * gap;
    return k_and_v_apart(kv);
  };
  expect(apart(8 * one, one, 4 * one), "k and v per page");
  expect(apart(8 * one, 2 * one, one), "k and v per block");
  expect(apart(8 * one, one, -4 * one), "v before k");
  expect(apart(4 * one, one, 24 * one), "two pools");
  expect(!apart(4 * one, one, 0), "one pool");
  expect(!apart(8 * one, one, 3 * one), "heads shared");
  expect(!apart(4 * one, one, 4 * one), "pages shared");
  expect(!apart(8 * one, 2 * one, 8), "blocks shared");
}

int main() {
  std::mt19937 rng(11);
  pages();
  rows();
  tiles(rng);
  splits(rng);
  strides();
  std::printf("{\"record\": \"pagedKv\", \"failures\": %d}\n", failures);
  return failures != 0;
}
