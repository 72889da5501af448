// The search of a row's or a tile's sequence (csrc/paged_kv.hpp last_of) on the CPU, with 64 lanes as a loop, against
// a walk over all sequences: numbers of sequences around the powers of 64, many of them without rows.
#include <cstdio>
#include <random>
#include <vector>

#include "../../moss-transcribe.cpp_amd/csrc/paged_kv.hpp"

using namespace mtg::paged;

static int failures = 0;
static void expect(bool ok, const char* what, long a, long b, long c) {
  if (ok) return;
  ++failures;
  std::fprintf(stderr, "FAILED: %s (%ld, %ld, %ld)\n", what, a, b, c);
}

template <class P>
static int search(int n, const P& pred) {
  return last_of(n, [&](int lo, int step, int count) {
    uint64_t yes = 0;
    for (int lane = 0; lane < 64; ++lane) {
      const int off = lane * step;
      if (off < count && lo + off < n && pred(lo + off)) yes |= 1ull << lane;
      expect(off >= count || lo + off < n, "a candidate outside", lo, step, count);
    }
    return yes;
  });
}

int main() {
  std::mt19937 rng(5);
  std::vector<int> sizes = {1, 2, 63, 64, 65, 127, 128, 129, 4095, 4096, 4097, 70000, 262143, 262144, 262145, 1 << 20};
  for (int i = 0; i < 200; ++i) sizes.push_back(1 + (int)(rng() % 9000));
  for (int n : sizes) {
    std::vector<int32_t> start(1, (int)(rng() % 3));
    for (int b = 0; b < n; ++b) start.push_back(start.back() + (rng() % 3 == 0 ? (int)(rng() % 5) : 0));
    const int n_tokens = start.back() + 2;
    // the rows' sequences, in order; a row before the first one has none
    const int rows = n > 10000 ? 300 : n_tokens;
    for (int i = 0; i < rows; ++i) {
      const int t = n > 10000 ? (int)(rng() % n_tokens) : i;
      int want = -1;
      for (int lo = 0, hi = n; lo < hi;) {  // the number of starts at or before t
        const int mid = (lo + hi) / 2;
        if (start[mid] <= t) want = mid, lo = mid + 1;
        else hi = mid;
      }
      expect(search(n, [&](int b) { return start[b] <= t; }) == want, "a row's sequence", n, t, want);
      const int group = 1 + (int)(rng() % 8), tile = rng() % 2 ? 16 : 128, at = first_tile(t, want < 0 ? 0 : want, n_tokens, group, tile);
      const int found = search(n, [&](int b) { return first_tile(start[b], b, n_tokens, group, tile) <= at; });
      const int by_halves = seq_of(start.data(), n, n_tokens, group, tile, at);
      expect(found == by_halves || (found < 0 && by_halves == 0), "a tile's sequence", n, at, found);
    }
  }
  for (int n : {1, 64, 65, 5000}) {
    expect(search(n, [](int) { return false; }) == -1, "none", n, 0, 0);
    expect(search(n, [](int) { return true; }) == n - 1, "all", n, 0, 0);
  }
  std::printf("{\"record\": \"seqSearch\", \"failures\": %d}\n", failures);
  return failures != 0;
}
