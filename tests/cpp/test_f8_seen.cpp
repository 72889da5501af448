// Which blocks of a cache in 8 bits some row of a tile sees (csrc/paged_kv.hpp), against all rows and keys one by one.
#include "../../moss-transcribe.cpp_amd/csrc/paged_kv.hpp"

#include <cstdio>
#include <random>

using namespace mtg::paged;

int main() {
  std::mt19937 rng(9);
  int failures = 0, unseen = 0;
  for (int turn = 0; turn < 20000; ++turn) {
    const int cap = 4096, window = rng() % 4 ? 1 + rng() % 300 : 0, sink = window ? rng() % (turn % 2 ? 400 : 20) : 0;
    const Rows rows{0, 1 + (int)(rng() % 40), (int)(rng() % 700) - 20};
    const int first = rng() % rows.n, last = first + rng() % (rows.n - first);
    int gap;
    const Keys keys = keys_of(rows, first, last, window, cap), axis = axis_of(keys, sink, &gap);
    const int oldest = oldest_of(rows.pos0 + first, window);
    for (int at = 0; at < axis.hi; at += MTG_F8_BLOCK) {
      const int block = key_at(at, sink, gap);
      bool seen = false;
      for (int key = block; key < block + MTG_F8_BLOCK; ++key)
        for (int i = first; i <= last; ++i) {
          const int pos = rows.pos0 + i;
          seen |= key <= pos && (!window || key > pos - window || key < sink);
        }
      unseen += !seen;
      if (block_seen(block, oldest, sink) != seen && ++failures < 20)
        std::fprintf(stderr, "block %d: rows %d to %d, window %d, sink %d\n", block, rows.pos0 + first, rows.pos0 + last, window, sink);
    }
  }
  if (unseen < 1000) ++failures;
  std::printf("{\"record\": \"f8Seen\", \"failures\": %d}\n", failures);
  return 0;
}
