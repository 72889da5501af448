// The rules for the scales of a cache in 8 bits (csrc/paged_kv.hpp): which blocks some row of a tile sees, against all rows and
// keys one by one, and codes as f16 numbers with what is left of their scale.
#include "../../moss-transcribe.cpp_amd/csrc/paged_kv.hpp"

#include <cmath>
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
  for (int most = 0; most <= 254; ++most)
    for (int byte = 0; byte <= most; ++byte) {
      const int e = code_exponent(byte, most), rest = scale_rest(byte, most);
      // from 448 down to 2^-9, four bits each: f16 numbers without a rounding
      const bool holds = 448.0 * std::ldexp(1.0, e) <= 65504.0 && e - 9 >= -24;
      const bool whole = e + rest == byte - most + kCodeLift;
      if ((!holds || !whole || rest > 0 || (rest == 0) != (most - byte <= kCodeSpan)) && ++failures < 20)
        std::fprintf(stderr, "byte %d of %d: %d %d\n", byte, most, e, rest);
    }
  for (int byte : {-1, 255}) {  // no page; counts as 254
    if (code_exponent(byte, 254) != (byte < 0 ? kCodeLift - kCodeSpan : kCodeLift) || scale_rest(255, 254) != 0) ++failures;
  }
  std::printf("{\"record\": \"f8Seen\", \"failures\": %d}\n", failures);
  return 0;
}
