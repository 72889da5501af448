// The index rules of a cache in 8 bits (csrc/paged_kv.hpp): every block that new rows lie in has a tile of its own, a
// block's scale is the least that holds its largest element, and which scales share bytes.
#include "../../moss-transcribe.cpp_amd/csrc/paged_kv.hpp"

#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

using namespace mtg::paged;

static int failures = 0;
#define CHECK(x)                                                        \
  do {                                                                  \
    if (!(x)) {                                                         \
      if (++failures < 20) std::fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #x); \
    }                                                                   \
  } while (0)

int main() {
  std::mt19937 rng(3);
  for (int turn = 0; turn < 2000; ++turn) {
    const int seqs = 1 + rng() % 9;
    std::vector<int> start{(int)(rng() % 3)}, pos;
    for (int b = 0; b < seqs; ++b) {
      start.push_back(start.back() + (int)(rng() % (turn % 2 ? 60 : 4)));
      pos.push_back((int)(rng() % 70) - 5);
    }
    const int n_tokens = start.back() + rng() % 3;
    for (int b = 0; b < seqs; ++b) {
      const int n = start[b + 1] - start[b];
      const int first = first_block(start[b], b, n_tokens), next = first_block(start[b + 1], b + 1, n_tokens);
      const int blocks = n ? ((pos[b] + n - 1) >> 4) - (pos[b] >> 4) + 1 : 0;
      CHECK(first + blocks <= next);
      CHECK(next <= blocks_bound(n_tokens, seqs));
    }
  }
  for (int i = 0; i < 200000; ++i) {
    uint32_t bits = rng() & 0x7fffffffu;
    if (i < 600) bits = ((uint32_t)(i / 3 + 20) << 23 | 0x600000u) + (i % 3) - 1;  // around 1.75 * 2^x
    if (bits >= 0x7f800000u) continue;
    float f;
    std::memcpy(&f, &bits, 4);
    const int e = scale_exponent(bits);
    CHECK(e >= -100 && e <= 120 && (double)f <= 448.0 * std::ldexp(1.0, e));
    CHECK(e == -100 || (double)f > 448.0 * std::ldexp(1.0, e - 1));
  }
  CHECK(scale_exponent(0) == -100);

  // the axis of a tile whose rows see the first keys too: every key that some row sees once, in order, blocks of 32 whole
  for (int turn = 0; turn < 20000; ++turn) {
    const int cap = 4096, window = rng() % 3 ? 1 + rng() % 300 : 0, sink = window ? rng() % (turn % 2 ? 400 : 5) : 0;
    Rows rows{0, 1 + (int)(rng() % 40), (int)(rng() % 700) - 20};
    const int first = rng() % rows.n, last = first + rng() % (rows.n - first);
    int gap;
    const Keys keys = keys_of(rows, first, last, window, cap), axis = axis_of(keys, sink, &gap);
    CHECK(axis.lo == 0 && axis.hi >= 0 && gap >= 0 && gap % 32 == 0 && axis.hi + gap == keys.hi);
    std::vector<char> on(cap, 0);
    for (int at = 0; at < axis.hi; ++at) {
      const int key = key_at(at, sink, gap);
      CHECK(key >= 0 && key < keys.hi && !on[key] && key == key_at(at & ~31, sink, gap) + (at & 31));
      on[key] = 1;
    }
    for (int i = first; i <= last; ++i)
      for (int key = 0; key <= rows.pos0 + i && key < cap; ++key)
        if (key >= oldest_of(rows.pos0 + i, window) || key < sink) CHECK(on[key]);
  }

  mtg_paged_kv kv{};
  std::vector<uint8_t> pool(1 << 16), scales(1 << 12);
  kv.k = pool.data(), kv.v = pool.data() + 8192;
  kv.page_size = 32, kv.n_pages = 2, kv.n_kv_heads = 2, kv.head_dim = 64, kv.head_stride = 2048, kv.page_stride = 4096;
  kv.kv_type = MTG_TYPE_F8_E4M3;
  mtg_f8_scales s{scales.data(), scales.data() + 8, 4, 2};
  CHECK(scale_extent(kv, s) == 8 && !check_scales(kv, s, true));
  s.v = scales.data() + 7;  // the last of k's
  CHECK(check_scales(kv, s, true) && !check_scales(kv, s, false));
  s = {scales.data(), scales.data() + 4, 8, 2};  // k and v in turns, page by page
  CHECK(!check_scales(kv, s, true));
  s = {scales.data(), scales.data() + 2, 8, 4};  // head by head
  CHECK(!check_scales(kv, s, true));
  s = {scales.data(), scales.data() + 100, 1, 2};
  CHECK(check_scales(kv, s, true));
  s = {scales.data(), pool.data() + 8191, 4, 2};
  CHECK(check_scales(kv, s, true) && check_scales(kv, s, false));
  s = {nullptr, scales.data(), 4, 2};
  CHECK(check_scales(kv, s, true));
  s = {scales.data(), scales.data() + 100, -4, 2};
  CHECK(check_scales(kv, s, true));
  s = {scales.data(), scales.data() + 100, (int64_t)1 << 62, 2};
  CHECK(check_scales(kv, s, true));
  std::printf("{\"record\": \"pagedF8\", \"failures\": %d}\n", failures);
  return 0;
}
