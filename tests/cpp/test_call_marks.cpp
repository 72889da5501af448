// The marks of calls whose workgroups join in the same launch (csrc/paged_kv.hpp next_mark): no half is 0, since a
// joined call leaves zeros in its workspace and a captured one looks for the same mark again.
#include <cstdio>
#include <set>

#include "../../moss-transcribe.cpp_amd/csrc/paged_kv.hpp"

using mtg::paged::next_mark;

static int failures = 0;
static void expect(bool ok, const char* what, unsigned long long x) {
  if (ok) return;
  ++failures;
  std::fprintf(stderr, "FAILED: %s (%llx)\n", what, x);
}

// x with x ^ (x >> by) = y, and 1 / a mod 2^64
static uint64_t unshift(uint64_t y, int by) {
  uint64_t x = y;
  for (int done = by; done < 64; done += by) x = y ^ (x >> by);
  return x;
}
static uint64_t inverse(uint64_t a) {
  uint64_t x = a;
  for (int i = 0; i < 6; ++i) x *= 2 - a * x;
  return x;
}
// the counter from which splitmix64 makes `mark`
static uint64_t counter_of(uint64_t mark) {
  uint64_t x = unshift(mark, 31) * inverse(0x94d049bb133111ebull);
  x = unshift(x, 27) * inverse(0xbf58476d1ce4e5b9ull);
  return unshift(x, 30) - 0x9e3779b97f4a7c15ull;
}

int main() {
  const uint64_t whole = 0x123456789abcdef1ull;
  std::atomic<uint64_t> calls{counter_of(whole)};
  expect(next_mark(calls) == whole, "the counter of a mark", calls);
  for (uint64_t poor : {0ull, 1ull, 0xffffffffull, 0x12345678ull, 0x100000000ull, 0x1234567800000000ull, 0xffffffff00000000ull}) {
    calls = counter_of(poor);
    const uint64_t x = next_mark(calls);
    expect(x >> 32 && (uint32_t)x, "a mark with a half of 0", x);
  }
  std::set<uint64_t> seen;
  for (int i = 0; i < 100000; ++i) seen.insert(next_mark(calls));
  expect(seen.size() == 100000, "marks that differ", seen.size());
  std::printf("{\"record\": \"callMarks\", \"failures\": %d}\n", failures);
  return failures != 0;
}
