// CPU check of mlc-vla_amd/csrc/rows.h: whether two strided arrays share a byte, against marking every byte, built with the
// address and undefined-behaviour sanitizers by tests/test_rows.py.
#include <cstdio>
#include <random>
#include <set>

#include "../mlc-vla_amd/csrc/rows.h"

using namespace mlcv;

struct Case {
  int64_t at, n1, s1, n2, s2, n;
};
static Rows rows(const Case& c) {
  return Rows(reinterpret_cast<const void*>((uintptr_t)c.at), c.n1, c.s1, c.n2, c.s2, c.n);
}
static std::set<int64_t> bytes(const Case& c) {
  std::set<int64_t> s;
  for (int64_t i = 0; i < c.n1; ++i)
    for (int64_t j = 0; j < c.n2; ++j)
      for (int64_t k = 0; k < c.n; ++k) s.insert(c.at + i * c.s1 + j * c.s2 + k);
  return s;
}

int main() {
  std::mt19937 rng(7);
  auto in = [&](int lo, int hi) { return lo + (int64_t)(rng() % (uint32_t)(hi - lo + 1)); };
  int failures = 0, met = 0;
  const int all = 300000;
  for (int i = 0; i < all; ++i) {
    Case c[2];
    for (Case& x : c) {
      x = {1000 + in(0, 60), in(0, 12), in(-40, 40), in(0, 5), in(-30, 30), in(0, 6)};
      if (i % 3 == 0) x.s2 = x.n * in(1, 2);        // heads that follow one another
      if (i % 5 == 0) x.s1 = c[0].s1 ? c[0].s1 : 7;  // the same stride of tokens
      if (i % 7 == 0) x.n1 = in(20, 60), x.n2 = 1, x.s1 = in(3, 25);  // long lines of different strides
    }
    const std::set<int64_t> a = bytes(c[0]), b = bytes(c[1]);
    bool want = false;
    for (int64_t v : a) want = want || b.count(v);
    const Rows x = rows(c[0]), y = rows(c[1]);
    met += want;
    if (rows_meet(x, y) != want || rows_meet(y, x) != want) {
      if (failures++ < 5)
        for (const Case& k : c)
          std::fprintf(stderr, "at %ld n1 %ld s1 %ld n2 %ld s2 %ld n %ld (want %d)\n", (long)k.at, (long)k.n1, (long)k.s1,
                       (long)k.n2, (long)k.s2, (long)k.n, want);
    }
  }
  // large ones: two halves of rows 2^40 bytes long in all, and strides past the address space
  const int64_t T = 1 << 30;
  const Case q{1 << 20, T, 1024, 1, 0, 512}, k{(1 << 20) + 512, T, 1024, 1, 0, 512}, o{(1 << 20) + 511, T, 1024, 1, 0, 512};
  const Case far{1 << 20, 1 << 30, INT64_MAX, 3, INT64_MIN, 512};
  failures += rows_meet(rows(q), rows(k)) + !rows_meet(rows(q), rows(o)) + !rows_meet(rows(far), rows(q));
  const Case slow{1 << 20, T, 1025, 1, 0, 1}, fast{(1 << 20) + 1023, T, 1024, 1, 0, 1};  // meet at token 1023
  failures += !rows_meet(rows(slow), rows(fast));
  const Case even{1 << 20, T, 1026, 1, 0, 1};  // odd bytes only against even ones
  failures += rows_meet(rows(even), rows(fast));
  std::printf("checked %d, %d share memory, failures: %d\n", all, met, failures);
  return failures ? 1 : 0;
}
