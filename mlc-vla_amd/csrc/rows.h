// Whether two strided arrays of a call share memory: for outputs that must not lie over inputs or one another.  Host only.
#pragma once

#include <cstdint>
#include <utility>

namespace mlcv {

// n1 x n2 rows of n bytes each, s1 and s2 bytes apart (any sign) from `at` on
struct Rows {
  typedef __int128 Int;
  Int p, end;  // all of them
  int64_t n1, n2;
  Int s1, s2, n;
  Rows(const void* at, int64_t n1, Int s1, int64_t n2, Int s2, Int n)
      : p((Int)reinterpret_cast<uintptr_t>(at)), n1(n1), n2(n2), s1(s1), s2(s2), n(at && n1 > 0 && n2 > 0 ? n : 0) {
    flat(this->p, this->n1, this->s1);
    flat(this->p, this->n2, this->s2);
    // rows that follow one another are one
    for (int i = 0; i < 2; ++i) {
      if (this->n2 > 1 && this->s2 == this->n) this->n *= this->n2, this->n2 = 1, this->s2 = 0;
      if (this->n1 > 1 && this->s1 == this->n) this->n *= this->n1, this->n1 = 1, this->s1 = 0;
    }
    if (this->n1 < this->n2) std::swap(this->n1, this->n2), std::swap(this->s1, this->s2);
    end = p + (this->n1 - 1) * this->s1 + (this->n2 - 1) * this->s2 + this->n;
  }
  Rows(const void* at, int64_t bytes) : Rows(at, 1, 0, 1, 0, bytes) {}

 private:
  static void flat(Int& p, int64_t& n, Int& s) {  // strides of 0 or more
    if (n <= 1 || s == 0) n = 1, s = 0;
    if (s < 0) p += (n - 1) * s, s = -s;
  }
};

// The least x >= 0 with l <= a x mod m <= r (0 < l <= r < m, 0 <= a < m); -1 if there is none.  As in Euclid's algorithm: where
// no multiple of a is in the range, a x - m y is for the least y with m y mod a in the range's negative.
inline Rows::Int first_within(Rows::Int a, Rows::Int m, Rows::Int l, Rows::Int r) {
  if (a == 0) return -1;
  if (2 * a > m) return first_within(m - a, m, m - r, m - l);
  const Rows::Int x = (l + a - 1) / a;
  if (a * x <= r) return x;
  const Rows::Int y = first_within(m % a, a, a - r % a, a - l % a);
  return y < 0 ? -1 : (l + m * y + a - 1) / a;
}

// Whether rows of a bytes, sa apart, share a byte with rows of b bytes, sb apart, whose first begins d bytes before theirs
inline bool lines_meet(Rows::Int d, int64_t na, Rows::Int sa, Rows::Int a, int64_t nb, Rows::Int sb, Rows::Int b) {
  typedef Rows::Int Int;
  if (nb == 1) {
    if (na == 1) return -a < d && d < b;
    return lines_meet(-d, nb, sb, b, na, sa, a);
  }
  // row t of the one and u of the other share one where 0 <= v - u sb <= w, with
  const Int v0 = d + a - 1, w = a + b - 2;  // v = v0 + t sa
  const Int most = (nb - 1) * sb + w - v0;  // t sa at most, for the last u
  const Int t0 = v0 >= 0 ? 0 : sa ? (-v0 + sa - 1) / sa : na;
  if (most < 0 || t0 >= na) return false;
  const Int t1 = sa && most / sa < na - 1 ? most / sa : (Int)(na - 1);
  if (t0 > t1) return false;
  if (v0 + t1 * sa >= nb * sb) return true;  // the last u
  const Int at = (v0 + t0 * sa) % sb;
  if (at <= w) return true;
  const Int x = first_within(sa % sb, sb, sb - at, sb - at + w);
  return x >= 0 && x <= t1 - t0;
}

inline bool rows_meet(const Rows& a, const Rows& b) {
  if (a.n <= 0 || b.n <= 0 || a.end <= b.p || b.end <= a.p) return false;
  // no memory is that large; below, no product passes 127 bits
  if (a.end - a.p > (Rows::Int)1 << 62 || b.end - b.p > (Rows::Int)1 << 62) return true;
  for (int64_t i = 0; i < a.n2; ++i)
    for (int64_t j = 0; j < b.n2; ++j)
      if (lines_meet(a.p + i * a.s2 - b.p - j * b.s2, a.n1, a.s1, a.n, b.n1, b.s1, b.n)) return true;
  return false;
}

// Whether one of the first `outs` arrays shares memory with any other
inline bool any_meet(const Rows* r, int outs, int all) {
  for (int i = 0; i < outs; ++i)
    for (int j = i + 1; j < all; ++j)
      if (rows_meet(r[i], r[j])) return true;
  return false;
}

}  // namespace mlcv
