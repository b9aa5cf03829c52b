// Whether memory that is laid out in rows of evenly spaced parts meets itself or other such memory.  Host code, no CUDA.
//
// A layout is the bytes at + r row + o part + [0, inner) for r < rows and o < outer.  Two bytes ranges of layouts A and B meet where
//   -B.inner < (B.at - A.at) + dr row + do part < A.inner,
// so with equal strides only the differences dr and do count, and for one of them the other follows by a division: a few steps where one
// stride spans the other's range, which is what tensors have.  Strides that differ are walked through range by range.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace vsk {

struct Strided {
  int64_t at, rows, row, outer, part, inner;   // strides not negative, inner positive, last() within 64 bits
  int64_t in_row() const { return (outer - 1) * part + inner; }              // bytes from a row's first to behind its last
  int64_t last() const { return at + (rows - 1) * row + in_row(); }   // behind the last byte
};

namespace strided {

inline int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0 ? 1 : 0); }   // b > 0

// Whether some n of [n0, n1] has  lo < y + n stride < hi  (lo < hi).
inline bool some(int64_t y, int64_t stride, int64_t n0, int64_t n1, int64_t lo, int64_t hi) {
  if (n0 > n1) return false;
  if (stride == 0) return lo < y && y < hi;
  const int64_t n = std::max(n0, floor_div(lo - y, stride) + 1);   // the first one above lo
  return n <= n1 && y + n * stride < hi;
}

// Whether some n of [n0, n1] and m of [m0, m1], not both 0 if `other`, have  lo < y + n big + m small < hi.
inline bool some_pair(int64_t y, int64_t big, int64_t n0, int64_t n1, int64_t small, int64_t m0, int64_t m1, int64_t lo, int64_t hi, bool other) {
  if (big == 0) n0 = n1 = 0;
  if (small == 0) m0 = m1 = 0;
  if (big > 0) {   // those n that any m can bring into the range
    n0 = std::max(n0, floor_div(lo - y - m1 * small, big));
    n1 = std::min(n1, floor_div(hi - y - m0 * small, big) + 1);
  }
  for (int64_t n = n0; n <= n1; ++n) {
    const int64_t x = y + n * big;
    if (other && n == 0) {
      if (some(x, small, m0, -1, lo, hi) || some(x, small, 1, m1, lo, hi)) return true;
    } else if (some(x, small, m0, m1, lo, hi)) {
      return true;
    }
  }
  return false;
}

inline Strided plain(Strided a) {   // strides that move nothing are 0
  if (a.row == 0) a.rows = 1;
  if (a.part == 0) a.outer = 1;
  if (a.rows == 1) a.row = 0;
  if (a.outer == 1) a.part = 0;
  return a;
}

}  // namespace strided

// Whether two of its ranges meet.  (rows and outer as given: a stride of 0 under more than one of them does.)
inline bool meets_itself(const Strided& s) {
  if ((s.row == 0 && s.rows > 1) || (s.part == 0 && s.outer > 1)) return true;
  const Strided a = strided::plain(s);
  const bool rows_wide = a.row >= a.part;
  const int64_t big = rows_wide ? a.row : a.part, n = (rows_wide ? a.rows : a.outer) - 1;
  const int64_t small = rows_wide ? a.part : a.row, m = (rows_wide ? a.outer : a.rows) - 1;
  return strided::some_pair(0, big, 0, n, small, -m, m, -a.inner, a.inner, true);   // (-n, -m) says the same as (n, m)
}

inline bool meet(const Strided& one, const Strided& two) {
  if (one.at >= two.last() || two.at >= one.last()) return false;
  Strided a = strided::plain(one), b = strided::plain(two);
  // a stride that only one of them has may be the other's as well
  if (a.rows == 1) a.row = b.row;
  if (b.rows == 1) b.row = a.row;
  if (a.outer == 1) a.part = b.part;
  if (b.outer == 1) b.part = a.part;
  if (a.row == b.row && a.part == b.part) {
    const bool rows_wide = a.row >= a.part;
    const int64_t n0 = 1 - (rows_wide ? a.rows : a.outer), n1 = (rows_wide ? b.rows : b.outer) - 1;
    const int64_t m0 = 1 - (rows_wide ? a.outer : a.rows), m1 = (rows_wide ? b.outer : b.rows) - 1;
    return strided::some_pair(b.at - a.at, std::max(a.row, a.part), n0, n1, std::min(a.row, a.part), m0, m1, -b.inner, a.inner, false);
  }
  if (a.row != b.row && a.part == b.part) {   // the same with the names changed
    std::swap(a.row, a.part);
    std::swap(a.rows, a.outer);
    std::swap(b.row, b.part);
    std::swap(b.rows, b.outer);
  }
  if (a.row == b.row) {
    // periods of one length whose contents lie apart
    const int64_t period = a.row, in_a = (a.outer - 1) * a.part + a.inner, in_b = (b.outer - 1) * b.part + b.inner;
    if (period >= std::max(in_a, in_b)) {
      const int64_t d = (b.at - a.at) - strided::floor_div(b.at - a.at, period) * period;
      if (d >= in_a && d + in_b <= period) return false;
    }
    for (int64_t o = 0; o < a.outer; ++o)
      if (strided::some_pair(b.at - (a.at + o * a.part), period, 1 - a.rows, b.rows - 1, b.part, 0, b.outer - 1, -b.inner, a.inner, false)) return true;
    return false;
  }
  if (a.rows * a.outer > b.rows * b.outer) std::swap(a, b);
  for (int64_t r = 0; r < a.rows; ++r)
    for (int64_t o = 0; o < a.outer; ++o) {
      const int64_t y = b.at - (a.at + r * a.row + o * a.part);
      const bool rows_wide = b.row >= b.part;
      if (strided::some_pair(y, std::max(b.row, b.part), 0, (rows_wide ? b.rows : b.outer) - 1, std::min(b.row, b.part), 0, (rows_wide ? b.outer : b.rows) - 1,
                             -b.inner, a.inner, false))
        return true;
    }
  return false;
}

}  // namespace vsk
