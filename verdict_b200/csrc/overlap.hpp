// Whether two strided buffers share a byte.  Host only, exact for what the
// operators are given (rows at one or two strides, the outer one common to
// both, as views of one packed buffer have); otherwise it errs towards yes.
#pragma once

#include <algorithm>
#include <cstdint>
#include <numeric>
#include <utility>

namespace vd {

// n0 x n1 rows of `bytes`, s0 and s1 bytes apart; null: nothing.
struct ByteRows {
  const void* p = nullptr;
  int64_t bytes = 0, n0 = 1, s0 = 0, n1 = 1, s1 = 0;

  ByteRows() = default;
  ByteRows(const void* p, int64_t bytes) : p(p), bytes(bytes) {}
  ByteRows(const void* p, int64_t bytes, int64_t n0, int64_t s0, int64_t n1 = 1, int64_t s1 = 0)
      : p(p), bytes(bytes), n0(n0), s0(s0), n1(n1), s1(s1) {
    if (this->n0 <= 1 || s0 == 0) this->n0 = 1, this->s0 = 0;
    if (this->n1 <= 1 || s1 == 0) this->n1 = 1, this->s1 = 0;
    if (this->s0 < this->s1) std::swap(this->n0, this->n1), std::swap(this->s0, this->s1);  // s0: the outer stride
  }
  uintptr_t begin() const { return reinterpret_cast<uintptr_t>(p); }
  uintptr_t end() const { return begin() + static_cast<uintptr_t>((n0 - 1) * s0 + (n1 - 1) * s1 + bytes); }
};

// The same rows in the same order.
inline bool same_rows(const ByteRows& a, const ByteRows& b) {
  return a.p == b.p && a.bytes == b.bytes && a.n0 == b.n0 && a.s0 == b.s0 && a.n1 == b.n1 && a.s1 == b.s1;
}

inline bool overlap(const ByteRows& a, const ByteRows& b) {
  if (!a.p || !b.p || a.bytes <= 0 || b.bytes <= 0 || a.begin() >= b.end() || b.begin() >= a.end()) return false;
  const int64_t d = static_cast<int64_t>(b.begin() - a.begin());
  const int64_t s = std::max(a.s0, b.s0);
  if (s == 0) return true;  // one row each
  if ((a.n0 > 1 && a.s0 != s) || (b.n0 > 1 && b.s0 != s)) {
    // No outer stride in common: all rows of both lie on one lattice.
    int64_t g = 0;
    for (const int64_t t : {a.s0, a.s1, b.s0, b.s1}) g = std::gcd(g, t);
    const int64_t r = (d % g + g) % g;
    return r < a.bytes || g - r < b.bytes;
  }
  // A row of b that starts q after one of a, up to whole strides s: do any two
  // rows i of a and j of b with j - i = n meet, -a.bytes < q + n s < .. ?
  const auto meet = [&](int64_t q) {
    const int64_t r = (q % s + s) % s, n = (r - q) / s;
    return (r < a.bytes && n > -a.n0 && n < b.n0) || (s - r < b.bytes && n - 1 > -a.n0 && n - 1 < b.n0);
  };
  if (a.bytes > s || b.bytes > s) return true;  // rows that overlap themselves
  if (a.s1 == b.s1 || a.n1 == 1 || b.n1 == 1) {
    const int64_t t = std::max(a.s1, b.s1);
    for (int64_t k = -(a.n1 - 1); k < b.n1; ++k)
      if (meet(d + k * t)) return true;
    return false;
  }
  if (a.n1 * b.n1 > 65536) return true;
  for (int64_t i = 0; i < a.n1; ++i)
    for (int64_t j = 0; j < b.n1; ++j)
      if (meet(d + j * b.s1 - i * a.s1)) return true;
  return false;
}

}  // namespace vd
