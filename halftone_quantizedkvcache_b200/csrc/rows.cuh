// Rows of two strided dimensions in memory (tokens and heads, pages and heads), on the host: whether two
// arrays share a byte, and whether rows of one do.  What a kernel writes has rows of its own, apart from what
// it or another block may still read.
#pragma once

#include <algorithm>
#include <cstdint>
#include <cstdlib>

namespace hq {

struct Rows {
  const void* base;
  int64_t n[2];      // extents
  int64_t stride[2]; // bytes
  int64_t bytes;     // of a row
};
inline Rows rows_of(const void* base, int64_t n0, int64_t n1, int64_t stride0, int64_t stride1, int64_t bytes) {
  return Rows{base, {n0, n1}, {n0 > 1 ? stride0 : 0, n1 > 1 ? stride1 : 0}, bytes};
}
// [T, H, 128] of a 16-bit type, strides in elements
inline Rows packed_rows(const void* base, int64_t T, int64_t H, const int64_t stride[2]) {
  return rows_of(base, T, H, 2 * stride[0], 2 * stride[1], 256);
}
inline bool same_rows(const Rows& a, const Rows& b) {
  return a.base == b.base && a.n[0] == b.n[0] && a.n[1] == b.n[1] && a.stride[0] == b.stride[0] && a.stride[1] == b.stride[1];
}
// Whether -below < d + k s < above for a k of lo .. hi.
inline bool comes_near(int64_t d, int64_t s, int64_t lo, int64_t hi, int64_t below, int64_t above) {
  if (lo > hi) return false;
  auto hit = [&](int64_t k) { return -below < d + k * s && d + k * s < above; };
  if (s == 0) return hit(lo);
  const int64_t k = -d / s;  // d + k s is least in magnitude here or one beside it
  for (int64_t x = k - 1; x <= k + 1; ++x)
    if (hit(std::min(std::max(x, lo), hi))) return true;
  return false;
}
// Whether a row of a and one of b share a byte.  Exact; where one does not look it is that they share none, a few
// operations a pair of n[1], and times the smaller n[0] where the strides of n[0] differ.
inline bool rows_meet(const Rows& a, const Rows& b) {
  if (a.n[0] <= 0 || a.n[1] <= 0 || b.n[0] <= 0 || b.n[1] <= 0) return false;
  auto ends = [](const Rows& r, int64_t& from, int64_t& to) {
    from = to = reinterpret_cast<intptr_t>(r.base);
    for (int i = 0; i < 2; ++i) (r.stride[i] < 0 ? from : to) += (r.n[i] - 1) * r.stride[i];
    to += r.bytes;
  };
  int64_t a0, a1, b0, b1;
  ends(a, a0, a1);
  ends(b, b0, b1);
  if (a1 <= b0 || b1 <= a0) return false;
  const int64_t d = reinterpret_cast<intptr_t>(a.base) - reinterpret_cast<intptr_t>(b.base);
  const bool even = a.stride[0] == b.stride[0] || a.n[0] == 1 || b.n[0] == 1;
  if (a.stride[0] == b.stride[0] && a.stride[0] > 0 && a.stride[1] >= 0 && b.stride[1] >= 0) {
    // (columns of one array's rows)
    const int64_t s = a.stride[0], at = (d % s + s) % s;
    if (at >= (b.n[1] - 1) * b.stride[1] + b.bytes && at + (a.n[1] - 1) * a.stride[1] + a.bytes <= s) return false;
  }
  const Rows &few = a.n[0] <= b.n[0] ? a : b, &many = a.n[0] <= b.n[0] ? b : a;
  for (int64_t h = 0; h < a.n[1]; ++h)
    for (int64_t g = 0; g < b.n[1]; ++g) {
      const int64_t at = d + h * a.stride[1] - g * b.stride[1];  // a's row less b's
      if (even) {
        const int64_t s = a.n[0] == 1 ? b.stride[0] : a.stride[0];
        if (comes_near(at, s, 1 - b.n[0], a.n[0] - 1, a.bytes, b.bytes)) return true;
      } else {
        const int64_t x = &few == &a ? at : -at;                 // few's row less many's
        for (int64_t t = 0; t < few.n[0]; ++t)
          if (comes_near(x + t * few.stride[0], -many.stride[0], 0, many.n[0] - 1, few.bytes, many.bytes)) return true;
      }
    }
  return false;
}
// Whether two rows of a share a byte.
inline bool rows_meet(const Rows& a) {
  const int64_t s0 = std::abs(a.stride[0]), s1 = std::abs(a.stride[1]);
  if (a.n[0] > 1 && s0 < a.bytes) return true;
  if (a.n[0] <= 1 ? a.n[1] <= 1 || s1 >= a.bytes : s1 >= a.bytes && s0 >= (a.n[1] - 1) * s1 + a.bytes) return false;
  for (int64_t h = 1; h < a.n[1]; ++h)
    if (comes_near(h * a.stride[1], a.stride[0], 1 - a.n[0], a.n[0] - 1, a.bytes, a.bytes)) return true;
  return false;
}

}  // namespace hq
