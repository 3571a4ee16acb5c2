// kh_rows.h — checks of rows that are given by strides (host code).
#pragma once
#include <stdint.h>

namespace khm {
// Elements of a row that is asked for by 16 bytes.
inline bool rows_whole(int64_t n, int esize) { return n % (16 / esize) == 0; }

// Rows of `size` elements, n[i] of them s[i] elements apart in dimension i of D: does every one lie beside the others?  By strides that lie
// within one another, the shorter ones' rows in a gap of the next: what several dimensions write then never meets.
template <int D>
inline bool rows_apart(const int64_t (&n)[D], const int64_t (&s)[D], int64_t size) {
  uint64_t extent = (uint64_t)size;
  bool used[D] = {};
  for (int k = 0; k < D; ++k) {
    int at = -1;
    uint64_t least = 0;
    for (int i = 0; i < D; ++i) {
      const uint64_t step = s[i] < 0 ? 0 - (uint64_t)s[i] : (uint64_t)s[i];
      if (n[i] <= 1 || used[i] || (at >= 0 && step >= least)) continue;
      at = i;
      least = step;
    }
    if (at < 0) return true;  // the others have one row
    if (least < extent) return false;
    used[at] = true;
    uint64_t more;
    if (__builtin_mul_overflow(least, (uint64_t)(n[at] - 1), &more) || __builtin_add_overflow(extent, more, &extent)) extent = UINT64_MAX;
  }
  return true;
}
}  // namespace khm
