// Whether arguments of a call share memory: matrices with a distance between their rows may lie in one another's gaps.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace b2 {

// `rows` rows of `row` bytes, `ld` bytes from one to the next. written: by the call.
struct Extent {
  const char* name;
  uintptr_t at;
  size_t rows, row, ld;
  bool written;
  uintptr_t end() const { return rows && row ? at + (rows - 1) * ld + row : at; }
};
inline Extent extent(const char* name, const void* p, size_t rows, size_t row, size_t ld, bool written) {
  return Extent{name, reinterpret_cast<uintptr_t>(p), p ? rows : 0, row, ld, written};
}

inline bool overlap(Extent a, Extent b) {
  if (a.at == a.end() || b.at == b.end() || a.end() <= b.at || b.end() <= a.at) return false;
  if (a.rows > b.rows) std::swap(a, b);
  if (a.rows > 1 && a.ld == b.ld) {
    // rows j of b and i of a lie D + (j - i) ld apart: the two k = j - i with the least distance
    const long long ld = (long long)a.ld, d = (long long)(b.at - a.at);
    const long long k0 = -(d / ld) - (d % ld > 0 ? 1 : 0);  // the last k with d + k ld <= 0
    for (long long k = k0; k <= k0 + 1; ++k) {
      const long long apart = d + k * ld;
      if (k <= (long long)b.rows - 1 && -k <= (long long)a.rows - 1 && apart < (long long)a.row && -apart < (long long)b.row) return true;
    }
    return false;
  }
  for (size_t i = 0; i < a.rows; ++i) {
    const uintptr_t from = a.at + i * a.ld, to = from + a.row;
    if (to <= b.at) continue;
    if (from >= b.end()) break;
    size_t j = from < b.at || b.rows == 1 ? 0 : (from - b.at) / b.ld;  // the last row of b that begins at `from` or before it, or the first one
    if (j > b.rows - 1) j = b.rows - 1;
    if (b.at + j * b.ld + b.row <= from) ++j;
    if (j < b.rows && b.at + j * b.ld < to) return true;
  }
  return false;
}

// The first pair among n extents that overlap, at least one of them written, in *a and *b. Sorts them.
inline bool any_overlap(Extent* x, int n, const Extent** a, const Extent** b) {
  std::sort(x, x + n, [](const Extent& p, const Extent& q) { return p.at < q.at; });
  for (int i = 0; i < n; ++i)
    for (int j = i + 1; j < n && x[j].at < x[i].end(); ++j)
      if ((x[i].written || x[j].written) && overlap(x[i], x[j])) {
        *a = x + i;
        *b = x + j;
        return true;
      }
  return false;
}

}  // namespace b2
