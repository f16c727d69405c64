// Whether two matrices in memory share an element (host side; nothing of the device is needed).
#ifndef KALDI_AMD_CSRC_HIP_OVERLAP_H_
#define KALDI_AMD_CSRC_HIP_OVERLAP_H_

#include <stdint.h>

#include <algorithm>

namespace kh {

// `rows` rows of `cols` elements of 4 bytes, `ld` elements apart (an element of 8 bytes counts as two columns)
struct Area {
  const char *name;
  const void *p;
  long long rows, cols, ld;

  bool empty() const { return p == nullptr || rows <= 0 || cols <= 0; }
  // (one row is as long as its columns, whatever ld says)
  long long step() const { return 4 * (rows > 1 ? ld : cols); }
  uintptr_t begin() const { return (uintptr_t)p; }
  uintptr_t end() const { return begin() + (uintptr_t)((rows - 1) * step() + 4 * cols); }
};

// Exact: matrices that lie side by side in the rows of a larger one do not overlap.  Ranges of bytes that are apart, the usual
// case, cost two comparisons.
inline bool overlap(const Area &a, const Area &b) {
  if (a.empty() || b.empty() || a.end() <= b.begin() || b.end() <= a.begin()) return false;
  if (a.rows > b.rows) return overlap(b, a);
  // a's rows from the first that ends behind b's beginning: of b's rows that begin in front of its end, the last one ends last
  const long long first = b.begin() < a.begin() + 4 * a.cols ? 0 : (long long)((b.begin() - a.begin() - 4 * a.cols) / a.step() + 1);
  for (long long i = first; i < a.rows; ++i) {
    const uintptr_t from = a.begin() + (uintptr_t)(i * a.step()), to = from + (uintptr_t)(4 * a.cols);
    if (from >= b.end()) break;
    const long long j = std::min(b.rows - 1, (long long)((to - 1 - b.begin()) / b.step()));
    if (b.begin() + (uintptr_t)(j * b.step() + 4 * b.cols) > from) return true;
    if (a.step() == b.step()) break;  // (further rows lie as this one does)
  }
  return false;
}

}  // namespace kh
#endif
