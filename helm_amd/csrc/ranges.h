// Byte ranges of an entry point's operands: which outputs lie over what (host code).
#pragma once

#include <stdint.h>

namespace helm {

// `rows` rows of `bytes` bytes, `step` (>= bytes) apart.
struct Range {
  uintptr_t at;
  int64_t rows, bytes, step;
};
template <typename T>
Range range(const T* p, int64_t n, int64_t rows = 1, int64_t stride = 0) {
  const int64_t e = sizeof(T);
  return {reinterpret_cast<uintptr_t>(p), rows, n * e, (rows > 1 ? stride : n) * e};
}
// Whether a byte of x (one row) is one of y's.
inline bool overlap(const Range& x, const Range& y) {
  if (!x.bytes || !y.bytes || !y.rows || x.at + x.bytes <= y.at) return false;
  if (x.at < y.at + y.bytes) return true;
  const int64_t row = (int64_t)(x.at - y.at) / y.step;      // the last that starts at or before x
  if (row >= y.rows) return false;
  const int64_t in = (int64_t)(x.at - y.at) - row * y.step;
  return in < y.bytes || (row + 1 < y.rows && in + x.bytes > y.step);
}

}  // namespace helm
