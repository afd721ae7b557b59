// Operands that may not share memory (host code).
#pragma once

#include <stdint.h>

namespace glt {

// `rows` rows of `width` bytes, `ld` >= width bytes apart; one row for what is dense.
struct ByteRows {
  const void* at;
  int64_t rows, width, ld;
};
inline ByteRows dense_bytes(const void* p, int64_t n) { return {p, 1, n, n}; }

// Whether two operands share a byte. Columns of one buffer lie between each
// other's rows and share none.
inline bool overlap(const ByteRows& p, const ByteRows& q) {
  const int64_t d = static_cast<int64_t>(reinterpret_cast<uintptr_t>(q.at) - reinterpret_cast<uintptr_t>(p.at));
  if (p.rows <= 0 || q.rows <= 0 || p.width <= 0 || q.width <= 0) return false;
  if (d >= (p.rows - 1) * p.ld + p.width || -d >= (q.rows - 1) * q.ld + q.width) return false;
  if (p.ld == q.ld) {
    // q's row j starts r bytes into row j + k of p
    const int64_t r = ((d % p.ld) + p.ld) % p.ld, k = (d - r) / p.ld;
    auto meets = [&](int64_t by) { return by > -q.rows && by < p.rows; };  // some row j + by is p's
    return (r < p.width && meets(k)) || (r + q.width > p.ld && meets(k + 1));
  }
  if (p.rows > q.rows) return overlap(q, p);
  for (int64_t i = 0; i < p.rows; ++i) {
    const int64_t from = i * p.ld - d, to = from + p.width;  // from q.at
    const int64_t j = from < q.width ? 0 : (from - q.width) / q.ld + 1;  // q's first row that ends behind from
    if (j < q.rows && j * q.ld < to) return true;
  }
  return false;
}

}  // namespace glt
