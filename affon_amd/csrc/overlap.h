// Whether two operands share memory.
#pragma once

#include <algorithm>
#include <cstdint>

namespace affon {

// `rows` rows of `bytes` bytes, `stride` bytes apart (rows at stride 0: one).
struct Rows {
  const void* data;
  int64_t rows, bytes, stride;
};

inline Rows rows_of(const void* data, int64_t rows, int64_t bytes, int64_t stride) {
  return Rows{data, stride == 0 ? 1 : rows, bytes, stride};
}

inline bool same_rows(const Rows& a, const Rows& b) {
  return a.data == b.data && a.rows == b.rows && a.bytes == b.bytes && (a.rows == 1 || a.stride == b.stride);
}

// Whether any byte belongs to both. Columns of one wider tensor do not meet
// though their rows lie between each other, so that ranges alone do not tell.
inline bool rows_meet(const Rows& a, const Rows& b) {
  if (a.data == nullptr || b.data == nullptr || a.rows <= 0 || b.rows <= 0) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.data), pb = reinterpret_cast<uintptr_t>(b.data);
  const int64_t d = static_cast<int64_t>(pb - pa);  // from a's first byte to b's
  if (d >= (a.rows - 1) * a.stride + a.bytes || -d >= (b.rows - 1) * b.stride + b.bytes) return false;
  auto below = [](int64_t n, int64_t by) { return n / by - (n % by < 0); };  // floor(n / by)
  if (a.stride == b.stride && a.rows > 1 && b.rows > 1) {
    // Row j of b starts d + (j - i) stride after row i of a: the first such
    // difference that does not leave b's row behind a's.
    const int64_t k = std::max(below(-b.bytes - d, a.stride) + 1, 1 - a.rows);
    return k < b.rows && d + k * a.stride < a.bytes;
  }
  const Rows &few = a.rows <= b.rows ? a : b, &many = a.rows <= b.rows ? b : a;
  const int64_t off = a.rows <= b.rows ? d : -d;  // from few's first byte to many's
  for (int64_t i = 0; i < few.rows; ++i) {
    const int64_t at = i * few.stride - off;  // of this row after many's first byte
    const int64_t j = many.rows == 1 ? 0 : std::max<int64_t>(below(at - many.bytes, many.stride) + 1, 0);
    if (j < many.rows && j * many.stride < at + few.bytes && at < j * many.stride + many.bytes) return true;
  }
  return false;
}

}  // namespace affon
