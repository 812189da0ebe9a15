// Which memory the arguments of a call share: rows of equal length at a stride, compared in pairs.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>

namespace memt {

// `rows` rows of `width` bytes, `stride` >= width bytes from one to the next; null: none.
struct Rows {
  uintptr_t at;
  uint64_t width, stride, rows;
  Rows(const void* p, int64_t width_, int64_t stride_, int64_t rows_)
      : at(reinterpret_cast<uintptr_t>(p)), width(width_), stride(stride_), rows(p == nullptr ? 0 : rows_) {
    if (width == stride) {  // one run of memory
      width *= rows;
      rows = width > 0 ? 1 : 0;
    }
  }
  Rows(const void* p, int64_t bytes) : Rows(p, bytes, bytes, 1) {}
  uintptr_t end() const { return at + (rows - 1) * stride + width; }
};

// Whether two of them may share a byte: exact for runs and for rows of one stride (columns of one wider
// buffer); rows of different strides within one another's reach count as sharing.
inline bool overlap(const Rows& a, const Rows& b) {
  if (a.rows == 0 || b.rows == 0 || a.end() <= b.at || b.end() <= a.at) return false;
  if (a.rows == 1 && b.rows == 1) return true;
  if (a.rows == 1) return overlap(b, a);
  if (b.rows == 1) {  // the row that begins at or before the run, and the next one
    if (b.at < a.at) return true;
    const uint64_t row = (b.at - a.at) / a.stride, off = (b.at - a.at) % a.stride;
    return (row < a.rows && off < a.width) || (row + 1 < a.rows && off + b.width > a.stride);
  }
  if (a.stride != b.stride) return true;
  const uint64_t off =
      b.at >= a.at ? (b.at - a.at) % a.stride : (a.stride - (a.at - b.at) % a.stride) % a.stride;
  return off < a.width || off + b.width > a.stride;
}

inline bool overlaps_any(const Rows& a, std::initializer_list<Rows> others) {
  for (const Rows& b : others)
    if (overlap(a, b)) return true;
  return false;
}

}  // namespace memt
