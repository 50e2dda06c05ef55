// Which bytes the norms of rows that start anywhere copy (norm_sm100.cuh): plain integer code, kept apart from the CUDA sources
// so that a host-only checker can include it.
//
// A row is copied by whole granules of 16 bytes, whose bytes beyond the row belong to its neighbours.  Rows near either end of the
// matrix have none there: a granule may begin before the matrix or end behind it.  Of these only what lies inside the row is
// read, the rest of a granule element by element.
#pragma once

#include <cstdint>

namespace fsw {

// How many rows at either end of a matrix may share a granule with what lies outside it: one, unless rows are shorter than
// a granule.  Rows are at least `row_bytes` apart.
constexpr int edge_rows(int row_bytes) { return (14 + row_bytes) / row_bytes; }

// Of a row [begin, end): [lo, hi) goes by whole granules, the elements before and behind it one by one.  first, last: nothing
// before, behind the row may be read.
struct RowGranules {
  uint64_t granule, lo, hi;  // granule: where the row's first granule starts
  constexpr RowGranules(uint64_t begin, uint64_t end, bool first, bool last)
      : granule(begin & ~15ull), lo(first ? (begin + 15) & ~15ull : begin & ~15ull), hi(last ? end & ~15ull : (end + 15) & ~15ull) {}
  constexpr uint32_t bytes() const { return hi > lo ? static_cast<uint32_t>(hi - lo) : 0u; }
};

}  // namespace fsw
