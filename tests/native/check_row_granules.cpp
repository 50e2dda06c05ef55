// Host-only check of what the norms of rows that start anywhere copy (csrc/row_granules.h): for every alignment, width, pitch and
// row count, all that is read lies inside the matrix, every element of a row is read, and a row's granules fit their place.
#include <cstdio>

#include "row_granules.h"

namespace {

bool fail(const char* what, int size, int base, int d, int pitch, int M, int row) {
  std::printf("%s: size %d base %d d %d pitch %d M %d row %d\n", what, size, base, d, pitch, M, row);
  return false;
}

bool check(int size, int base, int d, int pitch, int M) {
  const int edge = fsw::edge_rows(d * size);
  const uint64_t first_byte = 4096 + base, end_byte = first_byte + static_cast<uint64_t>((M - 1) * pitch + d) * size;
  for (int row = 0; row < M; ++row) {
    const uint64_t begin = first_byte + static_cast<uint64_t>(row) * pitch * size, end = begin + static_cast<uint64_t>(d) * size;
    const bool first = row < edge, last = row >= M - edge;
    const fsw::RowGranules g(begin, end, first, last);
    if (g.lo % 16 || (g.bytes() > 0 && g.hi % 16)) return fail("not whole granules", size, base, d, pitch, M, row);
    if (g.bytes() > 0 && (g.lo < first_byte || g.hi > end_byte)) return fail("outside the matrix", size, base, d, pitch, M, row);
    if (g.bytes() > 0 && (g.lo < g.granule || g.hi - g.granule > static_cast<uint64_t>(d) * size + 30))
      return fail("outside its place", size, base, d, pitch, M, row);
    for (uint64_t q = begin; q < end; q += size) {
      const bool wide = g.bytes() > 0 && q >= g.lo && q < g.hi;
      const bool single = (first && q < g.lo) || (last && q >= g.hi);
      if (!wide && !single) return fail("an element is not read", size, base, d, pitch, M, row);
    }
  }
  return true;
}

}  // namespace

int main() {
  long long checked = 0;
  for (int size = 2; size <= 4; size += 2) {
    for (int base = 0; base < 16; base += size) {
      for (int d = 1; d <= 40; ++d) {
        for (int pitch = d; pitch <= d + 9; ++pitch) {
          for (int M = 1; M <= 24; ++M, ++checked) {
            if (!check(size, base, d, pitch, M)) return 1;
          }
        }
      }
    }
  }
  std::printf("ok %lld matrices\n", checked);
  return 0;
}
