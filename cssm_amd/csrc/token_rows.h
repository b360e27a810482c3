// Where a tile of the token-sequence kernels finds its rows.  Plain arithmetic, on the host too, where it is tested.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace cssm {

constexpr int kTokenTile = 128, kTokenRows = 8;   // rows of a tile, and of one thread in it

// An offset from a tile's first row.  Where a thread takes several channels (V > 1) 128 rows lie within 2^31 bytes, so
// that 32 bits hold it and a load is a scalar base and one register.
template <int V>
using TileOff = typename std::conditional<V == 1, size_t, uint32_t>::type;

// Offsets of the 8 rows of row group `sub`, `row` apart, from the tile's first row: rows behind the last one that there
// is, which lies `left` >= 0 rows below the first, give that one again.  `left` counts to the end of the sequence, so it
// is cut to the tile before anything is multiplied: the whole sequence need not fit the offset's bits.
template <typename O>
struct TileRows {
  O row, at, last;
  __host__ __device__ __forceinline__ TileRows(O row_, int sub, O c, int left)
      : row(row_), at(O(sub * kTokenRows) * row_ + c), last(O(left < kTokenTile ? left : kTokenTile - 1) * row_ + c) {}
  __host__ __device__ __forceinline__ O operator()(int i) const {
    const O o = at + O(i) * row;
    return o < last ? o : last;
  }
};

}  // namespace cssm
