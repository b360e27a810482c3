// The offsets of csrc/token_rows.h in 32 bits against 64-bit arithmetic, on the host: for each sequence length and row
// stride in bytes every row of the tiles where a wrapped end would fall, and of the first and last ones.
#include <stdio.h>

#include "token_rows.h"

using cssm::kTokenRows;
using cssm::kTokenTile;

template <int V>
static long long wrong(long long T, long long row, long long c) {
  using O = cssm::TileOff<V>;
  long long bad = 0;
  const long long tiles = (T + kTokenTile - 1) / kTokenTile, wrap = ((1LL << 32) + row - 1) / row;
  for (long long t = 0; t < tiles + 2; ++t) {       // and tiles wholly behind the last row
    const long long r0 = t * kTokenTile < T - 1 ? t * kTokenTile : T - 1, left = T - 1 - r0;
    const bool near = left % wrap < 2 * kTokenTile || t < 3 || t + 3 > tiles;
    if (!near) continue;
    for (int sub = 0; sub < kTokenTile / kTokenRows; ++sub) {
      const cssm::TileRows<O> at(O(row), sub, O(c), int(left));
      for (int i = 0; i < kTokenRows; ++i) {
        const long long r = sub * kTokenRows + i, want = (r < left ? r : left) * row + c;
        bad += (long long)at(i) != want;
      }
    }
  }
  return bad;
}

int main() {
  // float32 and bfloat16 slices of a 3 * 4096-wide projection, contiguous rows of 1024 and 2048 bfloat16 values, 8-bit
  // rows, the longest rows that 32 bits serve
  const struct { long long T, row, c; } cases[] = {
      {1, 2048, 0}, {127, 2048, 8}, {128, 2048, 8}, {129, 2048, 8}, {90000, 49152, 16384}, {180000, 24576, 8192}, {2200000, 2048, 2040},
      {(1 << 20) + 64, 4096, 4088}, {(1 << 20) + 64, 4096, 0}, {700, 1LL << 23, 8}, {400, 1LL << 24, 1 << 10}, {1100, 1LL << 22, 64},
      {2147483520, 8, 0}};
  for (const auto& k : cases) printf("%lld %lld %lld %lld\n", k.T, k.row, wrong<4>(k.T, k.row, k.c), wrong<1>(k.T, k.row, k.c));
  return 0;
}
