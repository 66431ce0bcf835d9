// A row's listed vocabulary columns (a teacher's entries) as the GEMM epilogues
// walk them.
#pragma once

#include <climits>

#include "kernels.cuh"

namespace cce {

// The listed columns of one row that fall into successive 32-column chunks of a
// kTopkTile-column tile: entries are sorted by column, so every chunk takes the
// next ones, as bits.  `open` only loads: it is called before the tile's products
// are there, so that its latencies pass meanwhile.
struct TopkCursor {
  const int32_t* ids;  // the row's sorted columns
  int p, end;          // next entry, end of the tile's entries
  int next;            // column of entry p, INT_MAX at the end
  __device__ __forceinline__ void open(const TopkView& t, int64_t row, bool ok, int64_t tile) {
    ids = t.sid + row * t.K;
    p = end = 0;
    if (ok && tile + 1 < t.tiles1) {
      const uint16_t* st = t.start + row * t.tiles1 + tile;
      p = __ldg(st);
      end = __ldg(st + 1);
    }
    next = p < end ? __ldg(ids + p) : INT_MAX;
  }
  // Bits of the entries in [col, col + 32); `first` is the entry of the lowest bit.
  __device__ __forceinline__ uint32_t take(int64_t col, int& first) {
    first = p;
    uint32_t m = 0;
    while (next < col + 32) {
      m |= 1u << (int)(next - col);
      ++p;
      next = p < end ? __ldg(ids + p) : INT_MAX;
    }
    return m;
  }
};

}  // namespace cce
