// The order in which the tiles of one run's product are walked, and the work units of runs that are split
// along their rows. (No CUDA in here: the tests compile it for the host too.)
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define MOE_ORDER_FN __host__ __device__ __forceinline__
#else
#define MOE_ORDER_FN inline
#endif

namespace moe {

// x / d for 0 <= x < 2^31 with inverse = ceil(2^32 / d): a multiplication, at most one too much, put right.
MOE_ORDER_FN uint32_t quotient_inverse(uint32_t d) { return uint32_t((0x100000000ull + d - 1) / d); }
MOE_ORDER_FN int quotient(int x, int d, uint32_t inverse) {
  if (d == 1) return x;
  const int q = int(uint64_t(uint32_t(x)) * inverse >> 32);
  return q * int64_t(d) > x ? q - 1 : q;
}

struct TileAt {
  int m, n;
};

// Tile `l` of an m_tiles x n_tiles product: bands of `band` row tiles, within a band all row tiles of one
// column tile after another. The units in flight at one time (a cluster takes every n-th unit) then
// cover a block of about band x in_flight / band tiles, and each loaded row or column strip serves that many.
MOE_ORDER_FN TileAt tile_in_bands(int l, int m_tiles, int n_tiles, int band) {
  const int b = l / (band * n_tiles);
  const int r = l - b * band * n_tiles;
  const int left = m_tiles - b * band;
  const int high = left < band ? left : band;
  TileAt t;
  t.n = r / high;
  t.m = b * band + (r - t.n * high);
  return t;
}

// Chunks of at most ks rows that a run of `rows` rows is cut into: at least one, a run without rows
// still has its (zero) result stored.
MOE_ORDER_FN int run_chunks(int rows, int ks) { return rows <= ks ? 1 : (rows + ks - 1) / ks; }

// Rows per chunk for runs of `rows` rows in all whose result has `tiles` tiles each: half of a cluster's
// share, a multiple of 64, at least 512.
MOE_ORDER_FN int64_t grouped_chunk_rows(int64_t rows, int64_t tiles, int clusters) {
  const int64_t share = (rows * tiles + int64_t(clusters) * 2 - 1) / (int64_t(clusters) * 2);
  const int64_t ks = (share + 63) / 64 * 64;
  return ks < 512 ? 512 : ks;
}

}  // namespace moe
