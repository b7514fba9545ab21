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
MOE_ORDER_FN int run_chunks(int rows, int ks) { return rows <= ks ? 1 : (rows - 1) / ks + 1; }

// Rows per chunk for n_groups runs of `rows` rows in all whose result has `tiles` tiles each. The runs being
// alike, `n` chunks each give rounds of all clusters that take (a 64-row step 0.5 us, a tile's end 2 us, all
// measured) some time, and cutting costs the partial tiles' way through L2 and the join: the cheapest n is
// taken, and a quarter more rows, so that a run a little longer than the rest is not cut for it. A run that is
// much longer than the rest is cut into pieces of two thirds of a cluster's share.
MOE_ORDER_FN int64_t grouped_chunk_rows(int64_t rows, int32_t n_groups, int64_t tiles, int clusters) {
  const int64_t run = (rows + n_groups - 1) / n_groups;
  double best = 0;
  int64_t chunks = 1;
  for (int64_t n = 1; n <= 32; ++n) {
    const int64_t units = n_groups * tiles * n;
    const double rounds = double((units + clusters - 1) / clusters);
    const double steps = double((run + n * 64 - 1) / (n * 64));
    const double us = rounds * (steps * 0.5 + 2.0) + (n > 1 ? 5.0 + double(units) * 0.1 : 0.0);
    if (n == 1 || us < best) {
      best = us;
      chunks = n;
    }
  }
  const int64_t typical = run * 5 / (chunks * 4);
  const int64_t share = rows * tiles * 2 / (int64_t(clusters) * 3);
  const int64_t most = chunks == 1 ? (share > typical ? share : typical) : typical;
  const int64_t ks = (most + 63) / 64 * 64;
  return ks < 256 ? 256 : ks;
}

}  // namespace moe
