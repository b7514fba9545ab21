// Products grouped by expert over ragged runs: rows start[g] .. start[g + 1] of x, back to back and of any
// length, with matrix g of a stack, for any widths that are multiples of 8 and both 16-bit float types.
//
//   grouped_rows_kernel   y[r] = x[r] @ w[g(r)]        (the forward, and with w transposed the gradient of x)
//   grouped_wgrad_kernel  dw[g] = x_g^T @ dy_g         (the contraction runs over the rows of a run)
//
// The block's own GEMMs (gemm.cuh) pad every run to 128 rows, so that a tile never meets a border. Here a
// tile may: in the first product the rows of a tile behind its run's end are other experts' rows, and as
// rows of a product do not mix, they are computed and not stored. In the second they would be summed, so
// the last stage of a run has its rows behind the end set to zero in shared memory, in both operands (a
// zero times an infinity of the next run would be NaN).
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <climits>

#include "../../include/moe_b200.h"
#include "act.cuh"
#include "grouped_order.cuh"
#include "half16.cuh"
#include "pair.cuh"
#include "pdl.cuh"
#include "per_device.cuh"
#include "ptx.cuh"
#include "runs.cuh"
#include "tma_map.cuh"

namespace moe {
namespace grouped {

constexpr int BM = 128;   // accumulator rows of a CTA: one TMEM lane per row
constexpr int BK = 64;    // 64 16-bit values = one 128-byte swizzle span
constexpr int EPI_WARPS = 8;
constexpr int A_BYTES = BM * BK * 2;
constexpr int BAND = 8;   // row tiles of a band (tile_in_bands)
constexpr int SHORT = 32; // rows of the smaller A box
constexpr int MAX_UNITS = INT_MAX - 1024;   // (the unit a cluster takes behind the last one, too)
constexpr int MAX_DIM = INT_MAX - 2 * BM;   // of rows and widths: what a tile has behind the last one is still an int
// MN-major operands, as in gemm.cuh: 64 x 64 boxes
constexpr uint32_t MN_LBO = 8192u, MN_SBO = 1024u, MN_KADV = 2048u;

__device__ __forceinline__ void store_v8(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
               "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Stores this lane's 32 values of a row at columns col .. col + 31 (row: the row's first value, null: not
// stored; odd lanes hold the row behind the even lane's, ld values further). wide: rows start on 32 bytes
// and all 32 columns exist; then lanes 2i and 2i + 1 swap halves so that an instruction covers 64 bytes of
// 16 rows instead of 32 bytes of 32. Otherwise 16-byte pieces, those that start below n_dim.
template <typename T>
__device__ __forceinline__ void store32(T* row, int64_t ld, int col, int n_dim, bool wide, const float* v) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = Half16<T>::pack(v[2 * i], v[2 * i + 1]);
  if (wide) {   // (uniform over the warp)
    const bool odd = threadIdx.x & 1;
    const bool ok = row != nullptr;
    const bool other = __shfl_xor_sync(0xffffffffu, ok, 1);
    const uint64_t mine = reinterpret_cast<uint64_t>(row);
    const uint64_t theirs = __shfl_xor_sync(0xffffffffu, mine, 1);
    uint32_t a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t x = __shfl_xor_sync(0xffffffffu, odd ? w[i] : w[8 + i], 1);
      a[i] = odd ? x : w[i];
      b[i] = odd ? w[8 + i] : x;
    }
    T* even_row = reinterpret_cast<T*>(odd ? theirs : mine);
    T* odd_row = reinterpret_cast<T*>(odd ? mine : theirs);
    if (odd ? other : ok) store_v8(even_row + col + (odd ? 16 : 0), a);
    if (odd ? ok : other) store_v8(odd_row + col + (odd ? 16 : 0), b);
  } else if (row != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + 8 * i < n_dim)
        *reinterpret_cast<uint4*>(row + col + 8 * i) =
            make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
}

// N chunks of 32 accumulator columns from column `col` of the result on, those that start below n_dim. (A loop: its
// code is fetched once; the next chunk's read under this one's stores gained nothing, other warps fill the wait.)
template <int N, typename Store>
__device__ __forceinline__ void store_columns(uint32_t taddr, int col, int n_dim, Store store) {
  const int n = min(N, (n_dim - col + 31) / 32);
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    float v[32];
    tmem_ld32(taddr + i * 32, v);
    tmem_ld_wait();
    store(col + i * 32, v);
  }
}

struct RowsArgs {
  const int32_t* offsets;
  int32_t n_groups, rows;
  int32_t num_k;      // k_dim / 64, rounded up: the tail reads as zeros
  int32_t n_dim, n_chunks;
  int32_t b_fused;    // MN-major w whose n_dim is a multiple of 64: one copy brings a stage of it
  void* out;          // [rows, n_dim]
  int32_t wide;       // rows of out start on 32 bytes
  int32_t* status;
};

template <int BN, int STAGES>
struct RowsSmem {
  static constexpr int B_BYTES = (BN / 2) * BK * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int BARS = STAGES * STAGE;
  static constexpr int MISC = BARS + 8 * (2 * STAGES + 4);
  static constexpr int TABLE = (MISC + 16 + 15) / 16 * 16;
  static constexpr int TOTAL = TABLE + int(sizeof(RunTable));
  static constexpr int DYNAMIC = TOTAL + 1024;
  static_assert(DYNAMIC <= 232448, "more shared memory than a CTA has");
};

// A CTA pair computes 256 x BN tiles (two 128-row tiles of one run, one column chunk): each CTA loads its own
// rows of x and half of the weight's columns, the leader issues one M = 256 MMA per 16 of k, the accumulators
// are double-buffered in TMEM and drained while the next tile is computed. Warps: 0 loads, 1 multiplies,
// 2 .. 9 store. Barriers as in gemm_rows2.cuh.
template <typename T, int BN, int STAGES, bool B_MN>
__global__ void __launch_bounds__(64 + EPI_WARPS * 32, 1)
    grouped_rows_kernel(const __grid_constant__ CUtensorMap tmA,
                        const __grid_constant__ CUtensorMap tmShort,
                        const __grid_constant__ CUtensorMap tmB, const RowsArgs p) {
  using L = RowsSmem<BN, STAGES>;
  constexpr uint32_t TMEM_BUF = BN <= 128 ? 128 : 256;
  constexpr uint32_t TMEM_COLS = 2 * TMEM_BUF;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  RunTable& table = *reinterpret_cast<RunTable*>(smem + L::TABLE);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int n_clusters = int(gridDim.x) >> 1;
  const int cluster = int(blockIdx.x) >> 1;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmShort);
    tma_prefetch_desc(&tmB);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar + s, 1);
      mbar_init(empty_bar + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar + b, 1);
      mbar_init(tempty_bar + b, 2 * EPI_WARPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  const uint32_t tmem_base = pair_start(tmem_slot, TMEM_COLS, warp);

  if (warp == 2) {
    const bool bad = load_run_starts(p.offsets, p.n_groups, p.rows, lane, table.start);
    if (bad && blockIdx.x == 0 && lane == 0) report_input(p.status, ST_BAD_OFFSETS);
    const int nc = p.n_chunks;
    count_run_units(table.start, p.n_groups, lane, table.first,
                    [nc](int rows) { return ((rows + 2 * BM - 1) / (2 * BM)) * nc; });
  }
  __syncthreads();

  const int n_units = table.first[p.n_groups];
  struct Unit {
    int group, row0, left, n0;   // first row of the pair's tile, rows of the run from there on
  };
  auto unit_of = [&](int u, int group) {
    Unit c;
    c.group = group;
    const int start = table.start[c.group], rows = table.start[c.group + 1] - start;
    const TileAt t = tile_in_bands(u - table.first[c.group], (rows + 2 * BM - 1) / (2 * BM),
                                   p.n_chunks, BAND);
    c.row0 = start + t.m * 2 * BM;
    c.left = rows - t.m * 2 * BM;
    c.n0 = t.n * BN;
    return c;
  };
  // bytes of x that CTA r of the pair loads per stage: nothing without rows, the short box for few
  auto a_bytes = [](int left, int r) {
    const int rows = left - r * BM;
    return rows <= 0 ? 0 : rows <= SHORT ? SHORT * BK * 2 : A_BYTES;
  };

  if (warp == 0) {
    if (elect_one()) {
      uint32_t it = 0;
      for (int u = cluster; u < n_units && !*abort_flag; u += n_clusters) {
        const Unit c = unit_of(u, run_of_unit(table.first, p.n_groups, u));
        const int own = a_bytes(c.left, int(rank));
        const uint32_t both = a_bytes(c.left, 0) + a_bytes(c.left, 1) + 2 * L::B_BYTES;
        const CUtensorMap* ma = own == A_BYTES ? &tmA : &tmShort;
        const int row = c.row0 + int(rank) * BM;
        const int n = c.n0 + int(rank) * (BN / 2);
        for (int kt = 0; kt < p.num_k; ++kt, ++it) {
          const int s = it % STAGES;
          const uint32_t use = it / STAGES;
          if (use > 0 && !mbar_wait(empty_bar + s, (use - 1) & 1, p.status)) {
            *abort_flag = 1;
            atomicExch(p.status, ST_WAIT_TIMEOUT);
            break;
          }
          uint8_t* sA = smem + s * L::STAGE;
          uint8_t* sB = sA + A_BYTES;
          if (rank == 0) mbar_expect_tx(full_bar + s, both);
          const int k = kt * BK;
          if (own > 0) tma_load_3d_2cta(sA, ma, full_bar + s, k, row, 0);
          if constexpr (!B_MN) {
            tma_load_3d_2cta(sB, &tmB, full_bar + s, k, n, c.group);
          } else if (p.b_fused) {
            tma_load_4d_2cta(sB, &tmB, full_bar + s, 0, k, n / 64, c.group);
          } else {
#pragma unroll
            for (int i = 0; i < BN / 128; ++i)
              tma_load_3d_2cta(sB + i * 64 * BK * 2, &tmB, full_bar + s, n + 64 * i, k, c.group);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc = umma_idesc(2 * BM, BN, false, B_MN, Half16<T>::UMMA_FMT);
      uint32_t it = 0;
      int j = 0;
      for (int u = cluster; u < n_units && !*abort_flag; u += n_clusters, ++j) {
        const int b = j & 1;
        const uint32_t use = uint32_t(j) >> 1;
        if (use > 0 && !mbar_wait(tempty_bar + b, (use - 1) & 1, p.status)) {
          *abort_flag = 1;
          atomicExch(p.status, ST_WAIT_TIMEOUT);
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + b * TMEM_BUF;
        for (int kt = 0; kt < p.num_k; ++kt, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(full_bar + s, (it / STAGES) & 1, p.status)) {
            *abort_flag = 1;
            atomicExch(p.status, ST_WAIT_TIMEOUT);
            break;
          }
          tc_fence_after();
          const uint32_t sA = smem_u32(smem + s * L::STAGE);
          const uint32_t sB = sA + A_BYTES;
#pragma unroll
          for (int k16 = 0; k16 < BK / 16; ++k16) {
            const uint64_t da = umma_desc(sA + k16 * 32, 16, 1024);
            const uint64_t db = B_MN ? umma_desc(sB + k16 * MN_KADV, MN_LBO, MN_SBO)
                                     : umma_desc(sB + k16 * 32, 16, 1024);
            umma_f16_2cta(d_tmem, da, db, idesc, (kt == 0 && k16 == 0) ? 0u : 1u);
          }
          umma_commit_2cta(empty_bar + s, 3);
        }
        umma_commit_2cta(tfull_bar + b, 3);
      }
      // (whoever gave up, nobody reads on from here; the leader's barriers count both CTAs' bytes, and the pair leaves
      // together)
      if (*abort_flag) mbar_drain(full_bar, it, STAGES);
    }
  } else {
    const int ew = warp - 2;
    const int q = warp & 3;            // the TMEM lanes this warp may read
    const int half = ew >> 2;          // its half of the columns
    const int row = q * 32 + lane;
    constexpr int NCH = BN / 32;
    const uint32_t tempty_leader = mapa_u32(smem_u32(tempty_bar), 0);
    T* out = static_cast<T*>(p.out);
    int j = 0, group = 0;
    for (int u = cluster; u < n_units; u += n_clusters, ++j) {
      group = run_of_unit_warp(table.first, p.n_groups, u, group, lane);
      const Unit c = unit_of(u, group);
      const int b = j & 1;
      if (!mbar_wait(tfull_bar + b, (uint32_t(j) >> 1) & 1, p.status))
        atomicExch(p.status, ST_WAIT_TIMEOUT);
      tc_fence_after();
      const uint32_t taddr = tmem_base + b * TMEM_BUF + (uint32_t(q * 32) << 16);
      const int r = int(rank) * BM + row;
      T* mine = r < c.left ? out + int64_t(c.row0 + r) * p.n_dim : nullptr;
      if (__any_sync(0xffffffffu, mine != nullptr)) {
        store_columns<NCH / 2>(taddr + half * (BN / 2), c.n0 + half * (BN / 2), p.n_dim,
                               [&](int col, const float* v) {
                                 store32(mine, p.n_dim, col, p.n_dim, p.wide && col + 32 <= p.n_dim, v);
                               });
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty_leader + b * 8);
    }
    // rows of no run are zero
    const int64_t pieces = p.n_dim / 8;
    const int64_t head = table.start[0] * pieces, tail0 = table.start[p.n_groups] * pieces;
    const int64_t n = head + p.rows * pieces - tail0;
    for (int64_t i = int64_t(blockIdx.x) * (EPI_WARPS * 32) + threadIdx.x - 64; i < n;
         i += int64_t(gridDim.x) * (EPI_WARPS * 32))
      static_cast<uint4*>(p.out)[i < head ? i : tail0 + (i - head)] = make_uint4(0, 0, 0, 0);
  }

  // Nobody leaves while the other CTA may still signal its barriers or read its shared memory.
  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) tmem_dealloc2(tmem_base, TMEM_COLS);
}

// ------------------------------------------------------------------------------ weight gradients
struct WgradArgs {
  const int32_t* offsets;
  int32_t n_groups, rows;
  int32_t ks;               // rows of a chunk
  int32_t m_dim, n_dim;     // one dw[g]
  int32_t m_tiles, n_tiles; // tiles of a CTA pair
  uint32_t tiles_inv;       // (quotient)
  int32_t a_fused, b_fused; // the operand's width is a multiple of 64: one copy brings a stage of it
  void* out;                // [n_groups, m_dim, n_dim]
  int32_t wide;
  float* partials;          // [chunks of split runs][tiles][2][BN / 8][128][8]: a CTA's tile, eight columns of all its
                            // rows together (a warp's store is then 1 KB in one piece)
  int32_t* status;
};

constexpr int MAX_SORTED = 512;   // chunks that are put in order of their length
constexpr int WGRAD_THREADS = 96 + EPI_WARPS * 32;

template <int BN, int STAGES>
struct WgradSmem {
  static constexpr int B_BYTES = (BN / 2) * BK * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int TAILS = STAGES * STAGE;             // two stages for the ends of runs
  static constexpr int BARS = TAILS + 2 * STAGE;
  static constexpr int MISC = BARS + 8 * (2 * STAGES + 10);
  static constexpr int TABLE = (MISC + 16 + 15) / 16 * 16;
  static constexpr int SPLIT = TABLE + int(sizeof(RunTable));   // first chunk of every split run
  static constexpr int LENGTHS = (SPLIT + (RUNS_MAX_GROUPS + 1) * 4 + 15) / 16 * 16;
  static constexpr int SORTED = LENGTHS + MAX_SORTED * 4;
  static constexpr int TOTAL = SORTED + MAX_SORTED * int(sizeof(int4));
  static constexpr int DYNAMIC = TOTAL + 1024;
  static_assert(STAGE % 1024 == 0, "stages must keep the 1024-byte swizzle alignment");
  static_assert(DYNAMIC <= 232448, "more shared memory than a CTA has");
};

// 256 x BN tiles of dw[g] on CTA pairs: each CTA loads 128 columns of the first operand and half of the
// second's, both MN-major (their rows are the contraction). A single CTA's 128 x 256 tile takes 48 KB for 512
// cycles of MMAs, more than an SM gets out of L2; the pair's takes 32 KB per CTA (32768 rows x 2048 x 4096 in
// 16 groups: 471 us, 1167 TFLOP/s, as pairs 400 to 420, 1310 to 1370, under the power cap). Small matrices are
// bound by the rows' bytes: 98304 rows x 576 x 256 in 76 groups 48 us, 3.9 TB/s, three rounds of tiles and a
// last one nearly empty.
//
// A run's last rows, fewer than a stage, go through two stages of their own: they land on a barrier of their
// CTA, a warp sets the rows behind the run's end to zero (up to the next 16, which is what an MMA takes) and
// tells the leader. That happens ahead of the MMAs and keeps them out of it. Warps: 0 loads, 1 multiplies (the
// leader's), 2 .. 9 store, 10 clears.
//
// Work items are chunks of runs (at most ks rows), longest first, every tile of one after another; the
// clusters take them in turns, back and forth, so that the long ones do not come last. The fp32 tiles of runs
// with several chunks are added in order by wgrad_join_kernel.
template <typename T, int BN, int STAGES>
__global__ void __launch_bounds__(WGRAD_THREADS, 1)
    grouped_wgrad_kernel(const __grid_constant__ CUtensorMap tmA,
                         const __grid_constant__ CUtensorMap tmB, const WgradArgs p) {
  using L = WgradSmem<BN, STAGES>;
  constexpr uint32_t TMEM_BUF = BN <= 128 ? 128 : 256;
  constexpr uint32_t TMEM_COLS = 2 * TMEM_BUF;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* landed_bar = tempty_bar + 2;    // a run's end is in this CTA's tail stage
  uint64_t* cleared_bar = landed_bar + 2;   // leader: and clean in both CTAs'
  uint64_t* used_bar = cleared_bar + 2;     // and multiplied
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  RunTable& table = *reinterpret_cast<RunTable*>(smem + L::TABLE);   // first: in chunks
  int* split_first = reinterpret_cast<int*>(smem + L::SPLIT);
  int* lengths = reinterpret_cast<int*>(smem + L::LENGTHS);
  int4* sorted_chunks = reinterpret_cast<int4*>(smem + L::SORTED);   // group, first row, length, part

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int n_clusters = int(gridDim.x) >> 1;
  const int cluster = int(blockIdx.x) >> 1;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar + s, 1);
      mbar_init(empty_bar + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar + b, 1);
      mbar_init(tempty_bar + b, 2 * EPI_WARPS);
      mbar_init(landed_bar + b, 1);
      mbar_init(cleared_bar + b, 2);
      mbar_init(used_bar + b, 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  const uint32_t tmem_base = pair_start(tmem_slot, TMEM_COLS, warp);

  const int tiles = p.m_tiles * p.n_tiles;
  if (warp == 2) {
    const bool bad = load_run_starts(p.offsets, p.n_groups, p.rows, lane, table.start);
    if (bad && blockIdx.x == 0 && lane == 0) report_input(p.status, ST_BAD_OFFSETS);
    const int ks = p.ks;
    count_run_units(table.start, p.n_groups, lane, table.first, [=](int rows) { return run_chunks(rows, ks); });
    count_run_units(table.start, p.n_groups, lane, split_first,
                    [=](int rows) { return rows > ks ? run_chunks(rows, ks) : 0; });
  }
  __syncthreads();
  // chunk i: its group, first row, length, and its place among the chunks of split runs (-1: it is its run's only
  // one)
  auto chunk_of = [&](int i) {
    const int g = run_of_unit(table.first, p.n_groups, i), at = i - table.first[g];
    const int start = table.start[g] + at * p.ks;
    return make_int4(g, start, min(p.ks, table.start[g + 1] - start),
                     split_first[g + 1] > split_first[g] ? split_first[g] + at : -1);
  };
  const int n_chunks = table.first[p.n_groups];
  const bool sorted = n_chunks <= MAX_SORTED;
  if (sorted) {
    int4 mine[(MAX_SORTED + WGRAD_THREADS - 1) / WGRAD_THREADS];
#pragma unroll
    for (int k = 0; k < int(sizeof(mine) / sizeof(int4)); ++k) {
      const int i = threadIdx.x + k * WGRAD_THREADS;
      if (i < n_chunks) {
        mine[k] = chunk_of(i);
        lengths[i] = mine[k].z;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < int(sizeof(mine) / sizeof(int4)); ++k) {
      const int i = threadIdx.x + k * WGRAD_THREADS;
      if (i >= n_chunks) break;
      int before = 0;
      for (int j = 0; j < n_chunks; ++j) before += lengths[j] > mine[k].z || (lengths[j] == mine[k].z && j < i);
      sorted_chunks[before] = mine[k];
    }
    __syncthreads();
  }

  const int n_units = n_chunks * tiles;
  const int n_rounds = (n_units + n_clusters - 1) / n_clusters;
  struct Unit {
    int group, row0, len, m0, n0;
    int part;   // its chunk among those of split runs, -1: the run's only one; -2: no unit in this round
    int tile;
  };
  auto unit_of = [&](int round) {
    Unit c;
    const int u = round * n_clusters + (round & 1 ? n_clusters - 1 - cluster : cluster);
    if (u >= n_units) {
      c.part = -2;
      c.len = 0;
      return c;
    }
    const int k = quotient(u, tiles, p.tiles_inv);
    const int4 ch = sorted ? sorted_chunks[k] : chunk_of(k);
    c.tile = u - k * tiles;
    const TileAt t = tile_in_bands(c.tile, p.m_tiles, p.n_tiles, BAND);
    c.group = ch.x;
    c.row0 = ch.y;
    c.len = ch.z;
    c.part = ch.w;
    c.m0 = (t.m * 2 + int(rank)) * BM;   // this CTA's rows of dw
    c.n0 = t.n * BN;
    return c;
  };

  if (warp == 0) {
    if (elect_one()) {
      uint32_t it = 0;
      int tails = 0;
      auto give_up = [&] {
        *abort_flag = 1;
        atomicExch(p.status, ST_WAIT_TIMEOUT);
      };
      for (int round = 0; round < n_rounds && !*abort_flag; ++round) {
        const Unit c = unit_of(round);
        const int full = c.len / BK, nb = c.n0 + int(rank) * (BN / 2);
        for (int kt = 0; kt < full; ++kt, ++it) {
          const int s = it % STAGES;
          const uint32_t use = it / STAGES;
          if (use > 0 && !mbar_wait(empty_bar + s, (use - 1) & 1, p.status)) {
            give_up();
            break;
          }
          uint8_t* sA = smem + s * L::STAGE;
          uint8_t* sB = sA + A_BYTES;
          if (rank == 0) mbar_expect_tx(full_bar + s, 2 * L::STAGE);
          const int row = c.row0 + kt * BK;
          if (p.a_fused) {
            tma_load_3d_2cta(sA, &tmA, full_bar + s, 0, row, c.m0 / 64);
          } else {
#pragma unroll
            for (int i = 0; i < BM / 64; ++i)
              tma_load_3d_2cta(sA + i * 64 * BK * 2, &tmA, full_bar + s, c.m0 + 64 * i, row, 0);
          }
          if (p.b_fused) {
            tma_load_3d_2cta(sB, &tmB, full_bar + s, 0, row, nb / 64);
          } else {
#pragma unroll
            for (int i = 0; i < BN / 128; ++i)
              tma_load_3d_2cta(sB + i * 64 * BK * 2, &tmB, full_bar + s, nb + 64 * i, row, 0);
          }
        }
        if (c.len % BK == 0 || *abort_flag) continue;
        const int b = tails & 1;
        const uint32_t use = uint32_t(tails) >> 1;
        if (use > 0 && !mbar_wait(used_bar + b, (use - 1) & 1, p.status)) {
          give_up();
          break;
        }
        ++tails;
        uint8_t* sA = smem + L::TAILS + b * L::STAGE;
        uint8_t* sB = sA + A_BYTES;
        mbar_expect_tx(landed_bar + b, L::STAGE);
        const int row = c.row0 + full * BK;
        if (p.a_fused) {
          tma_load_3d(sA, &tmA, landed_bar + b, 0, row, c.m0 / 64);
        } else {
#pragma unroll
          for (int i = 0; i < BM / 64; ++i)
            tma_load_3d(sA + i * 64 * BK * 2, &tmA, landed_bar + b, c.m0 + 64 * i, row, 0);
        }
        if (p.b_fused) {
          tma_load_3d(sB, &tmB, landed_bar + b, 0, row, nb / 64);
        } else {
#pragma unroll
          for (int i = 0; i < BN / 128; ++i)
            tma_load_3d(sB + i * 64 * BK * 2, &tmB, landed_bar + b, nb + 64 * i, row, 0);
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc = umma_idesc(2 * BM, BN, true, true, Half16<T>::UMMA_FMT);
      uint32_t it = 0;
      int j = 0, tails = 0;
      for (int round = 0; round < n_rounds && !*abort_flag; ++round) {
        const Unit c = unit_of(round);
        if (c.len <= 0) continue;
        const int b = j & 1;
        const uint32_t use = uint32_t(j) >> 1;
        ++j;
        bool ok = use == 0 || mbar_wait(tempty_bar + b, (use - 1) & 1, p.status);
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + b * TMEM_BUF;
        uint32_t more = 0;
        auto multiply = [&](uint32_t sA, int steps) {
          const uint32_t sB = sA + A_BYTES;
#pragma unroll
          for (int k16 = 0; k16 < BK / 16; ++k16)
            if (k16 < steps) {
              umma_f16_2cta(d_tmem, umma_desc(sA + k16 * MN_KADV, MN_LBO, MN_SBO),
                            umma_desc(sB + k16 * MN_KADV, MN_LBO, MN_SBO), idesc, more);
              more = 1;
            }
        };
        const int full = c.len / BK, tail = c.len % BK;
        for (int kt = 0; kt < full && ok; ++kt, ++it) {
          const int s = it % STAGES;
          ok = mbar_wait(full_bar + s, (it / STAGES) & 1, p.status);
          if (!ok) break;
          tc_fence_after();
          multiply(smem_u32(smem + s * L::STAGE), BK / 16);
          umma_commit_2cta(empty_bar + s, 3);
        }
        if (ok && tail > 0) {
          const int tb = tails & 1;
          ok = mbar_wait_cluster(cleared_bar + tb, (uint32_t(tails) >> 1) & 1, p.status);
          ++tails;
          if (ok) {
            tc_fence_after();
            multiply(smem_u32(smem + L::TAILS + tb * L::STAGE), (tail + 15) / 16);
            umma_commit_2cta(used_bar + tb, 3);
          }
        }
        if (!ok) {
          *abort_flag = 1;
          atomicExch(p.status, ST_WAIT_TIMEOUT);
          break;
        }
        umma_commit_2cta(tfull_bar + b, 3);
      }
      // (whoever gave up, nobody reads on from here; the leader's barriers count both CTAs' bytes, and the pair leaves
      // together)
      if (*abort_flag) mbar_drain(full_bar, it, STAGES);
    }
  } else if (warp == 2 + EPI_WARPS) {
    int tails = 0;
    for (int round = 0; round < n_rounds; ++round) {
      const int tail = unit_of(round).len % BK;
      if (tail == 0) continue;
      const int b = tails & 1;
      // (the lanes go on together or not at all)
      const bool ok = mbar_wait(landed_bar + b, (uint32_t(tails) >> 1) & 1, p.status);
      ++tails;
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) {
          *abort_flag = 1;
          atomicExch(p.status, ST_WAIT_TIMEOUT);
        }
        mbar_drain(landed_bar, tails - 1, 2);
        break;
      }
      // a 64 x 64 box keeps its row r in bytes r * 128 .. r * 128 + 127, in whatever order
      const uint32_t first = smem_u32(smem + L::TAILS + b * L::STAGE) + tail * 128;
      const int bytes = ((tail + 15) / 16 * 16 - tail) * 128;
#pragma unroll
      for (int box = 0; box < BM / 64 + BN / 128; ++box)
        for (int i = lane * 16; i < bytes; i += 512) st_shared_v4(first + box * (64 * BK * 2) + i, 0, 0, 0, 0);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive_release_cluster(mapa_u32(smem_u32(cleared_bar + b), 0));
    }
  } else {
    const int ew = warp - 2;
    const int q = warp & 3;
    const int half = ew >> 2;
    const int row = q * 32 + lane;
    constexpr int NCH = BN / 32;
    const uint32_t tempty_leader = mapa_u32(smem_u32(tempty_bar), 0);
    T* out = static_cast<T*>(p.out);
    const int64_t matrix = int64_t(p.m_dim) * p.n_dim;
    int j = 0;
    for (int round = 0; round < n_rounds; ++round) {
      const Unit c = unit_of(round);
      if (c.part == -2) continue;
      const bool have = c.len > 0;
      const int b = j & 1;
      if (have) {
        if (!mbar_wait(tfull_bar + b, (uint32_t(j) >> 1) & 1, p.status))
          atomicExch(p.status, ST_WAIT_TIMEOUT);
        tc_fence_after();
        ++j;
      }
      const uint32_t taddr = tmem_base + b * TMEM_BUF + (uint32_t(q * 32) << 16);
      const int m = c.m0 + row;
      const bool ok = m < p.m_dim;
      T* mine = ok ? out + c.group * matrix + int64_t(m) * p.n_dim : nullptr;
      const int col0 = c.n0 + half * (BN / 2);
      if (!have) {   // a run without rows: zeros, row by row
        const int pieces = min(BN / 2, p.n_dim - col0) / 8;
        constexpr int ACROSS = BN / 16, DOWN = 32 / ACROSS;   // lanes along a row, rows at a time
#pragma unroll 4
        for (int r = lane / ACROSS; r < 32; r += DOWN) {
          const int at = c.m0 + q * 32 + r;
          if (at < p.m_dim && lane % ACROSS < pieces)
            *reinterpret_cast<uint4*>(out + c.group * matrix + int64_t(at) * p.n_dim + col0 +
                                      lane % ACROSS * 8) = make_uint4(0, 0, 0, 0);
        }
      } else if (__any_sync(0xffffffffu, ok)) {
        if (c.part < 0) {
          store_columns<NCH / 2>(taddr + half * (BN / 2), col0, p.n_dim, [&](int col, const float* v) {
            store32(mine, p.n_dim, col, p.n_dim, p.wide && col + 32 <= p.n_dim, v);
          });
        } else {
          float* part = p.partials + ((int64_t(c.part) * tiles + c.tile) * 2 + rank) * (BM * BN) + row * 8;
          store_columns<NCH / 2>(taddr + half * (BN / 2), col0, p.n_dim, [&](int col, const float* v) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              store_v8(part + ((col - c.n0) / 8 + i) * (BM * 8), reinterpret_cast<const uint32_t*>(v) + 8 * i);
          });
        }
      }
      if (have) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tempty_leader + b * 8);
      }
    }
  }

  // Nobody leaves while the other CTA may still signal its barriers or read its shared memory.
  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) tmem_dealloc2(tmem_base, TMEM_COLS);
}

// dw[g] = sum of the fp32 partials of its chunks, in order, for the runs that were cut. The blocks share these
// runs' tiles in pieces of 128 rows x 32 columns; a warp takes 8 rows x 32 columns at a time, 256 bytes in one
// piece of each partial and 64 of a row of dw.
constexpr int JOIN_THREADS = 256;
template <typename T, int BN>
__global__ void __launch_bounds__(JOIN_THREADS) wgrad_join_kernel(const WgradArgs p) {
  __shared__ int start[RUNS_MAX_GROUPS + 1], split_first[RUNS_MAX_GROUPS + 1];
  pdl_trigger();
  pdl_wait();
  // is there a long run at all? (starts that are not in order go the long way too)
  bool maybe = false;
  for (int g = threadIdx.x; g < p.n_groups; g += JOIN_THREADS) {
    const int a = ld_prev(p.offsets + g), b = ld_prev(p.offsets + g + 1);
    maybe |= a < 0 || b < a || b > p.rows || b - a > p.ks;
  }
  if (!__syncthreads_or(maybe)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    const int ks = p.ks;
    load_run_starts(p.offsets, p.n_groups, p.rows, lane, start);
    count_run_units(start, p.n_groups, lane, split_first,
                    [=](int rows) { return rows > ks ? run_chunks(rows, ks) : 0; });
  }
  __syncthreads();
  const int64_t matrix = int64_t(p.m_dim) * p.n_dim;
  const int tiles = p.m_tiles * p.n_tiles;
  const int pieces = tiles * 2 * (BN / 32);   // of a run
  int g = -1;
  int64_t before = 0;   // pieces of the cut runs up to g
  for (int64_t piece = blockIdx.x;; piece += gridDim.x) {
    while (piece >= before) {   // the next cut run
      do ++g;
      while (g < p.n_groups && split_first[g + 1] == split_first[g]);
      if (g == p.n_groups) return;
      before += pieces;
    }
    const int i = int(piece - (before - pieces));
    const int chunk32 = i % (BN / 32), half_tile = i / (BN / 32);
    const TileAt t = tile_in_bands(half_tile >> 1, p.m_tiles, p.n_tiles, BAND);
    const int m0 = (t.m * 2 + (half_tile & 1)) * BM, col = t.n * BN + chunk32 * 32 + (lane >> 3) * 8;
    if (m0 >= p.m_dim || col >= p.n_dim) continue;
    const int n = split_first[g + 1] - split_first[g];
    const int64_t step = int64_t(tiles) * 2 * (BM * BN);
    const float* from = p.partials + split_first[g] * step + int64_t(half_tile) * (BM * BN) +
                        (chunk32 * 4 + (lane >> 3)) * (BM * 8);
    T* out = static_cast<T*>(p.out) + g * matrix + col;
#pragma unroll
    for (int h = 0; h < BM / 64; ++h) {
      const int row = h * 64 + warp * 8 + (lane & 7);
      if (m0 + row >= p.m_dim) break;
      const float4* at = reinterpret_cast<const float4*>(from + row * 8);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll 4
      for (int c = 0; c < n; ++c, at += step / 4) {
        const float4 x = at[0], y = at[1];
        a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
        b.x += y.x; b.y += y.y; b.z += y.z; b.w += y.w;
      }
      *reinterpret_cast<uint4*>(out + int64_t(m0 + row) * p.n_dim) =
          make_uint4(Half16<T>::pack(a.x, a.y), Half16<T>::pack(a.z, a.w), Half16<T>::pack(b.x, b.y),
                     Half16<T>::pack(b.z, b.w));
    }
  }
}

// -------------------------------------------------------------------------------------- the host side
static int current_device() {
  int dev = -1;
  return cudaGetDevice(&dev) == cudaSuccess ? dev : -1;
}
static int sm_count(int dev) {
  static PerDevice<int> counts;
  const int* n = counts.get(dev, [](int d) {
    int v = 0;
    return cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, d) == cudaSuccess && v > 0 ? v : 148;
  });
  return n ? *n : 148;
}

// x [rows, cols] with ld values between rows as the K-major A operand: boxes of 64 columns x `high` rows.
static bool map_x(CUtensorMap* m, const void* x, int64_t rows, int64_t ld, int64_t cols, int high) {
  const uint64_t dims[3] = {uint64_t(cols), uint64_t(rows), 1};
  const uint64_t strides[2] = {uint64_t(ld) * 2, uint64_t(ld) * 2};   // (there is one of the last)
  const uint32_t box[3] = {64, uint32_t(high), 1};
  return make_map(m, x, 3, dims, strides, box);
}
// w [groups][outer][inner], inner contiguous. K-major (inner is the contraction): 64 x `high` boxes. MN-major:
// 64 x 64 boxes, `boxes` of them per copy where inner is a multiple of 64.
static bool map_w_kmajor(CUtensorMap* m, const void* w, int64_t groups, int64_t gstride, int64_t outer,
                         int64_t ld, int64_t inner, int high) {
  const uint64_t dims[3] = {uint64_t(inner), uint64_t(outer), uint64_t(groups)};
  const uint64_t strides[2] = {uint64_t(ld) * 2, uint64_t(gstride) * 2};
  const uint32_t box[3] = {64, uint32_t(high), 1};
  return make_map(m, w, 3, dims, strides, box);
}
static bool map_w_mnmajor(CUtensorMap* m, const void* w, int64_t groups, int64_t gstride, int64_t outer,
                          int64_t ld, int64_t inner, int boxes, int32_t* fused) {
  *fused = inner % 64 == 0;
  if (*fused) {
    const uint64_t dims[4] = {64, uint64_t(outer), uint64_t(inner / 64), uint64_t(groups)};
    const uint64_t strides[3] = {uint64_t(ld) * 2, 128, uint64_t(gstride) * 2};
    const uint32_t box[4] = {64, 64, uint32_t(boxes), 1};
    return make_map(m, w, 4, dims, strides, box);
  }
  const uint64_t dims[3] = {uint64_t(inner), uint64_t(outer), uint64_t(groups)};
  const uint64_t strides[2] = {uint64_t(ld) * 2, uint64_t(gstride) * 2};
  const uint32_t box[3] = {64, 64, 1};
  return make_map(m, w, 3, dims, strides, box);
}
// A [rows, cols] matrix as an MN-major operand of the weight gradient: `boxes` 64 x 64 boxes per copy where cols
// is a multiple of 64.
static bool map_mn(CUtensorMap* m, const void* x, int64_t rows, int64_t ld, int64_t cols, int boxes,
                   int32_t* fused) {
  *fused = cols % 64 == 0;
  if (*fused) {
    const uint64_t dims[3] = {64, uint64_t(rows), uint64_t(cols / 64)};
    const uint64_t strides[2] = {uint64_t(ld) * 2, 128};
    const uint32_t box[3] = {64, 64, uint32_t(boxes)};
    return make_map(m, x, 3, dims, strides, box);
  }
  return map_x(m, x, rows, ld, cols, 64);
}

// Clusters of two of `kern` that are resident at once (fewer than half the SMs: they pair up inside a
// processing cluster); 0: it cannot be launched.
template <typename Kern>
static int pair_clusters(Kern kern, int threads, int smem, int dev) {
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(sm_count(dev) / 2 * 2));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  return cudaOccupancyMaxActiveClusters(&n, kern, &cfg) == cudaSuccess ? n : 0;
}

template <typename T, int BN, bool B_MN>
static int launch_rows(const CUtensorMap& tmA, const CUtensorMap& tmShort, const CUtensorMap& tmB,
                       const RowsArgs& args, int64_t max_units, int dev, cudaStream_t st) {
  constexpr int STAGES = BN == 256 ? 6 : 8;
  auto kern = grouped_rows_kernel<T, BN, STAGES, B_MN>;
  constexpr int smem = RowsSmem<BN, STAGES>::DYNAMIC;
  constexpr int threads = 64 + EPI_WARPS * 32;
  static PerDevice<int> clusters;
  const int* resident = clusters.get(dev, [&](int d) { return pair_clusters(kern, threads, smem, d); });
  if (resident == nullptr || *resident < 1) return MOE_B200_ERR_CUDA;
  const int64_t n = std::max<int64_t>(1, std::min<int64_t>(max_units, *resident));
  return launch_pdl_pairs(kern, dim3(unsigned(2 * n)), dim3(threads), size_t(smem), st, tmA, tmShort, tmB,
                          args) == cudaSuccess
             ? MOE_B200_OK
             : MOE_B200_ERR_CUDA;
}

template <typename T>
static int rows_product(const void* x, int64_t rows, int64_t ld_x, int32_t k_dim, const void* w,
                        int32_t n_groups, int64_t gstride, int64_t ld_w, int32_t n_inner, int32_t n_dim,
                        const int32_t* offsets, void* y, int32_t* status, cudaStream_t st) {
  const int dev = current_device();
  // pairs of row tiles: at most one partly filled per run
  const int64_t pairs = std::min<int64_t>(rows, rows / (2 * BM) + n_groups);
  // The wide tile loads less per product (1293 rows x 76, 256 -> 576: 46 us against the narrow one's 57); the
  // narrow one where the wide one would leave a quarter of the clusters without work (100 rows x 8, 1024 -> 1024:
  // 7.5 us against 9.6; at 64 tiles for 74 clusters, 2048^3, the wide one's 15.3 against 17.5).
  const bool wide_tile = n_dim > 128 && pairs * ((n_dim + 255) / 256) * 8 >= sm_count(dev) * 3;
  const int bn = wide_tile ? 256 : 128;
  RowsArgs a{};
  a.offsets = offsets;
  a.n_groups = n_groups;
  a.rows = int32_t(rows);
  a.num_k = (k_dim + BK - 1) / BK;
  a.n_dim = n_dim;
  a.n_chunks = (n_dim + bn - 1) / bn;
  a.out = y;
  a.wide = n_dim % 16 == 0 && reinterpret_cast<uintptr_t>(y) % 32 == 0;
  a.status = status;
  if (pairs * a.n_chunks > MAX_UNITS) return MOE_B200_ERR_UNSUPPORTED;
  CUtensorMap tmA, tmShort, tmB;
  if (!map_x(&tmA, x, rows, ld_x, k_dim, BM) || !map_x(&tmShort, x, rows, ld_x, k_dim, SHORT))
    return MOE_B200_ERR_TMA;
  const bool mapped = n_inner ? map_w_mnmajor(&tmB, w, n_groups, gstride, k_dim, ld_w, n_dim, bn / 128, &a.b_fused)
                              : map_w_kmajor(&tmB, w, n_groups, gstride, n_dim, ld_w, k_dim, bn / 2);
  if (!mapped) return MOE_B200_ERR_TMA;
  const int64_t units = pairs * a.n_chunks;
  if (wide_tile)
    return n_inner ? launch_rows<T, 256, true>(tmA, tmShort, tmB, a, units, dev, st)
                   : launch_rows<T, 256, false>(tmA, tmShort, tmB, a, units, dev, st);
  return n_inner ? launch_rows<T, 128, true>(tmA, tmShort, tmB, a, units, dev, st)
                 : launch_rows<T, 128, false>(tmA, tmShort, tmB, a, units, dev, st);
}

static int wgrad_bn(int32_t n_dim) { return n_dim > 128 ? 256 : 128; }
static int64_t wgrad_tiles(int32_t m_dim, int32_t n_dim) {
  const int bn = wgrad_bn(n_dim);
  return int64_t((m_dim + 2 * BM - 1) / (2 * BM)) * ((n_dim + bn - 1) / bn);
}
// (of every device alike: the scratch is sized before it is known where)
static int64_t wgrad_chunk(int64_t rows, int32_t n_groups, int64_t tiles) {
  return grouped_chunk_rows(rows, n_groups, tiles, 74);
}
// Chunks of the runs that are split: each has more than ks rows or is its run's last.
static int64_t split_chunks(int64_t rows, int64_t ks, int32_t n_groups) {
  return rows <= ks ? 0 : rows / ks + std::min<int64_t>(rows / ks, n_groups);
}

template <typename T, int BN>
static int launch_wgrad(const CUtensorMap& tmA, const CUtensorMap& tmB, const WgradArgs& args,
                        int64_t max_units, int dev, cudaStream_t st) {
  constexpr int STAGES = BN == 256 ? 4 : 6;
  auto kern = grouped_wgrad_kernel<T, BN, STAGES>;
  constexpr int smem = WgradSmem<BN, STAGES>::DYNAMIC;
  static PerDevice<int> clusters;
  const int* resident = clusters.get(dev, [&](int d) { return pair_clusters(kern, WGRAD_THREADS, smem, d); });
  if (resident == nullptr || *resident < 1) return MOE_B200_ERR_CUDA;
  const int64_t n = std::min<int64_t>(max_units, *resident);
  return launch_pdl_pairs(kern, dim3(unsigned(2 * n)), dim3(WGRAD_THREADS), size_t(smem), st, tmA, tmB, args) ==
                 cudaSuccess
             ? MOE_B200_OK
             : MOE_B200_ERR_CUDA;
}

template <typename T>
static int wgrad_product(const void* a, int64_t ld_a, int32_t m_dim, const void* b, int64_t ld_b,
                         int32_t n_dim, int64_t rows, const int32_t* offsets, int32_t n_groups, void* dw,
                         float* partials, int32_t* status, cudaStream_t st) {
  const int dev = current_device();
  const int bn = wgrad_bn(n_dim);
  const int64_t tiles = wgrad_tiles(m_dim, n_dim);
  const int64_t ks = std::min<int64_t>(wgrad_chunk(rows, n_groups, tiles), INT_MAX / 2);
  const int64_t units = (rows / ks + n_groups) * tiles;
  if (units > MAX_UNITS) return MOE_B200_ERR_UNSUPPORTED;
  WgradArgs p{};
  p.offsets = offsets;
  p.n_groups = n_groups;
  p.rows = int32_t(rows);
  p.ks = int32_t(ks);
  p.m_dim = m_dim;
  p.n_dim = n_dim;
  p.m_tiles = (m_dim + 2 * BM - 1) / (2 * BM);
  p.n_tiles = (n_dim + bn - 1) / bn;
  p.tiles_inv = quotient_inverse(uint32_t(tiles));
  p.out = dw;
  p.wide = n_dim % 16 == 0 && reinterpret_cast<uintptr_t>(dw) % 32 == 0;
  p.partials = partials;
  p.status = status;
  CUtensorMap tmA, tmB;
  if (!map_mn(&tmA, a, rows, ld_a, m_dim, BM / 64, &p.a_fused) ||
      !map_mn(&tmB, b, rows, ld_b, n_dim, bn / 128, &p.b_fused))
    return MOE_B200_ERR_TMA;
  const int rc = bn == 256 ? launch_wgrad<T, 256>(tmA, tmB, p, units, dev, st)
                           : launch_wgrad<T, 128>(tmA, tmB, p, units, dev, st);
  if (rc != MOE_B200_OK || rows <= p.ks) return rc;
  auto join = bn == 256 ? wgrad_join_kernel<T, 256> : wgrad_join_kernel<T, 128>;
  return launch_pdl(join, dim3(unsigned(sm_count(dev) * 4)), dim3(JOIN_THREADS), 0, st, p) == cudaSuccess
             ? MOE_B200_OK
             : MOE_B200_ERR_CUDA;
}

static bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace grouped
}  // namespace moe

using namespace moe;

extern "C" {

int moe_b200_grouped_mm(const void* x, int64_t rows, int64_t ld_x, int32_t k_dim, const void* w,
                        int32_t n_groups, int64_t w_group_stride, int64_t ld_w, int32_t n_inner,
                        int32_t n_dim, const int32_t* offsets, int32_t dtype, void* y, int32_t* status,
                        void* stream) {
  if (rows < 0 || rows > grouped::MAX_DIM || k_dim > grouped::MAX_DIM || n_dim > grouped::MAX_DIM || k_dim < 8 || k_dim % 8 || n_dim < 8 || n_dim % 8 || n_groups < 1 ||
      n_groups > RUNS_MAX_GROUPS || ld_x < k_dim || ld_x % 8 || w_group_stride % 8 || ld_w % 8 ||
      w_group_stride < 0 || ld_w < (n_inner ? n_dim : k_dim))
    return MOE_B200_ERR_SHAPE;
  if (dtype != MOE_B200_BF16 && dtype != MOE_B200_FP16) return MOE_B200_ERR_UNSUPPORTED;
  if (rows == 0) return MOE_B200_OK;
  if (!x || !w || !offsets || !y || !status) return MOE_B200_ERR_NULL;
  if (!grouped::aligned(x, 16) || !grouped::aligned(w, 16) || !grouped::aligned(y, 16) ||
      !grouped::aligned(offsets, 4))
    return MOE_B200_ERR_ALIGN;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MOE_B200_BF16
             ? grouped::rows_product<__nv_bfloat16>(x, rows, ld_x, k_dim, w, n_groups, w_group_stride, ld_w,
                                                    n_inner, n_dim, offsets, y, status, st)
             : grouped::rows_product<__half>(x, rows, ld_x, k_dim, w, n_groups, w_group_stride, ld_w, n_inner,
                                             n_dim, offsets, y, status, st);
}

size_t moe_b200_grouped_wgrad_scratch_bytes(int32_t m_dim, int32_t n_dim, int64_t rows, int32_t n_groups) {
  if (m_dim < 8 || n_dim < 8 || m_dim > grouped::MAX_DIM || n_dim > grouped::MAX_DIM || rows < 0 || n_groups < 1) return 0;
  const int64_t tiles = grouped::wgrad_tiles(m_dim, n_dim);
  if (tiles > INT_MAX) return 0;   // (refused)
  const int64_t ks = grouped::wgrad_chunk(rows, n_groups, tiles);
  return size_t(grouped::split_chunks(rows, ks, n_groups)) * size_t(tiles) * 2 * grouped::BM *
         size_t(grouped::wgrad_bn(n_dim)) * sizeof(float);
}

int moe_b200_grouped_wgrad(const void* a, int64_t ld_a, int32_t m_dim, const void* b, int64_t ld_b,
                           int32_t n_dim, int64_t rows, const int32_t* offsets, int32_t n_groups,
                           int32_t dtype, void* dw, void* scratch, size_t scratch_bytes, int32_t* status,
                           void* stream) {
  if (rows < 0 || rows > grouped::MAX_DIM || m_dim > grouped::MAX_DIM || n_dim > grouped::MAX_DIM || m_dim < 8 || m_dim % 8 || n_dim < 8 || n_dim % 8 || n_groups < 1 ||
      n_groups > RUNS_MAX_GROUPS || ld_a < m_dim || ld_a % 8 || ld_b < n_dim || ld_b % 8)
    return MOE_B200_ERR_SHAPE;
  if (dtype != MOE_B200_BF16 && dtype != MOE_B200_FP16) return MOE_B200_ERR_UNSUPPORTED;
  if (grouped::wgrad_tiles(m_dim, n_dim) > INT_MAX) return MOE_B200_ERR_UNSUPPORTED;
  if (!dw || !status) return MOE_B200_ERR_NULL;
  if (!grouped::aligned(dw, 16)) return MOE_B200_ERR_ALIGN;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0)
    return cudaMemsetAsync(dw, 0, size_t(n_groups) * size_t(m_dim) * size_t(n_dim) * 2, st) == cudaSuccess
               ? MOE_B200_OK
               : MOE_B200_ERR_CUDA;
  if (!a || !b || !offsets) return MOE_B200_ERR_NULL;
  if (!grouped::aligned(a, 16) || !grouped::aligned(b, 16) || !grouped::aligned(offsets, 4) ||
      !grouped::aligned(scratch, 32))
    return MOE_B200_ERR_ALIGN;
  const size_t need = moe_b200_grouped_wgrad_scratch_bytes(m_dim, n_dim, rows, n_groups);
  if (need > scratch_bytes || (need > 0 && !scratch)) return MOE_B200_ERR_SCRATCH;
  float* partials = static_cast<float*>(scratch);
  return dtype == MOE_B200_BF16
             ? grouped::wgrad_product<__nv_bfloat16>(a, ld_a, m_dim, b, ld_b, n_dim, rows, offsets, n_groups, dw,
                                                     partials, status, st)
             : grouped::wgrad_product<__half>(a, ld_a, m_dim, b, ld_b, n_dim, rows, offsets, n_groups, dw, partials,
                                              status, st);
}

}  // extern "C"
