// Runs of rows given by their starts: offsets[g] .. offsets[g + 1] are the rows of group g, back to back,
// with no padding and of any length. The table a kernel makes of them in shared memory, by one warp.
#pragma once
#include <stdint.h>

#include "pdl.cuh"

namespace moe {

constexpr int RUNS_MAX_GROUPS = 1024;

struct RunTable {
  int start[RUNS_MAX_GROUPS + 1];   // first row of every run, then the end of the last
  int first[RUNS_MAX_GROUPS + 1];   // first work unit of every run, then their number
};

// An exclusive prefix sum (or maximum, from 0 on) over the warp. As a loop: a kernel's first work waits for its
// code more than for anything else (the table of 76 runs in straight lines took 6000 cycles the first time and 600
// the second; as it stands, 2000).
template <bool MAX>
__device__ __forceinline__ int warp_prefix(int v, int lane, int* all) {
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = MAX ? max(v, u) : v + u;
  }
  *all = __shfl_sync(0xffffffffu, v, 31);
  const int before = __shfl_up_sync(0xffffffffu, v, 1);
  return lane ? before : 0;
}

constexpr int RUNS_PER_LANE = 4;

// Starts that decrease or leave [0, rows] cannot reach memory: a start is taken into that range and is at
// least every earlier one. True when any had to be changed (the caller reports it).
__device__ __forceinline__ bool load_run_starts(const int32_t* offsets, int n_groups, int rows, int lane,
                                                int* start) {
  int high = 0;
  bool changed = false;
#pragma unroll 1
  for (int base = lane * RUNS_PER_LANE; base - lane * RUNS_PER_LANE <= n_groups; base += 32 * RUNS_PER_LANE) {
    int raw[RUNS_PER_LANE], v[RUNS_PER_LANE];
#pragma unroll
    for (int i = 0; i < RUNS_PER_LANE; ++i) raw[i] = ld_prev(offsets + min(base + i, n_groups));
    int own = 0, all;
#pragma unroll
    for (int i = 0; i < RUNS_PER_LANE; ++i) v[i] = own = max(own, min(raw[i], rows));
    const int before = max(high, warp_prefix<true>(own, lane, &all));
#pragma unroll
    for (int i = 0; i < RUNS_PER_LANE; ++i) {
      v[i] = max(v[i], before);
      changed |= v[i] != raw[i];
      start[min(base + i, n_groups)] = v[i];   // (behind the last start: that one again)
    }
    high = max(high, all);
  }
  __syncwarp();
  return __any_sync(0xffffffffu, changed);
}

// first[g] = units of the runs before g, units_of(rows) for each; returns their number.
template <typename UnitsOf>
__device__ __forceinline__ int count_run_units(const int* start, int n_groups, int lane, int* first,
                                               UnitsOf units_of) {
  int before = 0;
#pragma unroll 1
  for (int base = lane * RUNS_PER_LANE; base - lane * RUNS_PER_LANE < n_groups; base += 32 * RUNS_PER_LANE) {
    int own = 0, all, v[RUNS_PER_LANE];
#pragma unroll
    for (int i = 0; i < RUNS_PER_LANE; ++i) {
      const int g = min(base + i, n_groups - 1);
      v[i] = own;
      own += base + i < n_groups ? units_of(start[g + 1] - start[g]) : 0;
    }
    const int upto = before + warp_prefix<false>(own, lane, &all);
#pragma unroll
    for (int i = 0; i < RUNS_PER_LANE; ++i)
      if (base + i < n_groups) first[base + i] = upto + v[i];
    before += all;
  }
  if (lane == 0) first[n_groups] = before;
  __syncwarp();
  return before;
}

// The run that unit u (below first[n_groups]) belongs to: the last one that starts there or before, which
// is never one without units.
__device__ __forceinline__ int run_of_unit(const int* first, int n_groups, int u) {
  int lo = 0, hi = n_groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= u) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The same by a warp together, from a run at or before it on.
__device__ __forceinline__ int run_of_unit_warp(const int* first, int n_groups, int u, int from, int lane) {
  for (;; from += 32) {
    const uint32_t behind = __ballot_sync(0xffffffffu, from + lane + 1 < n_groups && first[from + lane + 1] <= u);
    if (behind != 0xffffffffu) return from + __popc(behind);
  }
}

}  // namespace moe
