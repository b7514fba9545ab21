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

__device__ __forceinline__ int warp_prefix_sum(int v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ int warp_prefix_max(int v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = max(v, u);
  }
  return v;
}

// Starts that decrease or leave [0, rows] cannot reach memory: a start is taken into that range and is at
// least every earlier one. True when any had to be changed (the caller reports it).
__device__ __forceinline__ bool load_run_starts(const int32_t* offsets, int n_groups, int rows, int lane,
                                                int* start) {
  constexpr int AT_ONCE = 4;   // loads in flight: this is a kernel's first work
  int high = 0;
  bool changed = false;
  for (int base = 0; base <= n_groups; base += 32 * AT_ONCE) {
    int raw[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int g = base + 32 * i + lane;
      raw[i] = g <= n_groups ? ld_prev(offsets + g) : 0;
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int g = base + 32 * i + lane;
      const int v = max(high, warp_prefix_max(min(max(raw[i], 0), rows), lane));
      if (g <= n_groups) {
        start[g] = v;
        changed |= v != raw[i];
      }
      high = __shfl_sync(0xffffffffu, v, 31);   // (behind the last start the lanes repeat the highest)
    }
  }
  __syncwarp();
  return __any_sync(0xffffffffu, changed);
}

// first[g] = units of the runs before g, units_of(rows) for each; returns their number.
template <typename UnitsOf>
__device__ __forceinline__ int count_run_units(const int* start, int n_groups, int lane, int* first,
                                               UnitsOf units_of) {
  int before = 0;
  for (int base = 0; base < n_groups; base += 32) {
    const int g = base + lane;
    const int own = g < n_groups ? units_of(start[g + 1] - start[g]) : 0;
    const int upto = warp_prefix_sum(own, lane);
    if (g < n_groups) first[g] = before + upto - own;
    before += __shfl_sync(0xffffffffu, upto, 31);
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
