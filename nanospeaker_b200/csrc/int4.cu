// Products of few rows with weights held in 4 bits: W[k, n] = (level[k, n] - 8) * scale[k / group, n].
//
//   moe_b200_int4_mm       y = x @ W
//   moe_b200_int4_experts  the block's GLU experts (routed by top-k ids, and shared ones) for a batch that
//                          generates: up + GLU -> down -> weighted sum, three launches
//
// What bounds them is the weights' bytes, so a weight is read once and used for up to 32 rows from registers.
// The layout (nanospeaker_b200/int4.py packs it) is the matrix instruction's: a lane's 16 bytes are its A
// fragments (16 outputs x 16 inputs each) of 64 inputs, and the inputs are numbered within those 64 so that
// the B fragments of a row of x are two 16-byte pieces of it. Levels become 16-bit floats exactly (a byte
// operation and a subtraction per two), products are summed in fp32 over one scale group at a time, and the
// scale is applied to that sum: no rounding but the final one (and the GLU's result, which is held in the
// activations' type between the two products).
//
// A strip of 16 outputs is one contiguous piece, and so is a row's share of the inputs: both come to shared
// memory by bulk copies, which a warp of their own issues as far ahead as the ring holds.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/moe_b200.h"
#include "act.cuh"
#include "half16.cuh"
#include "pdl.cuh"
#include "per_device.cuh"
#include "ptx.cuh"

namespace moe {
namespace q4 {

constexpr int MAX_WARPS = 8;     // that multiply; one more copies
constexpr int STRIPS = 2;        // strips of 16 outputs a warp computes
constexpr int MAX_DEPTH = 6;     // stages of the ring
constexpr int PAIR_WINDOW = 1024;   // pairs whose expert ids are looked at in one go

// One matrix stack in the packed layout.
struct Stack {
  const uint4* levels;      // [groups][strips][kblocks][32 lanes]
  const uint32_t* scales;   // [groups][strips][kgroups][8]: outputs g and g + 8 of the strip
  int32_t groups;
};

enum Mode { DENSE = 0, GLU = 1, PAIRS = 2 };

struct Args {
  const void* x;
  int64_t ld_x;
  Stack routed, shared;
  int32_t k_dim, n_dim;        // valid inputs and outputs (GLU: outputs = the hidden width)
  int32_t kblocks, kgroups, strips;   // of both stacks
  int32_t group_shift;         // scale group = 32 << group_shift inputs
  int32_t wk, wn, kpb;         // warps that share a strip's inputs, pairs of strips per CTA, blocks of a warp
                               // in a stage
  int32_t n_stages, depth;     // stages of a pass, stages of the ring
  int32_t x_rows;              // rows of x that a stage has room for
  int32_t rows;                // DENSE: rows of x; else tokens
  // GLU / PAIRS: row p of the result is pair p of topk_idx, row n_pairs + s * rows + t token t of shared expert s
  const int64_t* topk_idx;
  int32_t n_pairs, top_k;
  int32_t row_chunks;          // CTAs that share the rows of a matrix all rows go to (DENSE, shared experts)
  int32_t eager;               // copy before it is known whether the expert has rows
  int32_t act;
  void* out;                   // DENSE [rows, n_dim], GLU [n_pairs + S * rows, n_dim] of T; PAIRS fp32
  int64_t ld_out;
  int32_t* status;
};

template <typename T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
  static constexpr uint32_t MAGIC = 0x43004300u;   // 128 + level, as a pair
  static __device__ __forceinline__ uint32_t less_bias(uint32_t a) {   // a * 1 - 136: one instruction
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(0x3F803F80u), "r"(0xC308C308u));
    return d;
  }
  static __device__ __forceinline__ void run(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void first(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  }
};
template <>
struct Mma<__half> {
  static constexpr uint32_t MAGIC = 0x64006400u;   // 1024 + level
  static __device__ __forceinline__ uint32_t less_bias(uint32_t a) {   // - 1032
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(0xE408E408u));
    return d;
  }
  static __device__ __forceinline__ void run(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void first(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  }
};

// A packed word's eight levels as the four registers of an A fragment, values -8 .. 7.
template <typename T>
__device__ __forceinline__ void levels_of(uint32_t word, uint32_t* a) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;   // (word >> 4 i) & 0x000F000F | MAGIC
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(word >> (4 * i)), "r"(0x000F000Fu), "r"(Mma<T>::MAGIC));
    a[i] = Mma<T>::less_bias(v);
  }
}

__device__ __forceinline__ float activation(int act, float g) {
  switch (act) {
    case ACT_SILU: return act_f<ACT_SILU>(g);
    case ACT_GELU: return act_f<ACT_GELU>(g);
    case ACT_RELU: return act_f<ACT_RELU>(g);
    case ACT_SIGMOID: return act_f<ACT_SIGMOID>(g);
    default: return act_f<ACT_TANH>(g);
  }
}

__device__ __forceinline__ void compute_sync(int nthreads) {
  asm volatile("bar.sync 1, %0;" ::"r"(nthreads) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// A stage of the ring, `blocks` blocks of 64 inputs: per strip their levels and scales, then the rows of x (64
// bytes behind each, so that the two rows that a quarter of a warp reads at a time lie in different banks).
struct StageShape {
  int strip, x, row, bytes;
  __host__ __device__ StageShape(int blocks, int strips, int rows)
      : strip(blocks * (512 + 64)), x(strips * strip), row(blocks * 128 + 64),
        bytes((x + rows * row + 127) / 128 * 128) {}
};

// CTAs that an SM holds (their registers and shared memory are sized for it): few warps each and many at a
// time, so that one CTA's start and end lie under the others' copies and the grid is one wave.
__host__ __device__ constexpr int ctas_per_sm(int nt) { return nt == 1 ? 4 : nt == 2 ? 3 : 2; }

// A CTA: wn pairs of strips of one matrix (GLU: a pair is a gate strip and its up strip), wk warps on each that
// share the inputs (a stage is a block of 64 for each) and add their sums in shared memory, and a warp that
// copies. NT: tiles of 8 rows per pass; more rows of one expert take more passes, which copy the weights
// again. FINE: scale groups of 32 inputs (two per block).
template <typename T, int NT, bool FINE, int MODE>
__global__ void __launch_bounds__((MAX_WARPS + 1) * 32, ctas_per_sm(NT)) int4_kernel(const Args p) {
  constexpr int ROWS = NT * 8, RED = ROWS + 1;   // (odd: a column of sums meets every bank)
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full_bar[MAX_DEPTH], empty_bar[MAX_DEPTH];
  __shared__ int list[MODE == DENSE ? 1 : PAIR_WINDOW];
  __shared__ int warp_count[MAX_WARPS + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_warps = p.wk * p.wn;
  const int span = p.wk * p.kpb;   // blocks of a stage
  const StageShape sh(span, p.wn * STRIPS, p.x_rows);
  float* red = reinterpret_cast<float*>(smem + p.depth * sh.bytes);   // [ceil(wk / 2)][wn][STRIPS * 16][RED]

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.depth; ++i) {
      mbar_init(full_bar + i, 1);
      mbar_init(empty_bar + i, n_warps);
    }
    fence_mbar_init();
  }
  __syncthreads();

  // which matrix, and which of its rows
  const bool all_rows = MODE == DENSE || int(blockIdx.y) >= p.routed.groups;
  const int y = MODE == DENSE ? blockIdx.y : int(blockIdx.y) - p.routed.groups;
  const int chunk = all_rows ? y % p.row_chunks : 0;
  const int e = MODE == DENSE ? 0 : all_rows ? y / p.row_chunks : int(blockIdx.y);
  const int strip_step = MODE == GLU ? p.strips / 2 : 1;
  const int n_stages = p.n_stages;
  // the row of the result, and of x, that row r of this expert is
  auto out_row = [&](int r) -> int64_t {
    if (MODE == DENSE) return r;
    return all_rows ? int64_t(p.n_pairs) + int64_t(e) * p.rows + r : list[r];
  };
  auto x_row = [&](int r) -> int64_t {
    return MODE == DENSE ? r : MODE == PAIRS ? out_row(r) : all_rows ? r : list[r] / p.top_k;
  };

  // ---- the copying warp's side, kept to few instructions a stage (a warp by itself takes a hundred cycles for
  // twenty): lane i has strip i of the CTA and row i of the pass. A pass is n_stages stages, the weights the
  // same ones in each; w_issued and x_issued count stages whose weights and rows have been asked for.
  const bool copies = warp == n_warps;
  const Stack w = MODE != DENSE && all_rows ? p.shared : p.routed;
  int w_issued = 0, w_stage = 0, w_slot = 0, w_phase = 1;   // (phase: of the slot's release before)
  int x_issued = 0, x_stage = 0, x_slot = 0;
  bool dead = false;
  int strip = p.strips;
  if (copies && lane < p.wn * STRIPS) {
    const int pair = blockIdx.x * p.wn + lane / STRIPS, s = lane % STRIPS;
    strip = MODE == GLU ? (pair < strip_step ? pair + s * strip_step : p.strips) : pair * STRIPS + s;
  }
  const int live_strips = __popc(__ballot_sync(0xffffffffu, strip < p.strips));
  const uint32_t ring = smem_u32(smem);
  const uint4* levels = w.levels + (int64_t(e) * p.strips + strip) * p.kblocks * 32;
  const uint32_t* scales = w.scales + (int64_t(e) * p.strips + strip) * p.kgroups * 8;
  auto groups = [&](int blocks) { return ((2 * blocks - 1) >> p.group_shift) + 1; };   // that blocks reach into
  const int last_blocks = p.kblocks - (n_stages - 1) * span;
  const int full_groups = groups(span), last_groups = groups(last_blocks);
  const int last_k = p.k_dim - (n_stages - 1) * span * 64;
  auto issue_weights = [&] {
    if (w_issued >= p.depth) {
      if (!mbar_wait(empty_bar + w_slot, w_phase, p.status)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
      if (dead) return;
    }
    if (strip < p.strips) {
      const bool last = w_stage == n_stages - 1;
      const uint32_t dst = ring + w_slot * sh.bytes + lane * sh.strip;
      bulk_load(dst, levels + int64_t(w_stage) * span * 32, (last ? last_blocks : span) * 512, full_bar + w_slot);
      bulk_load(dst + span * 512, scales + int64_t(w_stage) * full_groups * 8, (last ? last_groups : full_groups) * 32,
                full_bar + w_slot);
    }
    ++w_issued;
    if (++w_stage == n_stages) w_stage = 0;
    if (++w_slot == p.depth) {
      w_slot = 0;
      w_phase ^= 1;
    }
  };
  auto issue_rows = [&](const T* row, int rows) {   // (rows 0: the stage's weights alone)
    const bool last = x_stage == n_stages - 1;
    const uint32_t bytes = (last ? last_k : span * 64) * 2;
    if (lane == 0)
      mbar_expect_tx(full_bar + x_slot, live_strips * ((last ? last_blocks : span) * 512 +
                                                       (last ? last_groups : full_groups) * 32) + rows * bytes);
    __syncwarp();
    if (lane < rows)
      bulk_load(ring + x_slot * sh.bytes + sh.x + lane * sh.row, row + x_stage * span * 64, bytes,
                full_bar + x_slot);
    ++x_issued;
    if (++x_stage == n_stages) x_stage = 0;
    if (++x_slot == p.depth) x_slot = 0;
  };

  // The down projection's weights and ids are older than the kernel before it, whose result (the rows of
  // x) it waits for behind this: that kernel lets this one start when it has itself waited for all before it.
  if (MODE != PAIRS) pdl_wait();
  pdl_trigger();
  if (copies && (p.eager || all_rows))
    for (int i = min(p.depth, n_stages); i > 0; --i) issue_weights();

  const int windows = all_rows ? 1 : (p.n_pairs + PAIR_WINDOW - 1) / PAIR_WINDOW;
  bool waited = MODE != PAIRS;
  int slot = 0, phase = 0;
  for (int win = 0; win < windows; ++win) {
    int first = chunk * ROWS, n_rows = all_rows ? min(p.rows, first + ROWS) : 0;
    if (!all_rows) {
      // the pairs of this expert among the window's, in order: every warp looks at a share of them
      const int base = win * PAIR_WINDOW, n = min(PAIR_WINDOW, p.n_pairs - base);
      const int all = n_warps + 1;
      const int share = ((n + all - 1) / all + 31) / 32 * 32;
      const int lo = warp * share, hi = min(n, lo + share);
      int count = 0;
      for (int i = lo; i < hi; i += 32)
        count += __popc(__ballot_sync(0xffffffffu, i + lane < hi && p.topk_idx[base + i + lane] == e));
      if (win > 0) __syncthreads();     // (the list of the window before has been used)
      if (lane == 0) warp_count[warp] = count;
      __syncthreads();
      int at = 0;
      for (int i = 0; i < all; ++i) {
        at += i < warp ? warp_count[i] : 0;
        n_rows += warp_count[i];
      }
      if (count > 0) {
        for (int i = lo; i < hi; i += 32) {
          const bool mine = i + lane < hi && p.topk_idx[base + i + lane] == e;
          const uint32_t who = __ballot_sync(0xffffffffu, mine);
          if (mine) list[at + __popc(who & ((1u << lane) - 1))] = base + i + lane;
          at += __popc(who);
        }
      }
      __syncthreads();
    }
    if (n_rows <= first) continue;
    if (!waited) {
      pdl_wait();
      waited = true;
    }
    if (copies) {
      for (int r0 = first; r0 < n_rows && !dead; r0 += ROWS) {
        const int rows = min(ROWS, n_rows - r0);
        const T* row = static_cast<const T*>(p.x) + (lane < rows ? x_row(r0 + lane) * p.ld_x : 0);
        for (int i = 0; i < n_stages && !dead; ++i) {
          if (x_issued == w_issued) issue_weights();
          if (!dead) issue_rows(row, rows);
        }
      }
      if (dead && lane == 0) atomicExch(p.status, ST_WAIT_TIMEOUT);
      continue;
    }
    const int wn = warp / p.wk, wk = warp - wn * p.wk;
    const int g = lane >> 2, t = lane & 3;
    for (int r0 = first; r0 < n_rows; r0 += ROWS) {
      const int live = min(ROWS, n_rows - r0), tiles = (live + 7) / 8;
      float acc[STRIPS][NT][4];
#pragma unroll
      for (int s = 0; s < STRIPS; ++s)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[s][i][k] = 0.f;

      // where this lane's pieces of a stage are: levels, the rows of x (those that a tile lacks are taken from
      // its last one: their sums are not stored)
      const uint8_t* const q_at = smem + wn * STRIPS * sh.strip + wk * p.kpb * 512 + lane * 16;
      const uint8_t* const s_at = smem + wn * STRIPS * sh.strip + span * 512 + g * 4;
      const uint8_t* x_at[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i)
        x_at[i] = smem + sh.x + min(i * 8 + g, p.x_rows - 1) * sh.row + wk * p.kpb * 128 + t * 16;
      int kb = wk * p.kpb;   // this warp's block
      for (int st = 0; st < n_stages; ++st, kb += span - p.kpb) {
        if (!dead && !mbar_wait(full_bar + slot, phase, p.status)) {
          dead = true;
          atomicExch(p.status, ST_WAIT_TIMEOUT);
        }
        int off = slot * sh.bytes;
        // one block of 64 inputs; cut: it is the last, inputs from k_dim on were not copied and count as zero
        auto block = [&](int j, bool cut) {
          uint32_t a[STRIPS][4][4];
          uint32_t sc[STRIPS][FINE ? 2 : 1];
          const int lb = wk * p.kpb + j;
          const uint8_t* s_of = s_at + off + ((2 * lb) >> p.group_shift) * 32;
#pragma unroll
          for (int s = 0; s < STRIPS; ++s) {
            const uint4 q = *reinterpret_cast<const uint4*>(q_at + off + j * 512 + s * sh.strip);
#pragma unroll
            for (int h = 0; h < (FINE ? 2 : 1); ++h)
              sc[s][h] = *reinterpret_cast<const uint32_t*>(s_of + s * sh.strip + h * 32);
            levels_of<T>(q.x, a[s][0]);
            levels_of<T>(q.y, a[s][1]);
            levels_of<T>(q.z, a[s][2]);
            levels_of<T>(q.w, a[s][3]);
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            if (i > 0 && i >= tiles) break;
            uint4 b0 = *reinterpret_cast<const uint4*>(x_at[i] + off + j * 128);
            uint4 b1 = *reinterpret_cast<const uint4*>(x_at[i] + off + j * 128 + 64);
            if (cut) {
              const int k = kb * 64 + t * 8;
              if (k >= p.k_dim) b0 = make_uint4(0, 0, 0, 0);
              if (k + 32 >= p.k_dim) b1 = make_uint4(0, 0, 0, 0);
            }
            float c[STRIPS][4];
            auto scale_in = [&](int h) {
#pragma unroll
              for (int s = 0; s < STRIPS; ++s) {
                const float2 f = Half16<T>::unpack(sc[s][h]);
                acc[s][i][0] += f.x * c[s][0];
                acc[s][i][1] += f.x * c[s][1];
                acc[s][i][2] += f.y * c[s][2];
                acc[s][i][3] += f.y * c[s][3];
              }
            };
#pragma unroll
            for (int s = 0; s < STRIPS; ++s) Mma<T>::first(c[s], a[s][0], b0.x, b0.y);
#pragma unroll
            for (int s = 0; s < STRIPS; ++s) Mma<T>::run(c[s], a[s][1], b0.z, b0.w);
            if constexpr (FINE) {
              scale_in(0);
#pragma unroll
              for (int s = 0; s < STRIPS; ++s) Mma<T>::first(c[s], a[s][2], b1.x, b1.y);
            } else {
#pragma unroll
              for (int s = 0; s < STRIPS; ++s) Mma<T>::run(c[s], a[s][2], b1.x, b1.y);
            }
#pragma unroll
            for (int s = 0; s < STRIPS; ++s) Mma<T>::run(c[s], a[s][3], b1.z, b1.w);
            scale_in(FINE ? 1 : 0);
          }
        };
        for (int j = 0; j < p.kpb; ++j, ++kb) {
          if ((kb + 1) * 64 <= p.k_dim) block(j, false);
          else if (kb < p.kblocks) block(j, true);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty_bar + slot);
        if (++slot == p.depth) {
          slot = 0;
          phase ^= 1;
        }
      }

      // The warps' sums meet in shared memory, the upper half's added to the lower half's until one is left.
      auto red_at = [&](int k) { return red + ((k * p.wn + wn) * STRIPS * 16 + g) * RED + 2 * t; };
      auto each = [&](auto f) {
#pragma unroll
        for (int s = 0; s < STRIPS; ++s)
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) f(acc[s][i][k], (s * 16 + (k >> 1) * 8) * RED + i * 8 + (k & 1));
      };
      int n = p.wk;
      while (n > 1) {
        const int half = (n + 1) >> 1;
        if (wk >= half && wk < n) {
          float* to = red_at(wk - half);
          each([&](float& v, int o) { to[o] = v; });
        }
        compute_sync(n_warps * 32);
        if (wk < n - half) {
          const float* from = red_at(wk);
          each([&](float& v, int o) { v += from[o]; });
        }
        compute_sync(n_warps * 32);
        n = half;
      }
      if (wk == 0) {
        float* to = red_at(0);
        each([&](float& v, int o) { to[o] = v; });
      }
      compute_sync(n_warps * 32);
      constexpr int OUT = MODE == GLU ? 16 : STRIPS * 16;   // results of a pair of strips
      const int n_out = OUT * p.wn;
      for (int i = threadIdx.x; i < n_out * live; i += n_warps * 32) {
        const int r = i / n_out, c = i - r * n_out, o = c % OUT;
        const int col = blockIdx.x * n_out + c;
        if (col >= p.n_dim) continue;
        const float* v = red + (c / OUT * STRIPS * 16 + o) * RED + r;
        const int64_t to = out_row(r0 + r) * p.ld_out + col;
        if (MODE == GLU)
          static_cast<T*>(p.out)[to] = Half16<T>::from_float(activation(p.act, v[0]) * v[16 * RED]);
        else if (MODE == DENSE)
          static_cast<T*>(p.out)[to] = Half16<T>::from_float(v[0]);
        else
          static_cast<float*>(p.out)[to] = v[0];
      }
      compute_sync(n_warps * 32);
    }
  }
  // weights copied for rows that did not come: nobody leaves with a copy in flight
  if (copies) {
    while (x_issued < w_issued) {
      const int s = x_slot, use = x_issued / p.depth;
      issue_rows(nullptr, 0);
      for (int n = 0; n < 4096 && !mbar_try_wait(full_bar + s, use & 1); ++n) {
      }
    }
  }
  // (what comes behind this kernel counts on all before it being over: nobody leaves before its own wait)
  if (!waited) pdl_wait();
}

// out[t] = sum_j topk_w[t, j] * y[t * top_k + j] + sum_s y[n_pairs + s * n_tokens + t], fp32, in that order.
// A pair whose expert does not exist has no row: it adds nothing and is reported.
template <typename T>
__global__ void __launch_bounds__(256)
    int4_sum_kernel(const float* y, const T* topk_w, const int64_t* topk_idx, int32_t n_tokens, int32_t top_k,
                    int32_t n_experts, int32_t n_shared, int32_t d, T* out, int32_t* status) {
  pdl_trigger();
  pdl_wait();
  const int64_t n_pairs = int64_t(n_tokens) * top_k, n4 = int64_t(n_tokens) * (d / 4);
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n4; i += int64_t(gridDim.x) * 256) {
    const int64_t tok = i / (d / 4);
    const int c = int(i - tok * (d / 4)) * 4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = 0; j < top_k; ++j) {
      const int64_t pair = tok * top_k + j;
      const int64_t e = ld_prev(topk_idx + pair);
      if (e < 0 || e >= n_experts) {
        if (c == 0) atomicExch(status, ST_BAD_EXPERT);
        continue;
      }
      const float w = Half16<T>::to_float(ld_prev(topk_w + pair));
      const float4 v = *reinterpret_cast<const float4*>(y + pair * d + c);
      a.x += w * v.x; a.y += w * v.y; a.z += w * v.z; a.w += w * v.w;
    }
    for (int s = 0; s < n_shared; ++s) {
      const float4 v = *reinterpret_cast<const float4*>(y + (n_pairs + int64_t(s) * n_tokens + tok) * d + c);
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
    *reinterpret_cast<uint2*>(out + tok * d + c) =
        make_uint2(Half16<T>::pack(a.x, a.y), Half16<T>::pack(a.z, a.w));
  }
}

// How a CTA's warps divide the work: eight on a strip's inputs where it is long, else fewer on
// more strips. A stage is a multiple of every scale group, or the whole strip.
static void set_shape(Args& a, int32_t k_dim, int32_t n_dim, int32_t n_cols, int32_t group, bool glu) {
  a.k_dim = k_dim;
  a.n_dim = n_dim;
  a.kblocks = (k_dim + 63) / 64;
  a.kgroups = (a.kblocks * 64 + group - 1) / group;
  a.strips = (n_cols + 15) / 16;
  a.group_shift = group == 32 ? 0 : group == 64 ? 1 : 2;
  a.wk = a.kblocks >= 32 ? 8 : a.kblocks >= 4 ? 4 : a.kblocks >= 2 ? 2 : 1;
  a.kpb = a.kblocks >= 16 ? 2 : 1;
  const int pairs = glu ? a.strips / 2 : (a.strips + 1) / 2;
  a.wn = std::min(MAX_WARPS / a.wk, pairs);
  a.n_stages = (a.kblocks + a.wk * a.kpb - 1) / (a.wk * a.kpb);
}
static unsigned ctas_for(const Args& a, bool glu) {
  const int pairs = glu ? a.strips / 2 : (a.strips + 1) / 2;
  return unsigned((pairs + a.wn - 1) / a.wn);
}

template <typename T, int NT, bool FINE, int MODE>
static int launch(Args a, cudaStream_t st) {
  auto kern = int4_kernel<T, NT, FINE, MODE>;
  // shared memory of a CTA: an equal share for as many as the registers allow
  constexpr int share = 227 * 1024 / ctas_per_sm(NT) / 1024 * 1024 - 1024 - (MODE == DENSE ? 0 : 4 * PAIR_WINDOW) - 256;
  a.x_rows = MODE == DENSE ? std::min(a.rows, NT * 8) : NT * 8;
  const StageShape sh(a.wk * a.kpb, a.wn * STRIPS, a.x_rows);
  const int red = (a.wk + 1) / 2 * a.wn * STRIPS * 16 * (NT * 8 + 1) * int(sizeof(float));
  a.depth = std::max(1, std::min(std::min((share - red) / sh.bytes, a.n_stages), MAX_DEPTH));
  const int smem = a.depth * sh.bytes + red;
  static PerDevice<cudaError_t> ready;
  int dev = -1;
  const cudaError_t* ok = cudaGetDevice(&dev) != cudaSuccess ? nullptr : ready.get(dev, [&](int) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, share);
  });
  if (ok == nullptr || *ok != cudaSuccess || smem > share) return MOE_B200_ERR_CUDA;
  a.row_chunks = std::max(1, (a.rows + NT * 8 - 1) / (NT * 8));
  const int64_t ys = MODE == DENSE ? a.row_chunks : a.routed.groups + int64_t(a.shared.groups) * a.row_chunks;
  if (ys > 65535) return MOE_B200_ERR_UNSUPPORTED;
  return launch_pdl(kern, dim3(ctas_for(a, MODE == GLU), unsigned(ys)), dim3((a.wk * a.wn + 1) * 32), size_t(smem), st,
                    a) == cudaSuccess
             ? MOE_B200_OK
             : MOE_B200_ERR_CUDA;
}
template <typename T, int MODE>
static int launch_for(const Args& a, int64_t rows, cudaStream_t st) {
#define LAUNCH(N) (a.group_shift == 0 ? launch<T, N, true, MODE>(a, st) : launch<T, N, false, MODE>(a, st))
  if (rows <= 8) return LAUNCH(1);
  if (rows <= 16) return LAUNCH(2);
  return LAUNCH(4);
#undef LAUNCH
}

static bool group_ok(int32_t g) { return g == 32 || g == 64 || g == 128; }
static bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename T>
static int experts(const void* x, int64_t ld_x, int64_t n_tokens, int32_t d, int32_t h, const void* topk_w,
                   const int64_t* topk_idx, int32_t top_k, const Stack& in, const Stack& in_sh,
                   const Stack& down, const Stack& down_sh, int32_t group, int32_t act, void* out,
                   uint8_t* scratch, size_t hid_bytes, int32_t* status, cudaStream_t st) {
  const int32_t n_pairs = int32_t(n_tokens * top_k);
  float* y = reinterpret_cast<float*>(scratch + hid_bytes);
  // rows per pass: half as many again as an expert has on average
  const int64_t rows = (int64_t(n_pairs) * 3 / 2 + in.groups - 1) / in.groups;
  Args a{};
  a.x = x;
  a.ld_x = ld_x;
  a.routed = in;
  a.shared = in_sh;
  set_shape(a, d, h, 2 * h, group, true);
  a.rows = int32_t(n_tokens);
  a.topk_idx = topk_idx;
  a.n_pairs = n_pairs;
  a.top_k = top_k;
  a.eager = n_pairs >= in.groups;   // (then most experts have rows)
  a.act = act;
  a.out = scratch;
  a.ld_out = h;
  a.status = status;
  int rc = launch_for<T, GLU>(a, rows, st);
  if (rc != MOE_B200_OK) return rc;
  a.x = scratch;
  a.ld_x = h;
  a.routed = down;
  a.shared = down_sh;
  set_shape(a, h, d, d, group, false);
  a.out = y;
  a.ld_out = d;
  rc = launch_for<T, PAIRS>(a, rows, st);
  if (rc != MOE_B200_OK) return rc;
  const int64_t blocks = std::min<int64_t>((n_tokens * (d / 4) + 255) / 256, 148 * 8);
  return launch_pdl(int4_sum_kernel<T>, dim3(unsigned(blocks)), dim3(256), 0, st,
                    static_cast<const float*>(y), static_cast<const T*>(topk_w), topk_idx, int32_t(n_tokens),
                    top_k, in.groups, in_sh.groups, d, static_cast<T*>(out), status) == cudaSuccess
             ? MOE_B200_OK
             : MOE_B200_ERR_CUDA;
}

}  // namespace q4
}  // namespace moe

using namespace moe;

extern "C" {

int moe_b200_int4_mm(const void* x, int64_t rows, int64_t ld_x, int32_t k_dim, const void* levels,
                     const void* scales, int32_t group, int32_t n_dim, int32_t dtype, void* y, int32_t* status,
                     void* stream) {
  if (rows < 0 || rows > 0x7fffffff || k_dim < 8 || k_dim % 8 || n_dim < 1 || ld_x < k_dim || ld_x % 8 ||
      !q4::group_ok(group))
    return MOE_B200_ERR_SHAPE;
  if (dtype != MOE_B200_BF16 && dtype != MOE_B200_FP16) return MOE_B200_ERR_UNSUPPORTED;
  if (rows == 0) return MOE_B200_OK;
  if (!x || !levels || !scales || !y || !status) return MOE_B200_ERR_NULL;
  if (!q4::aligned(x, 16) || !q4::aligned(levels, 16) || !q4::aligned(scales, 16) || !q4::aligned(y, 2))
    return MOE_B200_ERR_ALIGN;
  q4::Args a{};
  a.x = x;
  a.ld_x = ld_x;
  a.routed = {static_cast<const uint4*>(levels), static_cast<const uint32_t*>(scales), 1};
  q4::set_shape(a, k_dim, n_dim, n_dim, group, false);
  a.rows = int32_t(rows);
  a.out = y;
  a.ld_out = n_dim;
  a.status = status;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MOE_B200_BF16 ? q4::launch_for<__nv_bfloat16, q4::DENSE>(a, rows, st)
                                : q4::launch_for<__half, q4::DENSE>(a, rows, st);
}

size_t moe_b200_int4_experts_scratch_bytes(int64_t n_tokens, int32_t top_k, int32_t n_shared, int32_t d_model,
                                           int32_t d_hidden) {
  if (n_tokens < 0 || top_k < 0 || n_shared < 0 || d_model < 1 || d_hidden < 1) return 0;
  const size_t rows = size_t(n_tokens) * size_t(top_k + n_shared);
  const size_t hid = (rows * size_t(d_hidden) * 2 + 255) / 256 * 256;
  return hid + rows * size_t(d_model) * sizeof(float);
}

int moe_b200_int4_experts(const void* x, int64_t n_tokens, int64_t ld_x, int32_t d_model, int32_t d_hidden,
                          const void* topk_w, const int64_t* topk_idx, int32_t top_k, int32_t n_experts,
                          const void* in_levels, const void* in_scales, const void* out_levels,
                          const void* out_scales, int32_t n_shared, const void* sh_in_levels,
                          const void* sh_in_scales, const void* sh_out_levels, const void* sh_out_scales,
                          int32_t group, int32_t activation, int32_t dtype, void* out, void* scratch,
                          size_t scratch_bytes, int32_t* status, void* stream) {
  if (n_tokens < 0 || top_k < 1 || n_experts < 1 || n_shared < 0 || n_experts + int64_t(n_shared) > 65535 ||
      d_model < 8 || d_model % 8 || d_hidden < 16 || d_hidden % 16 || ld_x < d_model || ld_x % 8 ||
      !q4::group_ok(group) || n_tokens * (int64_t(top_k) + n_shared) > 0x7fffffff)
    return MOE_B200_ERR_SHAPE;
  if (dtype != MOE_B200_BF16 && dtype != MOE_B200_FP16) return MOE_B200_ERR_UNSUPPORTED;
  if (activation < MOE_B200_ACT_SILU || activation > MOE_B200_ACT_TANH) return MOE_B200_ERR_UNSUPPORTED;
  if (n_tokens == 0) return MOE_B200_OK;
  if (!x || !topk_w || !topk_idx || !in_levels || !in_scales || !out_levels || !out_scales || !out || !status ||
      (n_shared > 0 && (!sh_in_levels || !sh_in_scales || !sh_out_levels || !sh_out_scales)))
    return MOE_B200_ERR_NULL;
  if (!q4::aligned(x, 16) || !q4::aligned(topk_w, 2) || !q4::aligned(topk_idx, 8) ||
      !q4::aligned(in_levels, 16) || !q4::aligned(out_levels, 16) || !q4::aligned(sh_in_levels, 16) ||
      !q4::aligned(sh_out_levels, 16) || !q4::aligned(in_scales, 16) || !q4::aligned(out_scales, 16) ||
      !q4::aligned(sh_in_scales, 16) || !q4::aligned(sh_out_scales, 16) || !q4::aligned(out, 16) ||
      !q4::aligned(scratch, 16))
    return MOE_B200_ERR_ALIGN;
  const size_t need = moe_b200_int4_experts_scratch_bytes(n_tokens, top_k, n_shared, d_model, d_hidden);
  if (!scratch || scratch_bytes < need) return MOE_B200_ERR_SCRATCH;
  const size_t hid = (size_t(n_tokens) * size_t(top_k + n_shared) * size_t(d_hidden) * 2 + 255) / 256 * 256;
  auto stack = [](const void* l, const void* s, int32_t n) {
    return q4::Stack{static_cast<const uint4*>(l), static_cast<const uint32_t*>(s), n};
  };
  const q4::Stack in = stack(in_levels, in_scales, n_experts), down = stack(out_levels, out_scales, n_experts);
  const q4::Stack in_sh = stack(sh_in_levels, sh_in_scales, n_shared);
  const q4::Stack down_sh = stack(sh_out_levels, sh_out_scales, n_shared);
  uint8_t* s = static_cast<uint8_t*>(scratch);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MOE_B200_BF16
             ? q4::experts<__nv_bfloat16>(x, ld_x, n_tokens, d_model, d_hidden, topk_w, topk_idx, top_k, in,
                                            in_sh, down, down_sh, group, activation, out, s, hid, status, st)
             : q4::experts<__half>(x, ld_x, n_tokens, d_model, d_hidden, topk_w, topk_idx, top_k, in, in_sh,
                                     down, down_sh, group, activation, out, s, hid, status, st);
}

}  // extern "C"
