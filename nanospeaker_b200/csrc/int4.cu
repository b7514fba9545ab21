// Products of few rows with weights held in 4 bits: W[k, n] = (level[k, n] - 8) * scale[k / group, n].
//
//   moe_b200_int4_mm       y = x @ W
//   moe_b200_int4_experts  the block's GLU experts (routed by top-k ids, and shared ones) for a batch that
//                          generates: up + GLU -> down -> weighted sum, three launches
//
// What they cannot do without is the weights' bytes, so a weight is read once and used for up to 32 rows from
// registers; what bounds them is the latency of a CTA's start and of its instructions.
// The layout (nanospeaker_b200/int4.py packs it) is the matrix instruction's: a lane's 16 bytes are its A
// fragments (16 outputs x 16 inputs each) of 64 inputs, and the inputs are numbered within those 64 so that
// the B fragments of a row of x are two 16-byte pieces of it. Levels become 16-bit floats exactly (a byte
// operation and a subtraction per two), products are summed in fp32 over one scale group at a time, and the
// scale is applied to that sum: no rounding but the final one. The GLU's result has to be an operand of the matrix
// instruction again: it is held as two bf16 numbers, its upper half and what is left (2^-15 of the value at most is
// lost, and fp32's range kept), and the down projection multiplies its levels, exact in bf16 too, with both. Held in
// the activations' type it cost as much again as the rounding of the result (relative error against 64 bits: bf16
// 0.0024 to 0.0027 in place of 0.0017, fp16 0.00029 in place of 0.00021).
//
// In a graph, us: one row of 4096 x 16384 12.9, 64 of 4096 x 4096 12.1; the experts of one token 8.8, of 64 14.9, of 200
// tokens of the wide block (32 experts of 1024 x 768, four a token) 57.6. Figures further down compare the two sides of
// one choice when it was made; the experts' are up to 5 us lower there, before hidden values had a second part.
//
// A chunk of 512 inputs of neighbouring strips (16 outputs each), levels and scales together, is one contiguous
// piece: it comes to shared memory by one bulk copy (which costs the SM's copy engine some 50 cycles however
// small it is). The rows of x, few, in any place and read by every CTA, come by 16-byte asynchronous copies.
// Warps of their own issue both as far ahead as the ring holds.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "../../include/moe_b200.h"
#include "act.cuh"
#include "grouped_order.cuh"
#include "half16.cuh"
#include "pdl.cuh"
#include "per_device.cuh"
#include "ptx.cuh"

namespace moe {
namespace q4 {

constexpr int MAX_WARPS = 4;     // of a CTA that multiply (copy_warps more copy)
constexpr int STRIPS = 2;        // strips of 16 outputs a warp computes
constexpr int MAX_DEPTH = 6;     // stages of the ring
constexpr int PAIR_WINDOW = 1024;   // pairs whose expert ids are looked at in one go

constexpr int CHUNK = 8;         // blocks of 64 inputs in a chunk
constexpr int MAX_WIDTH = 0x7fffffff - 256;   // what a block or a CTA's strips have behind the last is still an int

// A stack of matrices in the packed layout (include/moe_b200.h).
struct Stack {
  const uint8_t* data;
  int32_t groups;
};

enum Mode { DENSE = 0, GLU = 1, PAIRS = 2 };
// Numbers that a value of x is held in: the GLU's result, which the down projection reads, is two bf16 values.
__host__ __device__ constexpr int parts_of(int mode) { return mode == PAIRS ? 2 : 1; }

struct Args {
  const void* x;               // PAIRS: [k_dim upper halves | k_dim rests] a row
  int64_t ld_x;
  Stack routed, shared;
  int32_t k_dim, n_dim;        // valid inputs and outputs (GLU: outputs = the hidden width)
  int32_t kblocks, strips;     // of both stacks
  int32_t group_shift;         // scale group = 32 << group_shift inputs
  int32_t n_stages, depth;     // stages of a pass over a strip, each a chunk (halves: half of one); of the ring
  int32_t full_blocks, last_blocks;   // blocks of a stage, of the last one
  int32_t full, last;          // bytes of a strip's piece of a stage
  int32_t halves, chunk;       // bytes of a strip's piece of a whole chunk
  int64_t matrix;              // bytes of a matrix
  int32_t wk, wn, kpb;         // warps that share a strip's inputs, pairs of strips per CTA, blocks of a warp
                               // in a stage
  int32_t x_rows;              // rows of x that a stage has room for
  int32_t rows;                // DENSE: rows of x; else tokens
  // GLU / PAIRS: row p of the result is pair p of topk_idx, row n_pairs + s * rows + t token t of shared expert s
  const int64_t* topk_idx;
  int32_t n_pairs, top_k;
  uint32_t top_k_inv, row_chunks_inv;   // (quotient)
  int32_t row_chunks;          // CTAs that share the rows of a matrix all rows go to (DENSE, shared experts)
  int32_t eager;               // copy before it is known whether the expert has rows
  int32_t act;
  void* out;                   // DENSE [rows, n_dim] of T, GLU [n_pairs + S * rows, 2, n_dim] bf16; PAIRS fp32
  int64_t ld_out;
  int32_t* status;
};

template <typename T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
  static constexpr uint32_t MAGIC = 0x43004300u;   // 128 + level, as a pair
  static constexpr bool WIDE = false;              // (seven bits: no room for 16 * level)
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
  static constexpr bool WIDE = true;
  static __device__ __forceinline__ uint32_t less_bias(uint32_t a) {   // - 1032
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(0xE408E408u));
    return d;
  }
  static __device__ __forceinline__ uint32_t less_bias16(uint32_t a) {   // (1024 + 16 * level) / 16 - 72
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(0x2C002C00u), "r"(0xD480D480u));
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

// A packed word's eight levels as the four registers of an A fragment, values -8 .. 7: a level is laid into the lowest
// bits of a power of two, which is then subtracted (as Kim, Henry, Fahim, Awadalla describe for quantised weights, "Who
// Says Elephants Can't Run: Bringing Large Scale MoE Models into Cloud Scale Production", 2022). (fp16 has the bits for a
// level where it lies, times 16: of three shifts one is left. 200 tokens of the wide block 55.4 -> 54.3 us.)
template <typename T>
__device__ __forceinline__ void levels_of(uint32_t word, uint32_t* a) {
  auto lay = [](uint32_t w, uint32_t mask) {   // w & mask | MAGIC
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "r"(mask), "r"(Mma<T>::MAGIC));
    return v;
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Mma<T>::WIDE) {
      const uint32_t w = word >> (8 * (i / 2));
      a[i] = i % 2 ? Mma<T>::less_bias16(lay(w, 0x00F000F0u)) : Mma<T>::less_bias(lay(w, 0x000F000Fu));
    } else {
      a[i] = Mma<T>::less_bias(lay(word >> (4 * i), 0x000F000Fu));
    }
  }
}

// Four at a time, side by side: one after another they were a tenth of a CTA's time. (Called, not copied to every
// place: these kernels are over before much code has been fetched.) tanh is CUDA's own: the block's 2 / (1 + exp(-2 g))
// - 1 is off by 2^-24 however small g is, more than fp16's rounding below |g| = 2^-13.
template <int ACT>
__device__ __forceinline__ float4 act4(const float4& g) {
  if constexpr (ACT == ACT_TANH) return make_float4(tanhf(g.x), tanhf(g.y), tanhf(g.z), tanhf(g.w));
  return make_float4(act_f<ACT>(g.x), act_f<ACT>(g.y), act_f<ACT>(g.z), act_f<ACT>(g.w));
}
__device__ __noinline__ float4 activation(int act, float4 g) {
  switch (act) {
    case ACT_SILU: return act4<ACT_SILU>(g);
    case ACT_GELU: return act4<ACT_GELU>(g);
    case ACT_RELU: return act4<ACT_RELU>(g);
    case ACT_SIGMOID: return act4<ACT_SIGMOID>(g);
    default: return act4<ACT_TANH>(g);
  }
}

// Two values as pairs of bf16: their upper halves (cut, so that nothing finite becomes an infinity) and the rests,
// rounded (of an infinity nothing: it would be infinity less infinity).
__device__ __forceinline__ void split(const float2& v, uint32_t& upper, uint32_t& rest) {
  const uint32_t x = __float_as_uint(v.x), y = __float_as_uint(v.y);
  upper = __byte_perm(x, y, 0x7632);
  auto left = [](float f, uint32_t bits) { return isinf(f) ? 0.f : f - __uint_as_float(bits & 0xFFFF0000u); };
  rest = Half16<__nv_bfloat16>::pack(left(v.x, x), left(v.y, y));
}

__device__ __forceinline__ uint32_t ld_shared_b32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void compute_sync(int nthreads) {
  asm volatile("bar.sync 1, %0;" ::"r"(nthreads) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Bytes of a strip's piece of `blocks` blocks: levels, and scales of groups of 32 << group_shift inputs.
__host__ __device__ constexpr int piece_bytes(int blocks, int group_shift) {
  return blocks * 512 + (((2 * blocks - 1) >> group_shift) + 1) * 32;
}

// A stage of the ring, up to `blocks` blocks: the strips' pieces, then the rows of x. A row's 16-byte
// piece c lies at c, in odd rows at c ^ 4: the two rows that a quarter of a warp reads at a time then lie in
// different banks. A row of two parts has the second one behind the first.
struct StageShape {
  int x, row, bytes;
  __host__ __device__ StageShape(int blocks, int strips, int piece, int rows, int parts)
      : x((strips * piece + 127) / 128 * 128), row(blocks * 128 * parts), bytes((x + rows * row + 127) / 128 * 128) {}
};

// CTAs that an SM holds (their registers and shared memory are sized for it): many at a time, so that one's
// start and end lie under the others' work, but with the registers for two blocks in the works. One row of 4096 x
// 16384: at 5 CTAs 14.4 us, at 4 12.1, at 3 15.6. The up projection at 3 (its longer ring holds a pass; one token
// of the experts 8.4 us, 64 14.2) rather than 4 (8.8, 15.1), the down projection, short strips, at 4 rather than 3
// (64 tokens 14.8 and 15.4, though it leaves 24 to 60 bytes of a thread's registers in memory). Two tiles: dense at
// 3, the experts at 2 (64 tokens of the wide block 30.9 us, at 3, with 56 to 220 bytes in memory, 42.5). Four tiles at
// 2: at 3 32 rows took 21.8 us in place of 12.3.
__host__ __device__ constexpr int ctas_per_sm(int nt, int mode) {
  return nt == 1 ? (mode == GLU ? 3 : 4) : nt == 2 && mode == DENSE ? 3 : 2;
}
__host__ __device__ constexpr int copy_warps(int nt) { return nt == 1 ? 1 : 2; }

// A CTA: wn pairs of strips of one matrix (GLU: a pair is a gate strip and its up strip), wk warps on each that
// share the inputs (of a chunk, kpb blocks of 64 each) and add their sums in shared memory, and warps that
// copy. NT: tiles of 8 rows per pass; more rows of one expert take more passes, which copy the weights
// again. FINE: scale groups of 32 inputs (two per block).
template <typename T, int NT, bool FINE, int MODE>
__global__ void __launch_bounds__((MAX_WARPS + copy_warps(NT)) * 32, ctas_per_sm(NT, MODE)) int4_kernel(const Args p) {
  constexpr int ROWS = NT * 8, PARTS = parts_of(MODE);
  using X = std::conditional_t<MODE == PAIRS, __nv_bfloat16, T>;   // what the rows of x are held in
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full_bar[MAX_DEPTH], empty_bar[MAX_DEPTH];
  __shared__ uint16_t list[MODE == DENSE ? 1 : PAIR_WINDOW];   // places in the window
  __shared__ int n_found;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_warps = p.wk * p.wn;
  constexpr int COPY_WARPS = copy_warps(NT);
  const StageShape sh(p.full_blocks, p.wn * STRIPS, p.full, p.x_rows, PARTS);
  float4* red = reinterpret_cast<float4*>(smem + p.depth * sh.bytes);   // [wk - 1][wn][STRIPS * NT][32 lanes]

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.depth; ++i) {
      mbar_init(full_bar + i, 1 + 32 * COPY_WARPS);   // the weights' bytes, and every copying lane's rows
      mbar_init(empty_bar + i, n_warps);
    }
    n_found = 0;
    fence_mbar_init();
  }
  // The down projection's weights and ids are older than the kernel before it, whose result (the rows of
  // x) it waits for further down: that kernel lets this one start when it has itself waited for all before it.
  if (MODE == GLU) pdl_wait();
  // The ids that this thread looks at first, asked for ahead of all else (LOOKS in flight, a CTA's width apart: as
  // many as cover the pairs of a usual batch, no more, for their code has to be fetched first. Few rows an expert:
  // 2, one token 9.0 us, with 8 9.4; many rows: 5, 200 tokens 53.6, with 2 56.2, with 8 54.5).
  constexpr int LOOKS = NT == 1 ? 2 : 5;
  int64_t seen[LOOKS];
  auto look = [&](int base, int n, int from) {
#pragma unroll
    for (int i = 0; i < LOOKS; ++i) {
      const int at = from + i * int(blockDim.x) + lane;
      seen[i] = at < n ? p.topk_idx[base + at] : -1;
    }
  };
  const bool all_rows = MODE == DENSE || int(blockIdx.y) >= p.routed.groups;
  if (!all_rows) look(0, min(PAIR_WINDOW, p.n_pairs), warp * 32);
  __syncthreads();

  // which matrix, and which of its rows
  const int y = MODE == DENSE ? blockIdx.y : int(blockIdx.y) - p.routed.groups;
  const int e = MODE == DENSE ? 0 : all_rows ? quotient(y, p.row_chunks, p.row_chunks_inv) : int(blockIdx.y);
  const int chunk = all_rows ? y - e * p.row_chunks : 0;
  const int strip_step = MODE == GLU ? p.strips / 2 : 1;
  const int n_stages = p.n_stages;
  // the row of the result, and of x, that row r of this expert is
  int win = 0;
  auto out_row = [&](int r) -> int64_t {
    if (MODE == DENSE) return r;
    return all_rows ? int64_t(p.n_pairs) + int64_t(e) * p.rows + r : win * PAIR_WINDOW + list[r];
  };
  auto x_row = [&](int r) -> int64_t {
    if (MODE == PAIRS) return out_row(r);
    return all_rows ? r : quotient(win * PAIR_WINDOW + list[r], p.top_k, p.top_k_inv);
  };

  // ---- the copying warps' side. A pass is n_stages stages, the weights the same ones in each; the first of
  // them copies the weights too, w_issued and x_issued count stages whose weights and rows have been asked for.
  const int copier = warp - n_warps;   // negative: this warp multiplies
  const uint32_t ring = smem_u32(smem);
  const int first_strip = MODE == GLU ? blockIdx.x * p.wn : blockIdx.x * p.wn * STRIPS;
  // strips in one piece: the CTA's, or (GLU) its gate strips, with the up strips in a piece of their own
  const int live_strips = min(MODE == GLU ? p.wn : p.wn * STRIPS, (MODE == GLU ? strip_step : p.strips) - first_strip);
  const uint8_t* matrix = (MODE != DENSE && all_rows ? p.shared : p.routed).data + e * p.matrix;
  int w_issued = 0, w_stage = 0, w_slot = 0;
  int x_issued = 0, x_stage = 0, x_slot = 0, x_phase = 1;   // (phase: of the slot's release before)
  bool dead = false;
  auto issue_weights = [&] {   // (the slot is free)
    const bool last = w_stage == n_stages - 1;
    const int piece = last ? p.last : p.full;
    if (MODE == PAIRS && p.halves) {   // (a strip's levels and its scales lie apart)
      if (lane < 2 * live_strips) {
        const int at = w_stage >> 1, half = w_stage & 1, blocks = min(CHUNK, p.kblocks - at * CHUNK);
        const int strip = lane >> 1, levels = (last ? p.last_blocks : p.full_blocks) * 512;
        const uint8_t* from = matrix + int64_t(at) * p.strips * p.chunk +
                              int64_t(first_strip + strip) * piece_bytes(blocks, p.group_shift);
        const uint32_t to = ring + w_slot * sh.bytes + strip * piece;
        if (lane & 1)
          bulk_load(to + levels, from + blocks * 512 + half * (CHUNK >> p.group_shift) * 32, piece - levels,
                    full_bar + w_slot);
        else
          bulk_load(to, from + half * (CHUNK / 2 * 512), levels, full_bar + w_slot);
      }
    } else if (lane < (MODE == GLU ? 2 : 1)) {
      const uint8_t* from = matrix + int64_t(w_stage) * p.strips * p.full +
                            int64_t(first_strip + lane * strip_step) * piece;
      bulk_load(ring + w_slot * sh.bytes + lane * p.wn * p.full, from, live_strips * piece, full_bar + w_slot);
    }
    ++w_issued;
    if (++w_stage == n_stages) w_stage = 0;
    if (++w_slot == p.depth) w_slot = 0;
  };
  // `row`: lane r's row r of x; rows 0: the stage's weights alone
  auto issue_stage = [&](const X* row, int rows) {
    if (x_issued >= p.depth) {
      if (!mbar_wait(empty_bar + x_slot, x_phase, p.status)) dead = true;
      dead = __any_sync(0xffffffffu, dead);
      if (dead) return;
    }
    const bool last = x_stage == n_stages - 1;
    if (copier == 0) {
      if (w_issued == x_issued) issue_weights();
      if (lane == 0)
        mbar_expect_tx(full_bar + x_slot, (MODE == GLU ? 2 : 1) * live_strips * (last ? p.last : p.full));
    }
    const int at = x_stage * p.full_blocks * 64;
    const int pieces = min(p.full_blocks * 8, (p.k_dim - at) / 8);
    const uint32_t to = ring + x_slot * sh.bytes + sh.x;
    for (int r = copier; r < rows; r += COPY_WARPS) {
      const X* from = reinterpret_cast<const X*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(row), r)) + at;
#pragma unroll
      for (int part = 0; part < PARTS; ++part, from += p.k_dim)
#pragma unroll
        for (int h = 0; h < CHUNK * 8 / 32; ++h)
          if (lane + 32 * h < pieces)
            cp_async_16(to + r * sh.row + part * (p.full_blocks * 128) + (((lane + 32 * h) ^ ((r & 1) << 2)) << 4),
                        from + (lane + 32 * h) * 8, 16);
    }
    cp_async_arrive(full_bar + x_slot);
    ++x_issued;
    if (++x_stage == n_stages) x_stage = 0;
    if (++x_slot == p.depth) {
      x_slot = 0;
      x_phase ^= 1;
    }
  };

  if (MODE == DENSE) pdl_wait();
  pdl_trigger();
  if (copier == 0 && (p.eager || all_rows))
    for (int i = min(p.depth, n_stages); i > 0; --i) issue_weights();

  const int windows = all_rows ? 1 : (p.n_pairs + PAIR_WINDOW - 1) / PAIR_WINDOW;
  bool waited = MODE != PAIRS;
  int slot = 0, phase = 0;
  for (; win < windows; ++win) {
    int first = chunk * ROWS, n_rows = all_rows ? min(p.rows, first + ROWS) : 0;
    if (!all_rows) {
      // The pairs of this expert among the window's, in whatever order the warps come: rows do not mix, a row's
      // result is the same in any place.
      const int base = win * PAIR_WINDOW, n = min(PAIR_WINDOW, p.n_pairs - base);
      if (win > 0) {
        __syncthreads();     // (the list of the window before has been used)
        if (threadIdx.x == 0) n_found = 0;
        __syncthreads();
      }
      for (int from = warp * 32; from < n; from += LOOKS * int(blockDim.x)) {
        if (win > 0 || from != warp * 32) look(base, n, from);
        uint32_t who[LOOKS];
        int count = 0, at = 0;
#pragma unroll
        for (int i = 0; i < LOOKS; ++i) {
          who[i] = __ballot_sync(0xffffffffu, seen[i] == e);
          count += __popc(who[i]);
        }
        if (count == 0) continue;
        if (lane == 0) at = atomicAdd(&n_found, count);
        at = __shfl_sync(0xffffffffu, at, 0);
#pragma unroll
        for (int i = 0; i < LOOKS; ++i) {
          if ((who[i] >> lane) & 1)
            list[at + __popc(who[i] & ((1u << lane) - 1))] = uint16_t(from + i * int(blockDim.x) + lane);
          at += __popc(who[i]);
        }
      }
      __syncthreads();
      n_rows = n_found;
    }
    if (n_rows <= first) continue;
    if (!waited) {
      pdl_wait();
      waited = true;
    }
    if (copier >= 0) {
      for (int r0 = first; r0 < n_rows && !dead; r0 += ROWS) {
        const int rows = min(ROWS, n_rows - r0);
        const X* row = static_cast<const X*>(p.x) + (lane < rows ? x_row(r0 + lane) * p.ld_x : 0);
        for (int i = 0; i < n_stages && !dead; ++i) issue_stage(row, rows);
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

      uint32_t x_at[NT];   // (rows that a tile lacks are taken from its last one: their sums are not stored)
      uint32_t other[NT];  // from a lane's first piece of a block's row to its second
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int r = min(i * 8 + g, p.x_rows - 1);
        x_at[i] = ring + sh.x + r * sh.row + wk * p.kpb * 128 + (r & 1) * 64 + t * 16 + slot * sh.bytes;
        other[i] = (r & 1) ? uint32_t(-64) : 64u;
      }
      for (int st = 0; st < n_stages; ++st) {
        if (!dead && !mbar_wait(full_bar + slot, phase, p.status)) {
          dead = true;
          atomicExch(p.status, ST_WAIT_TIMEOUT);
          mbar_drain(full_bar, phase * p.depth + slot, p.depth);
        }
        // this warp's blocks of the chunk, and where its strips' pieces are
        const bool last = st == n_stages - 1;
        const int blocks = last ? p.last_blocks : p.full_blocks, piece = last ? p.last : p.full;
        const int lb0 = wk * p.kpb;
        const uint32_t mine = ring + slot * sh.bytes + wn * (MODE == GLU ? 1 : STRIPS) * piece;
        const uint32_t strip = MODE == GLU ? p.wn * p.full : piece;   // from a pair's first to its second
        const uint32_t q_at = mine + lb0 * 512 + lane * 16, s_at = mine + blocks * 512 + g * 4;
        int kb = st * p.full_blocks + lb0;
        // one block of 64 inputs; cut: it is the last, inputs from k_dim on were not copied and count as zero
        auto block = [&](int j, bool cut) {
          uint32_t a[STRIPS][4][4];
          uint32_t sc[STRIPS][FINE ? 2 : 1];
          const uint32_t s_of = s_at + ((2 * (lb0 + j)) >> p.group_shift) * 32;
#pragma unroll
          for (int s = 0; s < STRIPS; ++s) {
            uint32_t q[4];
            ld_shared_v4(q_at + j * 512 + s * strip, q[0], q[1], q[2], q[3]);
#pragma unroll
            for (int h = 0; h < (FINE ? 2 : 1); ++h) sc[s][h] = ld_shared_b32(s_of + s * strip + h * 32);
#pragma unroll
            for (int k = 0; k < 4; ++k) levels_of<X>(q[k], a[s][k]);
          }
          // Tiles whose products, independent of one another, are in the works together. Two where all tiles mostly
          // have rows (64 rows x 4096^2: 13.3 us with one, 12.8 with two); an expert's last tile would often have no
          // partner (200 tokens: 57.9 us with one, 58.7 with two).
          constexpr int AT = MODE == DENSE && NT > 1 ? 2 : 1;
#pragma unroll
          for (int i0 = 0; i0 < NT; i0 += AT) {
            if (i0 > 0 && i0 >= tiles) break;
            uint4 x[2][PARTS][AT];   // a lane's pieces of the block's first and second half
            float c[AT][STRIPS][4] = {};
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
#pragma unroll
              for (int i = 0; i < AT; ++i) {
                const uint32_t at = x_at[i0 + i] + j * 128 + part * (p.full_blocks * 128);
                uint4 &u = x[0][part][i], &v = x[1][part][i];
                ld_shared_v4(at, u.x, u.y, u.z, u.w);
                ld_shared_v4(at + other[i0 + i], v.x, v.y, v.z, v.w);
                if (cut) {
                  const int k = kb * 64 + t * 8;
                  if (k >= p.k_dim) u = make_uint4(0, 0, 0, 0);
                  if (k + 32 >= p.k_dim) v = make_uint4(0, 0, 0, 0);
                }
              }
            auto each = [&](auto f) {
#pragma unroll
              for (int i = 0; i < AT; ++i)
#pragma unroll
                for (int s = 0; s < STRIPS; ++s) f(i, s);
            };
            auto scale_in = [&](int h) {
              each([&](int i, int s) {
                const float2 f = Half16<T>::unpack(sc[s][h]);
                acc[s][i0 + i][0] += f.x * c[i][s][0];
                acc[s][i0 + i][1] += f.x * c[i][s][1];
                acc[s][i0 + i][2] += f.y * c[i][s][2];
                acc[s][i0 + i][3] += f.y * c[i][s][3];
              });
            };
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (FINE && k == 2) scale_in(0);
#pragma unroll
              for (int part = 0; part < PARTS; ++part)
                each([&](int i, int s) {
                  const uint4& v = x[k / 2][part][i];
                  const uint32_t lo = k % 2 ? v.z : v.x, hi = k % 2 ? v.w : v.y;
                  if (part == 0 && (k == 0 || (FINE && k == 2))) Mma<X>::first(c[i][s], a[s][k], lo, hi);
                  else Mma<X>::run(c[i][s], a[s][k], lo, hi);
                });
            }
            scale_in(FINE ? 1 : 0);
          }
        };
        // Two blocks side by side where that pays: in long strips as the one way there is (one row 12.1 us, with the
        // loop 13.0, as a loop of two 12.9), in experts of few rows as a loop of two (64 tokens 15.1 us, one by one
        // 15.4; of many rows 53.7 and 52.9).
        if (MODE == DENSE && p.kpb == 2 && lb0 + 2 <= blocks && (kb + 2) * 64 <= p.k_dim) {
          block(0, false);
          block(1, false);
        } else {
          int j = 0;
          if (MODE != DENSE && NT == 1)
            for (; j + 2 <= p.kpb && lb0 + j + 2 <= blocks && (kb + 2) * 64 <= p.k_dim; j += 2, kb += 2) {
              block(j, false);
              block(j + 1, false);
            }
          for (; j < p.kpb && lb0 + j < blocks; ++j, ++kb) block(j, (kb + 1) * 64 > p.k_dim);
        }
        __syncwarp();
        if (lane == 0 && !dead) mbar_arrive(empty_bar + slot);   // (a stage that was not seen is not filled again)
        int by = sh.bytes;
        if (++slot == p.depth) {
          slot = 0;
          phase ^= 1;
          by -= p.depth * sh.bytes;
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) x_at[i] += by;
      }

      // A tile of 8 rows is finished by one of the warps that share a strip's inputs, warp i % wk: the others leave
      // it their sums in shared memory. A lane adds what the same lane of another warp has, of four warps 0 and 2, 1
      // and 3, then both: whichever of them finishes, the bits are the same. It has outputs g and g + 8 of rows 2 t
      // and 2 t + 1; with the lane of the next g it trades one row's for the other's, so that it stores two outputs
      // side by side.
      float4* sums = red + wn * (STRIPS * NT * 32) + lane;   // of the warp d - 1 places behind the tile's own
      const int sums_step = p.wn * (STRIPS * NT * 32);
      if (p.wk > 1) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const int d = (wk - i) & (p.wk - 1);
          if (i >= tiles || d == 0) continue;
#pragma unroll
          for (int s = 0; s < STRIPS; ++s)
            sums[(d - 1) * sums_step + (s * NT + i) * 32] =
                make_float4(acc[s][i][0], acc[s][i][1], acc[s][i][2], acc[s][i][3]);
        }
        compute_sync(n_warps * 32);
      }
      const int pair = blockIdx.x * p.wn + wn;
      const bool odd = g & 1;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (i >= tiles || (i & (p.wk - 1)) != wk) continue;
        float4 v[STRIPS];
#pragma unroll
        for (int s = 0; s < STRIPS; ++s) v[s] = make_float4(acc[s][i][0], acc[s][i][1], acc[s][i][2], acc[s][i][3]);
        const float4* from = sums + i * 32;
        auto add = [](float4& x, const float4& y) {
          x.x += y.x;
          x.y += y.y;
          x.z += y.z;
          x.w += y.w;
        };
        if (p.wk == 2) {
          float4 u[STRIPS];
#pragma unroll
          for (int s = 0; s < STRIPS; ++s) u[s] = from[s * (NT * 32)];
#pragma unroll
          for (int s = 0; s < STRIPS; ++s) add(v[s], u[s]);
        } else if (p.wk == 4) {
          float4 u[3][STRIPS];
#pragma unroll
          for (int d = 0; d < 3; ++d)
#pragma unroll
            for (int s = 0; s < STRIPS; ++s) u[d][s] = from[d * sums_step + s * (NT * 32)];
#pragma unroll
          for (int s = 0; s < STRIPS; ++s) {
            add(v[s], u[1][s]);
            add(u[0][s], u[2][s]);
            add(v[s], u[0][s]);
          }
        }
        if (MODE == GLU) {
          const float4 f = activation(p.act, v[0]);
          v[0] = make_float4(f.x * v[1].x, f.y * v[1].y, f.z * v[1].z, f.w * v[1].w);
        }
        constexpr int OUTS = MODE == GLU ? 1 : STRIPS;
        float2 o[OUTS][2];
#pragma unroll
        for (int s = 0; s < OUTS; ++s) {
          const float x = __shfl_xor_sync(0xffffffffu, odd ? v[s].x : v[s].y, 4);
          const float y = __shfl_xor_sync(0xffffffffu, odd ? v[s].z : v[s].w, 4);
          o[s][0] = odd ? make_float2(x, v[s].y) : make_float2(v[s].x, x);
          o[s][1] = odd ? make_float2(y, v[s].w) : make_float2(v[s].z, y);
        }
        const int r = i * 8 + 2 * t + odd;
        if (r < live && !dead) {
          const int col = pair * (16 * OUTS) + (g & 6);
          const int64_t to = out_row(r0 + r) * p.ld_out + col;
#pragma unroll
          for (int s = 0; s < OUTS; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int at = s * 16 + h * 8;
              if (col + at >= p.n_dim) continue;
              const float2 f = o[s][h];
              if (MODE == PAIRS) {   // (an even number of columns, in fp32)
                *reinterpret_cast<float2*>(static_cast<float*>(p.out) + to + at) = f;
              } else if (MODE == GLU) {
                __nv_bfloat16* h = static_cast<__nv_bfloat16*>(p.out) + to + at;
                split(f, *reinterpret_cast<uint32_t*>(h), *reinterpret_cast<uint32_t*>(h + p.n_dim));
              } else if (p.n_dim % 2 == 0) {
                *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + to + at) = Half16<T>::pack(f.x, f.y);
              } else {
                static_cast<T*>(p.out)[to + at] = Half16<T>::from_float(f.x);
                if (col + at + 1 < p.n_dim) static_cast<T*>(p.out)[to + at + 1] = Half16<T>::from_float(f.y);
              }
            }
        }
      }
      if (p.wk > 1) compute_sync(n_warps * 32);
    }
  }
  // weights copied for rows that did not come: nobody leaves with a copy in flight
  if (copier == 0) {
    for (int i = x_issued; i < w_issued; ++i) {   // (only ever a pass's first stages, each slot's first use)
      if (lane == 0)
        mbar_expect_tx(full_bar + i, (MODE == GLU ? 2 : 1) * live_strips * (i == n_stages - 1 ? p.last : p.full));
      for (int k = lane; k < 32 * COPY_WARPS; k += 32) mbar_arrive(full_bar + i);
      for (int n = 0; n < 4096 && !mbar_try_wait(full_bar + i, 0); ++n) {
      }
    }
  }
  // (what comes behind this kernel counts on all before it being over: nobody leaves before its own wait)
  if (!waited) pdl_wait();
}

// out[t] = sum_j topk_w[t, j] * y[t * top_k + j] + sum_s y[n_pairs + s * n_tokens + t], fp32, in that order.
// A pair whose expert does not exist has no row: it adds nothing and is reported. AT_ONCE pairs' ids, weights and
// then rows are asked for at once, no more than a token has (code that is fetched for nothing: of six pairs, at
// eight places, 0.2 us); the first ids and weights ahead of the wait (they are older than the kernel before this one,
// which started behind the one that waited for them).
template <typename T, int AT_ONCE>
__global__ void __launch_bounds__(128)
    int4_sum_kernel(const float* y, const T* topk_w, const int64_t* topk_idx, int32_t n_tokens, int32_t top_k,
                    int32_t n_experts, int32_t n_shared, int32_t d, T* out, int32_t* status) {
  pdl_trigger();
  bool waited = false, bad = false;
  const int64_t n_pairs = int64_t(n_tokens) * top_k, n4 = int64_t(n_tokens) * (d / 4);
  for (int64_t i = int64_t(blockIdx.x) * 128 + threadIdx.x; i < n4; i += int64_t(gridDim.x) * 128) {
    const int64_t tok = i / (d / 4);
    const int c = int(i - tok * (d / 4)) * 4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float w, const float4& v) {
      a.x += w * v.x;
      a.y += w * v.y;
      a.z += w * v.z;
      a.w += w * v.w;
    };
    for (int j0 = 0; j0 < top_k; j0 += AT_ONCE) {
      bool there[AT_ONCE];
      float w[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        there[j] = false;
        if (j0 + j < top_k) {
          const int64_t e = ld_prev(topk_idx + tok * top_k + j0 + j);
          w[j] = Half16<T>::to_float(ld_prev(topk_w + tok * top_k + j0 + j));
          there[j] = e >= 0 && e < n_experts;
          bad |= !there[j] && c == 0;
        }
      }
      if (!waited) {
        pdl_wait();
        waited = true;
      }
      float4 v[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j)
        if (there[j]) v[j] = *reinterpret_cast<const float4*>(y + (tok * top_k + j0 + j) * d + c);
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j)
        if (there[j]) add(w[j], v[j]);
    }
#pragma unroll 4
    for (int s = 0; s < n_shared; ++s)
      add(1.f, *reinterpret_cast<const float4*>(y + (n_pairs + int64_t(s) * n_tokens + tok) * d + c));
    *reinterpret_cast<uint2*>(out + tok * d + c) =
        make_uint2(Half16<T>::pack(a.x, a.y), Half16<T>::pack(a.z, a.w));
  }
  if (!waited) pdl_wait();
  if (bad) report_input(status, ST_BAD_EXPERT);   // (nothing is written ahead of the wait)
}

static void set_shape(Args& a, int mode, int32_t k_dim, int32_t n_dim, int32_t n_cols, int32_t group) {
  a.k_dim = k_dim;
  a.n_dim = n_dim;
  a.kblocks = (k_dim + 63) / 64;
  a.strips = (n_cols + 15) / 16;
  a.group_shift = group == 32 ? 0 : group == 64 ? 1 : 2;
  auto stages = [&](int blocks) {
    a.n_stages = (a.kblocks + blocks - 1) / blocks;
    a.full_blocks = std::min(blocks, a.kblocks);
    a.last_blocks = a.kblocks - (a.n_stages - 1) * blocks;
    a.full = piece_bytes(a.full_blocks, a.group_shift);
    a.last = piece_bytes(a.last_blocks, a.group_shift);
  };
  stages(CHUNK);
  a.chunk = a.full;
  a.matrix = int64_t(a.strips) * (int64_t(a.n_stages - 1) * a.full + a.last);
  // Rows in two parts fill a stage of whole chunks: of 32 rows one such stage fits, which is then copied and
  // multiplied in turns (200 tokens of the wide block 70.2 us; with halves, two of which are in the ring, 57.6).
  a.halves = mode == PAIRS && a.kblocks > CHUNK / 2;
  if (a.halves) stages(CHUNK / 2);
}
// How a CTA's warps divide the work: on a strip's inputs where it has that many blocks; on more strips, which
// share the rows of x, where the grid is more than the SMs hold at a time. False: no stage fits `memory`.
static bool set_warps(Args& a, int nt, int mode, int64_t matrices, int slots, int memory) {
  const int pairs = mode == GLU ? a.strips / 2 : (a.strips + 1) / 2;
  for (int wk = 4; wk > 0; wk /= 2) {
    if (wk > a.kblocks && wk > 1) continue;
    Args b = a;
    b.wk = wk;
    b.kpb = (a.full_blocks + wk - 1) / wk;
    b.wn = MAX_WARPS / wk;
    while (b.wn / 2 >= pairs) b.wn /= 2;
    const int64_t ctas = (pairs + b.wn - 1) / b.wn * matrices;
    const int red = (wk - 1) * b.wn * STRIPS * nt * 32 * int(sizeof(float4));
    const int fit = (memory - red) / StageShape(a.full_blocks, b.wn * STRIPS, a.full, a.x_rows, parts_of(mode)).bytes;
    b.depth = std::min(std::min(fit, a.n_stages), MAX_DEPTH);
    if (b.depth < std::min(2, a.n_stages) && a.wk > 0) break;   // (the ring of the last try is longer)
    if (b.depth < 1) return false;
    // A warp alone on its strips pays where the rows come in one pass (200 tokens of the wide block 57.6 us, with two
    // warps 60.1); in several passes only where the SMs stay full (256 tokens, two of eight experts of 1536 x 1024:
    // 79.7 us on 192 CTAs, 66.7 on 384).
    if (wk == 1 && a.wk > 0 && mode == PAIRS && a.n_pairs > a.routed.groups * nt * 8 && ctas < slots) break;
    a = b;
    if (ctas <= slots) break;
  }
  return true;
}
static unsigned ctas_for(const Args& a, bool glu) {
  const int pairs = glu ? a.strips / 2 : (a.strips + 1) / 2;
  return unsigned((pairs + a.wn - 1) / a.wn);
}

template <typename T, int NT, bool FINE, int MODE>
static int launch(Args a, cudaStream_t st) {
  auto kern = int4_kernel<T, NT, FINE, MODE>;
  // shared memory of a CTA: an equal share for as many as the registers allow
  constexpr int share =
      227 * 1024 / ctas_per_sm(NT, MODE) / 1024 * 1024 - 1024 - (MODE == DENSE ? 0 : 2 * PAIR_WINDOW) - 256;
  a.x_rows = MODE == DENSE ? std::min(a.rows, NT * 8) : NT * 8;
  a.row_chunks = std::max(1, (a.rows + NT * 8 - 1) / (NT * 8));
  a.row_chunks_inv = quotient_inverse(a.row_chunks);
  const int64_t ys = MODE == DENSE ? a.row_chunks : a.routed.groups + int64_t(a.shared.groups) * a.row_chunks;
  if (ys > 65535) return MOE_B200_ERR_UNSUPPORTED;
  if (!set_warps(a, NT, MODE, ys, 148 * ctas_per_sm(NT, MODE), share)) return MOE_B200_ERR_UNSUPPORTED;
  const int smem = a.depth * StageShape(a.full_blocks, a.wn * STRIPS, a.full, a.x_rows, parts_of(MODE)).bytes +
                   (a.wk - 1) * a.wn * STRIPS * NT * 32 * int(sizeof(float4));
  static PerDevice<cudaError_t> ready;
  int dev = -1;
  const cudaError_t* ok = cudaGetDevice(&dev) != cudaSuccess ? nullptr : ready.get(dev, [&](int) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, share);
  });
  if (ok == nullptr || *ok != cudaSuccess || smem > share) return MOE_B200_ERR_CUDA;
  return launch_pdl(kern, dim3(ctas_for(a, MODE == GLU), unsigned(ys)),
                    dim3((a.wk * a.wn + copy_warps(NT)) * 32), size_t(smem), st, a) == cudaSuccess
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
  set_shape(a, GLU, d, h, 2 * h, group);
  a.rows = int32_t(n_tokens);
  a.topk_idx = topk_idx;
  a.n_pairs = n_pairs;
  a.top_k = top_k;
  a.top_k_inv = quotient_inverse(top_k);
  a.eager = n_pairs >= in.groups;   // (then most experts have rows)
  a.act = act;
  a.out = scratch;
  a.ld_out = 2 * int64_t(h);
  a.status = status;
  int rc = launch_for<T, GLU>(a, rows, st);
  if (rc != MOE_B200_OK) return rc;
  a.x = scratch;
  a.ld_x = 2 * int64_t(h);
  a.routed = down;
  a.shared = down_sh;
  set_shape(a, PAIRS, h, d, d, group);
  a.out = y;
  a.ld_out = d;
  rc = launch_for<T, PAIRS>(a, rows, st);
  if (rc != MOE_B200_OK) return rc;
  const int64_t blocks = std::min<int64_t>((n_tokens * (d / 4) + 127) / 128, 148 * 16);
  auto sum = top_k <= 2 ? int4_sum_kernel<T, 2> : top_k <= 4 ? int4_sum_kernel<T, 4>
             : top_k <= 6 ? int4_sum_kernel<T, 6> : int4_sum_kernel<T, 8>;
  return launch_pdl(sum, dim3(unsigned(blocks)), dim3(128), 0, st, static_cast<const float*>(y),
                    static_cast<const T*>(topk_w), topk_idx, int32_t(n_tokens), top_k, in.groups, in_sh.groups, d,
                    static_cast<T*>(out), status) == cudaSuccess
             ? MOE_B200_OK
             : MOE_B200_ERR_CUDA;
}

}  // namespace q4
}  // namespace moe

using namespace moe;

extern "C" {

size_t moe_b200_int4_bytes(int32_t k_dim, int32_t n_dim, int32_t group) {
  if (k_dim < 8 || k_dim % 8 || k_dim > q4::MAX_WIDTH || n_dim < 1 || n_dim > q4::MAX_WIDTH || !q4::group_ok(group))
    return 0;
  q4::Args a{};
  q4::set_shape(a, q4::DENSE, k_dim, n_dim, n_dim, group);
  return size_t(a.matrix);
}

int moe_b200_int4_mm(const void* x, int64_t rows, int64_t ld_x, int32_t k_dim, const void* w, int32_t group,
                     int32_t n_dim, int32_t dtype, void* y, int32_t* status, void* stream) {
  if (rows < 0 || rows > 0x7fffffff || k_dim < 8 || k_dim % 8 || k_dim > q4::MAX_WIDTH || n_dim < 1 ||
      n_dim > q4::MAX_WIDTH || ld_x < k_dim || ld_x % 8 ||
      !q4::group_ok(group))
    return MOE_B200_ERR_SHAPE;
  if (dtype != MOE_B200_BF16 && dtype != MOE_B200_FP16) return MOE_B200_ERR_UNSUPPORTED;
  if (rows > 65535 * 32) return MOE_B200_ERR_UNSUPPORTED;   // (a grid of 32 rows each)
  if (rows == 0) return MOE_B200_OK;
  if (!x || !w || !y || !status) return MOE_B200_ERR_NULL;
  if (!q4::aligned(x, 16) || !q4::aligned(w, 16) || !q4::aligned(y, n_dim % 2 ? 2 : 4)) return MOE_B200_ERR_ALIGN;
  q4::Args a{};
  a.x = x;
  a.ld_x = ld_x;
  a.routed = {static_cast<const uint8_t*>(w), 1};
  q4::set_shape(a, q4::DENSE, k_dim, n_dim, n_dim, group);
  a.rows = int32_t(rows);
  a.out = y;
  a.ld_out = n_dim;
  a.status = status;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MOE_B200_BF16 ? q4::launch_for<__nv_bfloat16, q4::DENSE>(a, rows, st)
                                : q4::launch_for<__half, q4::DENSE>(a, rows, st);
}

static size_t int4_hidden_bytes(int64_t n_tokens, int32_t top_k, int32_t n_shared, int32_t d_hidden) {
  return (size_t(n_tokens) * (size_t(top_k) + size_t(n_shared)) * size_t(d_hidden) * 4 + 255) / 256 * 256;
}

size_t moe_b200_int4_experts_scratch_bytes(int64_t n_tokens, int32_t top_k, int32_t n_shared, int32_t d_model,
                                           int32_t d_hidden) {
  if (n_tokens < 0 || top_k < 0 || n_shared < 0 || d_model < 1 || d_hidden < 1) return 0;
  return int4_hidden_bytes(n_tokens, top_k, n_shared, d_hidden) +
         size_t(n_tokens) * (size_t(top_k) + size_t(n_shared)) * size_t(d_model) * sizeof(float);
}

int moe_b200_int4_experts(const void* x, int64_t n_tokens, int64_t ld_x, int32_t d_model, int32_t d_hidden,
                          const void* topk_w, const int64_t* topk_idx, int32_t top_k, int32_t n_experts,
                          const void* w_in, const void* w_out, int32_t n_shared, const void* w_sh_in,
                          const void* w_sh_out, int32_t group, int32_t activation, int32_t dtype, void* out,
                          void* scratch, size_t scratch_bytes, int32_t* status, void* stream) {
  if (n_tokens < 0 || top_k < 1 || n_experts < 1 || n_shared < 0 || n_experts + int64_t(n_shared) > 65535 ||
      d_model < 8 || d_model % 8 || d_model > q4::MAX_WIDTH || d_hidden < 16 || d_hidden % 16 ||
      d_hidden > q4::MAX_WIDTH / 2 || ld_x < d_model || ld_x % 8 ||
      !q4::group_ok(group) || n_tokens > 0x7fffffff ||
      n_tokens * (int64_t(top_k) + n_shared) > 0x7fffffff - q4::PAIR_WINDOW)
    return MOE_B200_ERR_SHAPE;
  if (dtype != MOE_B200_BF16 && dtype != MOE_B200_FP16) return MOE_B200_ERR_UNSUPPORTED;
  if (activation < MOE_B200_ACT_SILU || activation > MOE_B200_ACT_TANH) return MOE_B200_ERR_UNSUPPORTED;
  if (n_tokens == 0) return MOE_B200_OK;
  if (!x || !topk_w || !topk_idx || !w_in || !w_out || !out || !status || (n_shared > 0 && (!w_sh_in || !w_sh_out)))
    return MOE_B200_ERR_NULL;
  if (!q4::aligned(x, 16) || !q4::aligned(topk_w, 2) || !q4::aligned(topk_idx, 8) || !q4::aligned(w_in, 16) ||
      !q4::aligned(w_out, 16) || !q4::aligned(w_sh_in, 16) || !q4::aligned(w_sh_out, 16) || !q4::aligned(out, 16) ||
      !q4::aligned(scratch, 16))
    return MOE_B200_ERR_ALIGN;
  const size_t need = moe_b200_int4_experts_scratch_bytes(n_tokens, top_k, n_shared, d_model, d_hidden);
  if (!scratch || scratch_bytes < need) return MOE_B200_ERR_SCRATCH;
  const size_t hid = int4_hidden_bytes(n_tokens, top_k, n_shared, d_hidden);
  auto stack = [](const void* w, int32_t n) { return q4::Stack{static_cast<const uint8_t*>(w), n}; };
  const q4::Stack in = stack(w_in, n_experts), down = stack(w_out, n_experts);
  const q4::Stack in_sh = stack(w_sh_in, n_shared), down_sh = stack(w_sh_out, n_shared);
  uint8_t* s = static_cast<uint8_t*>(scratch);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MOE_B200_BF16
             ? q4::experts<__nv_bfloat16>(x, ld_x, n_tokens, d_model, d_hidden, topk_w, topk_idx, top_k, in,
                                            in_sh, down, down_sh, group, activation, out, s, hid, status, st)
             : q4::experts<__half>(x, ld_x, n_tokens, d_model, d_hidden, topk_w, topk_idx, top_k, in, in_sh,
                                     down, down_sh, group, activation, out, s, hid, status, st);
}

}  // extern "C"
