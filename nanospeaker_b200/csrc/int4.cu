// Products of few rows with weights held in 4 bits: W[k, n] = (level[k, n] - 8) * scale[k / group, n].
//
//   moe_b200_int4_mm       y = x @ W
//   moe_b200_int4_experts  the block's GLU experts (routed by top-k ids, and shared ones) for a batch that
//                          generates: up + GLU -> down -> weighted sum, three launches
//
// What bounds them is the weights' bytes, so a weight is read once, 16 bytes per lane, and used for up to 64
// rows from registers. The layout (nanospeaker_b200/int4.py packs it) is the matrix instruction's: a lane's 16 bytes are its A
// fragments (16 outputs x 16 inputs each) of 64 inputs, and the inputs are numbered within those 64 so that
// the B fragments of a row of x are two 16-byte pieces of it. Levels become 16-bit floats exactly (a byte
// operation and a subtraction per two), products are summed in fp32 over one scale group at a time, and the
// scale is applied to that sum: no rounding but the final one (and the GLU's result, which is held in the
// activations' type between the two products).
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/moe_b200.h"
#include "act.cuh"
#include "half16.cuh"
#include "pdl.cuh"
#include "per_device.cuh"

namespace moe {
namespace q4 {

constexpr int MAX_WARPS = 8;
constexpr int STRIPS = 2;        // strips of 16 outputs a CTA computes
constexpr int AHEAD = 4;         // weight blocks in flight per warp and strip
constexpr int PAIR_WINDOW = 2048;   // pairs whose expert ids are looked at in one go

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
  int32_t kblocks, kgroups, strips, group;   // of both stacks
  int32_t rows;                // DENSE: rows of x; else tokens
  // GLU / PAIRS: row p of the result is pair p of topk_idx, row n_pairs + s * rows + t token t of shared expert s
  const int64_t* topk_idx;
  int32_t n_pairs, top_k;
  int32_t act;
  void* out;                   // DENSE [rows, n_dim], GLU [n_pairs + S * rows, n_dim] of T; PAIRS fp32
  int64_t ld_out;
};

template <typename T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
  static constexpr uint32_t MAGIC = 0x43004300u, BIAS = 0x43084308u;   // 128 + level, 128 + 8
  static __device__ __forceinline__ uint32_t sub(uint32_t a) {
    const uint32_t bias = BIAS;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                     *reinterpret_cast<const __nv_bfloat162*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void run(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Mma<__half> {
  static constexpr uint32_t MAGIC = 0x64006400u, BIAS = 0x64086408u;   // 1024 + level, 1024 + 8
  static __device__ __forceinline__ uint32_t sub(uint32_t a) {
    const uint32_t bias = BIAS;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a),
                              *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void run(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// A packed word's eight levels as the four registers of an A fragment, values -8 .. 7.
template <typename T>
__device__ __forceinline__ void levels_of(uint32_t word, uint32_t* a) {
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = Mma<T>::sub(((word >> (4 * i)) & 0x000F000Fu) | Mma<T>::MAGIC);
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

// A CTA: two strips of one matrix (GLU: a gate strip and its up strip), its warps share the inputs (warp w takes
// the blocks w, w + warps, ... of 64) and add their sums in shared memory. NT: tiles of 8 rows per pass; more
// rows take more passes, which read the weights again. FINE: scale groups of 32 inputs (two per block).
template <typename T, int NT, bool FINE, int MODE>
__global__ void __launch_bounds__(MAX_WARPS * 32) int4_kernel(const Args p) {
  constexpr int ROWS = NT * 8;
  extern __shared__ float red[];        // [warps][STRIPS * 16][ROWS]
  __shared__ int list[MODE == DENSE ? 1 : PAIR_WINDOW];
  __shared__ int warp_count[MAX_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int warps = blockDim.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  pdl_trigger();
  pdl_wait();

  const int e = blockIdx.y;
  const bool shared = MODE != DENSE && e >= p.routed.groups;
  const Stack w = shared ? p.shared : p.routed;
  const int we = shared ? e - p.routed.groups : e;
  const int strip0 = MODE == GLU ? blockIdx.x : blockIdx.x * STRIPS;
  const int strip_step = MODE == GLU ? p.strips / 2 : 1;
  const bool two = strip0 + strip_step < p.strips;
  const uint4* levels[STRIPS];
  const uint32_t* scales[STRIPS];
#pragma unroll
  for (int s = 0; s < STRIPS; ++s) {
    const int64_t at = int64_t(we) * p.strips + strip0 + (s == 0 || two ? s * strip_step : 0);
    levels[s] = w.levels + at * p.kblocks * 32 + lane;
    scales[s] = w.scales + at * p.kgroups * 8 + g;
  }
  const T* x = static_cast<const T*>(p.x);

  const int windows = MODE == DENSE || shared ? 1 : (p.n_pairs + PAIR_WINDOW - 1) / PAIR_WINDOW;
  for (int win = 0; win < windows; ++win) {
    int n_rows = p.rows;
    if (MODE != DENSE && !shared) {
      // the pairs of this expert among the window's, in order: every warp looks at a share of them
      const int base = win * PAIR_WINDOW, n = min(PAIR_WINDOW, p.n_pairs - base);
      const int share = ((n + warps - 1) / warps + 31) / 32 * 32;
      const int lo = warp * share, hi = min(n, lo + share);
      int count = 0;
      for (int i = lo; i < hi; i += 32)
        count += __popc(__ballot_sync(0xffffffffu, i + lane < hi && p.topk_idx[base + i + lane] == e));
      __syncthreads();                  // (the list of the window before has been used)
      if (lane == 0) warp_count[warp] = count;
      __syncthreads();
      int at = 0;
      n_rows = 0;
      for (int i = 0; i < warps; ++i) {
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

    for (int r0 = 0; r0 < n_rows; r0 += ROWS) {
      const int tiles = min(NT, (n_rows - r0 + 7) / 8);
      // where a row of x is, and the row of the result
      auto out_row = [&](int r) -> int64_t {
        if (MODE == DENSE) return r;
        return shared ? int64_t(p.n_pairs) + int64_t(we) * p.rows + r : list[r];
      };
      const T* xr[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int r = r0 + 8 * i + g;
        xr[i] = nullptr;
        if (r < n_rows) {
          const int64_t at = MODE == DENSE ? r : MODE == PAIRS ? out_row(r) : shared ? r : list[r] / p.top_k;
          xr[i] = x + at * p.ld_x;
        }
      }
      float acc[STRIPS][NT][4];
#pragma unroll
      for (int s = 0; s < STRIPS; ++s)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[s][i][k] = 0.f;

      auto scale_at = [&](int s, int kb, int half) {
        return scales[s][int64_t((kb * 64 + half * 32) / p.group) * 8];
      };
      uint4 next[AHEAD][STRIPS];
      uint32_t next_scale[AHEAD][STRIPS][FINE ? 2 : 1];
      auto fetch = [&](int slot, int kb) {
        if (kb < p.kblocks) {
#pragma unroll
          for (int s = 0; s < STRIPS; ++s) {
            next[slot][s] = levels[s][int64_t(kb) * 32];
            next_scale[slot][s][0] = scale_at(s, kb, 0);
            if constexpr (FINE) next_scale[slot][s][1] = scale_at(s, kb, 1);
          }
        }
      };
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) fetch(i, warp + i * warps);
      for (int kb0 = warp; kb0 < p.kblocks; kb0 += AHEAD * warps) {
#pragma unroll
        for (int slot = 0; slot < AHEAD; ++slot) {
          const int kb = kb0 + slot * warps;
          if (kb >= p.kblocks) break;
          uint4 q[STRIPS];
          uint32_t sc[STRIPS][FINE ? 2 : 1];
#pragma unroll
          for (int s = 0; s < STRIPS; ++s) {
            q[s] = next[slot][s];
            sc[s][0] = next_scale[slot][s][0];
            if constexpr (FINE) sc[s][1] = next_scale[slot][s][1];
          }
          fetch(slot, kb + AHEAD * warps);
          uint32_t a[STRIPS][4][4];
#pragma unroll
          for (int s = 0; s < STRIPS; ++s) {
            levels_of<T>(q[s].x, a[s][0]);
            levels_of<T>(q[s].y, a[s][1]);
            levels_of<T>(q[s].z, a[s][2]);
            levels_of<T>(q[s].w, a[s][3]);
          }
          const int k = kb * 64 + 8 * t;
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            if (i >= tiles) break;
            uint4 b0 = make_uint4(0, 0, 0, 0), b1 = b0;
            if (xr[i] != nullptr) {
              if (k < p.k_dim) b0 = *reinterpret_cast<const uint4*>(xr[i] + k);
              if (k + 32 < p.k_dim) b1 = *reinterpret_cast<const uint4*>(xr[i] + k + 32);
            }
#pragma unroll
            for (int s = 0; s < STRIPS; ++s) {
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              float2 f = Half16<T>::unpack(sc[s][0]);
              Mma<T>::run(c, a[s][0], b0.x, b0.y);
              Mma<T>::run(c, a[s][1], b0.z, b0.w);
              if constexpr (FINE) {
                acc[s][i][0] += f.x * c[0];
                acc[s][i][1] += f.x * c[1];
                acc[s][i][2] += f.y * c[2];
                acc[s][i][3] += f.y * c[3];
                c[0] = c[1] = c[2] = c[3] = 0.f;
                f = Half16<T>::unpack(sc[s][FINE ? 1 : 0]);
              }
              Mma<T>::run(c, a[s][2], b1.x, b1.y);
              Mma<T>::run(c, a[s][3], b1.z, b1.w);
              acc[s][i][0] += f.x * c[0];
              acc[s][i][1] += f.x * c[1];
              acc[s][i][2] += f.y * c[2];
              acc[s][i][3] += f.y * c[3];
            }
          }
        }
      }
      // the warps' sums meet in shared memory: [warp][output][row]
#pragma unroll
      for (int s = 0; s < STRIPS; ++s)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float* to = red + ((warp * STRIPS + s) * 16 + g) * ROWS + i * 8 + 2 * t;
          *reinterpret_cast<float2*>(to) = make_float2(acc[s][i][0], acc[s][i][1]);
          *reinterpret_cast<float2*>(to + 8 * ROWS) = make_float2(acc[s][i][2], acc[s][i][3]);
        }
      __syncthreads();
      const int live = min(ROWS, n_rows - r0);
      auto sum = [&](int o, int r) {
        float v = 0.f;
        for (int i = 0; i < warps; ++i) v += red[(i * STRIPS * 16 + o) * ROWS + r];
        return v;
      };
      if (MODE == GLU) {
        for (int i = threadIdx.x; i < 16 * live; i += blockDim.x) {
          const int o = i & 15, r = i >> 4;
          const float h = activation(p.act, sum(o, r)) * sum(16 + o, r);
          static_cast<T*>(p.out)[out_row(r0 + r) * p.ld_out + strip0 * 16 + o] = Half16<T>::from_float(h);
        }
      } else {
        for (int i = threadIdx.x; i < STRIPS * 16 * live; i += blockDim.x) {
          const int o = i % (STRIPS * 16), r = i / (STRIPS * 16);
          const int n = strip0 * 16 + o;
          if (n < p.n_dim) {
            const int64_t at = out_row(r0 + r) * p.ld_out + n;
            if (MODE == DENSE) static_cast<T*>(p.out)[at] = Half16<T>::from_float(sum(o, r));
            else static_cast<float*>(p.out)[at] = sum(o, r);
          }
        }
      }
      __syncthreads();
    }
  }
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

// Warps that share kblocks blocks so that none has more than another by more than the last round.
static int warps_for(int kblocks) {
  const int rounds = (kblocks + MAX_WARPS - 1) / MAX_WARPS;
  return (kblocks + rounds - 1) / rounds;
}

template <typename T, int NT, bool FINE, int MODE>
static int launch(const Args& a, unsigned ctas, unsigned experts, cudaStream_t st) {
  auto kern = int4_kernel<T, NT, FINE, MODE>;
  const int warps = warps_for(a.kblocks);
  constexpr size_t per_warp = size_t(STRIPS) * 16 * NT * 8 * sizeof(float);
  const size_t smem = size_t(warps) * per_warp;
  if constexpr (MAX_WARPS * per_warp > 32 * 1024) {   // (the default limit, 48 KB, counts the list too)
    static PerDevice<cudaError_t> ready;
    int dev = -1;
    const cudaError_t* ok = cudaGetDevice(&dev) != cudaSuccess ? nullptr : ready.get(dev, [&](int) {
      return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  int(MAX_WARPS * per_warp));
    });
    if (ok == nullptr || *ok != cudaSuccess) return MOE_B200_ERR_CUDA;
  }
  return launch_pdl(kern, dim3(ctas, experts), dim3(warps * 32), smem, st, a) == cudaSuccess
             ? MOE_B200_OK
             : MOE_B200_ERR_CUDA;
}
template <typename T, int MODE>
static int launch_for(const Args& a, int64_t rows, unsigned ctas, unsigned experts, cudaStream_t st) {
  const bool fine = a.group == 32;
#define LAUNCH(N) (fine ? launch<T, N, true, MODE>(a, ctas, experts, st) : launch<T, N, false, MODE>(a, ctas, experts, st))
  if (rows <= 8) return LAUNCH(1);
  if (rows <= 16) return LAUNCH(2);
  if (rows <= 32) return LAUNCH(4);
  return LAUNCH(8);
#undef LAUNCH
}

static void set_shape(Args& a, int32_t k_dim, int32_t n_dim, int32_t n_cols, int32_t group) {
  a.k_dim = k_dim;
  a.n_dim = n_dim;
  a.kblocks = (k_dim + 63) / 64;
  a.kgroups = (a.kblocks * 64 + group - 1) / group;
  a.strips = (n_cols + 15) / 16;
  a.group = group;
}
static bool group_ok(int32_t g) { return g == 32 || (g >= 64 && g % 64 == 0); }
static bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename T>
static int experts(const void* x, int64_t ld_x, int64_t n_tokens, int32_t d, int32_t h, const void* topk_w,
                   const int64_t* topk_idx, int32_t top_k, const Stack& in, const Stack& in_sh,
                   const Stack& down, const Stack& down_sh, int32_t group, int32_t act, void* out,
                   uint8_t* scratch, size_t hid_bytes, int32_t* status, cudaStream_t st) {
  const int32_t n_pairs = int32_t(n_tokens * top_k);
  const unsigned ne = unsigned(in.groups + in_sh.groups);
  float* y = reinterpret_cast<float*>(scratch + hid_bytes);
  // rows an expert has, with room for an uneven load
  const int64_t mean = in.groups ? (int64_t(n_pairs) + in.groups - 1) / in.groups : 0;
  const int64_t rows = std::max<int64_t>(mean > 4 ? 2 * mean : mean, in_sh.groups ? std::min<int64_t>(n_tokens, 64) : 1);
  Args a{};
  a.x = x;
  a.ld_x = ld_x;
  a.routed = in;
  a.shared = in_sh;
  set_shape(a, d, h, 2 * h, group);
  a.rows = int32_t(n_tokens);
  a.topk_idx = topk_idx;
  a.n_pairs = n_pairs;
  a.top_k = top_k;
  a.act = act;
  a.out = scratch;
  a.ld_out = h;
  int rc = launch_for<T, GLU>(a, rows, unsigned(h / 16), ne, st);
  if (rc != MOE_B200_OK) return rc;
  a.x = scratch;
  a.ld_x = h;
  a.routed = down;
  a.shared = down_sh;
  set_shape(a, h, d, d, group);
  a.out = y;
  a.ld_out = d;
  rc = launch_for<T, PAIRS>(a, rows, unsigned((a.strips + STRIPS - 1) / STRIPS), ne, st);
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
                     const void* scales, int32_t group, int32_t n_dim, int32_t dtype, void* y, void* stream) {
  if (rows < 0 || rows > 0x7fffffff || k_dim < 8 || k_dim % 8 || n_dim < 1 || ld_x < k_dim || ld_x % 8 ||
      !q4::group_ok(group))
    return MOE_B200_ERR_SHAPE;
  if (dtype != MOE_B200_BF16 && dtype != MOE_B200_FP16) return MOE_B200_ERR_UNSUPPORTED;
  if (rows == 0) return MOE_B200_OK;
  if (!x || !levels || !scales || !y) return MOE_B200_ERR_NULL;
  if (!q4::aligned(x, 16) || !q4::aligned(levels, 16) || !q4::aligned(scales, 4) || !q4::aligned(y, 2))
    return MOE_B200_ERR_ALIGN;
  q4::Args a{};
  a.x = x;
  a.ld_x = ld_x;
  a.routed = {static_cast<const uint4*>(levels), static_cast<const uint32_t*>(scales), 1};
  q4::set_shape(a, k_dim, n_dim, n_dim, group);
  a.rows = int32_t(rows);
  a.out = y;
  a.ld_out = n_dim;
  const unsigned ctas = unsigned((a.strips + q4::STRIPS - 1) / q4::STRIPS);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MOE_B200_BF16 ? q4::launch_for<__nv_bfloat16, q4::DENSE>(a, rows, ctas, 1, st)
                                : q4::launch_for<__half, q4::DENSE>(a, rows, ctas, 1, st);
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
      !q4::aligned(sh_out_levels, 16) || !q4::aligned(in_scales, 4) || !q4::aligned(out_scales, 4) ||
      !q4::aligned(sh_in_scales, 4) || !q4::aligned(sh_out_scales, 4) || !q4::aligned(out, 16) ||
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
