// Dropout whose mask is a function of the element's index and of a state (seed, call) in device memory, so
// that it is made where it is used, forward and backward, and never stored:
//
//   out[i] = residual[i] + (word(i) >= threshold ? x[i] * scale : 0),   scale = 1 / (1 - p)
//
// word(i) is word i % 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", 2011) at counter (i / 4, call) under the key seed. Indexes count elements of the whole tensor in
// row-major order, whatever its row length. The backward is the same kernel on the gradient, without a
// residual.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/moe_b200.h"
#include "half16.cuh"
#include "pdl.cuh"
#include "philox.cuh"

namespace moe {

constexpr int DROP_THREADS = 256;

// 16 bytes of type T as floats and back.
template <typename T>
struct Piece {
  static constexpr int N = 8;
  static __device__ __forceinline__ void to_float(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = Half16<T>::unpack(w[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ uint4 from_float(const float* f) {
    return make_uint4(Half16<T>::pack(f[0], f[1]), Half16<T>::pack(f[2], f[3]), Half16<T>::pack(f[4], f[5]),
                      Half16<T>::pack(f[6], f[7]));
  }
};
template <>
struct Piece<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void to_float(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 from_float(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <typename T>
__device__ __forceinline__ float one_to_float(T v) { return Half16<T>::to_float(v); }
template <>
__device__ __forceinline__ float one_to_float<float>(float v) { return v; }
template <typename T>
__device__ __forceinline__ T one_from_float(float v) { return Half16<T>::from_float(v); }
template <>
__device__ __forceinline__ float one_from_float<float>(float v) { return v; }

// `pieces` 16-byte pieces (0 where a pointer is not aligned); the rest goes one by one. A thread has 16
// elements at a time, in pieces a block's width apart: four counters. A dropped element adds nothing, whatever
// its value (a product would make NaN of an infinity). SMALL: no counter passes 32 bits; its upper word and
// the call's are then the same for all threads, and the products of theirs in the first rounds are made once.
template <typename T, bool RES, bool SMALL>
__global__ void __launch_bounds__(DROP_THREADS)
    dropout_kernel(const T* x, const T* residual, const int64_t* rng, int64_t* used, T* out, int64_t n,
                   int64_t pieces, uint32_t threshold, float scale) {
  constexpr int N = Piece<T>::N, PIECES = 16 / N, QUADS = N / 4;
  pdl_trigger();
  pdl_wait();
  const int64_t seed = ld_prev(rng), call = ld_prev(rng + 1);
  if (used != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
    used[0] = seed;
    used[1] = call;
  }
  auto counter = [](int64_t quad) { return SMALL ? uint64_t(uint32_t(quad)) : uint64_t(quad); };
  const int64_t block = int64_t(DROP_THREADS) * PIECES;
  for (int64_t at = blockIdx.x * block + threadIdx.x; at < pieces; at += gridDim.x * block) {
    uint4 a[PIECES], r[PIECES];
    uint64_t low[4];
#pragma unroll
    for (int h = 0; h < PIECES; ++h) {
      const int64_t i = at + h * DROP_THREADS;
      if (i < pieces) {
        a[h] = reinterpret_cast<const uint4*>(x)[i];
        if constexpr (RES) r[h] = reinterpret_cast<const uint4*>(residual)[i];
      }
#pragma unroll
      for (int q = 0; q < QUADS; ++q) low[h * QUADS + q] = counter(i * QUADS + q);
    }
    uint32_t word[4][4];
    philox4x32<4>(low, uint64_t(call), uint64_t(seed), word);
#pragma unroll
    for (int h = 0; h < PIECES; ++h) {
      const int64_t i = at + h * DROP_THREADS;
      if (i >= pieces) break;
      float f[N], o[N];
      Piece<T>::to_float(a[h], f);
      if constexpr (RES) Piece<T>::to_float(r[h], o);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const bool keep = word[h * QUADS + k / 4][k % 4] >= threshold;
        if constexpr (RES) o[k] = keep ? fmaf(f[k], scale, o[k]) : o[k];
        else o[k] = keep ? f[k] * scale : 0.f;
      }
      reinterpret_cast<uint4*>(out)[i] = Piece<T>::from_float(o);
    }
  }
  const int64_t first = int64_t(blockIdx.x) * DROP_THREADS + threadIdx.x;
  for (int64_t i = pieces * N + first; i < n; i += int64_t(gridDim.x) * DROP_THREADS) {
    uint32_t word[1][4];
    const uint64_t low = counter(i >> 2);
    philox4x32<1>(&low, uint64_t(call), uint64_t(seed), word);
    const uint32_t mine = (i & 2) ? ((i & 1) ? word[0][3] : word[0][2]) : ((i & 1) ? word[0][1] : word[0][0]);
    float o = 0.f;
    if constexpr (RES) o = one_to_float<T>(residual[i]);
    if (mine >= threshold) o = fmaf(one_to_float<T>(x[i]), scale, o);
    out[i] = one_from_float<T>(o);
  }
}

template <typename T>
static int launch_dropout(const void* x, const void* residual, const int64_t* rng, int64_t* used, void* out,
                          int64_t n, uint32_t threshold, float scale, cudaStream_t st) {
  const uintptr_t any = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
                        reinterpret_cast<uintptr_t>(out);
  if (any % sizeof(T)) return MOE_B200_ERR_ALIGN;
  constexpr int N = Piece<T>::N;
  const int64_t pieces = any % 16 ? 0 : n / N;
  const int64_t work = std::max((pieces * N + 15) / 16, n - pieces * N);
  const int64_t blocks = std::min<int64_t>((work + DROP_THREADS - 1) / DROP_THREADS, 148 * 8);
  const bool small = n <= int64_t(4) << 32;
  auto kern = residual ? (small ? dropout_kernel<T, true, true> : dropout_kernel<T, true, false>)
                       : (small ? dropout_kernel<T, false, true> : dropout_kernel<T, false, false>);
  return launch_pdl(kern, dim3(unsigned(blocks)), dim3(DROP_THREADS), 0, st, static_cast<const T*>(x),
                    static_cast<const T*>(residual), rng, used, static_cast<T*>(out), n, pieces, threshold,
                    scale) == cudaSuccess
             ? MOE_B200_OK
             : MOE_B200_ERR_CUDA;
}

}  // namespace moe

using namespace moe;

extern "C" int moe_b200_dropout(const void* x, const void* residual, int64_t n, int32_t dtype, double p,
                                const int64_t* rng, int64_t* used, void* out, void* stream) {
  if (n < 0 || !(p >= 0.0 && p < 1.0)) return MOE_B200_ERR_SHAPE;
  if (dtype != MOE_B200_BF16 && dtype != MOE_B200_FP16 && dtype != MOE_B200_FP32)
    return MOE_B200_ERR_UNSUPPORTED;
  if (n == 0 && used == nullptr) return MOE_B200_OK;
  if (!rng || (n > 0 && (!x || !out))) return MOE_B200_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(rng) % 8 || reinterpret_cast<uintptr_t>(used) % 8)
    return MOE_B200_ERR_ALIGN;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (n == 0)
    return cudaMemcpyAsync(used, rng, 16, cudaMemcpyDeviceToDevice, st) == cudaSuccess ? MOE_B200_OK
                                                                                       : MOE_B200_ERR_CUDA;
  const uint32_t threshold = dropout_threshold(p);
  const float scale = float(1.0 / (1.0 - p));
  if (dtype == MOE_B200_BF16)
    return launch_dropout<__nv_bfloat16>(x, residual, rng, used, out, n, threshold, scale, st);
  if (dtype == MOE_B200_FP16)
    return launch_dropout<__half>(x, residual, rng, used, out, n, threshold, scale, st);
  return launch_dropout<float>(x, residual, rng, used, out, n, threshold, scale, st);
}
