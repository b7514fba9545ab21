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

// 8 values of type T, as loaded and stored: one or two 16-byte pieces.
template <typename T>
struct Eight {
  uint4 v[1];
  __device__ __forceinline__ void to_float(float* f) const {
    const uint32_t w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = Half16<T>::unpack(w[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  __device__ __forceinline__ void from_float(const float* f) {
    v[0] = make_uint4(Half16<T>::pack(f[0], f[1]), Half16<T>::pack(f[2], f[3]),
                      Half16<T>::pack(f[4], f[5]), Half16<T>::pack(f[6], f[7]));
  }
};
template <>
struct Eight<float> {
  uint4 v[2];
  __device__ __forceinline__ void to_float(float* f) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[4 * i] = __uint_as_float(v[i].x);
      f[4 * i + 1] = __uint_as_float(v[i].y);
      f[4 * i + 2] = __uint_as_float(v[i].z);
      f[4 * i + 3] = __uint_as_float(v[i].w);
    }
  }
  __device__ __forceinline__ void from_float(const float* f) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      v[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]),
                        __float_as_uint(f[4 * i + 2]), __float_as_uint(f[4 * i + 3]));
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

// n8 = elements / 8 that lie in whole, 16-byte aligned pieces (0 where a pointer is not aligned); the rest
// goes one by one. A dropped element adds nothing, whatever its value (a product would make NaN of an
// infinity).
template <typename T, bool RES>
__global__ void __launch_bounds__(DROP_THREADS)
    dropout_kernel(const T* x, const T* residual, const int64_t* rng, int64_t* used, T* out, int64_t n,
                   int64_t n8, uint32_t threshold, float scale) {
  pdl_trigger();
  pdl_wait();
  const int64_t seed = ld_prev(rng), call = ld_prev(rng + 1);
  const int64_t first = int64_t(blockIdx.x) * DROP_THREADS + threadIdx.x;
  const int64_t step = int64_t(gridDim.x) * DROP_THREADS;
  if (used != nullptr && first == 0) {
    used[0] = seed;
    used[1] = call;
  }
  for (int64_t i = first; i < n8; i += step) {
    const Eight<T> a = reinterpret_cast<const Eight<T>*>(x)[i];
    Eight<T> r;
    if constexpr (RES) r = reinterpret_cast<const Eight<T>*>(residual)[i];
    uint32_t word[8];
    philox4x32(uint64_t(2 * i), uint64_t(call), uint64_t(seed), word);
    philox4x32(uint64_t(2 * i + 1), uint64_t(call), uint64_t(seed), word + 4);
    float f[8], o[8];
    a.to_float(f);
    if constexpr (RES) {
      r.to_float(o);
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = word[k] >= threshold ? fmaf(f[k], scale, o[k]) : o[k];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = word[k] >= threshold ? f[k] * scale : 0.f;
    }
    Eight<T> to;
    to.from_float(o);
    reinterpret_cast<Eight<T>*>(out)[i] = to;
  }
  for (int64_t i = n8 * 8 + first; i < n; i += step) {
    uint32_t word[4];
    philox4x32(uint64_t(i >> 2), uint64_t(call), uint64_t(seed), word);
    const uint32_t mine = (i & 2) ? ((i & 1) ? word[3] : word[2]) : ((i & 1) ? word[1] : word[0]);
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
  const int64_t n8 = any % 16 ? 0 : n / 8;
  const int64_t work = std::max(n8, n - n8 * 8);
  const int64_t blocks = std::min<int64_t>((work + DROP_THREADS - 1) / DROP_THREADS, 148 * 8);
  auto kern = residual ? dropout_kernel<T, true> : dropout_kernel<T, false>;
  return launch_pdl(kern, dim3(unsigned(blocks)), dim3(DROP_THREADS), 0, st, static_cast<const T*>(x),
                    static_cast<const T*>(residual), rng, used, static_cast<T*>(out), n, n8, threshold,
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
