// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): ten rounds
// of two 32 x 32 bit products on a 128-bit counter, a 64-bit key. (No CUDA in here: the tests compile it for
// the host too.)
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define MOE_PHILOX_FN __host__ __device__ __forceinline__
#else
#define MOE_PHILOX_FN inline
#endif

namespace moe {

// The words at counters (low[j], high) under `key`, four each: N counters side by side, so that they share the
// key's schedule and fill each other's waits.
template <int N>
MOE_PHILOX_FN void philox4x32(const uint64_t* low, uint64_t high, uint64_t key, uint32_t (*word)[4]) {
  uint32_t k0 = uint32_t(key), k1 = uint32_t(key >> 32);
#ifdef __CUDACC__
#pragma unroll
#endif
  for (int j = 0; j < N; ++j) {
    word[j][0] = uint32_t(low[j]);
    word[j][1] = uint32_t(low[j] >> 32);
    word[j][2] = uint32_t(high);
    word[j][3] = uint32_t(high >> 32);
  }
#ifdef __CUDACC__
#pragma unroll
#endif
  for (int i = 0; i < 10; ++i) {
#ifdef __CUDACC__
#pragma unroll
#endif
    for (int j = 0; j < N; ++j) {
      uint32_t* c = word[j];
      const uint64_t p0 = uint64_t(0xD2511F53u) * c[0], p1 = uint64_t(0xCD9E8D57u) * c[2];
      c[0] = uint32_t(p1 >> 32) ^ c[1] ^ k0;
      c[1] = uint32_t(p1);
      c[2] = uint32_t(p0 >> 32) ^ c[3] ^ k1;
      c[3] = uint32_t(p0);
    }
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// An element whose word is below this is dropped: p in [0, 1) in units of 2^-32, to the nearest (ties to
// even), at most 2^32 - 1.
inline uint32_t dropout_threshold(double p) {
  const double scaled = p * 4294967296.0;
  const double whole = double(uint64_t(scaled));
  const double rest = scaled - whole;
  const uint64_t t = uint64_t(whole) + (rest > 0.5 || (rest == 0.5 && (uint64_t(whole) & 1)) ? 1 : 0);
  return uint32_t(t > 0xFFFFFFFFull ? 0xFFFFFFFFull : t);
}

}  // namespace moe
