// Shared by the norm kernels: a thread's elements of a row, and reductions over a row's threads.
#pragma once

#include "lf_common.h"
#include "lf_internal.h"

namespace lfamd {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A thread's V = 16 / sizeof(T) adjacent elements from column c on: one 16-byte access at any
// alignment, single elements at the row's end (zeros behind it).
template <typename T> struct Pack {
  static constexpr int V = 16 / (int)sizeof(T);
  T e[V];
  __device__ __forceinline__ static Pack load(const T* row, int c, int width) {
    u32x4 v = {0, 0, 0, 0};  // one register block on both paths, so that the load stays whole
    if (c + V <= width) {
      __builtin_memcpy(&v, row + c, 16);
    } else {
#pragma unroll
      for (int j = 0; j < V - 1; ++j)
        if (c + j < width) {
          if constexpr (V == 8) v[j >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, row[c + j]) << (16 * (j & 1));
          else v[j] = __builtin_bit_cast(uint32_t, row[c + j]);
        }
    }
    return __builtin_bit_cast(Pack, v);
  }
  __device__ __forceinline__ void store(T* row, int c, int width) const {
    const u32x4 v = __builtin_bit_cast(u32x4, *this);
    if (c + V <= width) {
      __builtin_memcpy(row + c, &v, 16);
    } else {
#pragma unroll
      for (int j = 0; j < V - 1; ++j)
        if (c + j < width) row[c + j] = e[j];
    }
  }
};

// Sum over the TPR threads of a row, in every one of them. lds: one float per wave.
template <int TPR, bool MAX> __device__ __forceinline__ float row_reduce(float v, float* lds) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) v = MAX ? fmaxf(v, __shfl_xor(v, s)) : v + __shfl_xor(v, s);
  if constexpr (TPR > 64) {
    __syncthreads();  // the values of the reduction before have been read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < TPR / 64; ++i) v = MAX ? fmaxf(v, lds[i]) : v + lds[i];
  }
  return v;
}

}  // namespace lfamd
