// 16-byte loads and stores of fp32 or bf16 rows as fp32 values, shared by the
// element-wise and row-wise kernels.

#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace fh {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N elements from p; N = 1, or a multiple of a 16-byte vector with p 16-byte aligned.
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[N]) {
  constexpr int E = 16 / sizeof(T);
  if constexpr (N == 1) {
    v[0] = to_f32(*p);
  } else {
    static_assert(N % E == 0, "whole vectors");
#pragma unroll
    for (int q = 0; q < N / E; ++q) {
      const uint4 x = reinterpret_cast<const uint4*>(p)[q];
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) {
          v[q * E + k] = __uint_as_float(w[k]);
        } else {  // two bf16: the high half of an fp32 each
          v[q * E + 2 * k] = __uint_as_float(w[k] << 16);
          v[q * E + 2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        }
      }
    }
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[N]) {
  constexpr int E = 16 / sizeof(T);
  if constexpr (N == 1) {
    *p = from_f32<T>(v[0]);
  } else {
    static_assert(N % E == 0, "whole vectors");
#pragma unroll
    for (int q = 0; q < N / E; ++q) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) {
          w[k] = __float_as_uint(v[q * E + k]);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[q * E + 2 * k], v[q * E + 2 * k + 1]);
          w[k] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      reinterpret_cast<uint4*>(p)[q] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

inline bool vec_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace fh
