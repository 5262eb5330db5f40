// Vectors of N elements of bf16, fp16 or fp32 held as fp32, moved with 16-byte accesses where N elements fill them.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace mb {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half(v); }

// Raw bits of N elements: 16-byte pieces, or single elements for N = 1.
template <typename T, int N>
struct Vec {
  static_assert(N == 1 || (N * sizeof(T)) % 16 == 0, "whole 16-byte pieces");
  static constexpr int kPieces = N == 1 ? 1 : static_cast<int>(N * sizeof(T) / 16);
  union {
    uint4 piece[kPieces];
    uint32_t word[4 * kPieces];
    T at[N];
  };
  __device__ __forceinline__ Vec() {}
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) piece[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (N == 1) {
      at[0] = *p;
    } else {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) piece[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    }
  }
  // for data that is read once: leaves L1 to what is read again
  __device__ __forceinline__ void load_once(const T* p) {
    if constexpr (N == 1) {
      at[0] = *p;
    } else {
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(piece[i].x), "=r"(piece[i].y), "=r"(piece[i].z), "=r"(piece[i].w)
                     : "l"(reinterpret_cast<const uint4*>(p) + i));
    }
  }
  __device__ __forceinline__ void load_shared(const T* p) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) piece[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (N == 1) {
      *p = at[0];
    } else {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) reinterpret_cast<uint4*>(p)[i] = piece[i];
    }
  }
  __device__ __forceinline__ float get(int i) const { return to_float(at[i]); }
  __device__ __forceinline__ void set(int i, float v) { at[i] = from_float<T>(v); }
};

}  // namespace mb
