// Element types of the operators on learned values (fp32, fp16, bf16) and vectors of them.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/gsb200.h"

namespace gsb {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Whether p (null included) is a multiple of `bytes`: what the entry points ask of every pointer.
inline bool at_multiple(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
inline size_t value_bytes(int dtype) { return dtype == GSB_F32 ? 4 : 2; }

template <typename T> struct IsBf16 { static constexpr bool value = false; };
template <> struct IsBf16<__nv_bfloat16> { static constexpr bool value = true; };

template <int BYTES> struct Raw;
template <> struct Raw<2> { typedef unsigned short type; };
template <> struct Raw<4> { typedef unsigned int type; };
template <> struct Raw<8> { typedef uint2 type; };
template <> struct Raw<16> { typedef uint4 type; };

// N elements moved by one access (two of 16 bytes for the 32-byte ones)
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
  static constexpr int BYTES = (int)sizeof(T) * N;
  static constexpr int PIECE = BYTES < 16 ? BYTES : 16;
  typedef typename Raw<PIECE>::type raw;
  T v[N];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < BYTES / PIECE; ++i) reinterpret_cast<raw*>(v)[i] = __ldg(reinterpret_cast<const raw*>(p) + i);
  }
  // from memory that this kernel also writes
  __device__ __forceinline__ void load_written(const T* p) {
#pragma unroll
    for (int i = 0; i < BYTES / PIECE; ++i) reinterpret_cast<raw*>(v)[i] = reinterpret_cast<const raw*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < BYTES / PIECE; ++i) reinterpret_cast<raw*>(p)[i] = reinterpret_cast<const raw*>(v)[i];
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = from_float<T>(0.f);
  }
};

}  // namespace gsb
