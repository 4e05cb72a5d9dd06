// Shared by the two forms of the vocabulary cross entropy (gsb_loss.cu).
#pragma once
#include "gsb_common.cuh"

namespace gsb {

constexpr float LOG2E = 1.4426950408889634f;

struct LossArgs {
  const void* x;
  i64 ldx, N;
  const void* w;
  i64 ldw, V, D;
  const i64* target;
  i64 ignore;
  float scale;
  float* loss;   // [N]
  float* lse2;   // [N], base 2
  const float* g;  // [N] upstream gradient of every row's loss, 0 where it does not count
  const u32* top;  // bits of the largest |g|
  void *dx, *dw;
  void* ws;
  int* err;
  cudaStream_t st;
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

}  // namespace gsb
