// Shared by the two forms of the vocabulary cross entropy (gsb_loss.cu, gsb_loss_tc.cu).
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

// The tensor-core form (gsb_loss_tc.cu): 16-bit types, up to 256 columns.
bool tc_loss_takes(int dtype, i64 N, i64 V, i64 D);
bool tc_loss_packs(const void* w, i64 ldw);  // whether the rows of W have to be copied for it
size_t tc_loss_workspace(i64 N, i64 V, i64 D, bool pull, bool pack_w);
size_t tc_loss_grad_workspace(i64 N, i64 V, i64 D, bool pack_w);
template <typename T>
int tc_loss_forward(const LossArgs& a, float* pull);
template <typename T>
int tc_loss_grad_w(const LossArgs& a);
template <typename T>
void tc_loss_dx(const LossArgs& a, const float* pull);

}  // namespace gsb
