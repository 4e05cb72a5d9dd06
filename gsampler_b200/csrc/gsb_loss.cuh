// Shared by the two forms of the vocabulary cross entropy (gsb_loss.cu, gsb_loss_tc.cu).
#pragma once
#include <atomic>

#include "gsb_common.cuh"
#include "gsb_types.cuh"

namespace gsb {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int FWD_SHIFT = 7;    // the forward pass holds p at 2^7 times its value relative to the row's reference
// The backward pass holds g (p - target) at 2^14 / max |g| times its value for dW, whose sums run over the rows; for
// dx g is a factor of the row, and fp16 holds p at 2^14 times its value.
constexpr int GRAD_SHIFT = 14;
// Every addition into a 32-bit accumulator of the matrix units truncates, 16 products at a time: a sum of one sign
// loses 0.3 units in the last place each time (262144 terms in a row were off by 6e-4 of their sum, 65536
// columns by 4e-4 of the logit).  So a run of additions ends after this many terms, and its sum goes on in
// 32-bit additions that round: at most 2^-13 of the sum is lost, 2^-17 for fp32.  The streamed form lets
// bf16, whose half step is eight times fp16's, run eight times as long.
constexpr int RUN_TERMS = 16384, RUN_TERMS_F32 = 1024;
template <typename T>
constexpr int streamed_run() { return sizeof(T) == 4 ? RUN_TERMS_F32 : IsBf16<T>::value ? 8 * RUN_TERMS : RUN_TERMS; }
constexpr float MOVE_REFERENCE = 8.f;  // a row's reference moves when its maximum passes it by 2^8

// Factor from x . w to a base-2 logit, |scale| log2 e (the sign goes into x).  Not zero, so that a
// masked logit of -inf stays one; times any finite product 1e-38 is as good as zero.
inline float logit_factor(float scale) { return fmaxf(fabsf(scale) * LOG2E, 1e-38f); }

// Lets a kernel use `bytes` of shared memory; asked once a device, `done` is the kernel's own word.
template <typename K>
inline bool allow_shared(K kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

inline size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
inline int blocks_for(i64 threads) {
  const i64 b = (threads + 255) / 256, most = (i64)sm_count() * 16;
  return (int)(b < 1 ? 1 : b < most ? b : most);
}

// In how many parts the tiles B are split among the CTAs of one group of rows A.  `groups` CTAs cover
// the rows; the time is (rounds of CTAs on the SMs' `slots`) x (tiles of one + about 3 for its start and
// end), so for each number of rounds the split that just fills them is the only one worth a look.
inline int split_count(i64 groups, i64 tiles, i64 slots) {
  const i64 first = (groups + slots - 1) / slots;
  int best = 1;
  double best_t = (double)first * (double)(tiles + 3);
  for (i64 rounds = first; rounds <= 3; ++rounds) {
    i64 s = rounds * slots / groups;
    if (s < 1) continue;
    const i64 per = tiles <= s ? 1 : (tiles + s - 1) / s;
    s = (tiles + per - 1) / per;
    const double t = (double)((groups * s + slots - 1) / slots) * (double)(per + 3);
    if (t < best_t * 0.999) { best_t = t; best = (int)s; }
  }
  return best;
}

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
  int per_row;     // whether rows have gradients of their own
  const float* g;  // [N] upstream gradient of every row's loss, 0 where it does not count
  const float* miss;  // [N] 1 - p of the row's target
  const u32* top;  // bits of the largest finite |g|: one row's infinity or NaN is not a factor of the others
  void *dx, *dw;
  void* ws;
  int* err;
  cudaStream_t st;
};

template <typename T>
constexpr int dtype_of() { return sizeof(T) == 4 ? GSB_F32 : IsBf16<T>::value ? GSB_BF16 : GSB_F16; }

// How a type reaches the tensor cores: as it is, or as three bf16 planes (h + m + l, 8 bits each).
template <typename S> struct Planes { typedef S type; static constexpr int count = 1; };
template <> struct Planes<float> { typedef __nv_bfloat16 type; static constexpr int count = 3; };
// dst[plane][r, :] = the planes of +-src[r, :], rows of packed_ld(D) elements; with g and lse2, rows whose g is zero
// and whose lse2 is not finite as zeros; with top, rows times 2^small_rows (gsb_loss_gemm.cu)
template <typename S>
void make_planes(const void* src, i64 ld, i64 rows, i64 D, bool negate, const float* g, const float* lse2, const u32* top, void* dst,
                 cudaStream_t st);

// Where one array of g (p - target) serves both dx and dW, a row whose |g| is below 2^-16 of the largest would
// lose its digits in fp16.  Such a row is held times a power of two, 2^-small_rows, that brings it there (to at
// most top / 2^15), and its row of x takes the power back for dW.
template <typename T>
__device__ __forceinline__ int small_rows(float g, float top) {
  if (sizeof(T) != 2 || IsBf16<T>::value || !(fabsf(g) < INFINITY) || g == 0.f || top == 0.f) return 0;
  const int e = ilogbf(g) - ilogbf(top) + 16;
  return e < 0 ? e : 0;
}
__device__ __forceinline__ float times_power(float v, int e) { return e == 0 ? v : scalbnf(v, e); }

// Rounding to nearest would make the first plane of a finite value above this infinite (and the next ones
// infinite the other way): it stays at the largest bf16, and the next planes hold the rest.
__device__ __forceinline__ float first_plane(float v) {
  constexpr float MOST = 3.3895313892515355e38f;  // (2 - 2^-7) 2^127
  return fabsf(v) < INFINITY ? fminf(fmaxf(v, -MOST), MOST) : v;
}
// The two accumulators of plane products.  An infinite value is in its first plane and the others are
// NaN, so the accumulator of the two first planes alone decides: what is not finite there stays what
// it is, and the other counts as finite.
__device__ __forceinline__ float finite_part(float low) {
  float r;  // the smaller magnitude with low's sign: one instruction, where clamping takes two
  asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(low), "f"(3.402823466e38f));
  return r;
}
__device__ __forceinline__ float add_planes(float low, float high) { return high + finite_part(low); }

// The streamed form (gsb_loss_tc.cu): 16-bit types of up to 256 columns, fp32 of up to 128.
bool tc_loss_takes(int dtype, i64 D);
bool tc_loss_pulls(int dtype, i64 V);  // whether the forward pass delivers what dx is made from, or dx makes the logits again
bool tc_loss_packs(const void* w, i64 ldw);  // whether the rows of W have to be copied for it
size_t tc_loss_workspace(int dtype, i64 N, i64 V, i64 D, bool pull, bool pack_w);
size_t tc_loss_grad_workspace(int dtype, i64 N, i64 V, i64 D, bool dx, bool dw);
// The general form (gsb_loss_gemm.cu).
size_t gemm_loss_workspace(int dtype, i64 N, i64 V, i64 D, bool pack_w);
size_t gemm_loss_grad_workspace(int dtype, i64 N, i64 V, i64 D, bool dx, bool dw, bool pack_w);
template <typename T>
int gemm_loss_forward(const LossArgs& a);
template <typename T>
int gemm_loss_backward(const LossArgs& a);
// losses (and pulls) of all rows from the parts of their statistics, which leave the targets out, and hot, the
// targets' products (gsb_loss_tc.cu)
template <typename T>
void launch_loss_join(const LossArgs& a, const float2* part_ms, int parts, const float* part_o, const float* hot, float* pull);

template <typename T>
int tc_loss_forward(const LossArgs& a, float* pull);
template <typename T>
int tc_loss_grad_w(const LossArgs& a);
template <typename T>
int tc_loss_grad_x(const LossArgs& a);
template <typename T>
void tc_loss_dx(const LossArgs& a, const float* pull);

}  // namespace gsb
