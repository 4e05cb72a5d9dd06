// Softmax cross entropy of x W^T over a vocabulary of V rows, without keeping the logits:
//
//   l_ij = s x_i . w_j      lse_i = log sum_j exp l_ij      loss_i = lse_i - l_{i,t_i}
//   dx_i = g_i s (sum_j p_ij w_j - w_{t_i})     dW_j = s sum_i g_i (p_ij - [t_i = j]) x_i
//   p_ij = exp(l_ij - lse_i)
//
// Entry points, and the small kernels around two forms of the products: gsb_loss_tc.cu for 16-bit
// types of up to 256 columns and fp32 of up to 128, gsb_loss_gemm.cu for wider rows.
#include "gsb_common.cuh"
#include "gsb_loss.cuh"
#include "gsb_types.cuh"

namespace gsb {

// Sum of the rows' losses (in 64 bits) and the number of rows that count: CTA b adds its share to
// part[b], or finishes when it is the only one; then one CTA adds the parts in order.
__device__ __forceinline__ void block_total(double s, double c, double* shared, double* out_s, double* out_c) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, d);
    c += __shfl_xor_sync(0xffffffffu, c, d);
  }
  if ((threadIdx.x & 31) == 0) { shared[threadIdx.x >> 5] = s; shared[32 + (threadIdx.x >> 5)] = c; }
  __syncthreads();
  *out_s = *out_c = 0;
  for (int k = 0; k < (int)blockDim.x / 32; ++k) { *out_s += shared[k]; *out_c += shared[32 + k]; }
}
__device__ __forceinline__ void write_total(double s, double c, int mean, float* total, float* count) {
  if (c < 1) c = 1;  // no row counts: the loss is 0, and so are the gradients
  *total = (float)(mean ? s / c : s);
  *count = (float)c;
}
__global__ void __launch_bounds__(512)
loss_total_kernel(const float* __restrict__ loss, const i64* __restrict__ target, i64 ignore, i64 V, i64 N, int mean,
                  double2* __restrict__ part, float* __restrict__ total, float* __restrict__ count) {
  __shared__ double shared[64];
  double s = 0, c = 0;
  for (i64 i = (i64)blockIdx.x * 512 + threadIdx.x; i < N; i += (i64)gridDim.x * 512) {
    s += loss[i];
    const i64 t = target[i];
    c += t != ignore && t >= 0 && t < V ? 1.0 : 0.0;
  }
  double all_s, all_c;
  block_total(s, c, shared, &all_s, &all_c);
  if (threadIdx.x == 0) {
    if (gridDim.x == 1) write_total(all_s, all_c, mean, total, count);
    else part[blockIdx.x] = make_double2(all_s, all_c);
  }
}
__global__ void __launch_bounds__(512)
loss_total_join_kernel(const double2* __restrict__ part, int parts, int mean, float* __restrict__ total, float* __restrict__ count) {
  __shared__ double shared[64];
  const double2 mine = (int)threadIdx.x < parts ? part[threadIdx.x] : make_double2(0, 0);
  double all_s, all_c;
  block_total(mine.x, mine.y, shared, &all_s, &all_c);
  if (threadIdx.x == 0) write_total(all_s, all_c, mean, total, count);
}
// up to 8192 rows take one CTA less time than a second launch
static int total_blocks(i64 N) {
  if (N <= 8192) return 1;
  const i64 b = (N + 4095) / 4096;
  return (int)(b < 512 ? b : 512);
}

// 1 - p_t of every row that counts, from its loss.
__device__ __forceinline__ float miss_of_loss(float loss) { return -expm1f(-loss); }

// The same from the log-sum-exp and the target's logit made once more, a warp a row: to about 1e-6, the units in
// the last place of both.
template <typename T>
__global__ void __launch_bounds__(256)
loss_miss_kernel(const T* __restrict__ x, i64 ldx, i64 N, const T* __restrict__ w, i64 ldw, i64 V, int D, float scale, const i64* __restrict__ target,
                 i64 ignore, const float* __restrict__ lse2, float* __restrict__ miss) {
  const i64 r = ((i64)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (r >= N) return;
  const i64 t = target[r];
  float l = 0.f;
  if (t != ignore && t >= 0 && t < V)
    for (int d = lane; d < D; d += 32) l = fmaf(to_float(x[r * ldx + d]), to_float(w[t * ldw + d]), l);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  if (lane == 0) {
    const float d = lse2[r] * 0.6931471805599453f - l * scale;
    miss[r] = miss_of_loss(d < 0.f ? 0.f : d);
  }
}

// g[i] = upstream gradient of row i's loss (divided by the count for the mean), 0 where the row
// does not count; with loss, miss[i] = 1 - p_t; top = bits of the largest finite magnitude (an integer maximum: no order matters).
__global__ void loss_row_grad_kernel(const float* __restrict__ up, int per_row, const float* __restrict__ count,
                                     const i64* __restrict__ target, i64 ignore, i64 V, i64 N, const float* __restrict__ loss,
                                     float* __restrict__ g, float* __restrict__ miss, u32* top) {
  constexpr u32 INFINITE = 0x7F800000u;
  u32 mine = 0;
  for (i64 i = (i64)blockIdx.x * blockDim.x + threadIdx.x; i < N; i += (i64)gridDim.x * blockDim.x) {
    const i64 t = target[i];
    float v = 0.f;
    if (t != ignore && t >= 0 && t < V) v = per_row ? up[i] : (count ? *up / *count : *up);
    g[i] = v;
    if (loss) miss[i] = miss_of_loss(loss[i]);
    const u32 b = __float_as_uint(fabsf(v));
    mine = b > mine && b < INFINITE ? b : mine;
  }
  if (!per_row) {  // the same for every row that counts
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      const u32 b = __float_as_uint(fabsf(count ? *up / *count : *up));
      *top = b < INFINITE ? b : 0;
    }
    return;
  }
  mine = __reduce_max_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0 && mine) atomicMax(top, mine);
}

}  // namespace gsb

using namespace gsb;

static bool loss_sizes_ok(i64 N, i64 V, i64 D, i64 ldx, i64 ldw) {
  return N >= 0 && N <= (1ll << 30) && V >= 1 && V <= (1ll << 30) && D >= 1 && D <= GSB_LOSS_MAX_D && (N < 2 || ldx >= D) &&
         (V < 2 || ldw >= D);
}

extern "C" int gsb_linear_ce_has_pull(int dtype, int64_t V, int64_t D) { return tc_loss_takes(dtype, D) && tc_loss_pulls(dtype, V); }

extern "C" size_t gsb_linear_ce_workspace_bytes(int dtype, const void* weight, int64_t ldw, int64_t N, int64_t V, int64_t D,
                                                int want_pull) {
  if (!loss_sizes_ok(N, V, D, D, D)) return 0;
  if (tc_loss_takes(dtype, D)) return tc_loss_workspace(dtype, N, V, D, want_pull != 0, tc_loss_packs(weight, ldw));
  return gemm_loss_workspace(dtype, N, V, D, tc_loss_packs(weight, ldw));
}

extern "C" int gsb_linear_ce(const void* x, int dtype, int64_t ldx, int64_t N, const void* weight, int64_t ldw, int64_t V,
                             int64_t D, const int64_t* target, int64_t ignore, float scale, float* loss, float* lse2,
                             float* pull, void* workspace, size_t workspace_bytes, int* d_err, void* cuda_stream) {
  if (!loss_sizes_ok(N, V, D, ldx, ldw) || !(scale - scale == 0.f)) return GSB_ERR_INVALID;
  if (dtype != GSB_F32 && dtype != GSB_F16 && dtype != GSB_BF16) return GSB_ERR_INVALID;
  if (pull && !gsb_linear_ce_has_pull(dtype, V, D)) return GSB_ERR_UNSUPPORTED;
  if (N == 0) return GSB_OK;
  if (!x || !weight || !target || !loss || !lse2) return GSB_ERR_INVALID;
  if (!at_multiple(x, value_bytes(dtype)) || !at_multiple(weight, value_bytes(dtype)) || !at_multiple(target, 8) ||
      !at_multiple(loss, 4) || !at_multiple(lse2, 4) || !at_multiple(pull, 4) || !at_multiple(workspace, 16) || !at_multiple(d_err, 4))
    return GSB_ERR_INVALID;
  if (!workspace || workspace_bytes < gsb_linear_ce_workspace_bytes(dtype, weight, ldw, N, V, D, pull != nullptr))
    return GSB_ERR_WORKSPACE;
  LossArgs a = {};
  a.x = x; a.ldx = ldx; a.N = N; a.w = weight; a.ldw = ldw; a.V = V; a.D = D;
  a.target = (const i64*)target; a.ignore = ignore; a.scale = scale; a.loss = loss; a.lse2 = lse2;
  a.ws = workspace; a.err = d_err; a.st = (cudaStream_t)cuda_stream;
  int rc = GSB_OK;
  if (tc_loss_takes(dtype, D))
    rc = dtype == GSB_F32 ? tc_loss_forward<float>(a, pull)
         : dtype == GSB_F16 ? tc_loss_forward<__half>(a, pull) : tc_loss_forward<__nv_bfloat16>(a, pull);
  else
    rc = dtype == GSB_F32 ? gemm_loss_forward<float>(a)
         : dtype == GSB_F16 ? gemm_loss_forward<__half>(a) : gemm_loss_forward<__nv_bfloat16>(a);
  if (rc != GSB_OK) return rc;
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}

extern "C" size_t gsb_linear_ce_total_workspace_bytes(int64_t N) { return sizeof(double2) * (size_t)total_blocks(N); }

extern "C" int gsb_linear_ce_total(const float* loss, const int64_t* target, int64_t ignore, int64_t V, int64_t N,
                                   int mean, float* total, float* count, void* workspace, size_t workspace_bytes,
                                   void* cuda_stream) {
  if (N < 0 || !total || !count || (N > 0 && (!loss || !target))) return GSB_ERR_INVALID;
  if (!at_multiple(loss, 4) || !at_multiple(target, 8) || !at_multiple(total, 4) || !at_multiple(count, 4) || !at_multiple(workspace, 16))
    return GSB_ERR_INVALID;
  const int blocks = total_blocks(N);
  if (blocks > 1 && (!workspace || workspace_bytes < gsb_linear_ce_total_workspace_bytes(N))) return GSB_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)cuda_stream;
  {
    LaunchScope ls(KID_LOSS_JOIN, st);
    loss_total_kernel<<<blocks, 512, 0, st>>>(loss, (const i64*)target, ignore, V, N, mean, (double2*)workspace, total, count);
  }
  if (blocks > 1) {
    LaunchScope ls(KID_LOSS_JOIN, st);
    loss_total_join_kernel<<<1, 512, 0, st>>>((const double2*)workspace, blocks, mean, total, count);
  }
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}

extern "C" size_t gsb_linear_ce_grad_workspace_bytes(int dtype, const void* weight, int64_t ldw, int64_t N, int64_t V, int64_t D,
                                                     int have_pull, int want_dx, int want_dw) {
  if (!loss_sizes_ok(N, V, D, D, D)) return 0;
  const size_t head = 2 * up256(4 * (size_t)N) + 256;
  if (!tc_loss_takes(dtype, D))
    return head + gemm_loss_grad_workspace(dtype, N, V, D, want_dx != 0, want_dw != 0, tc_loss_packs(weight, ldw));
  return head + tc_loss_grad_workspace(dtype, N, V, D, want_dx && !have_pull, want_dw != 0);
}

extern "C" int gsb_linear_ce_grad(const void* x, int dtype, int64_t ldx, int64_t N, const void* weight, int64_t ldw,
                                  int64_t V, int64_t D, const int64_t* target, int64_t ignore, float scale,
                                  const float* lse2, const float* pull, const float* upstream, int per_row,
                                  const float* count, void* dx, void* dw, void* workspace, size_t workspace_bytes,
                                  int* d_err, void* cuda_stream) {
  return gsb_linear_ce_grad_rows(x, dtype, ldx, N, weight, ldw, V, D, target, ignore, scale, nullptr, lse2, pull, upstream, per_row, count, dx,
                                 dw, workspace, workspace_bytes, d_err, cuda_stream);
}

extern "C" int gsb_linear_ce_grad_rows(const void* x, int dtype, int64_t ldx, int64_t N, const void* weight, int64_t ldw,
                                       int64_t V, int64_t D, const int64_t* target, int64_t ignore, float scale,
                                       const float* loss, const float* lse2, const float* pull, const float* upstream,
                                       int per_row, const float* count, void* dx, void* dw, void* workspace,
                                       size_t workspace_bytes, int* d_err, void* cuda_stream) {
  if (!loss_sizes_ok(N, V, D, ldx, ldw) || !(scale - scale == 0.f)) return GSB_ERR_INVALID;
  if (dtype != GSB_F32 && dtype != GSB_F16 && dtype != GSB_BF16) return GSB_ERR_INVALID;
  if (!at_multiple(x, value_bytes(dtype)) || !at_multiple(weight, value_bytes(dtype)) || !at_multiple(target, 8) ||
      !at_multiple(loss, 4) || !at_multiple(lse2, 4) || !at_multiple(pull, 4) || !at_multiple(upstream, 4) || !at_multiple(count, 4) ||
      !at_multiple(dx, value_bytes(dtype)) || !at_multiple(dw, value_bytes(dtype)) || !at_multiple(workspace, 16) || !at_multiple(d_err, 4))
    return GSB_ERR_INVALID;
  cudaStream_t st = (cudaStream_t)cuda_stream;
  if (N == 0) {
    if (dw) GSB_CUDA_OK(cudaMemsetAsync(dw, 0, (size_t)V * D * (dtype == GSB_F32 ? 4 : 2), st));
    return GSB_OK;
  }
  if (!dx && !dw) return GSB_OK;
  if (!x || !weight || !target || !lse2 || !upstream) return GSB_ERR_INVALID;
  if (!workspace || workspace_bytes < gsb_linear_ce_grad_workspace_bytes(dtype, weight, ldw, N, V, D, pull != nullptr,
                                                                         dx != nullptr, dw != nullptr))
    return GSB_ERR_WORKSPACE;
  char* ws = (char*)workspace;
  float* g = (float*)ws;
  float* miss = (float*)(ws + up256(4 * (size_t)N));
  u32* top = (u32*)(ws + 2 * up256(4 * (size_t)N));
  if (per_row) GSB_CUDA_OK(cudaMemsetAsync(top, 0, 4, st));
  {
    LaunchScope ls(KID_LOSS_JOIN, st);
    i64 blocks = (N + 255) / 256;
    if (blocks > sm_count() * 4) blocks = sm_count() * 4;
    loss_row_grad_kernel<<<(int)blocks, 256, 0, st>>>(upstream, per_row, count, (const i64*)target, ignore, V, N, loss, g, miss, top);
  }
  if (!loss && (dw || !pull)) {
    LaunchScope ls(KID_LOSS_JOIN, st);
    const int blocks = ceil_div_i(N, 8);
    auto launch = [&](auto* xs, auto* rows_w) {
      loss_miss_kernel<<<blocks, 256, 0, st>>>(xs, ldx, N, rows_w, ldw, V, (int)D, scale, (const i64*)target, ignore, lse2, miss);
    };
    if (dtype == GSB_F32) launch((const float*)x, (const float*)weight);
    else if (dtype == GSB_F16) launch((const __half*)x, (const __half*)weight);
    else launch((const __nv_bfloat16*)x, (const __nv_bfloat16*)weight);
  }
  LossArgs a = {};
  a.x = x; a.ldx = ldx; a.N = N; a.w = weight; a.ldw = ldw; a.V = V; a.D = D;
  a.target = (const i64*)target; a.ignore = ignore; a.scale = scale; a.lse2 = const_cast<float*>(lse2);
  a.per_row = per_row; a.g = g; a.miss = miss; a.top = top; a.dx = dx; a.dw = dw; a.ws = ws + 2 * up256(4 * (size_t)N) + 256; a.err = d_err; a.st = st;
  int rc = GSB_OK;
  if (!tc_loss_takes(dtype, D)) {
    rc = dtype == GSB_F32 ? gemm_loss_backward<float>(a)
         : dtype == GSB_F16 ? gemm_loss_backward<__half>(a) : gemm_loss_backward<__nv_bfloat16>(a);
  } else {
    if (a.dx && pull) {
      if (dtype == GSB_F16) tc_loss_dx<__half>(a, pull);
      else tc_loss_dx<__nv_bfloat16>(a, pull);
      a.dx = nullptr;  // what is left below
    } else if (a.dx) {
      rc = dtype == GSB_F32 ? tc_loss_grad_x<float>(a)
           : dtype == GSB_F16 ? tc_loss_grad_x<__half>(a) : tc_loss_grad_x<__nv_bfloat16>(a);
    }
    if (rc == GSB_OK && a.dw)
      rc = dtype == GSB_F32 ? tc_loss_grad_w<float>(a)
           : dtype == GSB_F16 ? tc_loss_grad_w<__half>(a) : tc_loss_grad_w<__nv_bfloat16>(a);
  }
  if (rc != GSB_OK) return rc;
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}
