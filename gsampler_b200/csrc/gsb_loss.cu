// Softmax cross entropy of x W^T over a vocabulary of V rows, without keeping the logits:
//
//   l_ij = s x_i . w_j      lse_i = log sum_j exp l_ij      loss_i = lse_i - l_{i,t_i}
//   dx_i = g_i s (sum_j p_ij w_j - w_{t_i})     dW_j = s sum_i g_i (p_ij - [t_i = j]) x_i
//   p_ij = exp(l_ij - lse_i)
//
// Entry points, and the small kernels around two forms of the products: gsb_loss_tc.cu for 16-bit
// types of up to 256 columns, gsb_loss_gemm.cu for fp32 and for wider rows.
#include "gsb_common.cuh"
#include "gsb_loss.cuh"
#include "gsb_types.cuh"

namespace gsb {

// One CTA: sum of the rows' losses (in 64 bits) and the number of rows that count.
__global__ void __launch_bounds__(1024)
loss_total_kernel(const float* __restrict__ loss, const i64* __restrict__ target, i64 ignore, i64 V, i64 N, int mean,
                  float* __restrict__ total, float* __restrict__ count) {
  __shared__ double ws[32];
  __shared__ i64 wc[32];
  double s = 0;
  i64 c = 0;
  for (i64 i = threadIdx.x; i < N; i += 1024) {
    s += loss[i];
    const i64 t = target[i];
    c += t != ignore && t >= 0 && t < V;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  c = warp_sum(c);
  if ((threadIdx.x & 31) == 0) { ws[threadIdx.x >> 5] = s; wc[threadIdx.x >> 5] = c; }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0;
    c = 0;
    for (int k = 0; k < 32; ++k) { s += ws[k]; c += wc[k]; }
    if (c < 1) c = 1;  // no row counts: the loss is 0, and so are the gradients
    *total = (float)(mean ? s / (double)c : s);
    *count = (float)c;
  }
}

// g[i] = upstream gradient of row i's loss (divided by the count for the mean), 0 where the row
// does not count; top = bits of the largest magnitude (an integer maximum: no order matters).
__global__ void loss_row_grad_kernel(const float* __restrict__ up, int per_row, const float* __restrict__ count,
                                     const i64* __restrict__ target, i64 ignore, i64 V, i64 N, float* __restrict__ g,
                                     u32* top) {
  u32 mine = 0;
  for (i64 i = (i64)blockIdx.x * blockDim.x + threadIdx.x; i < N; i += (i64)gridDim.x * blockDim.x) {
    const i64 t = target[i];
    float v = 0.f;
    if (t != ignore && t >= 0 && t < V) v = per_row ? up[i] : (count ? *up / *count : *up);
    g[i] = v;
    const u32 b = __float_as_uint(fabsf(v));
    mine = b > mine ? b : mine;
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

extern "C" int gsb_linear_ce_has_pull(int dtype, int64_t N, int64_t V, int64_t D) { return tc_loss_takes(dtype, N, V, D); }

extern "C" size_t gsb_linear_ce_workspace_bytes(int dtype, const void* weight, int64_t ldw, int64_t N, int64_t V, int64_t D,
                                                int want_pull) {
  if (!loss_sizes_ok(N, V, D, D, D)) return 0;
  if (tc_loss_takes(dtype, N, V, D)) return tc_loss_workspace(N, V, D, want_pull != 0, tc_loss_packs(weight, ldw));
  return gemm_loss_workspace(dtype, N, V, D, tc_loss_packs(weight, ldw));
}

extern "C" int gsb_linear_ce(const void* x, int dtype, int64_t ldx, int64_t N, const void* weight, int64_t ldw, int64_t V,
                             int64_t D, const int64_t* target, int64_t ignore, float scale, float* loss, float* lse2,
                             float* pull, void* workspace, size_t workspace_bytes, int* d_err, void* cuda_stream) {
  if (!loss_sizes_ok(N, V, D, ldx, ldw) || !(scale - scale == 0.f)) return GSB_ERR_INVALID;
  if (dtype != GSB_F32 && dtype != GSB_F16 && dtype != GSB_BF16) return GSB_ERR_INVALID;
  if (pull && !gsb_linear_ce_has_pull(dtype, N, V, D)) return GSB_ERR_UNSUPPORTED;
  if (N == 0) return GSB_OK;
  if (!x || !weight || !target || !loss || !lse2) return GSB_ERR_INVALID;
  if (!workspace || workspace_bytes < gsb_linear_ce_workspace_bytes(dtype, weight, ldw, N, V, D, pull != nullptr))
    return GSB_ERR_WORKSPACE;
  LossArgs a = {};
  a.x = x; a.ldx = ldx; a.N = N; a.w = weight; a.ldw = ldw; a.V = V; a.D = D;
  a.target = (const i64*)target; a.ignore = ignore; a.scale = scale; a.loss = loss; a.lse2 = lse2;
  a.ws = workspace; a.err = d_err; a.st = (cudaStream_t)cuda_stream;
  int rc = GSB_OK;
  if (tc_loss_takes(dtype, N, V, D))
    rc = dtype == GSB_F16 ? tc_loss_forward<__half>(a, pull) : tc_loss_forward<__nv_bfloat16>(a, pull);
  else
    rc = dtype == GSB_F32 ? gemm_loss_forward<float>(a)
         : dtype == GSB_F16 ? gemm_loss_forward<__half>(a) : gemm_loss_forward<__nv_bfloat16>(a);
  if (rc != GSB_OK) return rc;
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}

extern "C" int gsb_linear_ce_total(const float* loss, const int64_t* target, int64_t ignore, int64_t V, int64_t N,
                                   int mean, float* total, float* count, void* cuda_stream) {
  if (N < 0 || !total || !count || (N > 0 && (!loss || !target))) return GSB_ERR_INVALID;
  cudaStream_t st = (cudaStream_t)cuda_stream;
  LaunchScope ls(KID_LOSS_JOIN, st);
  loss_total_kernel<<<1, 1024, 0, st>>>(loss, (const i64*)target, ignore, V, N, mean, total, count);
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}

extern "C" size_t gsb_linear_ce_grad_workspace_bytes(int dtype, const void* weight, int64_t ldw, int64_t N, int64_t V, int64_t D,
                                                     int have_pull, int want_dx, int want_dw) {
  if (!loss_sizes_ok(N, V, D, D, D)) return 0;
  const size_t head = up256(4 * (size_t)N) + 256;
  const bool tc = tc_loss_takes(dtype, N, V, D);
  const bool rest_dx = want_dx && !(tc && have_pull), rest_dw = want_dw && !tc, pack = tc_loss_packs(weight, ldw);
  size_t need = rest_dx || rest_dw ? gemm_loss_grad_workspace(dtype, N, V, D, rest_dx, rest_dw, pack) : 0;
  if (tc && want_dw) {
    const size_t b = tc_loss_grad_workspace(N, V, D, pack);
    if (b > need) need = b;
  }
  return head + need;
}

extern "C" int gsb_linear_ce_grad(const void* x, int dtype, int64_t ldx, int64_t N, const void* weight, int64_t ldw,
                                  int64_t V, int64_t D, const int64_t* target, int64_t ignore, float scale,
                                  const float* lse2, const float* pull, const float* upstream, int per_row,
                                  const float* count, void* dx, void* dw, void* workspace, size_t workspace_bytes,
                                  int* d_err, void* cuda_stream) {
  if (!loss_sizes_ok(N, V, D, ldx, ldw) || !(scale - scale == 0.f)) return GSB_ERR_INVALID;
  if (dtype != GSB_F32 && dtype != GSB_F16 && dtype != GSB_BF16) return GSB_ERR_INVALID;
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
  u32* top = (u32*)(ws + up256(4 * (size_t)N));
  GSB_CUDA_OK(cudaMemsetAsync(top, 0, 4, st));
  {
    LaunchScope ls(KID_LOSS_JOIN, st);
    i64 blocks = (N + 255) / 256;
    if (blocks > sm_count() * 4) blocks = sm_count() * 4;
    loss_row_grad_kernel<<<(int)blocks, 256, 0, st>>>(upstream, per_row, count, (const i64*)target, ignore, V, N, g, top);
  }
  LossArgs a = {};
  a.x = x; a.ldx = ldx; a.N = N; a.w = weight; a.ldw = ldw; a.V = V; a.D = D;
  a.target = (const i64*)target; a.ignore = ignore; a.scale = scale; a.lse2 = const_cast<float*>(lse2);
  a.g = g; a.top = top; a.dx = dx; a.dw = dw; a.ws = ws + up256(4 * (size_t)N) + 256; a.err = d_err; a.st = st;
  if (tc_loss_takes(dtype, N, V, D)) {
    const bool half = dtype == GSB_F16;
    if (a.dx && pull) {
      if (half) tc_loss_dx<__half>(a, pull);
      else tc_loss_dx<__nv_bfloat16>(a, pull);
      a.dx = nullptr;
    }
    if (a.dw) {
      const int rc = half ? tc_loss_grad_w<__half>(a) : tc_loss_grad_w<__nv_bfloat16>(a);
      if (rc != GSB_OK) return rc;
      a.dw = nullptr;
    }
  }
  if (a.dx || a.dw) {
    const int rc = dtype == GSB_F32 ? gemm_loss_backward<float>(a)
                   : dtype == GSB_F16 ? gemm_loss_backward<__half>(a) : gemm_loss_backward<__nv_bfloat16>(a);
    if (rc != GSB_OK) return rc;
  }
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}
