// Dropout whose mask is a function of the element's place: kept elements are multiplied by
// 65536 / (65536 - T), the others become zero, T = the drop probability in 1/65536.
//
// Element e belongs to block g = e / 8; the block's eight 16-bit numbers are the halfwords (low
// one first) of Philox4x32-10 with counter {g lo, g hi, 0, stream} and key = seed, the same
// counter-based streams the samplers draw from.  The element is dropped when its number is below
// T.  The backward pass is the same map on the gradient, so no mask is ever stored.
//
// Bound by the copy (read x, write y).  Sixteen bits an element and not 32: ten rounds cost about
// sixty instructions a block, which for eight 2-byte elements stays below the time of their 32
// bytes of traffic and for four would not.
#include "gsb_common.cuh"
#include "gsb_types.cuh"

namespace gsb {

template <typename T, bool VECTOR>
__global__ void __launch_bounds__(256)
dropout_kernel(const T* __restrict__ x, i64 n, u32 threshold, float scale, u64 seed, u32 stream,
               const i64* __restrict__ stream_dev, T* __restrict__ y) {
  if (stream_dev) stream += (u32)__ldg(stream_dev);
  const i64 blocks = (n + 7) / 8, step = (i64)gridDim.x * blockDim.x;
  for (i64 g = (i64)blockIdx.x * blockDim.x + threadIdx.x; g < blocks; g += step) {
    Pack<T, 8> v;
    const i64 e = g * 8;
    const bool whole = VECTOR && e + 8 <= n;
    if (whole) {
      v.load(x + e);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (e + j < n) v.v[j] = x[e + j];
    }
    const Philox4 r = stream_block(seed, stream, (u64)g, 0);
    const u32 w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const u32 u = (j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu;
      // a selection, not a product: what is dropped is zero even where x is not finite
      v.v[j] = u >= threshold ? from_float<T>(to_float(v.v[j]) * scale) : from_float<T>(0.f);
    }
    if (whole) {
      v.store(y + e);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (e + j < n) y[e + j] = v.v[j];
    }
  }
}

template <typename T>
static void launch_dropout(const void* x, i64 n, u32 threshold, float scale, u64 seed, u32 stream,
                           const i64* stream_dev, void* y, cudaStream_t st) {
  i64 blocks = ((n + 7) / 8 + 255) / 256;
  if (blocks > (i64)sm_count() * 32) blocks = (i64)sm_count() * 32;
  LaunchScope ls(KID_DROPOUT, st);
  if ((((uintptr_t)x | (uintptr_t)y) & 15) == 0)
    dropout_kernel<T, true><<<(int)blocks, 256, 0, st>>>((const T*)x, n, threshold, scale, seed, stream, stream_dev, (T*)y);
  else
    dropout_kernel<T, false><<<(int)blocks, 256, 0, st>>>((const T*)x, n, threshold, scale, seed, stream, stream_dev, (T*)y);
}

}  // namespace gsb

using namespace gsb;

extern "C" int gsb_dropout(const void* x, int dtype, int64_t n, double p, uint64_t seed, uint32_t stream,
                           const int64_t* stream_dev, void* y, void* cuda_stream) {
  if (n < 0 || !(p >= 0.0 && p <= 1.0)) return GSB_ERR_INVALID;
  if (n == 0) return GSB_OK;
  if (!x || !y) return GSB_ERR_INVALID;
  const u32 threshold = (u32)(p * 65536.0 + 0.5);
  const float scale = threshold >= 65536u ? 0.f : (float)(65536.0 / (65536.0 - threshold));
  cudaStream_t st = (cudaStream_t)cuda_stream;
  if (dtype == GSB_F32) launch_dropout<float>(x, n, threshold, scale, seed, stream, (const i64*)stream_dev, y, st);
  else if (dtype == GSB_F16) launch_dropout<__half>(x, n, threshold, scale, seed, stream, (const i64*)stream_dev, y, st);
  else if (dtype == GSB_BF16) launch_dropout<__nv_bfloat16>(x, n, threshold, scale, seed, stream, (const i64*)stream_dev, y, st);
  else return GSB_ERR_INVALID;
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}
