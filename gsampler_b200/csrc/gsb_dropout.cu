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

__device__ __forceinline__ u32 scale_pair(u32 v, float scale, const __half*) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  const __half2 r = __floats2half2_rn(f.x * scale, f.y * scale);
  return *reinterpret_cast<const u32*>(&r);
}
__device__ __forceinline__ u32 scale_pair(u32 v, float scale, const __nv_bfloat16*) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(__uint_as_float(v << 16) * scale, __uint_as_float(v & 0xFFFF0000u) * scale);
  return *reinterpret_cast<const u32*>(&r);
}

// the eight elements of block g; a selection, not a product: what is dropped is zero even where x is
// not finite
template <typename T>
__device__ __forceinline__ void drop_block(Pack<T, 8>& v, i64 g, u32 threshold, float scale, u64 seed, u32 stream) {
  const Philox4 r = stream_block(seed, stream, (u64)g, 0);
  const u32 w[4] = {r.x, r.y, r.z, r.w};
  // threshold 65536 drops everything: its comparisons would wrap
  const u32 high = threshold < 65536u ? threshold << 16 : 0xFFFFFFFFu;
  const bool none = threshold >= 65536u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool keep_lo = (w[j] << 16) >= high && !none, keep_hi = w[j] >= high && !none;
    if constexpr (sizeof(T) == 2) {  // two elements a word
      u32* p = reinterpret_cast<u32*>(v.v) + j;
      *p = scale_pair(*p, scale, (const T*)nullptr) & ((keep_lo ? 0xFFFFu : 0u) | (keep_hi ? 0xFFFF0000u : 0u));
    } else {
      v.v[2 * j] = keep_lo ? v.v[2 * j] * scale : 0.f;
      v.v[2 * j + 1] = keep_hi ? v.v[2 * j + 1] * scale : 0.f;
    }
  }
}

// U blocks of eight a thread, all requested first; no grid-stride loop, whose last round leaves most of
// a launch of a few rounds idle.  The copy needs about 35 KB in flight an SM: 4 M x 100 bf16 in 319 us
// with U = 1, 267 with 2, 253 with 4 (6.3 TB/s); a small tensor has more CTAs with U = 1.
// y may be x: a thread loads all its elements before it stores the first, and nobody else touches them.
template <typename T, bool VECTOR, int U>
__global__ void __launch_bounds__(256)
dropout_kernel(const T* x, i64 n, u32 threshold, float scale, u64 seed, u32 stream, const i64* __restrict__ stream_dev, T* y) {
  const i64 g0 = (i64)blockIdx.x * (256 * U) + threadIdx.x;
  if (VECTOR && ((i64)blockIdx.x + 1) * (256 * U) * 8 <= n) {  // whole blocks only
    Pack<T, 8> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].load_written(x + (g0 + u * 256) * 8);
    if (stream_dev) stream += (u32)__ldg(stream_dev);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      drop_block(v[u], g0 + u * 256, threshold, scale, seed, stream);
      v[u].store(y + (g0 + u * 256) * 8);
    }
    return;
  }
  if (stream_dev) stream += (u32)__ldg(stream_dev);
  for (int u = 0; u < U; ++u) {
    const i64 g = g0 + u * 256, e = g * 8;
    if (e >= n) return;
    Pack<T, 8> v;
    const bool whole = VECTOR && e + 8 <= n;
    if (whole) {
      v.load_written(x + e);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v.v[j] = e + j < n ? x[e + j] : from_float<T>(0.f);
    }
    drop_block(v, g, threshold, scale, seed, stream);
    if (whole) {
      v.store(y + e);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (e + j < n) y[e + j] = v.v[j];
    }
  }
}

template <typename T, bool VECTOR, int U>
static void launch_dropout_u(const void* x, i64 n, u32 threshold, float scale, u64 seed, u32 stream, const i64* stream_dev,
                             void* y, cudaStream_t st) {
  const i64 blocks = ((n + 7) / 8 + 256 * U - 1) / (256 * U);
  LaunchScope ls(KID_DROPOUT, st);
  dropout_kernel<T, VECTOR, U><<<(unsigned)blocks, 256, 0, st>>>((const T*)x, n, threshold, scale, seed, stream, stream_dev, (T*)y);
}
template <typename T>
static void launch_dropout(const void* x, i64 n, u32 threshold, float scale, u64 seed, u32 stream, const i64* stream_dev, void* y,
                           cudaStream_t st) {
  if ((((uintptr_t)x | (uintptr_t)y) & 15) != 0) launch_dropout_u<T, false, 1>(x, n, threshold, scale, seed, stream, stream_dev, y, st);
  else if (n >= (i64)sm_count() * 8 * 8192) launch_dropout_u<T, true, 4>(x, n, threshold, scale, seed, stream, stream_dev, y, st);
  else launch_dropout_u<T, true, 1>(x, n, threshold, scale, seed, stream, stream_dev, y, st);
}

}  // namespace gsb

using namespace gsb;

extern "C" int gsb_dropout(const void* x, int dtype, int64_t n, double p, uint64_t seed, uint32_t stream,
                           const int64_t* stream_dev, void* y, void* cuda_stream) {
  if (n < 0 || n > (1ll << 40) || !(p >= 0.0 && p <= 1.0)) return GSB_ERR_INVALID;  // the grid's limit
  if (n == 0) return GSB_OK;
  if (!x || !y) return GSB_ERR_INVALID;
  if (!at_multiple(x, value_bytes(dtype)) || !at_multiple(y, value_bytes(dtype)) || !at_multiple(stream_dev, 8)) return GSB_ERR_INVALID;
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
