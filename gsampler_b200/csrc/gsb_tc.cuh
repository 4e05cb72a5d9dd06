// The instructions that the tensor-core kernels are written in: mbarriers with bounded waits, TMA
// loads, tcgen05 products and TMEM accesses, and the descriptors they take.
#pragma once
#include <cuda.h>

#include "gsb_common.cuh"
#include "gsb_types.cuh"

namespace gsb {

__device__ __forceinline__ u32 smem_addr(const void* p) { return (u32)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(u32 bar, u32 count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(u32 bar, u32 bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(u32 bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(u32 bar, u32 parity) {
  u32 ok;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.b32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Every wait ends: after two seconds, or once another warp of the CTA gave up, it reports and the
// kernel runs out without touching anything more.
static __device__ __noinline__ bool bar_wait_slow(u32 bar, u32 parity, volatile int* gave_up, int* err) {
  u64 t0;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
  for (;;) {
    for (int k = 0; k < 64; ++k)
      if (bar_try(bar, parity)) return true;
    u64 now;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
    if (*gave_up) return false;
    if (now - t0 > 2000000000ull) {
      *gave_up = 1;
      raise(err, ERRBIT_LOOKBACK_TIMEOUT);
      return false;
    }
  }
}
__device__ __forceinline__ bool bar_wait(u32 bar, u32 parity, volatile int* gave_up, int* err) {
  if (bar_try(bar, parity)) return true;
  return bar_wait_slow(bar, parity, gave_up, err);
}

__device__ __forceinline__ void tma_tile(u32 dst, const CUtensorMap* map, int x, int y, int plane, u32 bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(plane), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void bulk_copy(u32 dst, const void* src, u32 bytes, u32 bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tc_commit(u32 bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_mma(u32 d, u64 a, u64 b, u32 idesc, bool add) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a),
               "l"(b), "r"(idesc), "r"((u32)add)
               : "memory");
}
__device__ __forceinline__ void tc_mma_ta(u32 d, u32 a, u64 b, u32 idesc, bool add) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a),
               "l"(b), "r"(idesc), "r"((u32)add)
               : "memory");
}
// one lane of a warp that runs together: the products' descriptors then stay in uniform registers
__device__ __forceinline__ bool elect_one() {
  u32 ok;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}" : "=r"(ok));
  return ok != 0;
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define GSB_R4(a, i) "=f"(a[i]), "=f"(a[i + 1]), "=f"(a[i + 2]), "=f"(a[i + 3])
#define GSB_R16(a, i) GSB_R4(a, i), GSB_R4(a, i + 4), GSB_R4(a, i + 8), GSB_R4(a, i + 12)
__device__ __forceinline__ void tc_ld32(float* v, u32 addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : GSB_R16(v, 0), GSB_R16(v, 16)
      : "r"(addr));
}
__device__ __forceinline__ void tc_ld16(float* v, u32 addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : GSB_R16(v, 0)
      : "r"(addr));
}
#define GSB_U4(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3])
#define GSB_U16(a, i) GSB_U4(a, i), GSB_U4(a, i + 4), GSB_U4(a, i + 8), GSB_U4(a, i + 12)
__device__ __forceinline__ void tc_st16(u32 addr, const u32* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      GSB_U16(v, 0)
      : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle.  Along rows (K-major): 8-row groups 1024 bytes
// apart.  Across rows (MN-major): 64-element pieces `lead` bytes apart, 8-row groups 1024 bytes apart.
__device__ __forceinline__ u64 tc_desc(u32 addr, u32 lead) {
  return (u64)((addr & 0x3FFFF) >> 4) | ((u64)(lead >> 4) << 16) | ((u64)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor of kind::f16 with a 32-bit accumulator and M = 128; `across` operands are
// MN-major.
__device__ __forceinline__ u32 tc_idesc(bool bf16, u32 n, bool a_across, bool b_across) {
  const u32 t = bf16 ? 1 : 0;
  return (1u << 4) | (t << 7) | (t << 10) | ((a_across ? 1u : 0u) << 15) | ((b_across ? 1u : 0u) << 16) | ((n >> 3) << 17) |
         ((128u >> 4) << 24);
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// two 32-bit operations an instruction
__device__ __forceinline__ u64 join2(float lo, float hi) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void part2(u64 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 both(float v) { return join2(v, v); }
// 2^x of two values on the multiply-add pipe, for the share of them that would otherwise queue for
// the special-function unit (16 results a cycle and SM).  x = n + f with n the nearest integer, which
// the addition of 1.5 2^23 leaves in the low bits (127 more makes them an exponent field); 2^f by
// the polynomial of degree 5 that is nearest to it in relative error on [-1/2, 1/2] (weighted least
// squares on Chebyshev points; 1.5e-7 with its coefficients in 32 bits, 2.1e-7 with the roundings of its
// evaluation).  x below -126
// gives 2^-126; a NaN and an infinity give NaN.  x < 128.
__device__ __forceinline__ void ex2_poly(float& lo, float& hi) {
  const u64 x = join2(max_nan(lo, -126.f), max_nan(hi, -126.f));
  const u64 t = add2(x, both(12582912.f + 127.f));
  const u64 f = fma2(add2(t, both(-12582912.f - 127.f)), both(-1.f), x);
  u64 r = fma2(f, both(0.0013276472f), both(0.009675541f));
  r = fma2(r, f, both(0.05550713f));
  r = fma2(r, f, both(0.2402212f));
  r = fma2(r, f, both(0.69314694f));
  r = fma2(r, f, both(1.0000001f));
  float tl, th;
  part2(t, tl, th);
  part2(mul2(r, join2(__uint_as_float(__float_as_uint(tl) << 23), __uint_as_float(__float_as_uint(th) << 23))), lo, hi);
}
template <typename T>
__device__ __forceinline__ u32 pack2(float lo, float hi);
template <>
__device__ __forceinline__ u32 pack2<__half>(float lo, float hi) {
  u32 r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ u32 pack2<__nv_bfloat16>(float lo, float hi) {
  u32 r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// ---------------------------------------------------------------- tensor maps
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeFn tc_encode_fn() {
  static EncodeFn fn = []() -> EncodeFn {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    return (EncodeFn)f;
  }();
  return fn;
}

// Map of `planes` matrices of 16-bit elements [rows, cols], rows ld elements apart, planes behind one
// another; boxes of box_cols (128 bytes, the swizzle's width) x box_rows x 1, zeros outside.
inline bool tc_map(CUtensorMap* map, const void* p, bool bf16, i64 rows, i64 cols, i64 ld, int planes, int box_cols, int box_rows,
                   i64 plane_rows = 0) {
  EncodeFn fn = tc_encode_fn();
  if (!fn) return false;
  if (!plane_rows) plane_rows = rows;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)ld * 2 * plane_rows};
  const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1}, step[3] = {1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p), dims, strides,
            box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// what a map's base and row step have to satisfy
inline bool tma_ready(const void* p, i64 ld) { return ((uintptr_t)p & 15) == 0 && ld * 2 % 16 == 0; }
inline i64 packed_ld(i64 cols) { return (cols + 7) / 8 * 8; }

}  // namespace gsb
