// The vocabulary cross entropy of 16-bit types on the tensor cores (tcgen05, TMA, TMEM).
//
// Both passes are one shape of computation: a tile of 128 rows A stays in shared memory, tiles B of
// the other matrix stream past it, and for each
//     S = A B^T   ->   P = f(S)   ->   O += P B
// where one copy of the B tile in shared memory serves both products (read along its rows for S,
// across them for O).  S, P (16-bit, in the place of S) and O live in TMEM.
//   forward   A = rows of x, B = the vocabulary.  P = exp2(l - m) against a running reference m;
//             O / sum P is the expected row of W, which is all that dx needs; log2 sum P + m is
//             the log-sum-exp.  Without a gradient for x there is no second product.
//   dW        A = rows of W, B = rows of x.  P = g (p - target) with the known log-sum-exp.
// So training costs four products of N V D multiply-adds (the logits twice, dx, dW) and no array of
// N x V values exists anywhere.
//
// The reference m moves only when a row's maximum passes it by 2^8, because moving it rescales O;
// P stays below 2^15, which fp16 holds.  Sums and O are 32 bits; P is rounded to the type, half a
// step each, which is the rounding that the tensor cores' operands ask for.
#include <cuda.h>

#include "gsb_common.cuh"
#include "gsb_loss.cuh"
#include "gsb_types.cuh"

namespace gsb {

enum { TC_STATS = 0, TC_PULL = 1, TC_GRAD_W = 2 };

constexpr int FWD_SHIFT = 7;    // P is held at 2^7 times its value relative to the reference
constexpr int GRAD_SHIFT = 14;  // g (p - target) is held at 2^14 / max |g| times its value
constexpr float MOVE_REFERENCE = 8.f;

// ---------------------------------------------------------------- instructions
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
__device__ __noinline__ bool bar_wait_slow(u32 bar, u32 parity, volatile int* gave_up, int* err) {
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

__device__ __forceinline__ void tma_tile(u32 dst, const CUtensorMap* map, int x, int y, u32 bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(bar)
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
#define GSB_U4(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3])
#define GSB_U16(a, i) GSB_U4(a, i), GSB_U4(a, i + 4), GSB_U4(a, i + 8), GSB_U4(a, i + 12)
__device__ __forceinline__ void tc_st16(u32 addr, const u32* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      GSB_U16(v, 0)
      : "memory");
}
__device__ __forceinline__ void tc_st32(u32 addr, const u32* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      GSB_U16(v, 0), GSB_U16(v, 16)
      : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle.  Along rows (K-major): 8-row groups 1024 bytes
// apart.  Across rows (MN-major): 64-element pieces `lead` bytes apart, 8-row groups 1024 bytes apart.
__device__ __forceinline__ u64 tc_desc(u32 addr, u32 lead) {
  return (u64)((addr & 0x3FFFF) >> 4) | ((u64)(lead >> 4) << 16) | ((u64)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor of kind::f16 with a 32-bit accumulator and M = 128.
__device__ __forceinline__ u32 tc_idesc(bool bf16, u32 n, bool b_across) {
  const u32 t = bf16 ? 1 : 0;
  return (1u << 4) | (t << 7) | (t << 10) | ((b_across ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
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

// ---------------------------------------------------------------- shapes of the kernel
// DP    columns a row may have (64, 128, 256)
// NA    tiles A a CTA works on at once, WG  warpgroups that turn S into P
// NB    S buffers, BT  rows of a tile B, ST  stages of the B pipeline, CTAS  CTAs an SM
// An item is (tile B j, tile A a), numbered w = j NA + a; it uses buffer w % NB and warpgroup w % WG.
template <int MODE_, int DP_, int NA_, int WG_, int NB_, int BT_, int ST_, int CTAS_>
struct TcShape {
  static constexpr int MODE = MODE_, DP = DP_, NA = NA_, WG = WG_, NB = NB_, BT = BT_, ST = ST_, CTAS = CTAS_;
  static constexpr bool SECOND = MODE != TC_STATS;  // the product with P
  static constexpr int SUBS = DP / 64;
  static constexpr int A_BYTES = SUBS * 128 * 128, B_BYTES = SUBS * BT * 128;
  static constexpr int META = MODE == TC_GRAD_W ? BT * 14 : 0;
  static constexpr int O_COL = NB * BT;
  static constexpr int USED = O_COL + (SECOND ? NA * DP : 0);
  static constexpr int COLS = USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
  static constexpr int THREADS = WG * 128 + 64;
  static constexpr int OFF_B = NA * A_BYTES, OFF_META = OFF_B + ST * B_BYTES;
  static constexpr int OFF_BAR = (OFF_META + ST * META + 15) / 16 * 16;
  static constexpr int BARS = 2 * ST + 2 * NB + 3;
  static constexpr int BYTES = OFF_BAR + 8 * BARS + 16 + 1024;  // and room to align the base
  static_assert(USED <= 512 && COLS * CTAS <= 512, "TMEM");
  static_assert(BYTES * CTAS <= 227 * 1024, "shared memory");
  static_assert(WG % NA == 0 || NA % WG == 0, "a tile A keeps its warpgroup");
  static_assert(MODE != TC_PULL || WG == NA, "a row's running state has one owner");
};

struct TcParams {
  int rows_a, rows_b, D;
  int tiles_per_split;      // tiles B a CTA runs over
  float c;                  // |scale| log2 e
  const unsigned char* meta;  // TC_GRAD_W: BT * 14 bytes a tile B
  float2* part_ms;          // TC_STATS / TC_PULL: [parts][rows_a] reference and sum
  float* part_o;            // TC_PULL: [splits][rows_a][D]; TC_GRAD_W with splits: the same
  void* out;                // TC_GRAD_W without splits: [rows_a][D]
  const u32* top;           // TC_GRAD_W: bits of max |g|
  float out_scale;          // |scale| 2^-GRAD_SHIFT
  int* err;
};

template <typename T, typename C>
__global__ void __launch_bounds__(C::THREADS, C::CTAS)
loss_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const TcParams p) {
  extern __shared__ unsigned char smem_raw[];
  const u32 base = (smem_addr(smem_raw) + 1023) & ~1023u;
  unsigned char* smem = smem_raw + (base - smem_addr(smem_raw));
  const u32 bar0 = base + C::OFF_BAR;
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (C::ST + s); };
  auto s_full = [&](int b) { return bar0 + 8 * (2 * C::ST + b); };
  auto p_full = [&](int b) { return bar0 + 8 * (2 * C::ST + C::NB + b); };
  const u32 a_full = bar0 + 8 * (2 * C::ST + 2 * C::NB), o_full = a_full + 8, pv_done = a_full + 16;
  u32* tmem_slot = reinterpret_cast<u32*>(smem + C::OFF_BAR + 8 * C::BARS);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = blockIdx.x * (128 * C::NA);
  const int tiles = (p.rows_b + C::BT - 1) / C::BT;
  const int t0 = blockIdx.y * p.tiles_per_split;
  const int my_tiles = min(p.tiles_per_split, tiles - t0);
  const int items = my_tiles * C::NA;
  const int subs = (p.D + 63) / 64, ksteps = (p.D + 15) / 16;

  if (warp == C::WG * 4 && lane == 0) {
    for (int s = 0; s < C::ST; ++s) { bar_init(full(s), 1); bar_init(empty(s), 1); }
    for (int b = 0; b < C::NB; ++b) { bar_init(s_full(b), 1); bar_init(p_full(b), 4); }
    bar_init(a_full, 1);
    bar_init(o_full, 1);
    bar_init(pv_done, 1);
    *gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == C::WG * 4 + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"((u32)C::COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const u32 tmem = *tmem_slot;

  if (warp == C::WG * 4) {
    // ------------------------------------------------ loads
    if (lane == 0 && my_tiles > 0) {
      bar_expect(a_full, (u32)(C::NA * subs * 16384));
      for (int a = 0; a < C::NA; ++a)
        for (int s = 0; s < subs; ++s) tma_tile(base + a * C::A_BYTES + s * 16384, &map_a, s * 64, row0 + a * 128, a_full);
      int issued = 0;
      for (int j = 0; j < my_tiles; ++j) {
        const int st = j % C::ST;
        if (j >= C::ST && !bar_wait(empty(st), ((j / C::ST) - 1) & 1, gave_up, p.err)) break;
        bar_expect(full(st), (u32)(subs * C::BT * 128 + C::META));
        for (int s = 0; s < subs; ++s)
          tma_tile(base + C::OFF_B + st * C::B_BYTES + s * (C::BT * 128), &map_b, s * 64, (t0 + j) * C::BT, full(st));
        if (C::META) bulk_copy(base + C::OFF_META + st * C::META, p.meta + (i64)(t0 + j) * C::META, C::META, full(st));
        ++issued;
      }
      // no copy may be in flight when the CTA ends (only after a wait that gave up can one be)
      bar_wait(a_full, 0, gave_up, p.err);
      for (int j = issued > C::ST ? issued - C::ST : 0; j < issued; ++j)
        for (int k = 0; k < (1 << 16) && !bar_try(full(j % C::ST), (j / C::ST) & 1); ++k) __nanosleep(32);
    }
  } else if (warp == C::WG * 4 + 1) {
    // ------------------------------------------------ products
    if (lane == 0 && my_tiles > 0) {
      const bool bf = IsBf16<T>::value;
      const u32 id_s = tc_idesc(bf, C::BT, false), id_o = tc_idesc(bf, (u32)ksteps * 16, true);
      bool ok = bar_wait(a_full, 0, gave_up, p.err);
      auto product_s = [&](int w) {
        const int j = w / C::NA, a = w % C::NA, st = j % C::ST;
        if (a == 0 || C::NA == 1) ok = ok && bar_wait(full(st), (j / C::ST) & 1, gave_up, p.err);
        if (!ok) return;
        tc_after();
        const u32 A = base + a * C::A_BYTES, B = base + C::OFF_B + st * C::B_BYTES, d = tmem + (w % C::NB) * C::BT;
        for (int k = 0; k < ksteps; ++k)
          tc_mma(d, tc_desc(A + (k >> 2) * 16384 + (k & 3) * 32, 16), tc_desc(B + (k >> 2) * (C::BT * 128) + (k & 3) * 32, 16), id_s, k > 0);
        tc_commit(s_full(w % C::NB));
        if (!C::SECOND && a == C::NA - 1) tc_commit(empty(st));
      };
      for (int w = 0; w < C::NB && w < items; ++w) product_s(w);
      for (int w = 0; w < items && ok; ++w) {
        const int j = w / C::NA, a = w % C::NA, st = j % C::ST, b = w % C::NB;
        ok = bar_wait(p_full(b), (w / C::NB) & 1, gave_up, p.err);
        if (!ok) break;
        if (C::SECOND) {
          tc_after();
          const u32 B = base + C::OFF_B + st * C::B_BYTES, P = tmem + b * C::BT, d = tmem + C::O_COL + a * C::DP;
          for (int k = 0; k < C::BT / 16; ++k) tc_mma_ta(d, P + k * 8, tc_desc(B + k * 2048, C::BT * 128), id_o, j > 0 || k > 0);
          if (a == C::NA - 1) tc_commit(empty(st));
          if (C::MODE == TC_PULL && C::NA == 1 && C::NB > 1) tc_commit(pv_done);
        }
        if (w + C::NB < items) product_s(w + C::NB);
      }
      tc_commit(o_full);
      // the products that were issued end by themselves; a bounded look keeps the order when a wait gave up
      for (int k = 0; k < (1 << 16) && !bar_try(o_full, 0); ++k) __nanosleep(32);
    }
  } else {
    // ------------------------------------------------ S -> P
    const int wg = warp >> 2, quarter = warp & 3;
    const u32 lanes = (u32)(quarter * 32) << 16;
    const int a_mine = C::NA == 1 ? 0 : wg;
    const int row = row0 + a_mine * 128 + quarter * 32 + lane;
    const bool warp_live = row0 + a_mine * 128 + quarter * 32 < p.rows_a;
    float m = -INFINITY, sum = 0.f;
    bool ok = true;
    for (int w = wg; w < items; w += C::WG) {
      const int j = w / C::NA, st = j % C::ST, b = w % C::NB;
      ok = bar_wait(s_full(b), (w / C::NB) & 1, gave_up, p.err);
      if (C::META) ok = ok && bar_wait(full(st), (j / C::ST) & 1, gave_up, p.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_after();
      if (warp_live) {
        const u32 S = tmem + b * C::BT + lanes;
        float v[C::BT];
#pragma unroll
        for (int k = 0; k < C::BT; k += 32) tc_ld32(v + k, S + k);
        tc_wait_ld();
        if constexpr (C::MODE == TC_GRAD_W) {
          const unsigned char* meta = smem + C::OFF_META + st * C::META;
          const float4* bias = reinterpret_cast<const float4*>(meta);
#pragma unroll
          for (int k = 0; k < C::BT / 4; ++k) {
            const float4 q = bias[k];
            v[4 * k] = ex2(fmaf(v[4 * k], p.c, -q.x));
            v[4 * k + 1] = ex2(fmaf(v[4 * k + 1], p.c, -q.y));
            v[4 * k + 2] = ex2(fmaf(v[4 * k + 2], p.c, -q.z));
            v[4 * k + 3] = ex2(fmaf(v[4 * k + 3], p.c, -q.w));
          }
          const int* tgt = reinterpret_cast<const int*>(meta + 4 * C::BT);
          const float* gs = reinterpret_cast<const float*>(meta + 8 * C::BT);
          bool near = false;
#pragma unroll
          for (int k = 0; k < C::BT / 32; ++k) near |= (u32)(tgt[k * 32 + lane] - (row - lane)) < 32u;
          if (__any_sync(0xffffffffu, near)) {  // some row's target is one of this warp's vocabulary rows
#pragma unroll
            for (int k = 0; k < C::BT; ++k)
              if (tgt[k] == row) v[k] -= gs[k];
          }
        } else {
          const int col0 = (t0 + j) * C::BT;
          if (col0 + C::BT > p.rows_b) {
#pragma unroll
            for (int k = 0; k < C::BT; ++k)
              if (col0 + k >= p.rows_b) v[k] = -INFINITY;
          }
          float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int k = 4; k < C::BT; k += 4) {
#pragma unroll
            for (int q = 0; q < 4; ++q) top[q] = fmaxf(top[q], v[k + q]);
          }
          const float t = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.c;
          const bool move = t > m + MOVE_REFERENCE || (m == -INFINITY && t > m);
          if (__any_sync(0xffffffffu, move)) {
            const float f = move ? (m == -INFINITY ? 0.f : ex2(m - t)) : 1.f;
            sum *= f;
            if (move) m = t;
            if (C::MODE == TC_PULL && w >= C::WG) {
              // O was made against the old reference
              if (C::NA == 1 && C::NB > 1) {
                ok = bar_wait(pv_done, (w - 1) & 1, gave_up, p.err);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_after();
              }
              for (int k = 0; k < ksteps * 16; k += 32) {
                float o[32];
                const u32 at = tmem + C::O_COL + a_mine * C::DP + k + lanes;
                tc_ld32(o, at);
                tc_wait_ld();
#pragma unroll
                for (int q = 0; q < 32; ++q) o[q] *= f;
                tc_st32(at, reinterpret_cast<const u32*>(o));
              }
            }
          }
          const float off = (float)FWD_SHIFT - (m == -INFINITY ? 0.f : m);
          float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < C::BT; ++k) {
            v[k] = ex2(fmaf(v[k], p.c, off));
            add[k & 3] += v[k];
          }
          sum += (add[0] + add[1]) + (add[2] + add[3]);
        }
        if constexpr (C::SECOND) {
#pragma unroll
          for (int k = 0; k < C::BT; k += 32) {
            u32 h[16];
#pragma unroll
            for (int q = 0; q < 16; ++q) h[q] = pack2<T>(v[k + 2 * q], v[k + 2 * q + 1]);
            if constexpr (C::MODE == TC_GRAD_W) {
              // rows with a negative upstream gradient: the sign of their whole column
              const u32* sign = reinterpret_cast<const u32*>(smem + C::OFF_META + st * C::META + 12 * C::BT) + k / 2;
              const u32 own = sign[lane & 15];
              if (__any_sync(0xffffffffu, own != 0)) {
#pragma unroll
                for (int q = 0; q < 16; ++q) h[q] ^= sign[q];
              }
            }
            tc_st16(S + k / 2, h);
          }
          tc_wait_st();
        }
      }
      tc_before();
      __syncwarp();
      if (lane == 0) bar_arrive(p_full(b));
    }
    if (C::MODE != TC_GRAD_W && row < p.rows_a && ok) {
      const int part = blockIdx.y * (C::WG / C::NA) + (C::NA == 1 ? wg : 0);
      p.part_ms[(i64)part * p.rows_a + row] = make_float2(m, sum);
    }
    if (C::SECOND && my_tiles > 0) {
      ok = ok && bar_wait(o_full, 0, gave_up, p.err);
      ok = __all_sync(0xffffffffu, ok);
      if (ok && warp_live) {
        tc_after();
        const float f = C::MODE == TC_GRAD_W ? p.out_scale * __uint_as_float(*p.top) : 1.f;
        // with two warpgroups and one tile each takes half the columns
        const int step = C::WG > C::NA ? 64 : 32;
        for (int k = C::WG > C::NA ? wg * 32 : 0; k < p.D; k += step) {
          float o[32];
          tc_ld32(o, tmem + C::O_COL + a_mine * C::DP + k + lanes);
          tc_wait_ld();
          if (row < p.rows_a) {
            const bool slab = C::MODE == TC_PULL || gridDim.y > 1;
            if (slab) {
              float* to = p.part_o + ((i64)blockIdx.y * p.rows_a + row) * p.D + k;
              if ((p.D & 3) == 0) {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                  if (k + 4 * q < p.D) reinterpret_cast<float4*>(to)[q] = make_float4(o[4 * q] * f, o[4 * q + 1] * f, o[4 * q + 2] * f, o[4 * q + 3] * f);
              } else {
#pragma unroll
                for (int q = 0; q < 32; ++q)
                  if (k + q < p.D) to[q] = o[q] * f;
              }
            } else {
              T* to = (T*)p.out + (i64)row * p.D + k;
              if ((p.D & 7) == 0) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  if (k + 8 * q < p.D)
                    reinterpret_cast<uint4*>(to)[q] = make_uint4(pack2<T>(o[8 * q] * f, o[8 * q + 1] * f), pack2<T>(o[8 * q + 2] * f, o[8 * q + 3] * f),
                                                                 pack2<T>(o[8 * q + 4] * f, o[8 * q + 5] * f), pack2<T>(o[8 * q + 6] * f, o[8 * q + 7] * f));
              } else {
#pragma unroll
                for (int q = 0; q < 32; ++q)
                  if (k + q < p.D) to[q] = from_float<T>(o[q] * f);
              }
            }
          }
        }
      }
    }
    tc_before();
  }
  __syncwarp();
  __syncthreads();
  tc_after();
  if (warp == C::WG * 4 + 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((u32)C::COLS) : "memory");
}

// ---------------------------------------------------------------- preparation and joins
// dst[r, :] = +-src[r, :] with rows of ldp elements (16-byte multiples, zeros behind D); rows whose
// g is zero become zeros, so that nothing they hold reaches a product.
template <typename T>
__global__ void loss_pack_kernel(const T* __restrict__ src, i64 ld, i64 rows, int D, int ldp, bool negate,
                                 const float* __restrict__ g, T* __restrict__ dst) {
  const int chunks = ldp / 8;
  const i64 total = rows * chunks;
  for (i64 e = (i64)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (i64)gridDim.x * blockDim.x) {
    const i64 r = e / chunks;
    const int c = (int)(e - r * chunks) * 8;
    const bool live = !g || g[r] != 0.f;
    Pack<T, 8> v;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      v.v[q] = from_float<T>(0.f);
      if (live && c + q < D) {
        v.v[q] = src[r * ld + c + q];
        if (negate) v.v[q] = -v.v[q];
      }
    }
    v.store(dst + r * ldp + c);
  }
}

// What the dW pass needs of every row of x, by tiles of BT rows: bias (p g = exp2(l - bias)), target,
// |g| as P holds it, and the sign as a mask of the packed element.  Rows that do not count, and the
// rows behind the last, have an infinite bias: P = 0.
__global__ void loss_meta_kernel(const float* __restrict__ lse2, const i64* __restrict__ target, const float* __restrict__ g,
                                 const u32* __restrict__ top, i64 N, i64 Npad, int BT, unsigned char* __restrict__ meta) {
  const i64 r = (i64)blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= Npad) return;
  unsigned char* tile = meta + r / BT * (BT * 14);
  const int k = (int)(r % BT);
  float bias = INFINITY, gs = 0.f;
  int t = -1;
  u32 sign = 0;
  if (r < N && g[r] != 0.f) {
    const float rel = fabsf(g[r]) / __uint_as_float(*top);
    gs = rel * (float)(1 << GRAD_SHIFT);
    bias = lse2[r] - log2f(rel) - (float)GRAD_SHIFT;
    t = (int)target[r];
    sign = g[r] < 0.f ? 0x8000u : 0u;
  }
  reinterpret_cast<float*>(tile)[k] = bias;
  reinterpret_cast<int*>(tile + 4 * BT)[k] = t;
  reinterpret_cast<float*>(tile + 8 * BT)[k] = gs;
  reinterpret_cast<unsigned short*>(tile + 12 * BT)[k] = (unsigned short)sign;
}

// A warp per row: joins the parts' statistics (and pulls), adds the target's logit.
//   pull_i = sum_j p_ij w_j - w_{t_i}      (zeros for a row that does not count)
template <typename T>
__global__ void __launch_bounds__(256)
loss_join_kernel(const float2* __restrict__ part, int parts, const float* __restrict__ part_o, const T* __restrict__ x, i64 ldx,
                 i64 N, const T* __restrict__ w, i64 ldw, i64 V, int D, float scale, const i64* __restrict__ target, i64 ignore,
                 float* __restrict__ loss, float* __restrict__ lse2, float* __restrict__ pull, int* err) {
  const i64 r = ((i64)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (r >= N) return;
  float m = -INFINITY;
  for (int k = lane; k < parts; k += 32) m = max_nan(m, part[(i64)k * N + r].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
  float s = 0.f;
  for (int k = lane; k < parts; k += 32) {
    const float2 q = part[(i64)k * N + r];
    // a part without a reference has either no finite logit (sum 0) or a NaN
    s += q.x == -INFINITY ? q.y : q.y * exp2f(q.x - m);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  const float total = m - (float)FWD_SHIFT + log2f(s);
  const i64 t = target[r];
  const bool counts = t != ignore && t >= 0 && t < V;
  if (t != ignore && !counts && lane == 0) raise(err, ERRBIT_BAD_INPUT);
  float dot = 0.f;
  if (counts)
    for (int d = lane; d < D; d += 32) dot = fmaf(to_float(x[r * ldx + d]), to_float(w[t * ldw + d]), dot);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
  if (lane == 0) {
    lse2[r] = total;
    loss[r] = counts ? total * 0.6931471805599453f - dot * scale : 0.f;
  }
  if (pull) {
    const float inv = 1.f / s;
    for (int d = lane; d < D; d += 32) {
      float v = 0.f;
      if (counts) {
        for (int k = 0; k < parts; ++k) {
          const float mk = part[(i64)k * N + r].x;
          v += part_o[((i64)k * N + r) * D + d] * (mk == -INFINITY ? 1.f : exp2f(mk - m));
        }
        v = v * inv - to_float(w[t * ldw + d]);
      }
      pull[r * D + d] = v;
    }
  }
}

template <typename T>
__global__ void loss_dx_kernel(const float* __restrict__ pull, const float* __restrict__ g, float scale, i64 N, int D,
                               T* __restrict__ dx) {
  for (i64 e = (i64)blockIdx.x * blockDim.x + threadIdx.x; e < N * D; e += (i64)gridDim.x * blockDim.x) {
    const float gi = g[e / D];
    dx[e] = from_float<T>(gi == 0.f ? 0.f : pull[e] * (gi * scale));
  }
}

template <typename T>
__global__ void loss_join_dw_kernel(const float* __restrict__ slab, i64 size, int slabs, T* __restrict__ out) {
  for (i64 e = (i64)blockIdx.x * blockDim.x + threadIdx.x; e < size; e += (i64)gridDim.x * blockDim.x) {
    float v = 0.f;
    for (int z = 0; z < slabs; ++z) v += slab[z * size + e];
    out[e] = from_float<T>(v);
  }
}

// ---------------------------------------------------------------- host side
static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
static int blocks_for(i64 threads) {
  const i64 b = (threads + 255) / 256, most = (i64)sm_count() * 16;
  return (int)(b < 1 ? 1 : b < most ? b : most);
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
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

static bool make_map(CUtensorMap* map, const void* p, bool bf16, i64 rows, i64 D, i64 ld, int box_rows) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, step[2] = {1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(p), dims, strides,
            box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static bool tma_ready(const void* p, i64 ld) { return ((uintptr_t)p & 15) == 0 && ld * 2 % 16 == 0; }
static i64 packed_ld(i64 D) { return (D + 7) / 8 * 8; }

// Tiles B a CTA runs over.  `groups` CTAs cover the rows A; the tiles are split until the CTAs fill
// the SMs' `slots` evenly: the time is (rounds of CTAs) x (tiles of one + about 3 for its start and end).
static int split_count(i64 groups, i64 tiles, i64 slots) {
  int best = 1;
  double best_t = 1e300;
  for (i64 s = 1; s <= tiles && s <= 2 * slots && (s == 1 || groups * s <= 3 * slots); ++s) {
    const i64 per = (tiles + s - 1) / s;
    if ((tiles + per - 1) / per != s) continue;  // the same as fewer splits
    const double t = (double)((groups * s + slots - 1) / slots) * (double)(per + 3);
    if (t < best_t * 0.999) { best_t = t; best = (int)s; }
  }
  return best;
}

struct TcPlan {
  int NA, BT, ctas, splits, per, parts;
  i64 groups;
};
// Few rows on the streaming side's partner make the pass a stream of B (forward, N <= 128) or of A (dW, N <= 256):
// then two small CTAs an SM overlap one's loads with the other's products.  Otherwise one large CTA.
template <typename C>
static TcPlan plan_of(i64 rows_a, i64 rows_b) {
  TcPlan p;
  if (rows_a < 1) rows_a = 1;  // sizes are asked for empty batches too
  if (rows_b < 1) rows_b = 1;
  p.NA = C::NA;
  p.BT = C::BT;
  p.ctas = C::CTAS;
  p.groups = (rows_a + 128 * C::NA - 1) / (128 * C::NA);
  const i64 tiles = (rows_b + C::BT - 1) / C::BT;
  const int s = split_count(p.groups, tiles, (i64)sm_count() * C::CTAS);
  p.per = (int)((tiles + s - 1) / s);
  p.splits = (int)((tiles + p.per - 1) / p.per);
  p.parts = p.splits * (C::MODE == TC_GRAD_W ? 1 : C::WG / C::NA);
  return p;
}

//                     MODE      DP  NA WG NB  BT ST CTAS
typedef TcShape<TC_STATS, 64, 2, 2, 4, 128, 6, 1> Stats64;
typedef TcShape<TC_STATS, 128, 2, 2, 4, 128, 4, 1> Stats128;
typedef TcShape<TC_STATS, 256, 1, 2, 4, 128, 2, 1> Stats256;
typedef TcShape<TC_STATS, 64, 1, 1, 2, 128, 4, 2> StatsFew64;
typedef TcShape<TC_STATS, 128, 1, 1, 2, 128, 2, 2> StatsFew128;
typedef TcShape<TC_PULL, 64, 2, 2, 2, 128, 6, 1> Pull64;
typedef TcShape<TC_PULL, 128, 2, 2, 2, 128, 4, 1> Pull128;
typedef TcShape<TC_PULL, 256, 1, 1, 2, 64, 4, 1> Pull256;
typedef TcShape<TC_PULL, 64, 1, 1, 1, 128, 4, 2> PullFew64;
typedef TcShape<TC_PULL, 128, 1, 1, 1, 128, 2, 2> PullFew128;
typedef TcShape<TC_GRAD_W, 64, 2, 2, 2, 128, 6, 1> Grad64;
typedef TcShape<TC_GRAD_W, 128, 2, 2, 2, 128, 4, 1> Grad128;
typedef TcShape<TC_GRAD_W, 256, 1, 2, 2, 64, 4, 1> Grad256;
typedef TcShape<TC_GRAD_W, 64, 1, 1, 1, 128, 4, 2> GradFew64;
typedef TcShape<TC_GRAD_W, 128, 1, 1, 1, 128, 2, 2> GradFew128;

// f(shape) for the shape that the sizes ask for
template <typename F>
static auto with_shape(int mode, i64 N, i64 D, F f) {
  if (mode == TC_STATS) {
    if (D > 128) return f(Stats256());
    if (N <= 128) return D > 64 ? f(StatsFew128()) : f(StatsFew64());
    return D > 64 ? f(Stats128()) : f(Stats64());
  }
  if (mode == TC_PULL) {
    if (D > 128) return f(Pull256());
    if (N <= 128) return D > 64 ? f(PullFew128()) : f(PullFew64());
    return D > 64 ? f(Pull128()) : f(Pull64());
  }
  if (D > 128) return f(Grad256());
  if (N <= 256) return D > 64 ? f(GradFew128()) : f(GradFew64());
  return D > 64 ? f(Grad128()) : f(Grad64());
}

static TcPlan tc_plan(int mode, i64 N, i64 V, i64 D) {
  return with_shape(mode, N, D, [&](auto shape) {
    return mode == TC_GRAD_W ? plan_of<decltype(shape)>(V, N) : plan_of<decltype(shape)>(N, V);
  });
}

bool tc_loss_takes(int dtype, i64 N, i64 V, i64 D) {
  // tile counts and coordinates stay in 31 bits, and the grid in its limits
  return dtype != GSB_F32 && D <= 256 && N < (1ll << 30) && V < (1ll << 30);
}

struct TcFwdLayout { size_t ms, o, x, w, bytes; };
static TcFwdLayout fwd_layout(i64 N, i64 V, i64 D, bool pull) {
  TcFwdLayout L;
  size_t o = 0;
  auto take = [&](size_t b) { const size_t at = o; o += up256(b); return at; };
  const TcPlan p = tc_plan(pull ? TC_PULL : TC_STATS, N, V, D);
  L.ms = take(8 * (size_t)p.parts * N);
  L.o = take(pull ? 4 * (size_t)p.splits * N * D : 0);
  L.x = take(2 * (size_t)N * packed_ld(D));
  // whether the rows of W have to be copied depends on its address and row step
  L.w = take(2 * (size_t)V * packed_ld(D));
  L.bytes = o;
  return L;
}
size_t tc_loss_workspace(i64 N, i64 V, i64 D, bool pull, bool pack_w) {
  const TcFwdLayout L = fwd_layout(N, V, D, pull);
  return pack_w ? L.bytes : L.w;
}

struct TcGradLayout { size_t meta, x, slab, w, bytes; };
static TcGradLayout grad_layout(i64 N, i64 V, i64 D) {
  TcGradLayout L;
  size_t o = 0;
  auto take = [&](size_t b) { const size_t at = o; o += up256(b); return at; };
  const TcPlan p = tc_plan(TC_GRAD_W, N, V, D);
  L.meta = take((size_t)((N + p.BT - 1) / p.BT) * p.BT * 14);
  L.x = take(2 * (size_t)N * packed_ld(D));
  L.slab = take(p.splits > 1 ? 4 * (size_t)p.splits * V * D : 0);
  L.w = take(2 * (size_t)V * packed_ld(D));
  L.bytes = o;
  return L;
}
size_t tc_loss_grad_workspace(i64 N, i64 V, i64 D, bool pack_w) {
  const TcGradLayout L = grad_layout(N, V, D);
  return pack_w ? L.bytes : L.w;
}
bool tc_loss_packs(const void* w, i64 ldw) { return !tma_ready(w, ldw); }

template <typename T>
static const T* pack_rows(const void* src, i64 ld, i64 rows, i64 D, bool negate, const float* g, void* dst, cudaStream_t st) {
  LaunchScope ls(KID_LOSS_JOIN, st);
  loss_pack_kernel<T><<<blocks_for(rows * packed_ld(D) / 8), 256, 0, st>>>((const T*)src, ld, rows, (int)D, (int)packed_ld(D), negate, g,
                                                                          (T*)dst);
  return (const T*)dst;
}

template <typename T, typename C>
static int launch_tc(const CUtensorMap& a, const CUtensorMap& b, const TcPlan& plan, const TcParams& p, int kid, cudaStream_t st) {
  // the attribute belongs to the device's copy of the kernel; setting it is cheap and not a stream operation
  GSB_CUDA_OK(cudaFuncSetAttribute(loss_tc_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::BYTES));
  LaunchScope ls(kid, st);
  loss_tc_kernel<T, C><<<dim3((unsigned)plan.groups, (unsigned)plan.splits), C::THREADS, C::BYTES, st>>>(a, b, p);
  return GSB_OK;
}

// not zero, so that a masked logit of -inf stays one; times any finite product it is as good as zero
static float logit_factor(float scale) { return fmaxf(fabsf(scale) * LOG2E, 1e-38f); }

template <typename T>
int tc_loss_forward(const LossArgs& a, float* pull) {
  const int mode = pull ? TC_PULL : TC_STATS;
  const TcPlan plan = tc_plan(mode, a.N, a.V, a.D);
  const TcFwdLayout L = fwd_layout(a.N, a.V, a.D, pull != nullptr);
  char* ws = (char*)a.ws;
  // l = |scale| (+-x) . w: the running maximum needs a factor that is not negative
  const bool negate = a.scale < 0.f;
  const T* x = (const T*)a.x;
  const T* w = (const T*)a.w;
  i64 ldx = a.ldx, ldw = a.ldw;
  if (negate || !tma_ready(x, ldx)) { x = pack_rows<T>(x, ldx, a.N, a.D, negate, nullptr, ws + L.x, a.st); ldx = packed_ld(a.D); }
  if (!tma_ready(w, ldw)) { w = pack_rows<T>(w, ldw, a.V, a.D, false, nullptr, ws + L.w, a.st); ldw = packed_ld(a.D); }
  CUtensorMap ma, mb;
  if (!make_map(&ma, x, IsBf16<T>::value, a.N, a.D, ldx, 128) || !make_map(&mb, w, IsBf16<T>::value, a.V, a.D, ldw, plan.BT)) return GSB_ERR_CUDA;
  TcParams p = {};
  p.rows_a = (int)a.N;
  p.rows_b = (int)a.V;
  p.D = (int)a.D;
  p.tiles_per_split = plan.per;
  p.c = logit_factor(a.scale);
  p.part_ms = (float2*)(ws + L.ms);
  p.part_o = (float*)(ws + L.o);
  p.err = a.err;
  const int rc = with_shape(mode, a.N, a.D, [&](auto shape) { return launch_tc<T, decltype(shape)>(ma, mb, plan, p, KID_LOSS, a.st); });
  if (rc != GSB_OK) return rc;
  LaunchScope ls(KID_LOSS_JOIN, a.st);
  loss_join_kernel<T><<<ceil_div_i(a.N, 8), 256, 0, a.st>>>(p.part_ms, plan.parts, p.part_o, (const T*)a.x, a.ldx, a.N, (const T*)a.w, a.ldw,
                                                            a.V, (int)a.D, a.scale, a.target, a.ignore, a.loss, a.lse2, pull, a.err);
  return GSB_OK;
}

template <typename T>
int tc_loss_grad_w(const LossArgs& a) {
  const TcPlan plan = tc_plan(TC_GRAD_W, a.N, a.V, a.D);
  const TcGradLayout L = grad_layout(a.N, a.V, a.D);
  char* ws = (char*)a.ws;
  const T* x = pack_rows<T>(a.x, a.ldx, a.N, a.D, a.scale < 0.f, a.g, ws + L.x, a.st);
  const T* w = (const T*)a.w;
  i64 ldw = a.ldw;
  if (!tma_ready(w, ldw)) { w = pack_rows<T>(w, ldw, a.V, a.D, false, nullptr, ws + L.w, a.st); ldw = packed_ld(a.D); }
  {
    const i64 npad = (a.N + plan.BT - 1) / plan.BT * plan.BT;
    LaunchScope ls(KID_LOSS_JOIN, a.st);
    loss_meta_kernel<<<ceil_div_i(npad, 256), 256, 0, a.st>>>(a.lse2, a.target, a.g, a.top, a.N, npad, plan.BT, (unsigned char*)(ws + L.meta));
  }
  CUtensorMap ma, mb;
  if (!make_map(&ma, w, IsBf16<T>::value, a.V, a.D, ldw, 128) || !make_map(&mb, x, IsBf16<T>::value, a.N, a.D, packed_ld(a.D), plan.BT))
    return GSB_ERR_CUDA;
  TcParams p = {};
  p.rows_a = (int)a.V;
  p.rows_b = (int)a.N;
  p.D = (int)a.D;
  p.tiles_per_split = plan.per;
  p.c = logit_factor(a.scale);
  p.meta = (const unsigned char*)(ws + L.meta);
  p.part_o = (float*)(ws + L.slab);
  p.out = a.dw;
  p.top = a.top;
  p.out_scale = fabsf(a.scale) / (float)(1 << GRAD_SHIFT);
  p.err = a.err;
  const int rc = with_shape(TC_GRAD_W, a.N, a.D, [&](auto shape) { return launch_tc<T, decltype(shape)>(ma, mb, plan, p, KID_LOSS_GRAD, a.st); });
  if (rc != GSB_OK) return rc;
  if (plan.splits > 1) {
    LaunchScope ls(KID_LOSS_JOIN, a.st);
    loss_join_dw_kernel<T><<<blocks_for(a.V * a.D), 256, 0, a.st>>>(p.part_o, a.V * a.D, plan.splits, (T*)a.dw);
  }
  return GSB_OK;
}

template <typename T>
void tc_loss_dx(const LossArgs& a, const float* pull) {
  LaunchScope ls(KID_LOSS_JOIN, a.st);
  loss_dx_kernel<T><<<blocks_for(a.N * a.D), 256, 0, a.st>>>(pull, a.g, a.scale, a.N, (int)a.D, (T*)a.dx);
}

template int tc_loss_forward<__half>(const LossArgs&, float*);
template int tc_loss_forward<__nv_bfloat16>(const LossArgs&, float*);
template int tc_loss_grad_w<__half>(const LossArgs&);
template int tc_loss_grad_w<__nv_bfloat16>(const LossArgs&);
template void tc_loss_dx<__half>(const LossArgs&, const float*);
template void tc_loss_dx<__nv_bfloat16>(const LossArgs&, const float*);

}  // namespace gsb
