// The vocabulary cross entropy of 16-bit types on the tensor cores (tcgen05, TMA, TMEM).
//
// Both passes are one shape of computation: a tile of 128 rows A stays in TMEM, tiles B of the other
// matrix stream past it, and for each
//     S = A B^T   ->   P = f(S)   ->   O += P B
// where one copy of the B tile in shared memory serves both products (read along its rows for S,
// across them for O).  S, P (16-bit, in the place of S) and O live in TMEM too.  A there, and not in
// shared memory, halves what a product reads from shared memory: S alone ran at 984 TFLOP/s with
// both operands in shared memory (128 x 128 tiles, 8192 x 300000 x 128), the second product, whose
// first operand was in TMEM already, at 2000.
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
#include "gsb_common.cuh"
#include "gsb_loss.cuh"
#include "gsb_tc.cuh"
#include "gsb_types.cuh"

namespace gsb {

enum { TC_STATS = 0, TC_PULL = 1, TC_GRAD_W = 2 };

// ---------------------------------------------------------------- shapes of the kernel
// DP    columns a row may have (64, 128, 256)
// NA    tiles A a CTA works on at once
// NB    S buffers, BT  rows of a tile B, ST  stages of the B pipeline, CTAS  CTAs an SM
// HV    warpgroups that turn an item's S into P, each an equal share of its columns
// ATM   tiles A in TMEM, where there is room beside O and two S buffers; else in shared memory
// An item is (tile B j, tile A a), numbered w = j NA + a; it uses buffer w % NB.
template <int MODE_, int DP_, int NA_, int NB_, int BT_, int ST_, int CTAS_, int HV_, bool ATM_>
struct TcShape {
  static constexpr int MODE = MODE_, DP = DP_, NA = NA_, NB = NB_, BT = BT_, ST = ST_, CTAS = CTAS_;
  static constexpr int HV = HV_;
  static constexpr int POLY = MODE == TC_STATS ? 8 : 0;
  static constexpr bool ATM = ATM_;  // tiles A in TMEM, else in shared memory
  static constexpr bool SECOND = MODE != TC_STATS;  // the product with P
  static constexpr int WG = NA * HV, HC = BT / HV;
  static constexpr int SUBS = DP / 64;
  static constexpr int B_BYTES = SUBS * BT * 128;
  static constexpr int META = MODE == TC_GRAD_W ? BT * 14 : 0;
  static constexpr int A_COL = NB * BT, O_COL = A_COL + (ATM ? NA * (DP / 2) : 0);
  static constexpr int USED = O_COL + (SECOND ? NA * DP : 0);
  static constexpr int COLS = USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
  static constexpr int THREADS = WG * 128 + 64;
  static constexpr int A_BYTES = ATM ? 0 : SUBS * 128 * 128;
  static constexpr int OFF_B = NA * A_BYTES, OFF_META = OFF_B + ST * B_BYTES;
  static constexpr int OFF_BAR = OFF_META + ST * META;
  static constexpr int BARS = 2 * ST + 2 * NB + 3;
  static constexpr int BYTES = OFF_BAR + 8 * BARS + 16 + 1024;  // and room to align the base
  static_assert(USED <= 512 && COLS * CTAS <= 512, "TMEM");
  static_assert(BYTES * CTAS <= 226 * 1024, "shared memory");
  static_assert(MODE != TC_PULL || HV == 1, "a row's running state has one owner");
  static_assert(HC % 32 == 0 && META % 16 == 0 && OFF_BAR % 8 == 0, "");
};

struct TcParams {
  const void* a;            // rows of lda elements, 16-byte aligned
  i64 lda;
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
loss_tc_kernel(const __grid_constant__ CUtensorMap map_b, const TcParams p) {
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
    for (int b = 0; b < C::NB; ++b) { bar_init(s_full(b), 1); bar_init(p_full(b), 4 * C::HV); }
    bar_init(a_full, 4 * C::WG);
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
  const u32 tmem = __reduce_max_sync(0xffffffffu, *tmem_slot);  // the same in every lane, and known to be

  if (warp == C::WG * 4) {
    // ------------------------------------------------ loads
    if (lane == 0 && my_tiles > 0) {
      int issued = 0;
      for (int j = 0; j < my_tiles; ++j) {
        const int st = j % C::ST;
        if (j >= C::ST && !bar_wait(empty(st), ((j / C::ST) - 1) & 1, gave_up, p.err)) break;
        bar_expect(full(st), (u32)(subs * C::BT * 128 + C::META));
        for (int s = 0; s < subs; ++s)
          tma_tile(base + C::OFF_B + st * C::B_BYTES + s * (C::BT * 128), &map_b, s * 64, (t0 + j) * C::BT, 0, full(st));
        if (C::META) bulk_copy(base + C::OFF_META + st * C::META, p.meta + (i64)(t0 + j) * C::META, C::META, full(st));
        ++issued;
      }
      // no copy may be in flight when the CTA ends (only after a wait that gave up can one be)
      for (int j = issued > C::ST ? issued - C::ST : 0; j < issued; ++j)
        for (int k = 0; k < (1 << 16) && !bar_try(full(j % C::ST), (j / C::ST) & 1); ++k) __nanosleep(32);
    }
  } else if (warp == C::WG * 4 + 1) {
    // ------------------------------------------------ products
    // The whole warp walks the items and one lane issues: unrolled, with descriptors that differ by
    // constants.  A product of 128 x 128 x 16 takes 64 cycles; issued from a divergent lane with its
    // descriptors made one by one it took 130.
    if (my_tiles > 0) {
      const bool bf = IsBf16<T>::value;
      const u32 id_s = tc_idesc(bf, C::BT, false, false), id_o = tc_idesc(bf, (u32)ksteps * 16, false, true);
      const bool leader = elect_one();
      bool ok = bar_wait(a_full, 0, gave_up, p.err);
      tc_after();
      auto product_s = [&](int w) {
        const int j = w / C::NA, a = w % C::NA, st = j % C::ST;
        if (a == 0) ok = ok && bar_wait(full(st), (j / C::ST) & 1, gave_up, p.err);
        if (!ok) return;
        tc_after();
        const u32 A = tmem + C::A_COL + a * (C::DP / 2), d = tmem + (w % C::NB) * C::BT;
        const u64 B = tc_desc(base + C::OFF_B + st * C::B_BYTES, 16), As = tc_desc(base + a * C::A_BYTES, 16);
        if (leader) {
#pragma unroll
          for (int k = 0; k < C::DP / 16; ++k)
            if (k < ksteps && C::ATM) tc_mma_ta(d, A + k * 8, B + ((k >> 2) * (C::BT * 128) + (k & 3) * 32) / 16, id_s, k > 0);
            else if (k < ksteps) tc_mma(d, As + ((k >> 2) * 16384 + (k & 3) * 32) / 16, B + ((k >> 2) * (C::BT * 128) + (k & 3) * 32) / 16, id_s, k > 0);
          tc_commit(s_full(w % C::NB));
          if (!C::SECOND && a == C::NA - 1) tc_commit(empty(st));
        }
      };
      for (int w = 0; w < C::NB && w < items; ++w) product_s(w);
      for (int w = 0; w < items && ok; ++w) {
        const int j = w / C::NA, a = w % C::NA, st = j % C::ST, b = w % C::NB;
        ok = bar_wait(p_full(b), (w / C::NB) & 1, gave_up, p.err);
        if (!ok) break;
        if (C::SECOND) {
          tc_after();
          const u32 P = tmem + b * C::BT, d = tmem + C::O_COL + a * C::DP;
          const u64 B = tc_desc(base + C::OFF_B + st * C::B_BYTES, C::BT * 128);
          if (leader) {
#pragma unroll
            for (int k = 0; k < C::BT / 16; ++k)
              tc_mma_ta(d, P + (k / (C::HC / 16)) * C::HC + (k % (C::HC / 16)) * 8, B + k * (2048 / 16), id_o, j > 0 || k > 0);
            if (a == C::NA - 1) tc_commit(empty(st));
            if (C::MODE == TC_PULL && C::NA == 1 && C::NB > 1) tc_commit(pv_done);
          }
        }
        if (w + C::NB < items) product_s(w + C::NB);
      }
      if (leader) tc_commit(o_full);
      // the products that were issued end by themselves; a bounded look keeps the order when a wait gave up
      for (int k = 0; k < (1 << 16) && !bar_try(o_full, 0); ++k) __nanosleep(32);
    }
  } else {
    // ------------------------------------------------ S -> P
    const int wg = warp >> 2, quarter = warp & 3, a = wg / C::HV, half = wg % C::HV;
    const u32 lanes = (u32)(quarter * 32) << 16;
    const int row = row0 + a * 128 + quarter * 32 + lane;
    const bool warp_live = row0 + a * 128 + quarter * 32 < p.rows_a;
    // the rows of A into TMEM: a thread its row, pairs of elements a column; zeros behind the last
    // column (nothing there may meet the zeros of B as a NaN) and row
    for (int k = half * 32; k < ksteps * 16; k += 32 * C::HV) {
      const T* from = (const T*)p.a + (i64)row * p.lda + k;
      Pack<T, 32> piece;
#pragma unroll
      for (int q = 0; q < 32; q += 8) {
        if (row < p.rows_a && k + q + 8 <= p.D) {
          reinterpret_cast<Pack<T, 8>*>(piece.v + q)->load(from + q);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) piece.v[q + e] = row < p.rows_a && k + q + e < p.D ? from[q + e] : from_float<T>(0.f);
        }
      }
      if constexpr (C::ATM) {
        tc_st16(tmem + C::A_COL + a * (C::DP / 2) + k / 2 + lanes, reinterpret_cast<const u32*>(piece.v));
      } else {  // as a swizzled tile: 16-byte piece c of row r lies at c ^ (r & 7)
        const int r = quarter * 32 + lane;
        unsigned char* to = smem + a * C::A_BYTES + (k >> 6) * 16384 + r * 128;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<uint4*>(to + ((((k & 63) >> 3) + q) ^ (r & 7)) * 16) = reinterpret_cast<const uint4*>(piece.v)[q];
      }
    }
    if (C::ATM) tc_wait_st();
    else asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_before();
    __syncwarp();
    if (lane == 0) bar_arrive(a_full);
    // one pair in POLY by the polynomial
    auto exponentials = [](float& lo, float& hi, int k) {
      if (C::POLY && (k / 2) % (C::POLY ? C::POLY : 1) == C::POLY - 1) {
        ex2_poly(lo, hi);
      } else {
        lo = ex2(lo);
        hi = ex2(hi);
      }
    };
    float m = -INFINITY, sum = 0.f;
    const u64 c2 = join2(p.c, p.c);
    bool ok = true;
    for (int w = a; w < items; w += C::NA) {
      const int j = w / C::NA, st = j % C::ST, b = w % C::NB;
      ok = bar_wait(s_full(b), (w / C::NB) & 1, gave_up, p.err);
      if (C::META) ok = ok && bar_wait(full(st), (j / C::ST) & 1, gave_up, p.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_after();
      if (warp_live) {
        const u32 S = tmem + b * C::BT + half * C::HC + lanes;
        float v[C::HC];
#pragma unroll
        for (int k = 0; k < C::HC; k += 32) tc_ld32(v + k, S + k);
        tc_wait_ld();
        if constexpr (C::MODE == TC_GRAD_W) {
          const unsigned char* meta = smem + C::OFF_META + st * C::META + half * C::HC * 4;
          const ulonglong2* bias = reinterpret_cast<const ulonglong2*>(meta);  // negative
#pragma unroll
          for (int k = 0; k < C::HC / 4; ++k) {
            const ulonglong2 q = bias[k];
            part2(fma2(join2(v[4 * k], v[4 * k + 1]), c2, q.x), v[4 * k], v[4 * k + 1]);
            part2(fma2(join2(v[4 * k + 2], v[4 * k + 3]), c2, q.y), v[4 * k + 2], v[4 * k + 3]);
          }
#pragma unroll
          for (int k = 0; k < C::HC; k += 2) exponentials(v[k], v[k + 1], k);
          const int* tgt = reinterpret_cast<const int*>(meta + 4 * C::BT);
          const float* gs = reinterpret_cast<const float*>(meta + 8 * C::BT);
          bool near = false;
#pragma unroll
          for (int k = 0; k < C::HC / 32; ++k) near |= (u32)(tgt[k * 32 + lane] - (row - lane)) < 32u;
          if (__any_sync(0xffffffffu, near)) {  // some row's target is one of this warp's vocabulary rows
#pragma unroll
            for (int k = 0; k < C::HC; ++k)
              if (tgt[k] == row) v[k] -= gs[k];
          }
        } else {
          const int col0 = (t0 + j) * C::BT + half * C::HC;
          if (col0 + C::HC > p.rows_b) {
#pragma unroll
            for (int k = 0; k < C::HC; ++k)
              if (col0 + k >= p.rows_b) v[k] = -INFINITY;
          }
          float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int k = 4; k < C::HC; k += 4) {
            const int q = (k >> 2) & 1 ? 2 : 0;
            top[q] = max3(top[q], v[k], v[k + 1]);
            top[q + 1] = max3(top[q + 1], v[k + 2], v[k + 3]);
          }
          const float t = fmaxf(max3(top[0], top[1], top[2]), top[3]) * p.c;
          const bool move = t > m + MOVE_REFERENCE;
          if (__any_sync(0xffffffffu, move)) {
            const float f = move ? (m == -INFINITY ? 0.f : ex2(m - t)) : 1.f;
            sum = m == -INFINITY ? sum : sum * f;
            if (move) m = t;
            if (C::MODE == TC_PULL && j > 0) {
              // O was made against the old reference
              if (C::NA == 1 && C::NB > 1) {
                ok = bar_wait(pv_done, (w - 1) & 1, gave_up, p.err);
                tc_after();
              }
              for (int k = 0; k < ksteps * 16; k += 16) {
                float o[16];
                const u32 at = tmem + C::O_COL + a * C::DP + k + lanes;
                tc_ld16(o, at);
                tc_wait_ld();
#pragma unroll
                for (int q = 0; q < 16; ++q) o[q] *= f;
                tc_st16(at, reinterpret_cast<const u32*>(o));
              }
            }
          }
          const float off = (float)FWD_SHIFT - (m == -INFINITY ? 0.f : m);
          const u64 off2 = join2(off, off);
          u64 add[2] = {0, 0};
#pragma unroll
          for (int k = 0; k < C::HC; k += 2) {
            part2(fma2(join2(v[k], v[k + 1]), c2, off2), v[k], v[k + 1]);
            exponentials(v[k], v[k + 1], k);
            add[(k >> 1) & 1] = add2(add[(k >> 1) & 1], join2(v[k], v[k + 1]));
          }
          float lo, hi;
          part2(add2(add[0], add[1]), lo, hi);
          sum += lo + hi;
        }
        if constexpr (C::SECOND) {
          // each half's P takes the first columns of the half's own S: a warp overwrites what it has read itself
          u32 h[C::HC / 2];
#pragma unroll
          for (int q = 0; q < C::HC / 2; ++q) h[q] = pack2<T>(v[2 * q], v[2 * q + 1]);
          if constexpr (C::MODE == TC_GRAD_W) {
            // rows with a negative upstream gradient: the sign of their whole column
            const u32* sign = reinterpret_cast<const u32*>(smem + C::OFF_META + st * C::META + 12 * C::BT) + half * (C::HC / 2);
            const u32 own = sign[lane % (C::HC / 2)];
            if (__any_sync(0xffffffffu, own != 0)) {
#pragma unroll
              for (int q = 0; q < C::HC / 2; ++q) h[q] ^= sign[q];
            }
          }
#pragma unroll
          for (int q = 0; q < C::HC / 2; q += 16) tc_st16(S + q, h + q);
          tc_wait_st();
        }
      }
      tc_before();
      __syncwarp();
      if (lane == 0) bar_arrive(p_full(b));
    }
    if (C::MODE == TC_STATS && row < p.rows_a && ok)
      p.part_ms[(i64)(blockIdx.y * C::HV + half) * p.rows_a + row] = make_float2(m, sum);
    if (C::MODE == TC_PULL && row < p.rows_a && ok) p.part_ms[(i64)blockIdx.y * p.rows_a + row] = make_float2(m, sum);
    if (C::SECOND && my_tiles > 0) {
      ok = ok && bar_wait(o_full, 0, gave_up, p.err);
      ok = __all_sync(0xffffffffu, ok);
      if (ok && warp_live) {
        tc_after();
        const float f = C::MODE == TC_GRAD_W ? p.out_scale * __uint_as_float(*p.top) : 1.f;
        for (int k = half * 32; k < p.D; k += 32 * C::HV) {
          float o[32];
          tc_ld32(o, tmem + C::O_COL + a * C::DP + k + lanes);
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

// What the dW pass needs of every row of x, by tiles of BT rows: -bias (p g = exp2(l - bias)), target,
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
  reinterpret_cast<float*>(tile)[k] = -bias;
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
  p.parts = p.splits * (C::MODE == TC_STATS ? C::HV : 1);
  return p;
}

//               MODE      DP  NA NB  BT ST CTAS HV ATM
typedef TcShape<TC_STATS, 64, 2, 3, 128, 6, 1, 2, true> Stats64;
typedef TcShape<TC_STATS, 128, 2, 3, 128, 5, 1, 2, true> Stats128;
typedef TcShape<TC_STATS, 256, 2, 2, 128, 3, 1, 2, true> Stats256;
typedef TcShape<TC_STATS, 64, 1, 3, 64, 8, 2, 2, true> StatsFew64;
typedef TcShape<TC_STATS, 128, 1, 3, 64, 6, 2, 2, true> StatsFew128;
typedef TcShape<TC_PULL, 64, 2, 2, 128, 6, 1, 1, true> Pull64;
typedef TcShape<TC_PULL, 128, 2, 2, 128, 4, 1, 1, false> Pull128;
typedef TcShape<TC_PULL, 256, 1, 2, 64, 5, 1, 1, true> Pull256;
typedef TcShape<TC_PULL, 64, 1, 2, 64, 8, 2, 1, true> PullFew64;
typedef TcShape<TC_PULL, 128, 1, 1, 64, 6, 2, 1, true> PullFew128;
typedef TcShape<TC_GRAD_W, 64, 2, 2, 128, 6, 1, 2, true> Grad64;
typedef TcShape<TC_GRAD_W, 128, 1, 2, 128, 4, 1, 2, true> Grad128;
typedef TcShape<TC_GRAD_W, 256, 1, 2, 64, 5, 1, 2, true> Grad256;
typedef TcShape<TC_GRAD_W, 64, 1, 2, 64, 8, 2, 2, true> GradFew64;
typedef TcShape<TC_GRAD_W, 128, 1, 1, 64, 6, 2, 2, true> GradFew128;

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
  (void)N;
  (void)V;
  return dtype != GSB_F32 && D <= 256;
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
static int launch_tc(const CUtensorMap& b, const TcPlan& plan, const TcParams& p, int kid, cudaStream_t st) {
  // the attribute belongs to the device's copy of the kernel; setting it is cheap and not a stream operation
  GSB_CUDA_OK(cudaFuncSetAttribute(loss_tc_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::BYTES));
  LaunchScope ls(kid, st);
  loss_tc_kernel<T, C><<<dim3((unsigned)plan.groups, (unsigned)plan.splits), C::THREADS, C::BYTES, st>>>(b, p);
  return GSB_OK;
}

template <typename T>
void launch_loss_join(const LossArgs& a, const float2* part_ms, int parts, const float* part_o, float* pull) {
  LaunchScope ls(KID_LOSS_JOIN, a.st);
  loss_join_kernel<T><<<ceil_div_i(a.N, 8), 256, 0, a.st>>>(part_ms, parts, part_o, (const T*)a.x, a.ldx, a.N, (const T*)a.w, a.ldw, a.V,
                                                            (int)a.D, a.scale, a.target, a.ignore, a.loss, a.lse2, pull, a.err);
}

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
  CUtensorMap mb;
  if (!tc_map(&mb, w, IsBf16<T>::value, a.V, a.D, ldw, 1, 64, plan.BT)) return GSB_ERR_CUDA;
  TcParams p = {};
  p.a = x;
  p.lda = ldx;
  p.rows_a = (int)a.N;
  p.rows_b = (int)a.V;
  p.D = (int)a.D;
  p.tiles_per_split = plan.per;
  p.c = logit_factor(a.scale);
  p.part_ms = (float2*)(ws + L.ms);
  p.part_o = (float*)(ws + L.o);
  p.err = a.err;
  const int rc = with_shape(mode, a.N, a.D, [&](auto shape) { return launch_tc<T, decltype(shape)>(mb, plan, p, KID_LOSS, a.st); });
  if (rc != GSB_OK) return rc;
  launch_loss_join<T>(a, p.part_ms, plan.parts, p.part_o, pull);
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
  CUtensorMap mb;
  if (!tc_map(&mb, x, IsBf16<T>::value, a.N, a.D, packed_ld(a.D), 1, 64, plan.BT))
    return GSB_ERR_CUDA;
  TcParams p = {};
  p.a = w;
  p.lda = ldw;
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
  const int rc = with_shape(TC_GRAD_W, a.N, a.D, [&](auto shape) { return launch_tc<T, decltype(shape)>(mb, plan, p, KID_LOSS_GRAD, a.st); });
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

template void launch_loss_join<float>(const LossArgs&, const float2*, int, const float*, float*);
template void launch_loss_join<__half>(const LossArgs&, const float2*, int, const float*, float*);
template void launch_loss_join<__nv_bfloat16>(const LossArgs&, const float2*, int, const float*, float*);
template int tc_loss_forward<__half>(const LossArgs&, float*);
template int tc_loss_forward<__nv_bfloat16>(const LossArgs&, float*);
template int tc_loss_grad_w<__half>(const LossArgs&);
template int tc_loss_grad_w<__nv_bfloat16>(const LossArgs&);
template void tc_loss_dx<__half>(const LossArgs&, const float*);
template void tc_loss_dx<__nv_bfloat16>(const LossArgs&, const float*);

}  // namespace gsb
