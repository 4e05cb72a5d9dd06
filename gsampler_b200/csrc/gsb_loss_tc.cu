// The vocabulary cross entropy on the tensor cores (tcgen05, TMA, TMEM): 16-bit types of up to 256
// columns, fp32 of up to 128 as three bf16 planes.
//
// Every pass is one shape of computation: a tile of 128 rows A stays on chip, tiles B of the other
// matrix stream past it, and for each
//     S = A B^T   ->   P = f(S)   ->   O += P B
// where one copy of the B tile in shared memory serves both products (read along its rows for S,
// across them for O).  S, P (16-bit, in the place of S) and O live in TMEM; so does A where there is
// room, which halves what the first product reads from shared memory.
//   forward   A = rows of x, B = the vocabulary.  P = exp2(l - m) against a running reference m;
//             O / sum P is the expected row of W, which is all that dx needs; log2 sum P + m is
//             the log-sum-exp.  Without a gradient for x there is no second product.
//   dW        A = rows of W, B = rows of x.  P = g (p - target) with the known log-sum-exp.
//   dx        (small vocabularies, fp32) A = rows of x, B = the vocabulary, P = p without the target's,
//             whose (p_t - 1) w_t is added in 32 bits; the row's g is a factor at the end, so that no row's
//             scale is another's.  Makes the logits once more instead of keeping the expected rows.
// The gradients are sum_{j != t} p_j w_j - (1 - p_t) w_t and the like: where the target is likely, all of it is of
// the size of 1 - p_t, and half a step of p_t, or a unit of its logit, would be many times that.  So p_t is never
// made: the forward pass leaves the target out of P and of the sum, the join adds it and has the row's loss as
// log(1 + others / target), and the backward passes take 1 - p_t from the loss.
// So training costs four products of N V D multiply-adds (five with dx by itself), and no array of
// N x V values exists anywhere.
//
// Bound by the hand-over from the tensor cores to the exponentials and back: at 128 columns both take
// 1024 cycles a tile of 128 x 128 and each is busy 58 - 60 % of the time (8192 x 60000, bf16); at 256
// columns the products are twice as long and run at 1430 (forward) and 1520 TFLOP/s (dW; 8192 x 300000).
//
// The reference m moves only when a row's maximum passes it by 2^8, because moving it rescales O;
// P stays below 2^15, which fp16 holds.  Sums and O are 32 bits; P is rounded to the type, half a
// step each, which is the rounding that the tensor cores' operands ask for.  O leaves its accumulator every
// streamed_run rows of B: fp32 keeps the sums in registers, 16-bit types in memory, 32 bits an element.
#include "gsb_common.cuh"
#include "gsb_loss.cuh"
#include "gsb_tc.cuh"
#include "gsb_types.cuh"

namespace gsb {

constexpr int WIPE = -2;  // in the place of a target: the row must be zeroed, and its P with it

enum { TC_STATS = 0, TC_PULL = 1, TC_GRAD_W = 2, TC_GRAD_X = 3 };

// ---------------------------------------------------------------- shapes of the kernel
// DP    columns a row may have (64, 128, 256)
// NA    tiles A a CTA works on at once
// NB    S buffers, BT  rows of a tile B, ST  stages of the B pipeline, CTAS  CTAs an SM
// HV    warpgroups that turn an item's S into P, each an equal share of its columns
// PL    planes: 1 for 16-bit values, 3 for fp32 as three bf16 planes and six plane products (see gsb_loss_gemm.cu)
// ATM   tiles A in TMEM, where there is room beside O and two S buffers; else in shared memory
// SHORT for at most RUN_TERMS rows of B
// An item is (tile B j, tile A a), numbered w = j NA + a; it uses buffer w % NB.
template <int MODE_, int DP_, int NA_, int NB_, int BT_, int ST_, int CTAS_, int HV_, bool ATM_, int PL_ = 1, bool SHORT_ = false>
struct TcShape {
  static constexpr int PL = PL_, ACCS = PL == 3 ? 2 : 1, SB = BT_ * ACCS;  // planes, accumulators, columns of an S buffer
  static constexpr int MODE = MODE_, DP = DP_, NA = NA_, NB = NB_, BT = BT_, ST = ST_, CTAS = CTAS_;
  static constexpr int HV = HV_;
  // one pair of exponentials in POLY by the polynomial, where no second product waits for them (0.667 ->
  // 0.622 ms for 8192 x 300000 x 128; with a second product, a quarter: 0.992 -> 1.038)
  static constexpr int POLY = MODE == TC_STATS ? 8 : 0;
  static constexpr bool ATM = ATM_;
  static constexpr bool SECOND = MODE != TC_STATS;  // the product with P
  static constexpr int WG = NA * HV, HC = BT / HV;
  static constexpr int SUBS = DP / 64;
  static constexpr int B_BYTES = PL * SUBS * BT * 128;
  static constexpr int META = MODE == TC_GRAD_W ? BT * 14 : 0;
  static constexpr int A_COL = NB * SB, O_COL = A_COL + (ATM ? NA * PL * (DP / 2) : 0);
  static constexpr int USED = O_COL + (SECOND ? NA * DP * ACCS : 0);
  static constexpr int COLS = USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
  // columns of an S buffer that plane pl of a half's P takes: the half's own, which its warp has read
  __host__ __device__ static constexpr int p_at(int pl, int half) {
    return pl < 2 ? half * HC + pl * (HC / 2) : BT + half * HC;
  }
  static constexpr bool WIPES = MODE == TC_GRAD_W && PL == 1;
  static constexpr int THREADS = WG * 128 + 64 + (WIPES ? 32 : 0);
  static constexpr int A_BYTES = ATM ? 0 : PL * SUBS * 128 * 128;
  // whether O is emptied into sums in memory; dx of 16-bit types has at most SMALL_V rows to run over
  static constexpr bool SPILLS = PL == 1 && !SHORT_ && (MODE == TC_PULL || MODE == TC_GRAD_W);
  static constexpr bool KEEPS = PL == 3 && SECOND;  // or in registers
  static constexpr int OFF_B = NA * A_BYTES, OFF_META = OFF_B + ST * B_BYTES;
  static constexpr int OFF_BAR = OFF_META + ST * META;
  static constexpr int BARS = 3 * ST + 2 * NB + 3;
  static constexpr int BYTES = OFF_BAR + 8 * BARS + 16 + 1024;  // and room to align the base
  static_assert(USED <= 512 && COLS * CTAS <= 512, "TMEM");
  static_assert(BYTES * CTAS <= 226 * 1024, "shared memory");
  static_assert(MODE != TC_PULL || HV == 1, "a row's running state has one owner");
  static_assert(MODE != TC_PULL || NB > 1, "a moved reference waits for the product before");
  static_assert(PL == 1 || (MODE != TC_PULL && NA == 1), "");
  static_assert(!SECOND || NA == 1, "runs count tiles");
  static_assert(HC % 32 == 0 && META % 16 == 0 && OFF_BAR % 8 == 0, "");
};

struct TcParams {
  const void* a;            // rows of lda elements
  i64 lda;
  int a_bytes;              // 16, 8, 4 or 2: what the address and step of a row are multiples of
  u32 a_sign;               // 0x80008000 where A is taken with the other sign, else 0
  int rows_a, rows_b, D;
  int tiles_per_split;      // tiles B a CTA runs over
  float c;                  // |scale| log2 e
  const unsigned char* meta;  // TC_GRAD_W: BT * 14 bytes a tile B
  const void* w;            // TC_GRAD_X: the vocabulary, for the targets' rows
  i64 ldw;
  int w_bytes;
  const float* lse2;        // TC_GRAD_X, by row
  const float* g;           // TC_GRAD_X
  const float* miss;        // TC_GRAD_X: 1 - p of the row's target
  const i64* target;        // TC_STATS, TC_PULL, TC_GRAD_X
  float* hot;               // TC_STATS, TC_PULL: [rows_a] the target's product, where the target lies in the vocabulary
  float2* part_ms;          // TC_STATS / TC_PULL: [parts][rows_a] reference and sum
  float* part_o;            // TC_PULL, gradients with splits: [splits][rows_a][D]
  void* out;                // gradients without splits: [rows_a][D]
  int out_bytes;            // 16, 8, 4 or 2: what the address and step of its rows are multiples of
  float4* run_sums;         // O of the runs before the last, where a CTA has several: [CTA][D / 4 up to whole 32s][128 rows]
  const u32* top;           // TC_GRAD_W: bits of the largest finite |g|
  float out_scale;          // scale over what P is held at
  int* err;
};

// PIECES times 32 elements of a row, `step` elements apart, of which `left` are there (zeros behind
// them); rows start at multiples of `bytes`.  All loads are requested before the first is used.
template <typename V, int PIECES>
__device__ __forceinline__ void row_pieces(Pack<V, 32> (&to)[PIECES], const V* from, int step, int left, int bytes) {
  constexpr int E = 16 / sizeof(V);
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
#pragma unroll
    for (int q = 0; q < 32 * (int)sizeof(V) / 4; ++q) reinterpret_cast<u32*>(to[i].v)[q] = 0;
  }
  if (bytes == 16) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
#pragma unroll
      for (int q = 0; q < 32; q += E)
        if (i * step + q + E <= left) reinterpret_cast<Pack<V, E>*>(to[i].v + q)->load(from + i * step + q);
    }
  } else if (bytes >= 4) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
#pragma unroll
      for (int q = 0; q < 32; q += E)
        if (i * step + q + E <= left) {
#pragma unroll
          for (int e = 0; e < 4; ++e) reinterpret_cast<u32*>(to[i].v + q)[e] = __ldg(reinterpret_cast<const u32*>(from + i * step + q) + e);
        }
    }
  }
  // what no whole piece of 16 bytes covers
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
#pragma unroll
    for (int q = 0; q < 32; q += E)
      if (i * step + q < left && (bytes < 4 || i * step + q + E > left)) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (i * step + q + e < left) to[i].v[q + e] = from[i * step + q + e];
      }
  }
}

// Pairs of values as packed 16-bit elements; with more planes to come, the values become what this
// plane does not hold.  `any`: values of any size, and this is their first plane.
template <typename T, int N>
__device__ __forceinline__ void take_plane(u32 (&h)[N], float* v, bool more, bool any) {
#pragma unroll
  for (int q = 0; q < N; ++q) {
    h[q] = any ? pack2<T>(first_plane(v[2 * q]), first_plane(v[2 * q + 1])) : pack2<T>(v[2 * q], v[2 * q + 1]);
    if (more) {
      const T* t = reinterpret_cast<const T*>(h + q);
      v[2 * q] -= to_float(t[0]);
      v[2 * q + 1] -= to_float(t[1]);
    }
  }
}

// what dx holds p times
template <typename T>
__host__ __device__ constexpr float dx_unit() { return IsBf16<T>::value ? 1.f : (float)(1 << GRAD_SHIFT); }

// T: type of the planes, V: of the values in memory
template <typename T, typename V, typename C>
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
  // a tile of B may be read: with dW, after the rows that do not count were wiped
  auto ready = [&](int s) { return C::WIPES ? a_full + 24 + 8 * s : full(s); };
  u32* tmem_slot = reinterpret_cast<u32*>(smem + C::OFF_BAR + 8 * C::BARS);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = blockIdx.x * (128 * C::NA);
  const int tiles = (p.rows_b + C::BT - 1) / C::BT;
  const int t0 = blockIdx.y * p.tiles_per_split;
  const int my_tiles = min(p.tiles_per_split, tiles - t0);
  const int items = my_tiles * C::NA;
  const int subs = (p.D + 63) / 64, ksteps = (p.D + 15) / 16;
  constexpr int RUN = C::SPILLS || C::KEEPS ? streamed_run<V>() / C::BT : 1 << 30;  // tiles B of a run

  if (warp == C::WG * 4 && lane == 0) {
    for (int s = 0; s < C::ST; ++s) {
      bar_init(full(s), 1);
      bar_init(empty(s), 1);
      if (C::WIPES) bar_init(ready(s), 1);
    }
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
        bar_expect(full(st), (u32)(C::PL * subs * C::BT * 128 + C::META));
        for (int pl = 0; pl < C::PL; ++pl)
          for (int s = 0; s < subs; ++s)
            tma_tile(base + C::OFF_B + st * C::B_BYTES + (pl * C::SUBS + s) * (C::BT * 128), &map_b, s * 64, (t0 + j) * C::BT, pl, full(st));
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
    // descriptors made one by one it took 130 (8192 x 300000 x 256: 2.84 -> 1.81 ms).
    if (my_tiles > 0) {
      const bool bf = IsBf16<T>::value;
      const u32 id_s = tc_idesc(bf, C::BT, false, false), id_o = tc_idesc(bf, (u32)ksteps * 16, false, true);
      constexpr int PAIRS = C::PL == 3 ? 6 : 1;
      constexpr int PA[6] = {2, 0, 1, 1, 0, 0}, PB[6] = {0, 2, 1, 0, 1, 0};
      const bool leader = elect_one();
      bool ok = bar_wait(a_full, 0, gave_up, p.err);
      tc_after();
      auto product_s = [&](int w) {
        const int j = w / C::NA, a = w % C::NA, st = j % C::ST;
        if (a == 0) ok = ok && bar_wait(ready(st), (j / C::ST) & 1, gave_up, p.err);
        if (!ok) return;
        tc_after();
        const u32 A = tmem + C::A_COL + a * (C::DP / 2), d = tmem + (w % C::NB) * C::SB;
        const u64 B = tc_desc(base + C::OFF_B + st * C::B_BYTES, 16), As = tc_desc(base + a * C::A_BYTES, 16);
        if (leader) {
#pragma unroll
          for (int q = 0; q < PAIRS; ++q) {
            const int pa = C::PL == 3 ? PA[q] : 0, pb = C::PL == 3 ? PB[q] : 0;
            const bool high = q == PAIRS - 1;  // the largest products have an accumulator of their own
            const u32 to = d + (high ? (C::ACCS - 1) * C::BT : 0);
#pragma unroll
            for (int k = 0; k < C::DP / 16; ++k) {
              const u64 b = B + ((pb * C::SUBS + (k >> 2)) * (C::BT * 128) + (k & 3) * 32) / 16;
              const bool add = k > 0 || (q > 0 && !high);
              if (k < ksteps && C::ATM) tc_mma_ta(to, A + pa * (C::DP / 2) + k * 8, b, id_s, add);
              else if (k < ksteps) tc_mma(to, As + ((pa * C::SUBS + (k >> 2)) * 16384 + (k & 3) * 32) / 16, b, id_s, add);
            }
          }
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
          const u32 P = tmem + b * C::SB, d = tmem + C::O_COL + a * C::DP;
          const u64 B = tc_desc(base + C::OFF_B + st * C::B_BYTES, C::BT * 128);
          const bool fresh = j % RUN == 0;
          if (leader) {
#pragma unroll
            for (int q = 0; q < PAIRS; ++q) {
              const int pa = C::PL == 3 ? PA[q] : 0, pb = C::PL == 3 ? PB[q] : 0;
              const bool high = q == PAIRS - 1;
#pragma unroll
              for (int k = 0; k < C::BT / 16; ++k)
                tc_mma_ta(d + (high ? (C::ACCS - 1) * C::DP : 0), P + C::p_at(pa, k / (C::HC / 16)) + (k % (C::HC / 16)) * 8,
                          B + (pb * C::SUBS * (C::BT * 128) + k * 2048) / 16, id_o, !fresh || k > 0 || (q > 0 && !high));
            }
            if (a == C::NA - 1) tc_commit(empty(st));
            // waited for where a run ends, and in the forward pass wherever a reference moves
            if (C::MODE == TC_PULL || (C::SECOND && (j + 1) % RUN == 0)) tc_commit(pv_done);
          }
        }
        if (w + C::NB < items) product_s(w + C::NB);
      }
      if (leader) tc_commit(o_full);
      // the products that were issued end by themselves; a bounded look keeps the order when a wait gave up
      for (int k = 0; k < (1 << 16) && !bar_try(o_full, 0); ++k) __nanosleep(32);
    }
  } else if (C::WIPES && warp == C::WG * 4 + 2) {
    // ------------------------------------------------ rows that do not count must not reach a product with a NaN
    // P is zero there, which is enough unless the row holds an infinity or a NaN, and then its
    // log-sum-exp is not finite either (every logit has a term that is not): only those are wiped.
    for (int j = 0; j < my_tiles; ++j) {
      const int st = j % C::ST;
      const bool ok = __all_sync(0xffffffffu, bar_wait(full(st), (j / C::ST) & 1, gave_up, p.err));
      if (!ok) break;
      const int* tgt = reinterpret_cast<const int*>(smem + C::OFF_META + st * C::META + 4 * C::BT);
      bool wiped = false;
      for (int r0 = 0; r0 < C::BT; r0 += 32) {
        u32 dead = __ballot_sync(0xffffffffu, tgt[r0 + lane] == WIPE);
        wiped |= dead != 0;
        for (; dead; dead &= dead - 1) {
          const int r = r0 + __ffs(dead) - 1;
          for (int k = lane; k < subs * 8; k += 32)
            *reinterpret_cast<uint4*>(smem + C::OFF_B + st * C::B_BYTES + (k >> 3) * (C::BT * 128) + r * 128 + (k & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
      }
      if (wiped) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(ready(st));
    }
  } else {
    // ------------------------------------------------ S -> P
    const int wg = warp >> 2, quarter = warp & 3, a = wg / C::HV, half = wg % C::HV;
    const u32 lanes = (u32)(quarter * 32) << 16;
    const int row = row0 + a * 128 + quarter * 32 + lane;
    const bool warp_live = row0 + a * 128 + quarter * 32 < p.rows_a;
    // the rows of A into TMEM: a thread its row, pairs of elements a column; zeros behind the last
    // column (nothing there may meet the zeros of B as a NaN) and row
    const bool row_live = row < p.rows_a && (C::MODE != TC_GRAD_X || p.g[row < p.rows_a ? row : 0] != 0.f);
    constexpr int PIECES = C::DP / (32 * C::HV);
    {
      Pack<V, 32> piece[PIECES];
      row_pieces(piece, (const V*)p.a + (i64)row * p.lda + half * 32, 32 * C::HV, row_live ? p.D - half * 32 : 0, p.a_bytes);
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int k = half * 32 + i * (32 * C::HV);
        if (k < ksteps * 16) {
#pragma unroll
          for (int pl = 0; pl < C::PL; ++pl) {
            u32 h[16];
            if constexpr (C::PL == 1) {
#pragma unroll
              for (int q = 0; q < 16; ++q) h[q] = reinterpret_cast<const u32*>(piece[i].v)[q];
            } else {
              take_plane<T>(h, reinterpret_cast<float*>(piece[i].v), pl + 1 < C::PL, pl == 0);
            }
#pragma unroll
            for (int q = 0; q < 16; ++q) h[q] ^= p.a_sign;
            if constexpr (C::ATM) {
              tc_st16(tmem + C::A_COL + (a * C::PL + pl) * (C::DP / 2) + k / 2 + lanes, h);
            } else {  // as a swizzled tile: 16-byte piece c of row r lies at c ^ (r & 7)
              const int r = quarter * 32 + lane;
              unsigned char* to = smem + a * C::A_BYTES + (pl * C::SUBS + (k >> 6)) * 16384 + r * 128;
#pragma unroll
              for (int q = 0; q < 4; ++q)
                *reinterpret_cast<uint4*>(to + ((((k & 63) >> 3) + q) ^ (r & 7)) * 16) = reinterpret_cast<const uint4*>(h)[q];
            }
          }
        }
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
    // the target, and for dx the row's gradient (an infinite bias: P = 0) and p - 1 at the target, held as P is:
    // p itself, and only for fp16 at 2^14 times that
    constexpr float UNIT = dx_unit<T>();
    int hot = -1;
    float row_grad = 0.f, row_bias = -INFINITY, coef = 0.f;
    if ((C::MODE == TC_STATS || C::MODE == TC_PULL) && row < p.rows_a) {
      const i64 t = p.target[row];
      if (t >= 0 && t < p.rows_b) hot = (int)t;
    }
    if (C::MODE == TC_GRAD_X && row_live) {
      hot = (int)p.target[row];  // in range: the row counts
      row_grad = p.g[row];
      row_bias = -p.lse2[row];
      coef = -UNIT * p.miss[row];
    }
    bool ok = true;
    float kept[C::KEEPS ? PIECES * 32 : 1];  // O of the runs before this one, this warp's columns of it
    float kept_m = -INFINITY;                // TC_PULL: the reference that run_sums were made against
    if constexpr (C::KEEPS) {
#pragma unroll
      for (int q = 0; q < PIECES * 32; ++q) kept[q] = 0.f;
    }
    auto keep = [&]() {  // both accumulators of O into the sums
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int k = half * 32 + i * (32 * C::HV);
        if (k < ksteps * 16) {
          float o[32], u[32];
          tc_ld32(o, tmem + C::O_COL + k + lanes);
          tc_ld32(u, tmem + C::O_COL + C::DP + k + lanes);
          tc_wait_ld();
#pragma unroll
          for (int q = 0; q < 32; ++q) kept[i * 32 + q] += add_planes(o[q], u[q]);
        }
      }
    };
    // run_sums: a thread its row, pieces of four columns, so that a warp's accesses are whole lines
    const int pieces4 = (p.D + 31) / 32 * 8;
    float4* own_sums = p.run_sums + ((i64)(blockIdx.y * gridDim.x + blockIdx.x) * pieces4) * 128 + quarter * 32 + lane;
    // how much what was summed against an older reference counts now
    auto since = [&]() { return C::MODE != TC_PULL || kept_m == m ? 1.f : kept_m == -INFINITY ? 0.f : ex2(kept_m - m); };
    auto add_sums = [&](float (&o)[32], int k, float old) {
      float4 h[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) h[q] = own_sums[(k / 4 + q) * 128];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        o[4 * q] = fmaf(h[q].x, old, o[4 * q]);
        o[4 * q + 1] = fmaf(h[q].y, old, o[4 * q + 1]);
        o[4 * q + 2] = fmaf(h[q].z, old, o[4 * q + 2]);
        o[4 * q + 3] = fmaf(h[q].w, old, o[4 * q + 3]);
      }
    };
    auto spill = [&](bool first) {
      const float old = since();
#pragma unroll 1
      for (int k = half * 32; k < p.D; k += 32 * C::HV) {
        float o[32];
        tc_ld32(o, tmem + C::O_COL + k + lanes);
        tc_wait_ld();
        if (!first) add_sums(o, k, old);
#pragma unroll
        for (int q = 0; q < 8; ++q) own_sums[(k / 4 + q) * 128] = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
      }
      kept_m = m;
    };
    for (int w = a, run = 0;; ++run) {
      const int run_end = C::SPILLS || C::KEEPS ? min(items, (run + 1) * RUN) : items;
      for (; w < run_end; w += C::NA) {
        const int j = w / C::NA, st = j % C::ST, b = w % C::NB;
        ok = bar_wait(s_full(b), (w / C::NB) & 1, gave_up, p.err);
        if (C::META) ok = ok && bar_wait(ready(st), (j / C::ST) & 1, gave_up, p.err);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_after();
        if (warp_live) {
          const u32 S = tmem + b * C::SB + half * C::HC + lanes;
          float v[C::HC];
#pragma unroll
          for (int k = 0; k < C::HC; k += 32) {
            tc_ld32(v + k, S + k);
            if constexpr (C::ACCS == 2) {
              float u[32];
              tc_ld32(u, S + C::BT + k);
              tc_wait_ld();
#pragma unroll
              for (int q = 0; q < 32; q += 2)
                part2(add2(join2(finite_part(v[k + q]), finite_part(v[k + q + 1])), join2(u[q], u[q + 1])), v[k + q], v[k + q + 1]);
            }
          }
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
            const float* at_target = reinterpret_cast<const float*>(meta + 8 * C::BT);
            bool near = false;
#pragma unroll
            for (int k = 0; k < C::HC / 32; ++k) {
              const int t = tgt[k * 32 + lane];
              near |= (u32)(t - (row - lane)) < 32u || t == WIPE;
            }
            // some row's target is one of this warp's vocabulary rows, or some row is zeros: times a masked class's
            // infinity that is a NaN
            if (__any_sync(0xffffffffu, near)) {
#pragma unroll
              for (int k = 0; k < C::HC; ++k) {
                const int t = tgt[k];
                if (t == row) v[k] = at_target[k];
                if (t == WIPE) v[k] = 0.f;
              }
            }
          } else if constexpr (C::MODE == TC_GRAD_X) {
            const int col0 = (t0 + j) * C::BT + half * C::HC;
            if (col0 + C::HC > p.rows_b) {  // behind the vocabulary: a logit of 0 may lie far above the row's own
#pragma unroll
              for (int k = 0; k < C::HC; ++k)
                if (col0 + k >= p.rows_b) v[k] = -INFINITY;
            }
            const u64 bias2 = both(row_bias);
#pragma unroll
            for (int k = 0; k < C::HC; k += 2) {
              part2(fma2(join2(v[k], v[k + 1]), c2, bias2), v[k], v[k + 1]);
              exponentials(v[k], v[k + 1], k);
              if (UNIT != 1.f) part2(mul2(join2(v[k], v[k + 1]), both(UNIT)), v[k], v[k + 1]);
            }
            const int at = hot - col0;  // the target is not a part of P (100000 x 1000 x 128: 77 us, with a branch around this 81)
#pragma unroll
            for (int k = 0; k < C::HC; ++k) v[k] = k == at ? 0.f : v[k];
          } else {
            const int col0 = (t0 + j) * C::BT + half * C::HC;
            const int at = hot - col0;
            if (__any_sync(0xffffffffu, (u32)at < (u32)C::HC)) {  // the target's product: not a part of the sums
              float mine = 0.f;
#pragma unroll
              for (int k = 0; k < C::HC; ++k) mine = k == at ? v[k] : mine;
#pragma unroll
              for (int k = 0; k < C::HC; ++k) v[k] = k == at ? -INFINITY : v[k];
              if ((u32)at < (u32)C::HC && row < p.rows_a) p.hot[row] = mine;
            }
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
            const float t = __fmul_rn(fmaxf(max3(top[0], top[1], top[2]), top[3]), p.c);
            const bool move = t > m + MOVE_REFERENCE;
            if (__any_sync(0xffffffffu, move)) {
              const float f = move ? (m == -INFINITY ? 0.f : ex2(m - t)) : 1.f;
              sum = m == -INFINITY ? sum : sum * f;
              if (move) m = t;
              if (C::MODE == TC_PULL && j > 0) {
                // O was made against the old reference; S of this item is issued behind the product before the last
                ok = bar_wait(pv_done, (w - 1) & 1, gave_up, p.err);
                tc_after();
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
#pragma unroll
            for (int pl = 0; pl < C::PL; ++pl) {
              u32 h[C::HC / 2];
              take_plane<T>(h, v, pl + 1 < C::PL, false);
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
              for (int q = 0; q < C::HC / 2; q += 16) tc_st16(tmem + b * C::SB + C::p_at(pl, half) + lanes + q, h + q);
            }
            tc_wait_st();
          }
        }
        tc_before();
        __syncwarp();
        if (lane == 0) bar_arrive(p_full(b));
      }
      if (!ok || run_end >= items) break;
      if constexpr (C::SPILLS || C::KEEPS) {  // the run's last product, then its sum; the next run's first waits for this warp
        // the forward pass counts every product: S of the next item says that all but the last are done, and the
        // parity is then the last one's
        if (C::MODE == TC_PULL) ok = bar_wait(s_full(w % C::NB), (w / C::NB) & 1, gave_up, p.err);
        ok = __all_sync(0xffffffffu, ok && bar_wait(pv_done, (C::MODE == TC_PULL ? w - 1 : run) & 1, gave_up, p.err));
        if (!ok) break;
        tc_after();
        if (warp_live) {
          if constexpr (C::KEEPS) keep();
          else spill(run == 0);
        }
        tc_before();
      }
    }
    if (C::MODE == TC_STATS && row < p.rows_a && ok)
      p.part_ms[(i64)(blockIdx.y * C::HV + half) * p.rows_a + row] = make_float2(m, sum);
    if (C::MODE == TC_PULL && row < p.rows_a && ok) p.part_ms[(i64)blockIdx.y * p.rows_a + row] = make_float2(m, sum);
    // dx: the target's own row is added in 32 bits, by the split that has met it
    constexpr int AHEAD = C::MODE == TC_GRAD_X && C::PL == 1 ? PIECES : 1;  // pieces of it requested before the wait
    Pack<V, 32> target_row[AHEAD];
    const bool here = C::MODE == TC_GRAD_X && hot >= t0 * C::BT && hot < (t0 + my_tiles) * C::BT;
    const V* target_at = (const V*)p.w + (i64)(here ? hot : 0) * p.ldw;
    if (C::MODE == TC_GRAD_X && C::PL == 1) row_pieces(target_row, target_at + half * 32, 32 * C::HV, here ? p.D - half * 32 : 0, p.w_bytes);
    if (C::SECOND && my_tiles > 0) {
      ok = ok && bar_wait(o_full, 0, gave_up, p.err);
      ok = __all_sync(0xffffffffu, ok);
      if (ok && warp_live) {
        tc_after();
        if constexpr (C::KEEPS) keep();
        const float old = since();
        const float f = C::MODE == TC_PULL ? 1.f : p.out_scale * (C::MODE == TC_GRAD_X ? row_grad : __uint_as_float(*p.top));
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const int k = half * 32 + i * (32 * C::HV);
          if (k >= p.D) break;
          float o[32];
          if constexpr (C::KEEPS) {
#pragma unroll
            for (int q = 0; q < 32; ++q) o[q] = kept[i * 32 + q];
          } else {
            tc_ld32(o, tmem + C::O_COL + a * C::DP + k + lanes);
            tc_wait_ld();
            if (C::SPILLS && my_tiles > RUN) add_sums(o, k, old);
          }
          if (row < p.rows_a) {
            const bool slab = C::MODE == TC_PULL || gridDim.y > 1;
            if (C::MODE == TC_GRAD_X) {
              if (C::PL == 3) row_pieces(target_row, target_at + k, 0, here ? p.D - k : 0, p.w_bytes);
              // a row that does not count is zero
#pragma unroll
              for (int q = 0; q < 32; ++q) o[q] = row_live ? fmaf(coef, to_float(target_row[AHEAD == 1 ? 0 : i].v[q]), o[q]) : 0.f;
            }
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
              V* to = (V*)p.out + (i64)row * p.D + k;
              if constexpr (C::PL == 3) {
                if (p.out_bytes == 16) {
#pragma unroll
                  for (int q = 0; q < 8; ++q)
                    if (k + 4 * q < p.D) reinterpret_cast<float4*>(to)[q] = make_float4(o[4 * q] * f, o[4 * q + 1] * f, o[4 * q + 2] * f, o[4 * q + 3] * f);
                } else {
#pragma unroll
                  for (int q = 0; q < 32; ++q)
                    if (k + q < p.D) to[q] = o[q] * f;
                }
              } else {
              u32 h[16];
#pragma unroll
              for (int q = 0; q < 16; ++q) h[q] = pack2<T>(o[2 * q] * f, o[2 * q + 1] * f);
              if (p.out_bytes == 16) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  if (k + 8 * q < p.D) reinterpret_cast<uint4*>(to)[q] = make_uint4(h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]);
              } else if (p.out_bytes == 8) {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                  if (k + 4 * q < p.D) reinterpret_cast<uint2*>(to)[q] = make_uint2(h[2 * q], h[2 * q + 1]);
              } else if (p.out_bytes == 4) {
#pragma unroll
                for (int q = 0; q < 16; ++q)
                  if (k + 2 * q < p.D) reinterpret_cast<u32*>(to)[q] = h[q];
              } else {
#pragma unroll
                for (int q = 0; q < 32; ++q)
                  if (k + q < p.D) to[q] = reinterpret_cast<const V*>(h)[q];
              }
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
// dst[r, :] = src[r, :] with rows of ldp elements (16-byte multiples, zeros behind D), for a matrix
// whose address or row step TMA does not take
template <typename T>
__global__ void loss_pack_kernel(const T* __restrict__ src, i64 ld, i64 rows, int D, int ldp, T* __restrict__ dst) {
  const int chunks = ldp / 8;
  const i64 total = rows * chunks;
  for (i64 e = (i64)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (i64)gridDim.x * blockDim.x) {
    const i64 r = e / chunks;
    const int c = (int)(e - r * chunks) * 8;
    Pack<T, 8> v;
#pragma unroll
    for (int q = 0; q < 8; ++q) v.v[q] = c + q < D ? src[r * ld + c + q] : from_float<T>(0.f);
    v.store(dst + r * ldp + c);
  }
}

// What the dW pass needs of every row of x, by tiles of BT rows: -bias (p g = exp2(l - bias)), target,
// |g| (p - 1) of the target as P holds it, and the sign of g as a mask of the packed element.  Rows that do not count, and the
// rows behind the last, have an infinite bias: P = 0.  That is not enough where the row is taken as zeros,
// behind the last and where it holds an infinity or a NaN: WIPE.
__global__ void loss_meta_kernel(const float* __restrict__ lse2, const float* __restrict__ miss, const i64* __restrict__ target, const float* __restrict__ g,
                                 const u32* __restrict__ top, i64 N, i64 Npad, int BT, unsigned char* __restrict__ meta) {
  const i64 r = (i64)blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= Npad) return;
  unsigned char* tile = meta + r / BT * (BT * 14);
  const int k = (int)(r % BT);
  float bias = INFINITY, at_target = 0.f;
  int t = -1;
  u32 sign = 0;
  if (r >= N || (g[r] == 0.f && !(fabsf(lse2[r]) < INFINITY))) t = WIPE;
  if (r < N && g[r] != 0.f) {
    const float rel = fabsf(g[r]) / __uint_as_float(*top);
    at_target = -miss[r] * (rel * (float)(1 << GRAD_SHIFT));
    bias = lse2[r] - log2f(rel) - (float)GRAD_SHIFT;
    t = (int)target[r];
    sign = g[r] < 0.f ? 0x8000u : 0u;
  }
  reinterpret_cast<float*>(tile)[k] = -bias;
  reinterpret_cast<int*>(tile + 4 * BT)[k] = t;
  reinterpret_cast<float*>(tile + 8 * BT)[k] = at_target;
  reinterpret_cast<unsigned short*>(tile + 12 * BT)[k] = (unsigned short)sign;
}

// The statistics of a row's parts, which leave its target out, joined with the target's logit l2 in base 2 (-inf:
// there is none): the log-sum-exp in base 2 (of values held at 2^FWD_SHIFT).
struct RowSums { float m, others, s; };  // reference, sum without the target, sum
__device__ __forceinline__ float join_parts(const float2* __restrict__ part, int parts, i64 N, i64 r, int first, int step, float l2, RowSums& q) {
  float m = l2;
  for (int k = first; k < parts; k += step) m = max_nan(m, part[(i64)k * N + r].x);
  if (step == 32) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
  }
  float others = 0.f;
  for (int k = first; k < parts; k += step) {
    const float2 mine = part[(i64)k * N + r];
    // a part without a reference has either no finite logit or a NaN
    others += mine.x == -INFINITY ? mine.y * 0.f : mine.y * exp2f(mine.x - m);
  }
  if (step == 32) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) others += __shfl_xor_sync(0xffffffffu, others, d);
  }
  q.m = m;
  q.others = others;
  q.s = l2 == -INFINITY ? others : others + exp2f(l2 - m + (float)FWD_SHIFT);
  return m + (log2f(q.s) - (float)FWD_SHIFT);
}
constexpr float LN2 = 0.6931471805599453f;
// -log p of the target: log(1 + others / its own), which has the digits of a small loss; from the difference of
// logarithms where its own is as good as nothing
__device__ __forceinline__ float row_loss(float total, float l2, const RowSums& q) {
  const float d = l2 - q.m;
  return d > -20.f ? log1pf(q.others * exp2f(-(float)FWD_SHIFT - d)) : (total - l2) * LN2;
}

// Losses from the parts and the targets' products that went past (hot, of +-x: times c >= 0 a logit in base 2): a
// thread a row, or a warp where there are many parts.
__global__ void __launch_bounds__(256)
loss_finish_kernel(const float2* __restrict__ part, int parts, int lanes, const float* __restrict__ hot, i64 N, i64 V, float c,
                   const i64* __restrict__ target, i64 ignore, float* __restrict__ loss, float* __restrict__ lse2, int* err) {
  const i64 e = (i64)blockIdx.x * blockDim.x + threadIdx.x;
  const i64 r = lanes == 32 ? e >> 5 : e;
  if (r >= N) return;
  const i64 t = target[r];
  const bool there = t >= 0 && t < V, counts = there && t != ignore;
  const float l2 = there ? __fmul_rn(hot[r], c) : -INFINITY;
  RowSums q;
  const float total = join_parts(part, parts, N, r, lanes == 32 ? (int)(e & 31) : 0, lanes, l2, q);
  if (lanes == 32 && (e & 31) != 0) return;
  if (t != ignore && !counts) raise(err, ERRBIT_BAD_INPUT);
  lse2[r] = total;
  loss[r] = counts ? row_loss(total, l2, q) : 0.f;
}

// The same with pulls, a warp a row:
//   pull_i = sum_{j != t} p_ij w_j - (1 - p_it) w_t      (zeros for a row that does not count)
template <typename T>
__global__ void __launch_bounds__(256)
loss_join_kernel(const float2* __restrict__ part, int parts, const float* __restrict__ part_o, i64 N, const T* __restrict__ w, i64 ldw, i64 V,
                 int D, float c, const i64* __restrict__ target, i64 ignore, const float* __restrict__ hot, float* __restrict__ loss,
                 float* __restrict__ lse2, float* __restrict__ pull, int* err) {
  const i64 r = ((i64)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (r >= N) return;
  const i64 t = target[r];
  const bool there = t >= 0 && t < V, counts = there && t != ignore;
  if (t != ignore && !counts && lane == 0) raise(err, ERRBIT_BAD_INPUT);
  const float l2 = there ? __fmul_rn(hot[r], c) : -INFINITY;
  RowSums q;
  const float total = join_parts(part, parts, N, r, lane, 32, l2, q);
  if (lane == 0) {
    lse2[r] = total;
    loss[r] = counts ? row_loss(total, l2, q) : 0.f;
  }
  {  // D <= 256: a lane has every 32nd column; the parts' weights go round the warp
    const float inv = 1.f / q.s, miss = q.others * inv;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    if (counts) {
      for (int k0 = 0; k0 < parts; k0 += 32) {
        const float mk = k0 + lane < parts ? part[(i64)(k0 + lane) * N + r].x : -INFINITY;
        const float weight = mk == -INFINITY ? 1.f : exp2f(mk - q.m);
        const int here = parts - k0 < 32 ? parts - k0 : 32;
        for (int k = 0; k < here; k += 4) {  // four parts requested before the first is added
          float o[4][8];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float* from = part_o + ((i64)(k0 + (k + u < here ? k + u : 0)) * N + r) * D;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[u][i] = i * 32 + lane < D ? __ldg(from + i * 32 + lane) : 0.f;
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            float f = __shfl_sync(0xffffffffu, weight, (k + u) & 31);
            if (k + u >= here) break;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fmaf(o[u][i], f, v[i]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = i * 32 + lane;
      if (d < D) pull[r * D + d] = counts ? fmaf(-miss, to_float(w[t * ldw + d]), v[i] * inv) : 0.f;
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

// dx[i] = sum over the slabs
template <typename T>
__global__ void loss_join_dx_kernel(const float* __restrict__ slab, i64 size, int slabs, T* __restrict__ dx) {
  for (i64 e = (i64)blockIdx.x * blockDim.x + threadIdx.x; e < size; e += (i64)gridDim.x * blockDim.x) {
    float v = 0.f;
    for (int z = 0; z < slabs; ++z) v += slab[z * size + e];
    dx[e] = from_float<T>(v);
  }
}

// out[e] = sum over the slabs: 32 elements a CTA, eight runs of slabs each, joined in order
template <typename T>
__global__ void __launch_bounds__(256) loss_join_dw_kernel(const float* __restrict__ slab, i64 size, int slabs, T* __restrict__ out) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5, per = (slabs + 7) / 8;
  for (i64 e0 = (i64)blockIdx.x * 32; e0 < size; e0 += (i64)gridDim.x * 32) {
    const i64 e = e0 + lane;
    float v = 0.f;
    if (e < size)
      for (int z = run * per; z < slabs && z < (run + 1) * per; ++z) v += slab[z * size + e];
    part[run][lane] = v;
    __syncthreads();
    if (run == 0 && e < size) {
      for (int q = 1; q < 8; ++q) v += part[q][lane];
      out[e] = from_float<T>(v);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- host side
struct TcPlan {
  int BT, splits, per, parts;
  bool spills;
  i64 groups;
};
template <typename C>
static TcPlan plan_of(i64 rows_a, i64 rows_b) {
  TcPlan p;
  if (rows_a < 1) rows_a = 1;  // sizes are asked for empty batches too
  if (rows_b < 1) rows_b = 1;
  p.BT = C::BT;
  p.groups = (rows_a + 128 * C::NA - 1) / (128 * C::NA);
  const i64 tiles = (rows_b + C::BT - 1) / C::BT;
  const int s = split_count(p.groups, tiles, (i64)sm_count() * C::CTAS);
  p.per = (int)((tiles + s - 1) / s);
  p.splits = (int)((tiles + p.per - 1) / p.per);
  p.parts = p.splits * (C::MODE == TC_STATS ? C::HV : 1);
  p.spills = C::SPILLS;
  return p;
}

//               MODE      DP  NA NB  BT ST CTAS HV ATM
typedef TcShape<TC_STATS, 64, 2, 3, 128, 6, 1, 2, true> Stats64;
typedef TcShape<TC_STATS, 128, 2, 3, 128, 5, 1, 2, true> Stats128;
typedef TcShape<TC_STATS, 256, 2, 2, 128, 3, 1, 2, true> Stats256;
typedef TcShape<TC_STATS, 64, 1, 3, 64, 8, 2, 2, true> StatsFew64;
typedef TcShape<TC_STATS, 128, 1, 2, 128, 2, 2, 2, false> StatsFew128;
typedef TcShape<TC_STATS, 256, 1, 1, 64, 2, 2, 2, true> StatsFew256;
typedef TcShape<TC_STATS, 128, 1, 1, 64, 2, 2, 2, true> StatsTile128;
typedef TcShape<TC_STATS, 256, 1, 2, 64, 3, 2, 2, true> StatsMid256;
typedef TcShape<TC_PULL, 64, 1, 2, 64, 8, 2, 1, false> Pull64;
typedef TcShape<TC_PULL, 128, 1, 2, 64, 4, 2, 1, false> Pull128;
typedef TcShape<TC_PULL, 256, 1, 2, 64, 5, 1, 1, true> Pull256;
typedef TcShape<TC_GRAD_X, 64, 1, 2, 64, 4, 2, 2, true> GradX64;
typedef TcShape<TC_GRAD_X, 128, 1, 1, 64, 4, 2, 2, true> GradX128;
typedef TcShape<TC_GRAD_X, 256, 1, 2, 64, 3, 1, 2, true> GradX256;
// fp32: the products are six times as many, so one tile A and small tiles B are enough to hide the rest
// (4000 x 50021 x 64, us: statistics with 64-row tiles 131, 128 rows 114; gradients 237 with 64, 330 with 128)
typedef TcShape<TC_STATS, 64, 1, 2, 128, 3, 1, 2, false, 3> StatsF64;
typedef TcShape<TC_STATS, 128, 1, 2, 64, 2, 1, 2, false, 3> StatsF128;
typedef TcShape<TC_GRAD_X, 64, 1, 2, 64, 5, 1, 2, true, 3> GradXF64;
typedef TcShape<TC_GRAD_X, 128, 1, 1, 64, 2, 1, 2, false, 3> GradXF128;
typedef TcShape<TC_GRAD_W, 64, 1, 2, 64, 5, 1, 2, true, 3> GradF64;
typedef TcShape<TC_GRAD_W, 128, 1, 1, 64, 2, 1, 2, false, 3> GradF128;
typedef TcShape<TC_GRAD_W, 64, 1, 2, 64, 8, 2, 2, true> Grad64;
typedef TcShape<TC_GRAD_W, 128, 1, 2, 128, 4, 1, 2, true> Grad128;
typedef TcShape<TC_GRAD_W, 256, 1, 2, 64, 5, 1, 2, true> Grad256;
typedef TcShape<TC_GRAD_W, 128, 1, 2, 64, 4, 2, 2, false, 1, true> GradFew128;

// A vocabulary of up to this many rows: dx by making the logits again (2 V multiply-adds an element of
// x more at 1.3 PFLOP/s, against writing and reading 16 bytes of pull at 5 TB/s: equal near 2080).
constexpr i64 SMALL_V = 2048;

// f(shape) for the shape that the sizes ask for; the figures are those of the choice, each shape's own time has
// moved by up to 5 % since.  Two small CTAs an SM overlap one's loads and stores
// with the other's products, and their hand-overs fall out of step by themselves; one large CTA reads B
// less often.  Measured (bf16, ms): forward with pulls, 128 columns, two small / one large: 1024 x 232965
// 0.107 / 0.116, 4096 x 100000 0.173 / 0.186, 8192 x 300000 0.956 / 0.975; 64 columns 8192 x 300000
// 0.886 / 1.040.  dW: 1024 x 232965 x 128 0.149 / 0.182, 8192 x 300000 x 128 0.993 / 0.982, x 64 0.854 / 1.035.
// Statistics alone: 8192 x 300000 x 128 0.692 / 0.620, but one row against 2.45 M 0.104 / 0.125; with a tile
// or a few to run over, one S buffer and a short pipeline start sooner (300007 x 47 x 128 0.038 against 0.062,
// x 256 0.065 / 0.085), with dozens they do not (300007 x 1000 x 256 0.204 / 0.179).
template <int PL, typename F>
static auto with_shape(int mode, i64 N, i64 V, i64 D, F f) {
  if constexpr (PL == 3) {
    if (mode == TC_STATS) return D > 64 ? f(StatsF128()) : f(StatsF64());
    if (mode == TC_GRAD_X) return D > 64 ? f(GradXF128()) : f(GradXF64());
    return D > 64 ? f(GradF128()) : f(GradF64());
  } else {
    if (mode == TC_STATS) {
      const bool few = N <= 128 || V <= SMALL_V, tiny = V <= 256;
      if (D > 128) return N <= 128 || tiny ? f(StatsFew256()) : few ? f(StatsMid256()) : f(Stats256());
      if (D > 64) return N > 128 && tiny ? f(StatsTile128()) : few ? f(StatsFew128()) : f(Stats128());
      return few ? f(StatsFew64()) : f(Stats64());
    }
    if (mode == TC_PULL) return D > 128 ? f(Pull256()) : D > 64 ? f(Pull128()) : f(Pull64());
    if (mode == TC_GRAD_X) return D > 128 ? f(GradX256()) : D > 64 ? f(GradX128()) : f(GradX64());
    if (D > 64 && D <= 128 && N <= 2048) return f(GradFew128());
    return D > 128 ? f(Grad256()) : D > 64 ? f(Grad128()) : f(Grad64());
  }
}

template <int PL>
static TcPlan tc_plan(int mode, i64 N, i64 V, i64 D) {
  return with_shape<PL>(mode, N, V, D, [&](auto shape) {
    return mode == TC_GRAD_W ? plan_of<decltype(shape)>(V, N) : plan_of<decltype(shape)>(N, V);
  });
}

static TcPlan tc_plan(int planes, int mode, i64 N, i64 V, i64 D) {
  return planes == 3 ? tc_plan<3>(mode, N, V, D) : tc_plan<1>(mode, N, V, D);
}

bool tc_loss_takes(int dtype, i64 D) { return D <= (dtype == GSB_F32 ? 128 : 256); }
// fp32 makes the logits once more instead (a row's state and its sums of O would not fit beside one another)
bool tc_loss_pulls(int dtype, i64 V) { return dtype != GSB_F32 && V > SMALL_V; }

// rows of a streamed matrix as TMA takes them: a copy where its address or row step does not do, planes for fp32
static size_t copy_bytes(int planes, i64 rows, i64 D) { return 2 * (size_t)planes * rows * packed_ld(D); }

static int planes_of(int dtype) { return dtype == GSB_F32 ? 3 : 1; }
// sums of the runs before a CTA's last
static size_t run_bytes(int dtype, const TcPlan& p, i64 D) {
  const int run = dtype == GSB_BF16 ? streamed_run<__nv_bfloat16>() : streamed_run<__half>();
  if (!p.spills || (i64)p.per * p.BT <= run) return 0;
  return (size_t)p.groups * p.splits * ((D + 31) / 32 * 32) * 128 * 4;
}

struct TcFwdLayout { size_t ms, hot, o, runs, w, bytes; };
static TcFwdLayout fwd_layout(int dtype, i64 N, i64 V, i64 D, bool pull) {
  const int planes = planes_of(dtype);
  TcFwdLayout L;
  size_t o = 0;
  auto take = [&](size_t b) { const size_t at = o; o += up256(b); return at; };
  const TcPlan p = tc_plan(planes, pull ? TC_PULL : TC_STATS, N, V, D);
  L.ms = take(8 * (size_t)p.parts * N);
  L.hot = take(4 * (size_t)N);
  L.o = take(pull ? 4 * (size_t)p.splits * N * D : 0);
  L.runs = take(run_bytes(dtype, p, D));
  L.w = take(copy_bytes(planes, V, D));
  L.bytes = o;
  return L;
}
size_t tc_loss_workspace(int dtype, i64 N, i64 V, i64 D, bool pull, bool pack_w) {
  const TcFwdLayout L = fwd_layout(dtype, N, V, D, pull);
  return pack_w || dtype == GSB_F32 ? L.bytes : L.w;
}

struct TcGradLayout { size_t meta, dw_slab, dw_runs, dx_slab, x, w, bytes; };
static TcGradLayout grad_layout(int dtype, i64 N, i64 V, i64 D, bool dx, bool dw) {
  const int planes = planes_of(dtype);
  TcGradLayout L;
  size_t o = 0;
  auto take = [&](size_t b) { const size_t at = o; o += up256(b); return at; };
  const TcPlan w = tc_plan(planes, TC_GRAD_W, N, V, D), x = tc_plan(planes, TC_GRAD_X, N, V, D);
  L.meta = take(dw ? (size_t)((N + w.BT - 1) / w.BT) * w.BT * 14 : 0);
  L.dw_slab = take(dw && w.splits > 1 ? 4 * (size_t)w.splits * V * D : 0);
  L.dw_runs = take(dw ? run_bytes(dtype, w, D) : 0);
  L.dx_slab = take(dx && x.splits > 1 ? 4 * (size_t)x.splits * N * D : 0);
  L.x = take(dw ? copy_bytes(planes, N, D) : 0);
  L.w = take(dx ? copy_bytes(planes, V, D) : 0);
  L.bytes = o;
  return L;
}
size_t tc_loss_grad_workspace(int dtype, i64 N, i64 V, i64 D, bool dx, bool dw) {
  return grad_layout(dtype, N, V, D, dx, dw).bytes;
}
bool tc_loss_packs(const void* w, i64 ldw) { return !tma_ready(w, ldw); }

template <typename T>
static const T* pack_rows(const T* src, i64 ld, i64 rows, i64 D, void* dst, cudaStream_t st) {
  LaunchScope ls(KID_LOSS_JOIN, st);
  loss_pack_kernel<T><<<blocks_for(rows * packed_ld(D) / 8), 256, 0, st>>>(src, ld, rows, (int)D, (int)packed_ld(D), (T*)dst);
  return (const T*)dst;
}
static int row_bytes(const void* p, i64 ld, int size) {
  const uintptr_t m = (uintptr_t)p | (uintptr_t)(ld * size);
  return m & 2 ? 2 : m & 4 ? 4 : m & 8 ? 8 : 16;
}

template <typename V, typename C>
static int launch_tc(const CUtensorMap& b, const TcPlan& plan, const TcParams& p, int kid, cudaStream_t st) {
  typedef typename Planes<V>::type T;
  static std::atomic<unsigned long long> done{0};
  if (!allow_shared(loss_tc_kernel<T, V, C>, C::BYTES, done)) return GSB_ERR_CUDA;
  LaunchScope ls(kid, st);
  loss_tc_kernel<T, V, C><<<dim3((unsigned)plan.groups, (unsigned)plan.splits), C::THREADS, C::BYTES, st>>>(b, p);
  return GSB_OK;
}

template <typename T>
void launch_loss_join(const LossArgs& a, const float2* part_ms, int parts, const float* part_o, const float* hot, float* pull) {
  LaunchScope ls(KID_LOSS_JOIN, a.st);
  const float c = logit_factor(a.scale);
  if (pull) {
    loss_join_kernel<T><<<ceil_div_i(a.N, 8), 256, 0, a.st>>>(part_ms, parts, part_o, a.N, (const T*)a.w, a.ldw, a.V, (int)a.D, c, a.target,
                                                              a.ignore, hot, a.loss, a.lse2, pull, a.err);
    return;
  }
  const int lanes = parts > 8 ? 32 : 1;
  loss_finish_kernel<<<ceil_div_i(a.N * lanes, 256), 256, 0, a.st>>>(part_ms, parts, lanes, hot, a.N, a.V, c, a.target, a.ignore, a.loss, a.lse2,
                                                                    a.err);
}

// what the forward pass and both gradients have in common
template <typename T>
static TcParams base_params(const LossArgs& a, const TcPlan& plan, bool vocabulary_side) {
  TcParams p = {};
  p.a = vocabulary_side ? a.w : a.x;
  p.lda = vocabulary_side ? a.ldw : a.ldx;
  p.a_bytes = row_bytes(p.a, p.lda, sizeof(T));
  // l = |scale| (+-A) . B: the running maximum needs a factor that is not negative
  p.a_sign = a.scale < 0.f ? 0x80008000u : 0u;
  p.rows_a = (int)(vocabulary_side ? a.V : a.N);
  p.rows_b = (int)(vocabulary_side ? a.N : a.V);
  p.D = (int)a.D;
  p.tiles_per_split = plan.per;
  p.c = logit_factor(a.scale);
  p.target = a.target;
  p.lse2 = a.lse2;
  p.g = a.g;
  p.top = a.top;
  p.out_scale = a.scale / (float)(1 << GRAD_SHIFT);
  p.err = a.err;
  return p;
}
// The map of the streamed matrix; rows that TMA does not take as they lie are copied to `copy` first.
// fp32 rows go there as planes, those that must not reach a product as zeros.
template <typename T>
static bool stream_map(CUtensorMap* map, const void* src, i64 ld, i64 rows, i64 D, int box_rows, const float* g, const float* lse2, void* copy,
                       cudaStream_t st) {
  constexpr int planes = Planes<T>::count;
  if constexpr (planes == 3) {
    make_planes<T>(src, ld, rows, D, false, g, lse2, nullptr, copy, st);
    src = copy;
    ld = packed_ld(D);
  } else if (!tma_ready(src, ld)) {
    src = pack_rows<T>((const T*)src, ld, rows, D, copy, st);
    ld = packed_ld(D);
  }
  return tc_map(map, src, IsBf16<typename Planes<T>::type>::value, rows, D, ld, planes, 64, box_rows);
}

template <typename T>
int tc_loss_forward(const LossArgs& a, float* pull) {
  const int mode = pull ? TC_PULL : TC_STATS;
  const TcPlan plan = tc_plan(Planes<T>::count, mode, a.N, a.V, a.D);
  const TcFwdLayout L = fwd_layout(dtype_of<T>(), a.N, a.V, a.D, pull != nullptr);
  char* ws = (char*)a.ws;
  CUtensorMap mb;
  if (!stream_map<T>(&mb, a.w, a.ldw, a.V, a.D, plan.BT, nullptr, nullptr, ws + L.w, a.st)) return GSB_ERR_CUDA;
  TcParams p = base_params<T>(a, plan, false);
  p.part_ms = (float2*)(ws + L.ms);
  p.part_o = (float*)(ws + L.o);
  p.hot = (float*)(ws + L.hot);
  p.run_sums = (float4*)(ws + L.runs);
  const int rc = with_shape<Planes<T>::count>(mode, a.N, a.V, a.D, [&](auto shape) { return launch_tc<T, decltype(shape)>(mb, plan, p, KID_LOSS, a.st); });
  if (rc != GSB_OK) return rc;
  launch_loss_join<T>(a, p.part_ms, plan.parts, p.part_o, p.hot, pull);
  return GSB_OK;
}

template <typename T>
int tc_loss_grad_w(const LossArgs& a) {
  const TcPlan plan = tc_plan(Planes<T>::count, TC_GRAD_W, a.N, a.V, a.D);
  const TcGradLayout L = grad_layout(dtype_of<T>(), a.N, a.V, a.D, a.dx != nullptr, true);
  char* ws = (char*)a.ws;
  {
    const i64 npad = (a.N + plan.BT - 1) / plan.BT * plan.BT;
    LaunchScope ls(KID_LOSS_JOIN, a.st);
    loss_meta_kernel<<<ceil_div_i(npad, 256), 256, 0, a.st>>>(a.lse2, a.miss, a.target, a.g, a.top, a.N, npad, plan.BT, (unsigned char*)(ws + L.meta));
  }
  CUtensorMap mb;
  if (!stream_map<T>(&mb, a.x, a.ldx, a.N, a.D, plan.BT, a.g, a.lse2, ws + L.x, a.st)) return GSB_ERR_CUDA;
  TcParams p = base_params<T>(a, plan, true);
  p.meta = (const unsigned char*)(ws + L.meta);
  p.part_o = (float*)(ws + L.dw_slab);
  p.run_sums = (float4*)(ws + L.dw_runs);
  p.out = a.dw;
  p.out_bytes = row_bytes(a.dw, a.D, sizeof(T));
  const int rc = with_shape<Planes<T>::count>(TC_GRAD_W, a.N, a.V, a.D, [&](auto shape) { return launch_tc<T, decltype(shape)>(mb, plan, p, KID_LOSS_GRAD, a.st); });
  if (rc != GSB_OK) return rc;
  if (plan.splits > 1) {
    LaunchScope ls(KID_LOSS_JOIN, a.st);
    loss_join_dw_kernel<T><<<blocks_for(a.V * a.D * 8), 256, 0, a.st>>>(p.part_o, a.V * a.D, plan.splits, (T*)a.dw);
  }
  return GSB_OK;
}

// dx by making the logits again
template <typename T>
int tc_loss_grad_x(const LossArgs& a) {
  const TcPlan plan = tc_plan(Planes<T>::count, TC_GRAD_X, a.N, a.V, a.D);
  const TcGradLayout L = grad_layout(dtype_of<T>(), a.N, a.V, a.D, true, a.dw != nullptr);
  char* ws = (char*)a.ws;
  CUtensorMap mb;
  if (!stream_map<T>(&mb, a.w, a.ldw, a.V, a.D, plan.BT, nullptr, nullptr, ws + L.w, a.st)) return GSB_ERR_CUDA;
  TcParams p = base_params<T>(a, plan, false);
  p.w = a.w;
  p.ldw = a.ldw;
  p.w_bytes = row_bytes(a.w, a.ldw, sizeof(T));
  p.miss = a.miss;
  p.out_scale = a.scale / dx_unit<typename Planes<T>::type>();
  p.out = a.dx;
  p.out_bytes = row_bytes(a.dx, a.D, sizeof(T));
  p.part_o = (float*)(ws + L.dx_slab);
  const int rc = with_shape<Planes<T>::count>(TC_GRAD_X, a.N, a.V, a.D, [&](auto shape) { return launch_tc<T, decltype(shape)>(mb, plan, p, KID_LOSS_GRAD, a.st); });
  if (rc != GSB_OK) return rc;
  if (plan.splits > 1) {
    LaunchScope ls(KID_LOSS_JOIN, a.st);
    loss_join_dx_kernel<T><<<blocks_for(a.N * a.D), 256, 0, a.st>>>(p.part_o, a.N * a.D, plan.splits, (T*)a.dx);
  }
  return GSB_OK;
}

template <typename T>
void tc_loss_dx(const LossArgs& a, const float* pull) {
  LaunchScope ls(KID_LOSS_JOIN, a.st);
  loss_dx_kernel<T><<<blocks_for(a.N * a.D), 256, 0, a.st>>>(pull, a.g, a.scale, a.N, (int)a.D, (T*)a.dx);
}

template void launch_loss_join<float>(const LossArgs&, const float2*, int, const float*, const float*, float*);
template void launch_loss_join<__half>(const LossArgs&, const float2*, int, const float*, const float*, float*);
template void launch_loss_join<__nv_bfloat16>(const LossArgs&, const float2*, int, const float*, const float*, float*);
template int tc_loss_forward<float>(const LossArgs&, float*);
template int tc_loss_forward<__half>(const LossArgs&, float*);
template int tc_loss_forward<__nv_bfloat16>(const LossArgs&, float*);
template int tc_loss_grad_w<float>(const LossArgs&);
template int tc_loss_grad_w<__half>(const LossArgs&);
template int tc_loss_grad_w<__nv_bfloat16>(const LossArgs&);
template int tc_loss_grad_x<float>(const LossArgs&);
template int tc_loss_grad_x<__half>(const LossArgs&);
template int tc_loss_grad_x<__nv_bfloat16>(const LossArgs&);
template void tc_loss_dx<__half>(const LossArgs&, const float*);
template void tc_loss_dx<__nv_bfloat16>(const LossArgs&, const float*);

}  // namespace gsb
