// The vocabulary cross entropy for more columns than gsb_loss_tc.cu takes: tiled products on the tensor
// cores, with the vocabulary taken in pieces in the backward pass.
//
//   statistics  tiles of x W^T whose epilogue keeps the running maximum and sum of every row, its target left out
//   piece       tiles of x W^T again, whose epilogue writes g (p - target), the target's element from the row's
//               1 - p_t, of at most PIECE_ELEMS
//               elements to a workspace: 64 MB of 16-bit values, which L2 holds, 192 MB of fp32's planes, which
//               it does not; at least 128 columns, of which 16-bit tiles of 256 waste half, from 262144 rows on
//   dx, dW      the piece times W, its transpose times x; long sums are split into 32-bit slabs that
//               are added in a fixed order
//
// fp32 values are taken apart into three bf16 planes (8 + 8 + 8 bits of the 24) and a product is the
// six plane products that reach 2^-24 of it: h h, h m, m h, m m, h l, l h.  Six bf16 products are
// still several times the rate of 32-bit multiply-adds (at most 233 TFLOP/s here, of 1399 sustained).
// A load of all planes of a 64-deep slice feeds all six, so the slice's bytes are read once:
// 96 KB per 1536 cycles of products.
#include "gsb_common.cuh"
#include "gsb_loss.cuh"
#include "gsb_tc.cuh"
#include "gsb_types.cuh"

namespace gsb {

enum { GM_STATS = 0, GM_PIECE = 1, GM_DX = 2, GM_DW = 3 };

constexpr i64 PIECE_ELEMS = 1ll << 25;

// RUN: blocks of depth (64 each) after which the accumulators' sums move on to registers, 0 where the depth is
// never more than RUN_TERMS
template <int MODE_, int PL_, int BN_, int ST_, int RUN_>
struct GmShape {
  static constexpr int MODE = MODE_, PL = PL_, BN = BN_, ST = ST_, RUN = RUN_;
  static constexpr bool A_ACROSS = MODE == GM_DW, B_ACROSS = MODE == GM_DX || MODE == GM_DW;
  static constexpr int A_PLANE = 128 * 128, B_PLANE = BN * 128;
  static constexpr int STAGE = PL * (A_PLANE + B_PLANE);
  // The products of two high planes have an accumulator of their own: every addition into a 32-bit
  // accumulator truncates, and the five small products would truncate the large sum five times more.
  static constexpr int ACCS = PL == 3 ? 2 : 1;
  static constexpr int COLS = 2 * ACCS * BN;
  static constexpr int THREADS = 8 * 32 + 64;
  static constexpr int OFF_OUT = ST * STAGE;  // GM_PIECE: 32 rows x 64 columns a warp on their way out
  static constexpr int OFF_BAR = OFF_OUT + (MODE == GM_PIECE ? 8 * 4096 : 0);
  static constexpr int BARS = 2 * ST + 4;
  static constexpr int BYTES = OFF_BAR + 8 * BARS + 16 + 1024;
  static_assert(BYTES <= 227 * 1024 && COLS >= 128 && COLS <= 512, "");
  static_assert(MODE != GM_PIECE || BN % 128 == 0, "");
  static_assert(!RUN || BN <= 128, "half a tile's columns in registers");
};

struct GmParams {
  int M, N, K;              // rows of A, rows of B (columns of the result), depth
  int m_tiles, n_tiles, units;
  int n_per_cta;            // GM_STATS: column tiles a CTA runs over (grid = m_tiles x splits)
  int k_per;                // depth of one slab, a multiple of 64
  float c;
  float2* part_ms;          // GM_STATS: [2 * splits][M]
  float* hot;               // GM_STATS: [M] the target's product, where the target lies in the vocabulary
  const float* lse2;        // GM_PIECE, by row
  const float* g;
  const float* miss;
  const i64* target;        // GM_STATS, GM_PIECE
  const u32* top;
  int v0;                   // GM_PIECE: id of the piece's first column
  void* piece;              // GM_PIECE: [PL][M][ld_piece]
  i64 ld_piece, plane;
  float* lost;              // GM_PIECE: [M] what rounding the target's element to 16 bits lost, for dx
  float* slab;              // GM_DX / GM_DW: [units along z][M][N]
  int add;
  int* err;
};

template <typename T, typename C>
__global__ void __launch_bounds__(C::THREADS, 1)
loss_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const GmParams p) {
  extern __shared__ unsigned char smem_raw[];
  const u32 base = (smem_addr(smem_raw) + 1023) & ~1023u;
  unsigned char* smem = smem_raw + (base - smem_addr(smem_raw));
  const u32 bar0 = base + C::OFF_BAR;
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (C::ST + s); };
  auto acc_full = [&](int b) { return bar0 + 8 * (2 * C::ST + b); };
  auto acc_empty = [&](int b) { return bar0 + 8 * (2 * C::ST + 2 + b); };
  u32* tmem_slot = reinterpret_cast<u32*>(smem + C::OFF_BAR + 8 * C::BARS);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // the tiles of this CTA: (m, n, z) of the i-th, false behind the last
  auto tile_at = [&](int i, int& m, int& n, int& z) {
    if (C::MODE == GM_STATS) {
      m = blockIdx.x;
      n = blockIdx.y * p.n_per_cta + i;
      z = 0;
      return i < p.n_per_cta && n < p.n_tiles;
    }
    const i64 u = (i64)blockIdx.x + (i64)i * gridDim.x;
    if (u >= p.units) return false;
    m = (int)(u % p.m_tiles);
    n = (int)(u / p.m_tiles % p.n_tiles);
    z = (int)(u / ((i64)p.m_tiles * p.n_tiles));
    return true;
  };
  auto depth = [&](int z, int& k0, int& blocks) {  // a slab without depth is a slab of zeros
    k0 = z * p.k_per;
    const int k1 = min(p.K, k0 + p.k_per);
    blocks = k1 > k0 ? (k1 - k0 + 63) / 64 : 0;
  };
  // a tile's products are made in runs, each in accumulators of its own
  auto runs_of = [](int blocks) { return C::RUN && blocks > C::RUN ? (blocks + C::RUN - 1) / (C::RUN ? C::RUN : 1) : 1; };

  if (warp == 8 && lane == 0) {
    for (int s = 0; s < C::ST; ++s) { bar_init(full(s), 1); bar_init(empty(s), 1); }
    for (int b = 0; b < 2; ++b) { bar_init(acc_full(b), 1); bar_init(acc_empty(b), 8); }
    *gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"((u32)C::COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const u32 tmem = __reduce_max_sync(0xffffffffu, *tmem_slot);  // the same in every lane, and known to be

  if (warp == 8) {
    // ------------------------------------------------ loads
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      int m, n, z;
      for (int i = 0; ok && tile_at(i, m, n, z); ++i) {
        int k0, blocks;
        depth(z, k0, blocks);
        for (int kb = 0; kb < blocks; ++kb, ++it) {
          const int st = it % C::ST, k = k0 + kb * 64;
          if (it >= C::ST && !bar_wait(empty(st), ((it / C::ST) - 1) & 1, gave_up, p.err)) { ok = false; break; }
          bar_expect(full(st), C::STAGE);
          const u32 A = base + st * C::STAGE, B = A + C::PL * C::A_PLANE;
#pragma unroll
          for (int pl = 0; pl < C::PL; ++pl) {
            if (C::A_ACROSS) {
              for (int h = 0; h < 2; ++h) tma_tile(A + pl * C::A_PLANE + h * 8192, &map_a, m * 128 + h * 64, k, pl, full(st));
            } else {
              tma_tile(A + pl * C::A_PLANE, &map_a, k, m * 128, pl, full(st));
            }
            if (C::B_ACROSS) {
              for (int h = 0; h < C::BN / 64; ++h) tma_tile(B + pl * C::B_PLANE + h * 8192, &map_b, n * C::BN + h * 64, k, pl, full(st));
            } else {
              tma_tile(B + pl * C::B_PLANE, &map_b, k, n * C::BN, pl, full(st));
            }
          }
        }
      }
      // no copy may be in flight when the CTA ends (only after a wait that gave up can one be)
      for (int j = it > C::ST ? it - C::ST : 0; j < it; ++j)
        for (int k = 0; k < (1 << 16) && !bar_try(full(j % C::ST), (j / C::ST) & 1); ++k) __nanosleep(32);
    }
  } else if (warp == 9) {
    // ------------------------------------------------ products (the warp together, one lane issues)
    const u32 id = tc_idesc(C::PL == 3 || IsBf16<T>::value, C::BN, C::A_ACROSS, C::B_ACROSS);
    const bool leader = elect_one();
    int it = 0, acc = 0;
    bool ok = true;
    int m, n, z;
    for (int i = 0; ok && tile_at(i, m, n, z); ++i) {
      int k0, blocks;
      depth(z, k0, blocks);
      for (int r = 0, runs = runs_of(blocks); ok && r < runs; ++r, ++acc) {
        const int b = acc & 1, first = r * C::RUN, last = r + 1 < runs ? first + C::RUN : blocks;
        if (acc >= 2) ok = bar_wait(acc_empty(b), ((acc >> 1) - 1) & 1, gave_up, p.err);
        tc_after();
        const u32 d = tmem + b * (C::ACCS * C::BN);
        for (int kb = first; ok && kb < last; ++kb, ++it) {
          const int st = it % C::ST;
          ok = bar_wait(full(st), (it / C::ST) & 1, gave_up, p.err);
          if (!ok) break;
          tc_after();
          const u64 A = tc_desc(base + st * C::STAGE, C::A_ACROSS ? 8192 : 16);
          const u64 B = tc_desc(base + st * C::STAGE + C::PL * C::A_PLANE, C::B_ACROSS ? 8192 : 16);
          constexpr int PAIRS = C::PL == 3 ? 6 : 1;
          constexpr int pa[6] = {2, 0, 1, 1, 0, 0}, pb[6] = {0, 2, 1, 0, 1, 0};
          if (leader) {
#pragma unroll
            for (int q = 0; q < PAIRS; ++q) {
              const bool high = q == PAIRS - 1;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                tc_mma(d + (high ? (C::ACCS - 1) * C::BN : 0), A + ((C::PL == 3 ? pa[q] : 0) * C::A_PLANE + k * (C::A_ACROSS ? 2048 : 32)) / 16,
                       B + ((C::PL == 3 ? pb[q] : 0) * C::B_PLANE + k * (C::B_ACROSS ? 2048 : 32)) / 16, id,
                       kb > first || k > 0 || (q > 0 && !high));
            }
            tc_commit(empty(st));
          }
        }
        if (ok && leader) tc_commit(acc_full(b));
      }
    }
    // what was issued ends by itself; a bounded look keeps the order when a wait gave up
    for (int j = acc > 2 ? acc - 2 : 0; j < acc; ++j)
      for (int k = 0; k < (1 << 16) && !bar_try(acc_full(j & 1), (j >> 1) & 1); ++k) __nanosleep(32);
  } else {
    // ------------------------------------------------ epilogue: a thread has a row and half the columns
    const int half = warp >> 2, quarter = warp & 3;
    const u32 lanes = (u32)(quarter * 32) << 16;
    float run_m = -INFINITY, run_s = 0.f;
    bool ok = true;
    int m, n, z;
    int acc = 0;
    float kept[C::RUN ? C::BN / 2 : 1];  // the runs before a tile's last
    for (int i = 0; ok && tile_at(i, m, n, z); ++i) {
      int k0, blocks;
      depth(z, k0, blocks);
      auto columns = [&](float* v, int q) {  // 32 of the tile's columns, the accumulators added
        const u32 from = tmem + (acc & 1) * (C::ACCS * C::BN) + q + lanes;
        tc_ld32(v, from);
        if constexpr (C::ACCS == 2) {
          float u[32];
          tc_ld32(u, from + C::BN);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = add_planes(v[j], u[j]);
        } else {
          tc_wait_ld();
        }
      };
      const int runs = runs_of(blocks);
      if constexpr (C::RUN != 0) {
#pragma unroll
        for (int j = 0; j < C::BN / 2; ++j) kept[j] = 0.f;
        for (int r = 0; r + 1 < runs; ++r, ++acc) {
          ok = __all_sync(0xffffffffu, bar_wait(acc_full(acc & 1), (acc >> 1) & 1, gave_up, p.err));
          if (!ok) break;
          tc_after();
#pragma unroll
          for (int q = 0; q < C::BN / 2; q += 32) {
            float v[32];
            columns(v, half * (C::BN / 2) + q);
#pragma unroll
            for (int j = 0; j < 32; ++j) kept[q + j] += v[j];
          }
          tc_before();
          __syncwarp();
          if (lane == 0) bar_arrive(acc_empty(acc & 1));
        }
        if (!ok) break;
      }
      const int b = acc & 1;
      ok = bar_wait(acc_full(b), (acc >> 1) & 1, gave_up, p.err);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_after();
      const int row = m * 128 + quarter * 32 + lane;
      float lse = INFINITY, gs = 0.f;
      int hot = -1;
      float at_target = 0.f;
      if (C::MODE == GM_STATS && row < p.M) {
        const i64 t = p.target[row];
        if (t >= 0 && t < p.N) hot = (int)t;
      }
      if (C::MODE == GM_PIECE && row < p.M && p.g[row] != 0.f) {
        lse = p.lse2[row];
        const float top = __uint_as_float(*p.top);
        gs = times_power(p.g[row], -small_rows<T>(p.g[row], top)) / top * (float)(1 << GRAD_SHIFT);
        hot = (int)(p.target[row] - p.v0);
        at_target = -p.miss[row] * gs;
      }
      if constexpr (C::MODE == GM_PIECE) {
        // 64 columns at a time through shared memory, so that they leave as whole lines: row by row a
        // warp's stores touch 32 lines an instruction (52 us for 4000 x 4096 columns of three planes)
#pragma unroll (C::RUN ? 4 : 1)
        for (int own = 0; own < C::BN / 2; own += 64) {
          const int q = half * (C::BN / 2) + own, col = n * C::BN + q;
          if (col >= p.N || m * 128 + quarter * 32 >= p.M) break;
          float v[64];
          columns(v, q);
          columns(v + 32, q + 32);
          if constexpr (C::RUN != 0) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] += kept[own + j];
          }
#pragma unroll
          for (int j = 0; j < 64; ++j) {
            v[j] = ex2(fmaf(v[j], p.c, -lse));
            v[j] = gs == 0.f ? 0.f : col + j == hot ? at_target : v[j] * gs;  // zeros for rows that do not count
          }
          if (C::PL == 1 && (u32)(hot - col) < 64u) {
            // g (p - 1) is as large as its row's other elements together: dx gets the lost part back
#pragma unroll
            for (int j = 0; j < 64; ++j)
              if (col + j == hot) p.lost[row] = v[j] - to_float(from_float<T>(v[j]));
          }
          const u32 out = base + C::OFF_OUT + warp * 4096;
          const int first = m * 128 + quarter * 32;
#pragma unroll
          for (int pl = 0; pl < C::PL; ++pl) {
            __syncwarp();  // the plane before has been read
#pragma unroll
            for (int j = 0; j < 64; j += 8) {
              u32 h[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                h[e] = pack2<T>(v[j + 2 * e], v[j + 2 * e + 1]);
                if (pl + 1 < C::PL) {  // what this plane does not hold
                  const T* t = reinterpret_cast<const T*>(h + e);
                  v[j + 2 * e] -= to_float(t[0]);
                  v[j + 2 * e + 1] -= to_float(t[1]);
                }
              }
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(out + lane * 128 + ((j / 8) ^ (lane & 7)) * 16), "r"(h[0]), "r"(h[1]),
                           "r"(h[2]), "r"(h[3])
                           : "memory");
            }
            __syncwarp();
            // eight lanes a row
            T* to = (T*)p.piece + pl * p.plane + (i64)(first + (lane >> 3)) * p.ld_piece + col + (lane & 7) * 8;
#pragma unroll
            for (int r = 0; r < 32; r += 4) {
              uint4 h;
              const int mine = r + (lane >> 3);
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(h.x), "=r"(h.y), "=r"(h.z), "=r"(h.w)
                           : "r"(out + mine * 128 + ((lane & 7) ^ (mine & 7)) * 16));
              // whole pieces of 8: a row has room for them (packed_ld), and nobody reads behind its last column
              if (first + mine < p.M && col + (lane & 7) * 8 < p.N) *reinterpret_cast<uint4*>(to + (i64)r * p.ld_piece) = h;
            }
          }
        }
      }
#pragma unroll (C::RUN ? 4 : 1)
      for (int own = 0; C::MODE != GM_PIECE && own < C::BN / 2; own += 32) {
        const int q = half * (C::BN / 2) + own, col = n * C::BN + q;
        if (col >= p.N) break;
        float v[32];
        columns(v, q);
        if constexpr (C::RUN != 0) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += kept[own + j];
        }
        if (blocks == 0) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0.f;
        }
        if (C::MODE == GM_STATS) {
          const int at = hot - col;
          if (__any_sync(0xffffffffu, (u32)at < 32u)) {
            float mine = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j == at) {
                mine = v[j];
                v[j] = -INFINITY;
              }
            if ((u32)at < 32u) p.hot[row] = mine;
          }
          float top = -INFINITY;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (col + j >= p.N) v[j] = -INFINITY;
            top = fmaxf(top, v[j]);
          }
          const float t = __fmul_rn(top, p.c);
          if (t > run_m + MOVE_REFERENCE) {
            run_s = run_m == -INFINITY ? run_s : run_s * ex2(run_m - t);
            run_m = t;
          }
          const float off = (float)FWD_SHIFT - (run_m == -INFINITY ? 0.f : run_m);
          float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 32; ++j) s[j & 3] += ex2(fmaf(v[j], p.c, off));
          run_s += (s[0] + s[1]) + (s[2] + s[3]);
        } else if (row < p.M) {
          float* to = p.slab + ((i64)z * p.M + row) * p.N + col;
          if (col + 32 <= p.N && (p.N & 3) == 0) {
            float4* to4 = reinterpret_cast<float4*>(to);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              float4 r = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
              if (p.add) {
                const float4 o = to4[j];
                r = make_float4(r.x + o.x, r.y + o.y, r.z + o.z, r.w + o.w);
              }
              to4[j] = r;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (col + j < p.N) to[j] = p.add ? to[j] + v[j] : v[j];
          }
        }
      }
      tc_before();
      __syncwarp();
      if (lane == 0) bar_arrive(acc_empty(b));
      ++acc;
    }
    if (C::MODE == GM_STATS && ok) {
      const int row = blockIdx.x * 128 + quarter * 32 + lane;
      if (row < p.M) p.part_ms[(i64)(blockIdx.y * 2 + half) * p.M + row] = make_float2(run_m, run_s);
    }
    tc_before();
  }
  __syncwarp();
  __syncthreads();
  tc_after();
  if (warp == 9)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((u32)C::COLS) : "memory");
}

// dst[plane][r, :] = the planes of +-src[r, :] (one plane: the values themselves), rows of ldp elements
// with zeros behind D.  Rows that do not count (g = 0) and hold what is not finite (lse2 is not, either)
// become zeros, so that it reaches no product; with top, a row takes back the power of two that its g was given.
template <typename S, typename T, int PL>
__global__ void loss_planes_kernel(const S* __restrict__ src, i64 ld, i64 rows, int D, int ldp, bool negate,
                                   const float* __restrict__ g, const float* __restrict__ lse2, const u32* __restrict__ top,
                                   T* __restrict__ dst) {
  const int chunks = ldp / 8;
  const i64 total = rows * chunks;
  for (i64 e = (i64)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (i64)gridDim.x * blockDim.x) {
    const i64 r = e / chunks;
    const int c = (int)(e - r * chunks) * 8;
    const bool live = !g || g[r] != 0.f || fabsf(lse2[r]) < INFINITY;
    const int small = top && live ? small_rows<T>(g[r], __uint_as_float(*top)) : 0;
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      v[q] = live && c + q < D ? to_float(src[r * ld + c + q]) : 0.f;
      if (negate) v[q] = -v[q];
      v[q] = times_power(v[q], small);
    }
#pragma unroll
    for (int pl = 0; pl < PL; ++pl) {
      Pack<T, 8> h;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        h.v[q] = from_float<T>(PL > 1 && pl == 0 ? first_plane(v[q]) : v[q]);
        v[q] -= to_float(h.v[q]);
      }
      h.store(dst + (i64)pl * rows * ldp + r * ldp + c);
    }
  }
}

// dx[i] = factor * (sum over the slabs + lost_i w_{t_i}); zeros for a row that does not count
template <typename T>
__global__ void loss_wide_dx_kernel(const float* __restrict__ slab, i64 N, i64 D, int slabs, float factor, const u32* __restrict__ top,
                                    const float* __restrict__ g, const float* __restrict__ lost, const i64* __restrict__ target,
                                    const T* __restrict__ w, i64 ldw, T* __restrict__ dx) {
  const float largest = __uint_as_float(*top);
  for (i64 e = (i64)blockIdx.x * blockDim.x + threadIdx.x; e < N * D; e += (i64)gridDim.x * blockDim.x) {
    const i64 r = e / D;
    float v = 0.f;
    if (g[r] != 0.f) {
      for (int z = 0; z < slabs; ++z) v += slab[z * (N * D) + e];
      if (lost) v = fmaf(lost[r], to_float(w[target[r] * ldw + (e - r * D)]), v);
      v *= factor * times_power(largest, small_rows<T>(g[r], largest));
    }
    dx[e] = from_float<T>(v);
  }
}

// out[e] = factor * sum over the slabs
template <typename T>
__global__ void loss_slabs_kernel(const float* __restrict__ slab, i64 size, int slabs, float factor, const u32* __restrict__ top,
                                  T* __restrict__ out) {
  const float f = factor * __uint_as_float(*top);
  for (i64 e = (i64)blockIdx.x * blockDim.x + threadIdx.x; e < size; e += (i64)gridDim.x * blockDim.x) {
    float v = 0.f;
    for (int z = 0; z < slabs; ++z) v += slab[z * size + e];
    out[e] = from_float<T>(v * f);
  }
}

// ---------------------------------------------------------------- host side
// A slab for every SM that would otherwise be idle, of at least 512 products; and for 16-bit types, whose
// accumulators are not emptied on the way, enough of them for RUN_TERMS products at most.
static int slab_count(int planes, i64 m, i64 n, i64 K, int bn) {
  const i64 tiles = ((m > 0 ? m + 127 : 128) / 128) * ((n + bn - 1) / bn);
  i64 z = (i64)sm_count() / tiles;
  const i64 most = K / 512;
  if (z > most) z = most;
  if (z > 64) z = 64;
  if (planes == 1 && z < (K + RUN_TERMS - 1) / RUN_TERMS) z = (K + RUN_TERMS - 1) / RUN_TERMS;
  return (int)(z < 1 ? 1 : z);
}
static i64 piece_columns(i64 N, i64 V) {
  i64 c = PIECE_ELEMS / (N < 1 ? 1 : N) / 128 * 128;
  if (c < 128) c = 128;
  return c < V ? c : V;
}
static int bn_of(int planes, i64 cols) { return planes == 3 ? (cols <= 64 ? 64 : 128) : 256; }  // dx, dW
// logits; a tile of 256 leaves no registers for the sums of several runs
static int bn_wide(int planes, i64 D) { return planes == 3 || D > RUN_TERMS ? 128 : 256; }

struct GmLayout {
  size_t ms, hot, x, x_dw, w, piece, lost, dx_slab, dw_slab, bytes;
  bool x_dw_taken;
  i64 cols, ldp;
  int dx_slabs, dw_slabs, splits, per;
};
static GmLayout gemm_layout(int dtype, i64 N, i64 V, i64 D, bool forward, bool dx, bool dw) {
  const int planes = dtype == GSB_F32 ? 3 : 1;
  GmLayout L = {};
  size_t o = 0;
  auto take = [&](size_t b) { const size_t at = o; o += up256(b); return at; };
  L.ldp = packed_ld(D);
  L.x = take(2 * (size_t)planes * N * L.ldp);
  if (forward) {
    const i64 tiles = (V + bn_wide(planes, D) - 1) / bn_wide(planes, D);
    const int s = split_count(N > 0 ? (N + 127) / 128 : 1, tiles, sm_count());
    L.per = (int)((tiles + s - 1) / s);
    L.splits = (int)((tiles + L.per - 1) / L.per);
    L.ms = take(8 * (size_t)2 * L.splits * N);
    L.hot = take(4 * (size_t)N);
  } else {
    L.cols = piece_columns(N, V);
    L.dx_slabs = slab_count(planes, N, D, L.cols, bn_of(planes, D));
    L.dw_slabs = slab_count(planes, L.cols, D, N, bn_of(planes, D));
    L.piece = take(2 * (size_t)planes * N * packed_ld(L.cols));
    L.lost = take(4 * (size_t)N);
    L.x_dw_taken = dw && dtype == GSB_F16;
    L.x_dw = take(L.x_dw_taken ? 2 * (size_t)N * L.ldp : 0);
    L.dx_slab = take(dx ? 4 * (size_t)L.dx_slabs * N * D : 0);
    L.dw_slab = take(dw ? 4 * (size_t)L.dw_slabs * L.cols * D : 0);
  }
  L.w = take(2 * (size_t)planes * V * L.ldp);
  L.bytes = o;
  return L;
}
size_t gemm_loss_workspace(int dtype, i64 N, i64 V, i64 D, bool pack_w) {
  const GmLayout L = gemm_layout(dtype, N, V, D, true, false, false);
  return dtype == GSB_F32 || pack_w ? L.bytes : L.w;
}
size_t gemm_loss_grad_workspace(int dtype, i64 N, i64 V, i64 D, bool dx, bool dw, bool pack_w) {
  const GmLayout L = gemm_layout(dtype, N, V, D, false, dx, dw);
  return dtype == GSB_F32 || pack_w ? L.bytes : L.w;
}

template <typename S>
void make_planes(const void* src, i64 ld, i64 rows, i64 D, bool negate, const float* g, const float* lse2, const u32* top, void* dst,
                 cudaStream_t st) {
  typedef typename Planes<S>::type T;
  LaunchScope ls(KID_LOSS_JOIN, st);
  loss_planes_kernel<S, T, Planes<S>::count><<<blocks_for(rows * packed_ld(D) / 8), 256, 0, st>>>(
      (const S*)src, ld, rows, (int)D, (int)packed_ld(D), negate, g, lse2, top, (T*)dst);
}

template <typename T, typename C>
static int launch_gemm(const CUtensorMap& a, const CUtensorMap& b, const GmParams& p, dim3 grid, int kid, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  if (!allow_shared(loss_gemm_kernel<T, C>, C::BYTES, done)) return GSB_ERR_CUDA;
  LaunchScope ls(kid, st);
  loss_gemm_kernel<T, C><<<grid, C::THREADS, C::BYTES, st>>>(a, b, p);
  return GSB_OK;
}
// the shape for `cols` columns of the result (dx and dW of few columns: 64 of them, with a stage more) and a depth
template <typename T, int MODE, int PL>
static int launch_mode(i64 cols, i64 depth, const CUtensorMap& a, const CUtensorMap& b, const GmParams& p, dim3 grid, int kid, cudaStream_t st) {
  if constexpr (PL == 3) {
    if constexpr (MODE == GM_DX || MODE == GM_DW)
      if (bn_of(3, cols) == 64) return launch_gemm<T, GmShape<MODE, 3, 64, 3, RUN_TERMS_F32 / 64>>(a, b, p, grid, kid, st);
    return launch_gemm<T, GmShape<MODE, 3, 128, 2, RUN_TERMS_F32 / 64>>(a, b, p, grid, kid, st);
  } else {
    if constexpr (MODE == GM_STATS || MODE == GM_PIECE)
      if (bn_wide(1, depth) == 128) return launch_gemm<T, GmShape<MODE, 1, 128, 4, RUN_TERMS / 64>>(a, b, p, grid, kid, st);
    return launch_gemm<T, GmShape<MODE, 1, 256, 4, 0>>(a, b, p, grid, kid, st);
  }
}

template <typename S>
int gemm_loss_forward(const LossArgs& a) {
  typedef typename Planes<S>::type T;
  constexpr int PL = Planes<S>::count;
  const GmLayout L = gemm_layout(dtype_of<S>(), a.N, a.V, a.D, true, false, false);
  char* ws = (char*)a.ws;
  const void *x = a.x, *w = a.w;
  i64 ldx = a.ldx, ldw = a.ldw;
  if (PL == 3 || a.scale < 0.f || !tma_ready(x, ldx)) { make_planes<S>(x, ldx, a.N, a.D, a.scale < 0.f, nullptr, nullptr, nullptr, ws + L.x, a.st); x = ws + L.x; ldx = L.ldp; }
  if (PL == 3 || !tma_ready(w, ldw)) { make_planes<S>(w, ldw, a.V, a.D, false, nullptr, nullptr, nullptr, ws + L.w, a.st); w = ws + L.w; ldw = L.ldp; }
  const int bn = bn_wide(PL, a.D);
  CUtensorMap ma, mb;
  if (!tc_map(&ma, x, IsBf16<T>::value, a.N, a.D, ldx, PL, 64, 128) || !tc_map(&mb, w, IsBf16<T>::value, a.V, a.D, ldw, PL, 64, bn)) return GSB_ERR_CUDA;
  GmParams p = {};
  p.M = (int)a.N;
  p.N = (int)a.V;
  p.K = (int)a.D;
  p.m_tiles = ceil_div_i(a.N, 128);
  p.n_tiles = ceil_div_i(a.V, bn);
  p.n_per_cta = L.per;
  p.k_per = (int)((a.D + 63) / 64 * 64);
  p.c = logit_factor(a.scale);
  p.part_ms = (float2*)(ws + L.ms);
  p.hot = (float*)(ws + L.hot);
  p.target = a.target;
  p.err = a.err;
  const int rc = launch_mode<T, GM_STATS, PL>(a.V, a.D, ma, mb, p, dim3(p.m_tiles, L.splits), KID_LOSS, a.st);
  if (rc != GSB_OK) return rc;
  launch_loss_join<S>(a, p.part_ms, 2 * L.splits, nullptr, p.hot, nullptr);
  return GSB_OK;
}

template <typename S>
int gemm_loss_backward(const LossArgs& a) {
  typedef typename Planes<S>::type T;
  constexpr int PL = Planes<S>::count;
  constexpr bool bf = IsBf16<T>::value;
  const GmLayout L = gemm_layout(dtype_of<S>(), a.N, a.V, a.D, false, a.dx != nullptr, a.dw != nullptr);
  char* ws = (char*)a.ws;
  // x for the logits, and where rows of fp16 may have small_rows' powers, with these for dW
  make_planes<S>(a.x, a.ldx, a.N, a.D, a.scale < 0.f, a.g, a.lse2, nullptr, ws + L.x, a.st);
  const T* x = (const T*)(ws + L.x);
  const T* x_dw = x;
  if (a.dw && L.x_dw_taken && a.per_row) {
    make_planes<S>(a.x, a.ldx, a.N, a.D, a.scale < 0.f, a.g, a.lse2, a.top, ws + L.x_dw, a.st);
    x_dw = (const T*)(ws + L.x_dw);
  }
  const T* w = (const T*)a.w;
  i64 ldw = a.ldw;
  if (PL == 3 || !tma_ready(w, ldw)) { make_planes<S>(a.w, a.ldw, a.V, a.D, false, nullptr, nullptr, nullptr, ws + L.w, a.st); w = (const T*)(ws + L.w); ldw = L.ldp; }
  void* piece = ws + L.piece;
  float* dxs = (float*)(ws + L.dx_slab);
  float* dws = (float*)(ws + L.dw_slab);
  const i64 ldq = packed_ld(L.cols);
  const int bn_d = bn_of(PL, a.D);
  const float unit = 1.f / (float)(1 << GRAD_SHIFT);
  auto units_grid = [&](GmParams& p, int z) {
    const i64 u = (i64)p.m_tiles * p.n_tiles * z;
    p.units = (int)u;
    return dim3((unsigned)(u < sm_count() ? u : sm_count()));
  };
  for (i64 v0 = 0; v0 < a.V; v0 += L.cols) {
    const i64 c = v0 + L.cols < a.V ? L.cols : a.V - v0;
    const T* wv = w + v0 * ldw;
    CUtensorMap ma, mb;
    {
      const int bn = bn_wide(PL, a.D);
      if (!tc_map(&ma, x, bf, a.N, a.D, L.ldp, PL, 64, 128) || !tc_map(&mb, wv, bf, c, a.D, ldw, PL, 64, bn, a.V)) return GSB_ERR_CUDA;
      GmParams p = {};
      p.M = (int)a.N;
      p.N = (int)c;
      p.K = (int)a.D;
      p.m_tiles = ceil_div_i(a.N, 128);
      p.n_tiles = ceil_div_i(c, bn);
      p.k_per = (int)((a.D + 63) / 64 * 64);
      p.c = logit_factor(a.scale);
      p.lse2 = a.lse2;
      p.g = a.g;
      p.miss = a.miss;
      p.target = a.target;
      p.top = a.top;
      p.v0 = (int)v0;
      p.piece = piece;
      p.ld_piece = ldq;
      p.plane = a.N * ldq;
      p.lost = (float*)(ws + L.lost);
      p.err = a.err;
      const dim3 grid = units_grid(p, 1);
      const int rc = launch_mode<T, GM_PIECE, PL>(c, a.D, ma, mb, p, grid, KID_LOSS_GRAD, a.st);
      if (rc != GSB_OK) return rc;
    }
    if (a.dx) {
      if (!tc_map(&ma, piece, bf, a.N, c, ldq, PL, 64, 128) || !tc_map(&mb, wv, bf, c, a.D, ldw, PL, 64, 64, a.V)) return GSB_ERR_CUDA;
      GmParams p = {};
      p.M = (int)a.N;
      p.N = (int)a.D;
      p.K = (int)c;
      p.m_tiles = ceil_div_i(a.N, 128);
      p.n_tiles = ceil_div_i(a.D, bn_d);
      p.k_per = (int)(((c + L.dx_slabs - 1) / L.dx_slabs + 63) / 64 * 64);
      p.slab = dxs;
      p.add = v0 > 0;
      p.err = a.err;
      const dim3 grid = units_grid(p, L.dx_slabs);
      const int rc = launch_mode<T, GM_DX, PL>(a.D, p.k_per, ma, mb, p, grid, KID_LOSS_GRAD, a.st);
      if (rc != GSB_OK) return rc;
    }
    if (a.dw) {
      if (!tc_map(&ma, piece, bf, a.N, c, ldq, PL, 64, 64) || !tc_map(&mb, x_dw, bf, a.N, a.D, L.ldp, PL, 64, 64)) return GSB_ERR_CUDA;
      GmParams p = {};
      p.M = (int)c;
      p.N = (int)a.D;
      p.K = (int)a.N;
      p.m_tiles = ceil_div_i(c, 128);
      p.n_tiles = ceil_div_i(a.D, bn_d);
      p.k_per = (int)(((a.N + L.dw_slabs - 1) / L.dw_slabs + 63) / 64 * 64);
      p.slab = dws;
      p.err = a.err;
      const dim3 grid = units_grid(p, L.dw_slabs);
      const int rc = launch_mode<T, GM_DW, PL>(a.D, p.k_per, ma, mb, p, grid, KID_LOSS_GRAD, a.st);
      if (rc != GSB_OK) return rc;
      LaunchScope ls(KID_LOSS_JOIN, a.st);
      loss_slabs_kernel<S><<<blocks_for(c * a.D), 256, 0, a.st>>>(dws, c * a.D, L.dw_slabs, fabsf(a.scale) * unit, a.top,
                                                                 (S*)a.dw + v0 * a.D);
    }
  }
  if (a.dx) {
    LaunchScope ls(KID_LOSS_JOIN, a.st);
    loss_wide_dx_kernel<S><<<blocks_for(a.N * a.D), 256, 0, a.st>>>(dxs, a.N, a.D, L.dx_slabs, a.scale * unit, a.top, a.g,
                                                                    PL == 1 ? (const float*)(ws + L.lost) : nullptr, a.target, (const S*)a.w,
                                                                    a.ldw, (S*)a.dx);
  }
  return GSB_OK;
}

template void make_planes<float>(const void*, i64, i64, i64, bool, const float*, const float*, const u32*, void*, cudaStream_t);
template int gemm_loss_forward<float>(const LossArgs&);
template int gemm_loss_forward<__half>(const LossArgs&);
template int gemm_loss_forward<__nv_bfloat16>(const LossArgs&);
template int gemm_loss_backward<float>(const LossArgs&);
template int gemm_loss_backward<__half>(const LossArgs&);
template int gemm_loss_backward<__nv_bfloat16>(const LossArgs&);

}  // namespace gsb
