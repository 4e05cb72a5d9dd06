// Softmax cross entropy of x W^T over a vocabulary of V rows, without keeping the logits:
//
//   l_ij = s x_i . w_j      lse_i = log sum_j exp l_ij      loss_i = lse_i - l_{i,t_i}
//   dx_i = g_i s (sum_j p_ij w_j - w_{t_i})     dW_j = s sum_i g_i (p_ij - [t_i = j]) x_i
//   p_ij = exp(l_ij - lse_i)
//
// This file has the form that takes every type and width (gsb_loss_tc.cu has the one for 16-bit
// types of up to 256 columns): products by 32-bit multiply-adds on 128 x 64 tiles.  The forward pass runs over the vocabulary once with the running maximum and
// sum of every row.  The backward pass takes the vocabulary in pieces: the logits of a piece are
// computed again, turned into g (p - target) in a workspace of at most PIECE_ELEMS values, and
// multiplied with W (for dx) and with x (for dW).  Bound by the 32-bit multiply-add rate.
// Long sums are split over CTAs into slabs that are added in a fixed order, never by atomics.
#include "gsb_common.cuh"
#include "gsb_loss.cuh"
#include "gsb_types.cuh"

namespace gsb {

constexpr int BM = 128, BN = 64, BK = 16;
constexpr i64 PIECE_ELEMS = 1ll << 26;

// One BK-deep slice of an operand into shared memory as [k][row].  Element (row, k) lies at
// p[row * ld + k] when KMAJOR, else at p[k * ld + row].  Zeros outside [0, rows) x [k0, k1), and
// for every k whose `live` is zero (rows that do not count may hold NaN).
template <typename T, bool KMAJOR, int ROWS>
struct SliceLoader {
  static constexpr int PER = ROWS * BK / 256;
  float v[PER];
  __device__ __forceinline__ void load(const T* __restrict__ p, i64 ld, i64 row0, i64 rows, i64 k0, i64 k1,
                                       const float* __restrict__ live) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = KMAJOR ? tid * PER + j : j * 256 + tid;
      const i64 r = row0 + (KMAJOR ? e / BK : e % ROWS);
      const i64 k = k0 + (KMAJOR ? e % BK : e / ROWS);
      const bool take = r < rows && k < k1 && (!live || live[k] != 0.f);
      v[j] = take ? to_float(p[KMAJOR ? r * ld + k : k * ld + r]) : 0.f;
    }
  }
  __device__ __forceinline__ void put(float (*s)[ROWS + 4]) const {
    const int tid = threadIdx.x;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = KMAJOR ? tid * PER + j : j * 256 + tid;
      if (KMAJOR) s[e % BK][e / BK] = v[j];
      else s[e / ROWS][e % ROWS] = v[j];
    }
  }
};

template <typename TA, typename TB, bool AK, bool BKM>
struct Tile {
  float a[2][BK][BM + 4], b[2][BK][BN + 4];
  // acc[8][4]: rows ty * 8 .., columns tx * 4 ..
  __device__ __forceinline__ void product(float (&acc)[8][4], const TA* A, i64 lda, i64 m0, i64 M, const TB* B,
                                          i64 ldb, i64 n0, i64 N, i64 k0, i64 k1,
                                          const float* live = nullptr) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    SliceLoader<TA, AK, BM> la;
    SliceLoader<TB, BKM, BN> lb;
    __syncthreads();
    if (k0 >= k1) return;
    la.load(A, lda, m0, M, k0, k1, nullptr);
    lb.load(B, ldb, n0, N, k0, k1, live);
    la.put(a[0]);
    lb.put(b[0]);
    __syncthreads();
    int cur = 0;
    for (i64 k = k0; k < k1; k += BK) {
      const bool more = k + BK < k1;
      if (more) {
        la.load(A, lda, m0, M, k + BK, k1, nullptr);
        lb.load(B, ldb, n0, N, k + BK, k1, live);
      }
#pragma unroll
      for (int kk = 0; kk < BK; ++kk) {
        float ra[8], rb[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) ra[i] = a[cur][kk][ty * 8 + i];
#pragma unroll
        for (int j = 0; j < 4; ++j) rb[j] = b[cur][kk][tx * 4 + j];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(ra[i], rb[j], acc[i][j]);
      }
      if (more) {
        la.put(a[cur ^ 1]);
        lb.put(b[cur ^ 1]);
        __syncthreads();
        cur ^= 1;
      }
    }
  }
};

// ---------------------------------------------------------------- forward statistics
// CTA = 128 rows x a range of column tiles; running maximum and sum (base 2) of its rows.
template <typename T>
__global__ void __launch_bounds__(256)
loss_stats_kernel(const T* __restrict__ x, i64 ldx, i64 N, const T* __restrict__ w, i64 ldw, i64 V, i64 D, float scale2,
                  i64 cols_per_split, float2* __restrict__ part) {
  __shared__ Tile<T, T, true, true> tile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const i64 m0 = (i64)blockIdx.x * BM;
  const i64 v0 = (i64)blockIdx.y * cols_per_split, v1 = v0 + cols_per_split < V ? v0 + cols_per_split : V;
  float m[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { m[i] = -INFINITY; s[i] = 0.f; }
  for (i64 v = v0; v < v1; v += BN) {
    float acc[8][4];
    tile.product(acc, x, ldx, m0, N, w, ldw, v, v1, 0, D);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[i][j] = v + tx * 4 + j < v1 ? acc[i][j] * scale2 : -INFINITY;
        top = max_nan(top, acc[i][j]);  // a NaN logit is not lost in the maximum
      }
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float m2 = max_nan(m[i], top);
      float add = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) add += acc[i][j] == -INFINITY ? 0.f : exp2f(acc[i][j] - m2);
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) add += __shfl_xor_sync(0xffffffffu, add, d);
      s[i] = (m[i] == -INFINITY ? 0.f : s[i] * exp2f(m[i] - m2)) + add;
      m[i] = m2;
    }
  }
  if (tx == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const i64 r = m0 + ty * 8 + i;
      if (r < N) part[(i64)blockIdx.y * N + r] = make_float2(m[i], s[i]);
    }
  }
}

// ---------------------------------------------------------------- probabilities of a piece
// prob[i, j - v0] = g_i (p_ij - [t_i = j])
template <typename T>
__global__ void __launch_bounds__(256)
loss_prob_kernel(const T* __restrict__ x, i64 ldx, i64 N, const T* __restrict__ w, i64 ldw, i64 v0, i64 v1, i64 D,
                 float scale2, const float* __restrict__ lse2, const float* __restrict__ g,
                 const i64* __restrict__ target, float* __restrict__ prob, i64 ldp) {
  __shared__ Tile<T, T, true, true> tile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const i64 m0 = (i64)blockIdx.x * BM, v = v0 + (i64)blockIdx.y * BN;
  float acc[8][4];
  tile.product(acc, x, ldx, m0, N, w, ldw, v, v1, 0, D);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const i64 r = m0 + ty * 8 + i;
    if (r >= N) break;
    const float gi = g[r], le = lse2[r];
    const i64 t = target[r];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const i64 c = v + tx * 4 + j;
      // a row that does not count is zero whatever its values are
      if (c < v1) prob[r * ldp + (c - v0)] = gi == 0.f ? 0.f : gi * (exp2f(acc[i][j] * scale2 - le) - (c == t ? 1.f : 0.f));
    }
  }
}

// ---------------------------------------------------------------- products with a piece
// slab[z][M][N] (+)= A B over the z-th range of k
template <typename TA, typename TB, bool AK, bool BKM>
__global__ void __launch_bounds__(256)
loss_product_kernel(const TA* __restrict__ A, i64 lda, i64 M, const TB* __restrict__ B, i64 ldb, i64 N, i64 K, i64 k_per,
                    const float* __restrict__ live, int add, float* __restrict__ slab) {
  __shared__ Tile<TA, TB, AK, BKM> tile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const i64 m0 = (i64)blockIdx.x * BM, n0 = (i64)blockIdx.y * BN, k0 = (i64)blockIdx.z * k_per;
  const i64 k1 = k0 + k_per < K ? k0 + k_per : K;
  float acc[8][4];
  tile.product(acc, A, lda, m0, M, B, ldb, n0, N, k0, k1, live);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const i64 r = m0 + ty * 8 + i;
    if (r >= M) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const i64 c = n0 + tx * 4 + j;
      if (c >= N) break;
      float* to = slab + ((i64)blockIdx.z * M + r) * N + c;
      *to = add ? *to + acc[i][j] : acc[i][j];
    }
  }
}

// out[e] = scale * sum over the slabs; rows whose `live` is zero are zeros
template <typename T>
__global__ void loss_slabs_kernel(const float* __restrict__ slab, i64 size, int slabs, float scale,
                                  const float* __restrict__ live, i64 D, T* __restrict__ out) {
  for (i64 e = (i64)blockIdx.x * blockDim.x + threadIdx.x; e < size; e += (i64)gridDim.x * blockDim.x) {
    float v = 0.f;
    if (!live || live[e / D] != 0.f)
      for (int z = 0; z < slabs; ++z) v += slab[z * size + e];
    out[e] = from_float<T>(v * scale);
  }
}

// ---------------------------------------------------------------- small kernels
// A warp per row: joins the splits' statistics, adds the target's logit.  lse2 is in base 2.
template <typename T>
__global__ void __launch_bounds__(256)
loss_rows_kernel(const float2* __restrict__ part, int splits, const T* __restrict__ x, i64 ldx, i64 N,
                 const T* __restrict__ w, i64 ldw, i64 V, i64 D, float scale, const i64* __restrict__ target, i64 ignore,
                 float* __restrict__ loss, float* __restrict__ lse2, int* err) {
  const i64 r = ((i64)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (r >= N) return;
  float m = -INFINITY;
  for (int k = lane; k < splits; k += 32) m = max_nan(m, part[(i64)k * N + r].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
  float s = 0.f;
  for (int k = lane; k < splits; k += 32) {
    const float2 p = part[(i64)k * N + r];
    if (p.x != -INFINITY) s += p.y * exp2f(p.x - m);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  const float total = m + log2f(s);
  const i64 t = target[r];
  const bool counts = t != ignore && t >= 0 && t < V;
  if (t != ignore && !counts && lane == 0) raise(err, ERRBIT_BAD_INPUT);
  float dot = 0.f;
  if (counts)
    for (i64 d = lane; d < D; d += 32) dot = fmaf(to_float(x[r * ldx + d]), to_float(w[t * ldw + d]), dot);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
  if (lane == 0) {
    lse2[r] = total;
    loss[r] = counts ? total * 0.6931471805599453f - dot * scale : 0.f;
  }
}

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

// ---------------------------------------------------------------- host side
static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

static int stat_splits(i64 N, i64 V) {
  const i64 rows = N > 0 ? (N + BM - 1) / BM : 1, cols = (V + BN - 1) / BN;
  i64 s = ((i64)sm_count() * 4 + rows - 1) / rows;
  if (s > cols) s = cols;
  return (int)(s < 1 ? 1 : s);
}
static i64 piece_columns(i64 N, i64 V) {
  i64 c = PIECE_ELEMS / (N < 1 ? 1 : N) / BN * BN;
  if (c < BN) c = BN;
  if (c > (1 << 21)) c = 1 << 21;  // a launch has at most 65535 tiles along the vocabulary
  return c < V ? c : V;
}
static int product_slabs(i64 M, i64 N, i64 K) {
  const i64 tiles = ((M > 0 ? M + BM - 1 : BM) / BM) * ((N + BN - 1) / BN);
  i64 z = ((i64)sm_count() * 3 + tiles - 1) / tiles;
  const i64 most = (K + 255) / 256;  // at least 256 products a slab
  if (z > most) z = most;
  if (z > 64) z = 64;
  return (int)(z < 1 ? 1 : z);
}

struct GradLayout {
  size_t prob, dx_slab, dw_slab, bytes;
  i64 cols;
  int dx_slabs, dw_slabs;
};
static GradLayout grad_layout(i64 N, i64 V, i64 D, bool dx, bool dw) {
  GradLayout L;
  size_t o = 0;
  auto take = [&](size_t b) { const size_t at = o; o += up256(b); return at; };
  L.cols = piece_columns(N, V);
  L.dx_slabs = product_slabs(N, D, L.cols);
  L.dw_slabs = product_slabs(L.cols, D, N);
  L.prob = take(4 * (size_t)N * L.cols);
  L.dx_slab = take(dx ? 4 * (size_t)L.dx_slabs * N * D : 0);
  L.dw_slab = take(dw ? 4 * (size_t)L.dw_slabs * L.cols * D : 0);
  L.bytes = o;
  return L;
}

size_t simt_loss_workspace(i64 N, i64 V, i64 D) {
  (void)D;
  return up256(8 * (size_t)stat_splits(N, V) * N);
}
size_t simt_loss_grad_workspace(i64 N, i64 V, i64 D, bool dx, bool dw) { return grad_layout(N, V, D, dx, dw).bytes; }

template <typename T>
static void launch_rows(const LossArgs& a, const float2* part, int splits) {
  LaunchScope ls(KID_LOSS_JOIN, a.st);
  loss_rows_kernel<T><<<ceil_div_i(a.N, 8), 256, 0, a.st>>>(part, splits, (const T*)a.x, a.ldx, a.N, (const T*)a.w, a.ldw,
                                                           a.V, a.D, a.scale, a.target, a.ignore, a.loss, a.lse2, a.err);
}

template <typename T>
static void simt_forward(const LossArgs& a) {
  const int splits = stat_splits(a.N, a.V);
  const i64 tiles = (a.V + BN - 1) / BN, per = (tiles + splits - 1) / splits * BN;
  float2* part = (float2*)a.ws;
  {
    LaunchScope ls(KID_LOSS, a.st);
    loss_stats_kernel<T><<<dim3(ceil_div_i(a.N, BM), splits), 256, 0, a.st>>>(
        (const T*)a.x, a.ldx, a.N, (const T*)a.w, a.ldw, a.V, a.D, a.scale * LOG2E, per, part);
  }
  launch_rows<T>(a, part, splits);
}

template <typename T>
static void simt_backward(const LossArgs& a) {
  const GradLayout L = grad_layout(a.N, a.V, a.D, a.dx != nullptr, a.dw != nullptr);
  char* ws = (char*)a.ws;
  float* prob = (float*)(ws + L.prob);
  float* dxs = (float*)(ws + L.dx_slab);
  float* dws = (float*)(ws + L.dw_slab);
  const T* x = (const T*)a.x;
  const T* w = (const T*)a.w;
  auto blocks = [](i64 n) { const i64 b = (n + 255) / 256, most = (i64)sm_count() * 16; return (int)(b < most ? b : most); };
  for (i64 v0 = 0; v0 < a.V; v0 += L.cols) {
    const i64 v1 = v0 + L.cols < a.V ? v0 + L.cols : a.V, c = v1 - v0;
    {
      LaunchScope ls(KID_LOSS_GRAD, a.st);
      loss_prob_kernel<T><<<dim3(ceil_div_i(a.N, BM), ceil_div_i(c, BN)), 256, 0, a.st>>>(
          x, a.ldx, a.N, w, a.ldw, v0, v1, a.D, a.scale * LOG2E, a.lse2, a.g, a.target, prob, L.cols);
    }
    if (a.dx) {
      const i64 per = ((c + L.dx_slabs - 1) / L.dx_slabs + BK - 1) / BK * BK;
      LaunchScope ls(KID_LOSS_GRAD, a.st);
      loss_product_kernel<float, T, true, false><<<dim3(ceil_div_i(a.N, BM), ceil_div_i(a.D, BN), L.dx_slabs), 256, 0, a.st>>>(
          prob, L.cols, a.N, w + v0 * a.ldw, a.ldw, a.D, c, per, nullptr, v0 > 0, dxs);
    }
    if (a.dw) {
      const i64 per = ((a.N + L.dw_slabs - 1) / L.dw_slabs + BK - 1) / BK * BK;
      {
        LaunchScope ls(KID_LOSS_GRAD, a.st);
        loss_product_kernel<float, T, false, false><<<dim3(ceil_div_i(c, BM), ceil_div_i(a.D, BN), L.dw_slabs), 256, 0, a.st>>>(
            prob, L.cols, c, x, a.ldx, a.D, a.N, per, a.g, 0, dws);
      }
      LaunchScope ls(KID_LOSS_JOIN, a.st);
      loss_slabs_kernel<T><<<blocks(c * a.D), 256, 0, a.st>>>(dws, c * a.D, L.dw_slabs, a.scale, nullptr, a.D, (T*)a.dw + v0 * a.D);
    }
  }
  if (a.dx) {
    LaunchScope ls(KID_LOSS_JOIN, a.st);
    loss_slabs_kernel<T><<<blocks(a.N * a.D), 256, 0, a.st>>>(dxs, a.N * a.D, L.dx_slabs, a.scale, a.g, a.D, (T*)a.dx);
  }
}

}  // namespace gsb

using namespace gsb;

static bool loss_sizes_ok(i64 N, i64 V, i64 D, i64 ldx, i64 ldw) {
  return N >= 0 && N < (1ll << 31) && V >= 1 && V < (1ll << 31) && D >= 1 && D <= GSB_LOSS_MAX_D && (N < 2 || ldx >= D) &&
         (V < 2 || ldw >= D);
}

extern "C" int gsb_linear_ce_has_pull(int dtype, int64_t N, int64_t V, int64_t D) { return tc_loss_takes(dtype, N, V, D); }

extern "C" size_t gsb_linear_ce_workspace_bytes(int dtype, const void* weight, int64_t ldw, int64_t N, int64_t V, int64_t D,
                                                int want_pull) {
  if (!loss_sizes_ok(N, V, D, D, D)) return 0;
  if (tc_loss_takes(dtype, N, V, D)) return tc_loss_workspace(N, V, D, want_pull != 0, tc_loss_packs(weight, ldw));
  return simt_loss_workspace(N, V, D);
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
  else if (dtype == GSB_F32) simt_forward<float>(a);
  else if (dtype == GSB_F16) simt_forward<__half>(a);
  else simt_forward<__nv_bfloat16>(a);
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
  const bool simt_dx = want_dx && !(tc && have_pull), simt_dw = want_dw && !tc;
  size_t need = simt_dx || simt_dw ? simt_loss_grad_workspace(N, V, D, simt_dx, simt_dw) : 0;
  if (tc && want_dw) {
    const size_t b = tc_loss_grad_workspace(N, V, D, tc_loss_packs(weight, ldw));
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
    if (dtype == GSB_F32) simt_backward<float>(a);
    else if (dtype == GSB_F16) simt_backward<__half>(a);
    else simt_backward<__nv_bfloat16>(a);
  }
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}
