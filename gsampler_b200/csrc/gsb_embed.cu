// Embedding lookup with scaling, and its gradient by sorted ids.
//
//   forward   out[i] = scale * W[idx[i]]          (zeros where idx[i] is the padding id)
//   gradient  dW[v]  = scale * sum over {i : idx[i] = v} of g[i], in ascending order of i
//
// The sum runs over positions sorted by (id, position), in consecutive runs whose sums are added in order, and where
// the runs are cut depends on the sizes, the type and the number of SMs alone -- not on the order in which
// anything executes, nor on addresses: same inputs, same bits.  Sums are held in 32 bits and rounded once.
// All of it is bound by memory traffic; nothing here has arithmetic to speak of.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gsb_common.cuh"
#include "gsb_types.cuh"

namespace gsb {

constexpr u32 NO_KEY = 0xFFFFFFFFu;

// ---------------------------------------------------------------- forward
// A row is D / VEC chunks of VEC elements (16 bytes where the alignment allows); consecutive
// threads take consecutive chunks, four chunks a thread with all four ids, then all four chunks
// requested before the first store, because each is a chain of two dependent loads.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
embed_rows_kernel(const T* __restrict__ w, i64 ld, i64 rows, u32 chunks, const i64* __restrict__ idx, i64 n,
                  float scale, i64 padding, T* __restrict__ out, int* err) {
  constexpr int U = 4;
  const i64 total = n * chunks, step = (i64)gridDim.x * blockDim.x;
  for (i64 g0 = (i64)blockIdx.x * blockDim.x + threadIdx.x; g0 < total; g0 += step * U) {
    i64 at[U];
    Pack<T, VEC> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const i64 g = g0 + u * step;
      at[u] = -1;
      if (g >= total) continue;
      i64 i;
      u32 c;
      if (total < (1ll << 32)) {  // a 32-bit division where it is enough
        i = (u32)g / chunks;
        c = (u32)g - (u32)i * chunks;
      } else {
        i = g / chunks;
        c = (u32)(g - i * chunks);
      }
      const i64 r = __ldg(idx + i);
      if (r != padding) {
        if (r >= 0 && r < rows) at[u] = r * ld + (i64)c * VEC;
        else raise(err, ERRBIT_BAD_INPUT);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u].clear();
      if (at[u] >= 0) v[u].load(w + at[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const i64 g = g0 + u * step;
      if (g >= total) break;
      if (scale != 1.0f) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[u].v[j] = from_float<T>(to_float(v[u].v[j]) * scale);
      }
      v[u].store(out + g * VEC);
    }
  }
}

// ---------------------------------------------------------------- sort of (id, position)
// Least significant digit first, 8 bits at most a pass, three kernels a pass: every tile of 4096 items
// counts its digits; one CTA a digit turns the tiles' counts into places; every tile ranks its items
// (warp by warp in item order, so the sort is stable), orders itself in shared memory and writes
// itself out in runs.  A pass in one kernel, the tiles passing their sums down a look-back chain, took
// 86 us for 4 M items against 33: the chain is hundreds of tiles long, a trip to L2 each sixteen.
constexpr int ST_THREADS = 512, ST_ITEMS = 8, ST_TILE = ST_THREADS * ST_ITEMS, ST_WARPS = ST_THREADS / 32;

__device__ __forceinline__ u32 key_of(i64 id, i64 rows, i64 padding, int* err) {
  if (id != padding) {
    if (id >= 0 && id < rows) return (u32)id;
    raise(err, ERRBIT_BAD_INPUT);
  }
  return (u32)rows;  // behind every real id
}

struct SortPlan {
  int passes;
  int shift[4], bits[4];
};

// counts[digit * tiles + tile]
__global__ void __launch_bounds__(ST_THREADS)
embed_digits_kernel(const i64* __restrict__ idx, i64 rows, i64 padding, const u32* __restrict__ key_in, i64 n, int shift, int bits,
                    u32* __restrict__ counts, int* err) {
  __shared__ u32 hist[256];
  const int tid = threadIdx.x;
  if (tid < 256) hist[tid] = 0;
  __syncthreads();
  const i64 base = (i64)blockIdx.x * ST_TILE;
  u32 digit[ST_ITEMS];
#pragma unroll
  for (int k = 0; k < ST_ITEMS; ++k) {
    const i64 i = base + k * ST_THREADS + tid;
    digit[k] = 256;
    if (i < n) digit[k] = ((idx ? key_of(__ldg(idx + i), rows, padding, err) : key_in[i]) >> shift) & ((1u << bits) - 1);
  }
#pragma unroll
  for (int k = 0; k < ST_ITEMS; ++k)
    if (digit[k] < 256) atomicAdd(&hist[digit[k]], 1u);
  __syncthreads();
  if (tid < 256) counts[(i64)tid * gridDim.x + blockIdx.x] = hist[tid];
}

// a CTA per digit: its tiles' counts become the sum of those before; totals[digit] = all of them
__global__ void __launch_bounds__(256)
embed_places_kernel(u32* __restrict__ counts, i64 tiles, u32* __restrict__ totals) {
  __shared__ u32 warp_tot[8];
  u32* mine = counts + (i64)blockIdx.x * tiles;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  u32 before = 0;
  for (i64 t0 = 0; t0 < tiles; t0 += 1024) {
    u32 v[4], sum = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const i64 t = t0 + threadIdx.x * 4 + q;
      v[q] = t < tiles ? mine[t] : 0;
      sum += v[q];
    }
    u32 inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const u32 o = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += o;
    }
    if (lane == 31) warp_tot[wid] = inc;
    __syncthreads();
    u32 at = before + inc - sum;
    for (int w = 0; w < wid; ++w) at += warp_tot[w];
    for (int w = 0; w < 8; ++w) before += warp_tot[w];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const i64 t = t0 + threadIdx.x * 4 + q;
      if (t < tiles) mine[t] = at;
      at += v[q];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

struct RankShared {
  unsigned short warp_hist[ST_WARPS][256];  // a warp has 256 items
  u32 local[256];                           // first place of the digit in the tile
  u32 warp_tot[9];
};

// exclusive scan of one value of each of the first 256 threads (all threads call it)
__device__ __forceinline__ u32 scan256(u32 v, u32* warp_tot) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  u32 inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    u32 t = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += t;
  }
  __syncthreads();
  if (lane == 31 && wid < 8) warp_tot[wid] = inc;
  __syncthreads();
  u32 before = 0;
#pragma unroll
  for (int w = 0; w < 7; ++w) before += w < wid ? warp_tot[w] : 0;
  return before + inc - v;
}

// Ranks the tile's items by `digit` (256 = no item).  On return place[k] is the item's place in
// the digit-ordered tile and sh.local the first place of each digit.
__device__ __forceinline__ void rank_tile(const u32 (&digit)[ST_ITEMS], u32 (&place)[ST_ITEMS], RankShared& sh) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, tid = threadIdx.x;
#pragma unroll
  for (int q = 0; q < 4; ++q) reinterpret_cast<u32*>(sh.warp_hist[wid])[q * 32 + lane] = 0;
  __syncwarp();
#pragma unroll
  for (int k = 0; k < ST_ITEMS; ++k) {
    const u32 d = digit[k];
    // the lanes with the same digit, a vote a bit (the match instruction took 4 times as long)
    unsigned same = __ballot_sync(0xffffffffu, d < 256);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const bool set = (d >> b) & 1;
      const unsigned m = __ballot_sync(0xffffffffu, set);
      same &= set ? m : ~m;
    }
    if (d < 256) place[k] = sh.warp_hist[wid][d] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (d < 256 && (same >> lane) == 1u) sh.warp_hist[wid][d] = (unsigned short)(place[k] + 1);  // the last lane of the group
    __syncwarp();
  }
  __syncthreads();
  u32 total = 0;
  if (tid < 256) {
#pragma unroll
    for (int w = 0; w < ST_WARPS; ++w) {
      const u32 c = sh.warp_hist[w][tid];
      sh.warp_hist[w][tid] = (unsigned short)total;
      total += c;
    }
  }
  const u32 first = scan256(total, sh.warp_tot);
  if (tid < 256) sh.local[tid] = first;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ST_ITEMS; ++k)
    if (digit[k] < 256) place[k] += sh.local[digit[k]] + sh.warp_hist[wid][digit[k]];
}

__global__ void __launch_bounds__(ST_THREADS)
embed_sort_pass_kernel(const i64* __restrict__ idx, i64 rows, i64 padding, const u32* __restrict__ key_in,
                       const u32* __restrict__ pos_in, u32* __restrict__ key_out, u32* __restrict__ pos_out,
                       i64 n, int shift, int bits, const u32* __restrict__ counts, const u32* __restrict__ totals) {
  __shared__ RankShared sh;
  __shared__ u32 skey[ST_TILE], spos[ST_TILE];
  __shared__ u32 start[256];  // global place of the digit's run minus its place in the tile
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const i64 base = (i64)blockIdx.x * ST_TILE;
  u32 key[ST_ITEMS], pos[ST_ITEMS], digit[ST_ITEMS], place[ST_ITEMS];
  const u32 digit_base = scan256(tid < 256 ? totals[tid] : 0, sh.warp_tot);
  const u32 before = tid < 256 ? counts[(i64)tid * gridDim.x + blockIdx.x] : 0;
#pragma unroll
  for (int k = 0; k < ST_ITEMS; ++k) {
    const i64 i = base + wid * (32 * ST_ITEMS) + k * 32 + lane;
    digit[k] = 256;
    if (i < n) {
      key[k] = idx ? key_of(__ldg(idx + i), rows, padding, nullptr) : key_in[i];
      pos[k] = idx ? (u32)i : pos_in[i];
      digit[k] = (key[k] >> shift) & ((1u << bits) - 1);
    }
  }
  rank_tile(digit, place, sh);
  if (tid < 256) start[tid] = digit_base + before - sh.local[tid];
#pragma unroll
  for (int k = 0; k < ST_ITEMS; ++k)
    if (digit[k] < 256) {
      skey[place[k]] = key[k];
      spos[place[k]] = pos[k];
    }
  __syncthreads();
  const int live = (int)(n - base < ST_TILE ? n - base : ST_TILE);
  for (int j = tid; j < live; j += ST_THREADS) {
    const u32 k = skey[j];
    const u32 to = start[(k >> shift) & ((1u << bits) - 1)] + j;
    key_out[to] = k;
    pos_out[to] = spos[j];
  }
}

// Up to one tile of items: all passes in one CTA, no counting kernel and no look-back.
__global__ void __launch_bounds__(ST_THREADS)
embed_sort_small_kernel(const i64* __restrict__ idx, i64 rows, i64 padding, u32* __restrict__ key_out,
                        u32* __restrict__ pos_out, int n, SortPlan plan, int* err) {
  __shared__ RankShared sh;
  __shared__ u32 skey[ST_TILE], spos[ST_TILE];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  u32 key[ST_ITEMS], pos[ST_ITEMS], digit[ST_ITEMS], place[ST_ITEMS];
#pragma unroll
  for (int k = 0; k < ST_ITEMS; ++k) {
    const int i = wid * (32 * ST_ITEMS) + k * 32 + lane;
    if (i < n) {
      key[k] = key_of(__ldg(idx + i), rows, padding, err);
      pos[k] = (u32)i;
    }
  }
  for (int p = 0; p < plan.passes; ++p) {
#pragma unroll
    for (int k = 0; k < ST_ITEMS; ++k) {
      const int i = wid * (32 * ST_ITEMS) + k * 32 + lane;
      digit[k] = 256;
      if (i < n) {
        if (p) { key[k] = skey[i]; pos[k] = spos[i]; }
        digit[k] = (key[k] >> plan.shift[p]) & ((1u << plan.bits[p]) - 1);
      }
    }
    rank_tile(digit, place, sh);  // its barriers separate the reads above from the writes below
#pragma unroll
    for (int k = 0; k < ST_ITEMS; ++k)
      if (digit[k] < 256) {
        skey[place[k]] = key[k];
        spos[place[k]] = pos[k];
      }
    __syncthreads();
  }
  for (int j = tid; j < n; j += ST_THREADS) {
    key_out[j] = skey[j];
    pos_out[j] = spos[j];
  }
}

// ---------------------------------------------------------------- distinct ids (sparse gradient)
// seg[i] = rank of the sorted item's id among the distinct ids (NO_KEY behind the last), ids[rank] = id.
__global__ void __launch_bounds__(256)
embed_segments_kernel(const u32* __restrict__ key, i64 n, u32 rows, u32* __restrict__ seg, i64* __restrict__ ids,
                      i64* d_num, u64* status, u32* ticket, int* err) {
  __shared__ i64 scratch[33];
  __shared__ i64 prefix_s;
  __shared__ u32 tile_s;
  constexpr int PER = 8;
  if (threadIdx.x == 0) tile_s = atomicAdd(ticket, 1u);
  __syncthreads();
  const i64 tile = tile_s, i0 = tile * 256 * PER + (i64)threadIdx.x * PER;
  u32 k[PER];
  int head[PER];
  u32 prev = (i0 > 0 && i0 <= n) ? key[i0 - 1] : NO_KEY;
  int mine = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    k[j] = i0 + j < n ? key[i0 + j] : NO_KEY;
    head[j] = k[j] < rows && k[j] != prev;
    prev = k[j];
    mine += head[j];
  }
  i64 total;
  const i64 off = block_exclusive_scan(mine, scratch, &total);
  if (threadIdx.x < 32) {
    const i64 p = chained_exclusive_prefix(status, (int)tile, total, err);
    if (threadIdx.x == 0) prefix_s = p;
  }
  __syncthreads();
  i64 rank = prefix_s + off;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (i0 + j >= n) break;
    if (head[j] && rank < n) ids[rank] = k[j];
    rank += head[j];
    seg[i0 + j] = k[j] < rows ? (u32)(rank - 1) : NO_KEY;
  }
  if (tile == (i64)gridDim.x - 1 && threadIdx.x == 255) *d_num = rank;
}

// ---------------------------------------------------------------- segmented sum
// A group of lanes owns `chunk` consecutive sorted items and walks them with the running sum of
// its columns in registers.  A segment that lies inside the chunk is finished: one rounding,
// one store.  What reaches beyond the chunk becomes a 32-bit partial row: slot 2c for a segment
// that began before chunk c, slot 2c + 1 for one that begins in it and goes on.  A second kernel adds
// the partials of a segment in the order of its chunks.  Four rows are requested before the first is
// added: bound by the latency of id -> position -> row, which the resident warps hide (4 M rows of 128
// bf16: 322 us with eight rows and fewer warps, 270 with four; ids handed round by shuffles 450).
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
embed_segsum_kernel(const u32* __restrict__ key, const u32* __restrict__ pos, i64 n, const T* __restrict__ grad, int D,
                    int log_group, int chunk, u32 limit, float scale, T* __restrict__ out, float* __restrict__ part,
                    i64 part_ld, u32* __restrict__ part_key) {
  constexpr int U = 4;
  const int lane = threadIdx.x & ((1 << log_group) - 1);
  const i64 c = ((i64)blockIdx.x * blockDim.x + threadIdx.x) >> log_group;
  const i64 begin = c * chunk;
  if (begin >= n) return;
  const i64 end = begin + chunk < n ? begin + chunk : n;
  const int col = (((int)blockIdx.y << log_group) + lane) * VEC;
  const bool live = col < D;
  auto key_at = [&](i64 i) {
    const u32 k = key[i];
    return k < limit ? k : NO_KEY;
  };
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  u32 cur = key_at(begin);
  bool began_before = cur != NO_KEY && begin > 0 && key_at(begin - 1) == cur;
  const bool goes_on_at_end = end < n && key_at(end) != NO_KEY && key_at(end) == key_at(end - 1);
  u32 from_before = NO_KEY, to_after = NO_KEY;

  auto partial = [&](int which) {
    if (!live) return;
    float* to = part + (2 * c + which) * part_ld + col;
#pragma unroll
    for (int j = 0; j < VEC; ++j) to[j] = acc[j];
  };
  auto close = [&](bool goes_on) {
    if (cur == NO_KEY) return;
    if (began_before) {
      partial(0);
      from_before = cur;
    } else if (goes_on) {
      partial(1);
      to_after = cur;
    } else if (live) {
      Pack<T, VEC> r;
#pragma unroll
      for (int j = 0; j < VEC; ++j) r.v[j] = from_float<T>(acc[j] * scale);
      r.store(out + (i64)cur * D + col);
    }
  };

  for (i64 i = begin; i < end; i += U) {
    u32 k[U];
    Pack<T, VEC> row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = i + u < end ? key_at(i + u) : NO_KEY;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k[u] != NO_KEY && live) row[u].load(grad + (i64)pos[i + u] * D + col);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= end) break;
      if (k[u] != cur) {
        close(false);
        cur = k[u];
        began_before = false;
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
      }
      if (k[u] != NO_KEY && live) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += to_float(row[u].v[j]);
      }
    }
  }
  close(goes_on_at_end);
  if (blockIdx.y == 0 && lane == 0) {
    part_key[2 * c] = from_before;
    part_key[2 * c + 1] = to_after;
  }
}

// A group per chunk in which a segment begins and goes on: adds the partials of the chunks behind it.
// Nearly all runs end within a chunk or two; a hub that fills thousands of chunks is left to the
// whole CTA, whose groups take equal shares of it that are then added in order; `shares` is the number of groups
// that rows at 16-byte boundaries have, so that NARROW accesses, with fewer groups, change no sum.
template <typename T, int VEC, bool NARROW>
__global__ void __launch_bounds__(256)
embed_join_kernel(const u32* __restrict__ part_key, const float* __restrict__ part, i64 part_ld, i64 chunks, int D, int log_group,
                  int shares, float scale, T* __restrict__ out) {
  constexpr int U = 8, SHORT = 32;
  __shared__ i64 long_run[256];
  __shared__ int longs;
  __shared__ i64 lo_s, hi_s;
  __shared__ float sums[256 * (NARROW ? 16 / sizeof(T) : VEC)];  // by share and column
  const int lane = threadIdx.x & ((1 << log_group) - 1), group = threadIdx.x >> log_group, groups = 256 >> log_group;
  const i64 c = (i64)blockIdx.x * groups + group;
  const int col = (((int)blockIdx.y << log_group) + lane) * VEC;
  const bool live = col < D;
  if (threadIdx.x == 0) longs = 0;
  __syncthreads();
  auto write = [&](u32 key, const float (&acc)[VEC]) {
    Pack<T, VEC> r;
#pragma unroll
    for (int j = 0; j < VEC; ++j) r.v[j] = from_float<T>(acc[j] * scale);
    r.store(out + (i64)key * D + col);
  };
  auto add_run = [&](float (&acc)[VEC], i64 from, i64 to, u32 key, bool look) {  // stops at another key when it has to look
    for (i64 k = from; k < to; k += U) {
      bool mine[U];
      float row[U][VEC];
#pragma unroll
      for (int u = 0; u < U; ++u) mine[u] = k + u < to && (!look || part_key[2 * (k + u)] == key);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (mine[u] && live) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) row[u][j] = part[2 * (k + u) * part_ld + col + j];
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!mine[u]) return;
        if (live) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += row[u][j];
        }
      }
    }
  };
  const u32 key = c < chunks ? part_key[2 * c + 1] : NO_KEY;
  if (key != NO_KEY) {
    if (c + SHORT < chunks && part_key[2 * (c + SHORT)] == key) {
      if (lane == 0) long_run[atomicAdd(&longs, 1)] = c;  // any order: every run has its own row
    } else {
      float acc[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] = live ? part[(2 * c + 1) * part_ld + col + j] : 0.f;
      add_run(acc, c + 1, c + SHORT < chunks ? c + SHORT : chunks, key, true);
      if (live) write(key, acc);
    }
  }
  __syncthreads();
  const int todo = longs;
  for (int q = 0; q < todo; ++q) {
    const i64 at = long_run[q];
    const u32 k0 = part_key[2 * at + 1];
    // the run's chunks are neighbours: its end by cutting the range into 256 until it is found
    i64 lo = at + 1, hi = chunks;  // chunk lo belongs to the run; hi does not, or is behind the last
    while (hi - lo > 1) {
      const i64 step = (hi - lo + 255) / 256, probe = lo + step * threadIdx.x;
      const int in = probe < hi && part_key[2 * probe] == k0;
      const int count = __syncthreads_count(in);  // threads 0 .. count - 1 are in
      if (threadIdx.x == 0) {
        lo_s = lo + step * (count - 1);
        hi_s = lo + step * count < hi ? lo + step * count : hi;
      }
      __syncthreads();
      lo = lo_s;
      hi = hi_s;
      __syncthreads();
    }
    if (!NARROW) shares = groups;
    const i64 len = hi - (at + 1), per = (len + shares - 1) / shares;
    float acc[VEC];
#pragma unroll 1
    for (int g = group; g < (NARROW ? shares : group + 1); g += groups) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
      const i64 from = at + 1 + g * per;
      add_run(acc, from, from + per < hi ? from + per : hi, k0, false);
#pragma unroll
      for (int j = 0; j < VEC; ++j) sums[((g << log_group) + lane) * VEC + j] = acc[j];
    }
    __syncthreads();
    if (group == 0 && live) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] = part[(2 * at + 1) * part_ld + col + j];
      for (int g = 0; g < shares; ++g) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += sums[((g << log_group) + lane) * VEC + j];
      }
      write(k0, acc);
    }
    __syncthreads();
  }
}

static SortPlan sort_plan(i64 rows) {
  int bits = 1;
  while (bits < 32 && (rows >> bits) != 0) ++bits;  // keys are 0 .. rows
  SortPlan p;
  p.passes = (bits + 7) / 8;
  int at = 0;
  for (int i = 0; i < 4; ++i) { p.shift[i] = 0; p.bits[i] = 1; }
  for (int i = 0; i < p.passes; ++i) {
    const int b = (bits - at + (p.passes - i) - 1) / (p.passes - i);
    p.shift[i] = at;
    p.bits[i] = b;
    at += b;
  }
  return p;
}

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// Sorted items a group takes at the first level: long chunks leave fewer partial rows (2 of
// `chunk` at worst), short ones give a small batch enough groups for every SM.
static int first_chunk(i64 n) {
  int chunk = 128;
  while (chunk > 8 && n / chunk < (i64)sm_count() * 64) chunk >>= 1;
  return chunk;
}

struct EmbedLayout {
  size_t key[2], pos[2], counts, totals, status, ticket, zero_bytes, part, part_key, bytes;
  i64 tiles, part_ld;
};

static EmbedLayout embed_layout(i64 n, i64 D, i64 rows) {
  EmbedLayout L;
  size_t o = 0;
  auto take = [&](size_t b) { const size_t at = o; o += up256(b); return at; };
  for (int k = 0; k < 2; ++k) { L.key[k] = take(4 * (size_t)n); L.pos[k] = take(4 * (size_t)n); }
  L.tiles = (n + ST_TILE - 1) / ST_TILE;
  L.counts = take(4 * 256 * (size_t)L.tiles);
  L.totals = take(4 * 256);
  L.ticket = take(4);
  L.status = take(8 * (size_t)((n + 2047) / 2048));  // look-back words of the distinct-id pass
  L.zero_bytes = o - L.ticket;
  L.part_ld = (D + 7) / 8 * 8;
  const i64 chunks = (n + first_chunk(n) - 1) / first_chunk(n);
  L.part = take(4 * (size_t)(2 * chunks) * L.part_ld);
  L.part_key = take(4 * (size_t)(2 * chunks));
  L.bytes = o;
  return L;
}

// sorts the positions by id; returns which buffer holds the result
static int launch_embed_sort(const i64* idx, i64 n, i64 rows, i64 padding, char* ws, const EmbedLayout& L,
                             int* d_err, cudaStream_t st, int* which) {
  const SortPlan plan = sort_plan(rows);
  u32* key[2] = {(u32*)(ws + L.key[0]), (u32*)(ws + L.key[1])};
  u32* pos[2] = {(u32*)(ws + L.pos[0]), (u32*)(ws + L.pos[1])};
  if (n <= ST_TILE) {
    LaunchScope ls(KID_EMBED_SORT, st);
    embed_sort_small_kernel<<<1, ST_THREADS, 0, st>>>(idx, rows, padding, key[0], pos[0], (int)n, plan, d_err);
    *which = 0;
    return GSB_OK;
  }
  u32* counts = (u32*)(ws + L.counts);
  u32* totals = (u32*)(ws + L.totals);
  for (int p = 0; p < plan.passes; ++p) {
    const i64* ids = p == 0 ? idx : nullptr;
    const u32 *key_in = key[(p + 1) & 1], *pos_in = pos[(p + 1) & 1];
    {
      LaunchScope ls(KID_EMBED_SORT, st);
      embed_digits_kernel<<<(int)L.tiles, ST_THREADS, 0, st>>>(ids, rows, padding, key_in, n, plan.shift[p], plan.bits[p], counts, d_err);
    }
    {
      LaunchScope ls(KID_EMBED_SORT, st);
      embed_places_kernel<<<256, 256, 0, st>>>(counts, L.tiles, totals);
    }
    LaunchScope ls(KID_EMBED_SORT, st);
    embed_sort_pass_kernel<<<(int)L.tiles, ST_THREADS, 0, st>>>(ids, rows, padding, key_in, pos_in, key[p & 1], pos[p & 1], n,
                                                                plan.shift[p], plan.bits[p], counts, totals);
  }
  *which = (plan.passes - 1) & 1;
  return GSB_OK;
}

// elements a thread moves at once: 16 bytes where row width and addresses allow
static int vec_of(const void* a, const void* b, i64 D, i64 ld, int size) {
  const uintptr_t m = (uintptr_t)a | (uintptr_t)b | (uintptr_t)(D * size) | (uintptr_t)(ld * size);
  int bytes = 16;
  while (bytes > size && (m & (uintptr_t)(bytes - 1))) bytes >>= 1;
  return bytes / size;
}
// log2 of the lanes that take a row of D elements, vec each
static int log_lanes(i64 D, int vec) {
  int lg = 0;
  while (lg < 5 && (1 << lg) < D / vec) ++lg;
  return lg;
}

template <typename T, int VEC>
static void launch_segsum(const u32* key, const u32* pos, i64 n, const void* grad, i64 D, u32 limit, float scale,
                          void* out, char* ws, const EmbedLayout& L, cudaStream_t st) {
  float* part = (float*)(ws + L.part);
  u32* part_key = (u32*)(ws + L.part_key);
  const int chunk = first_chunk(n);
  const i64 chunks = (n + chunk - 1) / chunk, per_row = D / VEC;
  const int widest = vec_of(nullptr, nullptr, D, D, sizeof(T)), lg = log_lanes(D, VEC), shares = 256 >> log_lanes(D, widest);
  const dim3 grid((unsigned)(((chunks << lg) + 255) / 256), (unsigned)((per_row + (1 << lg) - 1) >> lg));
  {
    LaunchScope ls(KID_EMBED_GRAD, st);
    embed_segsum_kernel<T, VEC><<<grid, 256, 0, st>>>(key, pos, n, (const T*)grad, (int)D, lg, chunk, limit, scale, (T*)out, part,
                                                      L.part_ld, part_key);
  }
  if (chunks > 1) {
    LaunchScope ls(KID_EMBED_GRAD, st);
    if (VEC * sizeof(T) < 16 && VEC < widest)
      embed_join_kernel<T, VEC, (VEC * sizeof(T) < 16)><<<grid, 256, 0, st>>>(part_key, part, L.part_ld, chunks, (int)D, lg, shares, scale, (T*)out);
    else
      embed_join_kernel<T, VEC, false><<<grid, 256, 0, st>>>(part_key, part, L.part_ld, chunks, (int)D, lg, shares, scale, (T*)out);
  }
}

}  // namespace gsb

using namespace gsb;

template <typename T, int VEC>
static void run_rows(const void* w, i64 ld, i64 rows, i64 D, const i64* idx, i64 n, float scale, i64 padding,
                     void* out, int* d_err, cudaStream_t st) {
  const i64 chunks = D / VEC;
  i64 blocks = (n * chunks + 1023) / 1024;
  if (blocks > (i64)sm_count() * 32) blocks = (i64)sm_count() * 32;
  LaunchScope ls(KID_EMBED, st);
  embed_rows_kernel<T, VEC><<<(int)blocks, 256, 0, st>>>((const T*)w, ld, rows, (u32)chunks, idx, n, scale, padding,
                                                         (T*)out, d_err);
}

extern "C" int gsb_embedding(const void* weight, int dtype, int64_t ld, int64_t rows, int64_t D, const int64_t* idx,
                             int64_t n, float scale, int64_t padding, void* out, int* d_err, void* cuda_stream) {
  if (n < 0 || rows < 0 || D < 0 || D > GSB_EMBED_MAX_D || (rows > 1 && ld < D) || !(scale - scale == 0.f)) return GSB_ERR_INVALID;
  if (n == 0 || D == 0) return GSB_OK;
  if (!idx || !out || (rows > 0 && !weight)) return GSB_ERR_INVALID;
  if (!at_multiple(weight, value_bytes(dtype)) || !at_multiple(out, value_bytes(dtype)) || !at_multiple(idx, 8) || !at_multiple(d_err, 4))
    return GSB_ERR_INVALID;
  cudaStream_t st = (cudaStream_t)cuda_stream;
  const i64* ix = (const i64*)idx;
#define GSB_ROWS(T, V) run_rows<T, V>(weight, ld, rows, D, ix, n, scale, padding, out, d_err, st)
  if (dtype == GSB_F32) {
    switch (vec_of(weight, out, D, ld, 4)) { case 4: GSB_ROWS(float, 4); break; case 2: GSB_ROWS(float, 2); break; default: GSB_ROWS(float, 1); }
  } else if (dtype == GSB_F16) {
    switch (vec_of(weight, out, D, ld, 2)) { case 8: GSB_ROWS(__half, 8); break; case 4: GSB_ROWS(__half, 4); break; case 2: GSB_ROWS(__half, 2); break; default: GSB_ROWS(__half, 1); }
  } else if (dtype == GSB_BF16) {
    switch (vec_of(weight, out, D, ld, 2)) { case 8: GSB_ROWS(__nv_bfloat16, 8); break; case 4: GSB_ROWS(__nv_bfloat16, 4); break; case 2: GSB_ROWS(__nv_bfloat16, 2); break; default: GSB_ROWS(__nv_bfloat16, 1); }
  } else {
    return GSB_ERR_INVALID;
  }
#undef GSB_ROWS
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}

static bool embed_sizes_ok(i64 n, i64 rows, i64 D) {
  return n >= 0 && n < (1ll << 31) && rows >= 0 && rows < (i64)NO_KEY && D >= 0 && D <= GSB_EMBED_MAX_D;
}

extern "C" size_t gsb_embedding_grad_workspace_bytes(int64_t n, int64_t rows, int64_t D) {
  if (!embed_sizes_ok(n, rows, D)) return 0;
  return embed_layout(n, D, rows).bytes;
}

static void segsum_any(int dtype, const u32* key, const u32* pos, i64 n, const void* grad, i64 D, u32 limit,
                       float scale, void* out, char* ws, const EmbedLayout& L, cudaStream_t st) {
#define GSB_SUM(T, V) launch_segsum<T, V>(key, pos, n, grad, D, limit, scale, out, ws, L, st)
  if (dtype == GSB_F32) {
    switch (vec_of(grad, out, D, D, 4)) { case 4: GSB_SUM(float, 4); break; case 2: GSB_SUM(float, 2); break; default: GSB_SUM(float, 1); }
  } else if (dtype == GSB_F16) {
    switch (vec_of(grad, out, D, D, 2)) { case 8: GSB_SUM(__half, 8); break; case 4: GSB_SUM(__half, 4); break; case 2: GSB_SUM(__half, 2); break; default: GSB_SUM(__half, 1); }
  } else {
    switch (vec_of(grad, out, D, D, 2)) { case 8: GSB_SUM(__nv_bfloat16, 8); break; case 4: GSB_SUM(__nv_bfloat16, 4); break; case 2: GSB_SUM(__nv_bfloat16, 2); break; default: GSB_SUM(__nv_bfloat16, 1); }
  }
#undef GSB_SUM
}

extern "C" int gsb_embedding_grad(const void* grad, int dtype, int64_t D, const int64_t* idx, int64_t n, int64_t rows,
                                  float scale, int64_t padding, void* out, void* workspace, size_t workspace_bytes,
                                  int* d_err, void* cuda_stream) {
  if (!embed_sizes_ok(n, rows, D) || !(scale - scale == 0.f) || (dtype != GSB_F32 && dtype != GSB_F16 && dtype != GSB_BF16)) return GSB_ERR_INVALID;
  if (rows == 0 || D == 0) return GSB_OK;
  if (!out || (n > 0 && (!grad || !idx))) return GSB_ERR_INVALID;
  if (!at_multiple(grad, value_bytes(dtype)) || !at_multiple(out, value_bytes(dtype)) || !at_multiple(idx, 8) ||
      !at_multiple(workspace, 16) || !at_multiple(d_err, 4))
    return GSB_ERR_INVALID;
  cudaStream_t st = (cudaStream_t)cuda_stream;
  GSB_CUDA_OK(cudaMemsetAsync(out, 0, (size_t)rows * D * (dtype == GSB_F32 ? 4 : 2), st));
  if (n == 0) return GSB_OK;
  const EmbedLayout L = embed_layout(n, D, rows);
  if (!workspace || workspace_bytes < L.bytes) return GSB_ERR_WORKSPACE;
  char* ws = (char*)workspace;
  int which = 0;
  launch_embed_sort((const i64*)idx, n, rows, padding, ws, L, d_err, st, &which);
  segsum_any(dtype, (u32*)(ws + L.key[which]), (u32*)(ws + L.pos[which]), n, grad, D, (u32)rows, scale, out, ws, L, st);
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}

extern "C" int gsb_embedding_sort(const int64_t* idx, int64_t n, int64_t rows, int64_t D, int64_t padding, int64_t* ids,
                                  int64_t* d_num, void* workspace, size_t workspace_bytes, int* d_err,
                                  void* cuda_stream) {
  if (!embed_sizes_ok(n, rows, D) || n == 0 || !idx || !ids || !d_num) return GSB_ERR_INVALID;
  if (!at_multiple(idx, 8) || !at_multiple(ids, 8) || !at_multiple(d_num, 8) || !at_multiple(workspace, 16) || !at_multiple(d_err, 4))
    return GSB_ERR_INVALID;
  const EmbedLayout L = embed_layout(n, D, rows);
  if (!workspace || workspace_bytes < L.bytes) return GSB_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)cuda_stream;
  char* ws = (char*)workspace;
  GSB_CUDA_OK(cudaMemsetAsync(ws + L.ticket, 0, L.zero_bytes, st));
  int which = 0;
  launch_embed_sort((const i64*)idx, n, rows, padding, ws, L, d_err, st, &which);
  u64* status = (u64*)(ws + L.status);
  {
    LaunchScope ls(KID_EMBED_SORT, st);
    // the ranks take the place of the other key buffer
    embed_segments_kernel<<<(int)((n + 2047) / 2048), 256, 0, st>>>(
        (u32*)(ws + L.key[which]), n, (u32)rows, (u32*)(ws + L.key[which ^ 1]), (i64*)ids, (i64*)d_num, status,
        (u32*)(ws + L.ticket), d_err);
  }
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}

extern "C" int gsb_embedding_grad_rows(const void* grad, int dtype, int64_t D, int64_t n, int64_t rows, int64_t num,
                                       float scale, void* out, void* workspace, size_t workspace_bytes,
                                       void* cuda_stream) {
  if (!embed_sizes_ok(n, rows, D) || num < 0 || num > n || !(scale - scale == 0.f) || (dtype != GSB_F32 && dtype != GSB_F16 && dtype != GSB_BF16))
    return GSB_ERR_INVALID;
  if (num == 0 || D == 0) return GSB_OK;
  if (!grad || !out) return GSB_ERR_INVALID;
  if (!at_multiple(grad, value_bytes(dtype)) || !at_multiple(out, value_bytes(dtype)) || !at_multiple(workspace, 16))
    return GSB_ERR_INVALID;
  const EmbedLayout L = embed_layout(n, D, rows);
  if (!workspace || workspace_bytes < L.bytes) return GSB_ERR_WORKSPACE;
  char* ws = (char*)workspace;
  const int which = n <= ST_TILE ? 0 : (sort_plan(rows).passes - 1) & 1;
  segsum_any(dtype, (u32*)(ws + L.key[which ^ 1]), (u32*)(ws + L.pos[which]), n, grad, D, (u32)num, scale, out, ws, L,
             (cudaStream_t)cuda_stream);
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}
