// Embedding lookup with scaling, and its gradient by sorted ids.
//
//   forward   out[i] = scale * W[idx[i]]          (zeros where idx[i] is the padding id)
//   gradient  dW[v]  = scale * sum over {i : idx[i] = v} of g[i], in ascending order of i
//
// The sum runs over positions sorted by (id, position), so it does not depend on the order in
// which anything executes: same inputs, same bits.  Sums are held in 32 bits and rounded once.
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
// Least significant digit first, 8 bits at most a pass, one kernel a pass: a tile of 4096 items
// ranks its items (warp by warp in item order, so the sort is stable), learns from its
// predecessors where its run of each digit starts (one look-back chain per digit, a thread each;
// the tiles take tickets so that a predecessor is always running or done), orders the tile in
// shared memory and writes it out in runs.  One kernel before all passes counts every digit.
constexpr int ST_THREADS = 256, ST_ITEMS = 16, ST_TILE = ST_THREADS * ST_ITEMS, ST_WARPS = ST_THREADS / 32;

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

__global__ void __launch_bounds__(256)
embed_digits_kernel(const i64* __restrict__ idx, i64 n, i64 rows, i64 padding, SortPlan plan,
                    u32* __restrict__ counts, int* err) {
  __shared__ u32 hist[4][256];
  for (int j = threadIdx.x; j < 1024; j += 256) (&hist[0][0])[j] = 0;
  __syncthreads();
  for (i64 i = (i64)blockIdx.x * 256 + threadIdx.x; i < n; i += (i64)gridDim.x * 256) {
    const u32 k = key_of(__ldg(idx + i), rows, padding, err);
    for (int p = 0; p < plan.passes; ++p)
      atomicAdd(&hist[p][(k >> plan.shift[p]) & ((1u << plan.bits[p]) - 1)], 1u);
  }
  __syncthreads();
  for (int j = threadIdx.x; j < plan.passes * 256; j += 256) {
    const u32 c = (&hist[0][0])[j];
    if (c) atomicAdd(counts + j, c);
  }
}

struct RankShared {
  u32 warp_hist[ST_WARPS][256];
  u32 local[256];  // first place of the digit in the tile
  u32 warp_tot[33];
};

// exclusive scan of one u32 a thread over 256 threads
__device__ __forceinline__ u32 scan256(u32 v, u32* warp_tot) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  u32 inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    u32 t = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += t;
  }
  __syncthreads();
  if (lane == 31) warp_tot[wid] = inc;
  __syncthreads();
  u32 before = 0;
  for (int w = 0; w < wid; ++w) before += warp_tot[w];
  return before + inc - v;
}

// Ranks the tile's items by `digit` (256 = no item).  On return place[k] is the item's place in
// the digit-ordered tile and sh.local the first place of each digit; returns the count of digit
// threadIdx.x.
__device__ __forceinline__ u32 rank_tile(const u32 (&digit)[ST_ITEMS], u32 (&place)[ST_ITEMS], RankShared& sh) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, tid = threadIdx.x;
  for (int w = 0; w < ST_WARPS; ++w) sh.warp_hist[w][tid] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ST_ITEMS; ++k) {
    const u32 d = digit[k];
    unsigned same = __ballot_sync(0xffffffffu, d < 256);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const unsigned m = __ballot_sync(0xffffffffu, (d >> b) & 1);
      same &= ((d >> b) & 1) ? m : ~m;
    }
    if (d < 256) place[k] = sh.warp_hist[wid][d] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (d < 256 && (same >> lane) == 1u) sh.warp_hist[wid][d] = place[k] + 1;  // the last lane of the group
    __syncwarp();
  }
  __syncthreads();
  u32 total = 0;
  for (int w = 0; w < ST_WARPS; ++w) {
    const u32 c = sh.warp_hist[w][tid];
    sh.warp_hist[w][tid] = total;
    total += c;
  }
  const u32 first = scan256(total, sh.warp_tot);
  sh.local[tid] = first;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ST_ITEMS; ++k)
    if (digit[k] < 256) place[k] += sh.local[digit[k]] + sh.warp_hist[wid][digit[k]];
  return total;
}

__global__ void __launch_bounds__(ST_THREADS)
embed_sort_pass_kernel(const i64* __restrict__ idx, i64 rows, i64 padding, const u32* __restrict__ key_in,
                       const u32* __restrict__ pos_in, u32* __restrict__ key_out, u32* __restrict__ pos_out,
                       i64 n, int shift, int bits, const u32* __restrict__ counts, u64* status, u32* ticket,
                       int* err) {
  __shared__ RankShared sh;
  __shared__ u32 skey[ST_TILE], spos[ST_TILE];
  __shared__ u32 start[256];  // global place of the digit's run minus its place in the tile
  __shared__ u32 tile_s;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  if (tid == 0) tile_s = atomicAdd(ticket, 1u);
  __syncthreads();
  const i64 tile = tile_s, base = tile * ST_TILE;
  u32 key[ST_ITEMS], pos[ST_ITEMS], digit[ST_ITEMS], place[ST_ITEMS];
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
  const u32 mine = rank_tile(digit, place, sh);
  // look-back: one chain per digit
  u64* st = status + tile * 256 + tid;
  u64 before = 0;
  if (tile == 0) {
    st_relaxed(st, LB_PREFIX | mine);
  } else {
    st_relaxed(st, LB_AGG | mine);
    for (i64 t = tile - 1; t >= 0; --t) {
      const u64* p = status + t * 256 + tid;
      u64 w = ld_relaxed(p);
      int spins = 0;
      while ((w >> 62) == 0 && ++spins < LB_SPIN_LIMIT) {
        __nanosleep(20);
        w = ld_relaxed(p);
      }
      if ((w >> 62) == 0) {  // every place is still below n: nothing is written out of range
        raise(err, ERRBIT_LOOKBACK_TIMEOUT);
        break;
      }
      before += w & LB_MASK;
      if ((w >> 62) == 2) break;
    }
    st_relaxed(st, LB_PREFIX | (before + mine));
  }
  const u32 digit_base = scan256(counts[tid], sh.warp_tot);
  start[tid] = digit_base + (u32)before - sh.local[tid];
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
    if (to < n) {
      key_out[to] = k;
      pos_out[to] = spos[j];
    }
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
// that began before chunk c, slot 2c + 1 for one that began in it and goes on (for one that does
// both, slot 2c has the sum and slot 2c + 1 zeros, so that a segment's partials are neighbours).
// The next level runs the same kernel over the slots, until one chunk holds them all: a hub that
// fills half the batch is summed by thousands of groups, and in an order that is always the same.
// Eight rows are requested before the first is added.
template <typename Tin, typename Tout, int VEC, bool FIRST>
__global__ void __launch_bounds__(256)
embed_segsum_kernel(const u32* __restrict__ key, const u32* __restrict__ pos, i64 n, const Tin* __restrict__ src,
                    i64 ld, int D, int log_group, int chunk, u32 limit, float scale, Tout* __restrict__ out,
                    float* __restrict__ part, i64 part_ld, u32* __restrict__ part_key) {
  constexpr int U = 8;
  const int lane = threadIdx.x & ((1 << log_group) - 1);
  const i64 c = ((i64)blockIdx.x * blockDim.x + threadIdx.x) >> log_group;
  const i64 begin = c * chunk;
  if (begin >= n) return;
  const i64 end = begin + chunk < n ? begin + chunk : n;
  const int col = (((int)blockIdx.y << log_group) + lane) * VEC;
  const bool live = col < D;
  const bool scribe = blockIdx.y == 0 && lane == 0;
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
  u32 slot_key0 = NO_KEY, slot_key1 = NO_KEY;

  auto partial = [&](int which, bool zeros) {
    if (!live) return;
    float* to = part + (2 * c + which) * part_ld + col;
#pragma unroll
    for (int j = 0; j < VEC; ++j) to[j] = zeros ? 0.f : acc[j];
  };
  auto finish = [&]() {
    if (!live) return;
    Pack<Tout, VEC> r;
#pragma unroll
    for (int j = 0; j < VEC; ++j) r.v[j] = from_float<Tout>(acc[j] * scale);
    r.store(out + (i64)cur * D + col);
  };

  for (i64 i = begin; i < end; i += U) {
    u32 k[U];
    Pack<Tin, VEC> row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = i + u < end ? key_at(i + u) : NO_KEY;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k[u] != NO_KEY && live) row[u].load(src + (FIRST ? (i64)pos[i + u] : i + u) * ld + col);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= end) break;
      if (k[u] != cur) {
        if (cur != NO_KEY) {
          if (began_before) { partial(0, false); slot_key0 = cur; }
          else finish();
        }
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
  if (cur != NO_KEY) {
    if (began_before) {
      partial(0, false);
      slot_key0 = cur;
      if (goes_on_at_end) { partial(1, true); slot_key1 = cur; }
    } else if (goes_on_at_end) {
      partial(1, false);
      slot_key1 = cur;
    } else {
      finish();
    }
  }
  if (scribe && part_key) {
    part_key[2 * c] = slot_key0;
    part_key[2 * c + 1] = slot_key1;
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
  int chunk = 64;
  while (chunk > 8 && n / chunk < (i64)sm_count() * 64) chunk >>= 1;
  return chunk;
}
constexpr int NEXT_CHUNK = 64;

struct EmbedLayout {
  size_t key[2], pos[2], counts, status, ticket, zero_begin, zero_bytes, part[2], part_key[2], bytes;
  i64 tiles, part_ld;
};

static EmbedLayout embed_layout(i64 n, i64 D, i64 rows) {
  EmbedLayout L;
  size_t o = 0;
  auto take = [&](size_t b) { const size_t at = o; o += up256(b); return at; };
  for (int k = 0; k < 2; ++k) { L.key[k] = take(4 * (size_t)n); L.pos[k] = take(4 * (size_t)n); }
  L.tiles = (n + ST_TILE - 1) / ST_TILE;
  const int passes = sort_plan(rows).passes;
  L.zero_begin = o;
  L.counts = take(4 * 1024);
  L.ticket = take(4 * 8);
  // the sort's look-back words; the distinct-id pass has its own behind them
  L.status = take(8 * ((size_t)passes * L.tiles * 256 + (size_t)(n + 2047) / 2048));
  L.zero_bytes = o - L.zero_begin;
  L.part_ld = (D + 7) / 8 * 8;
  const i64 chunks0 = (n + first_chunk(n) - 1) / first_chunk(n);
  const i64 slots0 = 2 * chunks0, slots1 = 2 * ((slots0 + NEXT_CHUNK - 1) / NEXT_CHUNK);
  const i64 slots[2] = {slots0, slots1};
  for (int k = 0; k < 2; ++k) {
    L.part[k] = take(4 * (size_t)slots[k] * L.part_ld);
    L.part_key[k] = take(4 * (size_t)slots[k]);
  }
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
  u32* ticket = (u32*)(ws + L.ticket);
  u64* status = (u64*)(ws + L.status);
  {
    i64 blocks = (n + 2047) / 2048;
    if (blocks > sm_count() * 8) blocks = sm_count() * 8;
    LaunchScope ls(KID_EMBED_SORT, st);
    embed_digits_kernel<<<(int)blocks, 256, 0, st>>>(idx, n, rows, padding, plan, counts, d_err);
  }
  for (int p = 0; p < plan.passes; ++p) {
    LaunchScope ls(KID_EMBED_SORT, st);
    embed_sort_pass_kernel<<<(int)L.tiles, ST_THREADS, 0, st>>>(
        p == 0 ? idx : nullptr, rows, padding, key[(p + 1) & 1], pos[(p + 1) & 1], key[p & 1], pos[p & 1], n,
        plan.shift[p], plan.bits[p], counts + 256 * p, status + (size_t)p * L.tiles * 256, ticket + p, d_err);
  }
  *which = (plan.passes - 1) & 1;
  return GSB_OK;
}

template <typename Tin, typename Tout, int VEC, bool FIRST>
static void launch_level(const u32* key, const u32* pos, i64 n, const void* src, i64 ld, i64 D, int chunk,
                         u32 limit, float scale, void* out, float* part, i64 part_ld, u32* part_key,
                         cudaStream_t st) {
  const i64 per_row = D / VEC;
  int lg = 0;
  while (lg < 5 && (1 << lg) < per_row) ++lg;
  const i64 groups = (n + chunk - 1) / chunk, threads = groups << lg;
  dim3 grid((unsigned)((threads + 255) / 256), (unsigned)((per_row + (1 << lg) - 1) >> lg));
  LaunchScope ls(KID_EMBED_GRAD, st);
  embed_segsum_kernel<Tin, Tout, VEC, FIRST><<<grid, 256, 0, st>>>(key, pos, n, (const Tin*)src, ld, (int)D, lg,
                                                                   chunk, limit, scale, (Tout*)out, part, part_ld,
                                                                   part_key);
}

template <typename T, int VEC>
static void launch_segsum(const u32* key, const u32* pos, i64 n, const void* grad, i64 D, u32 limit, float scale,
                          void* out, char* ws, const EmbedLayout& L, cudaStream_t st) {
  float* part[2] = {(float*)(ws + L.part[0]), (float*)(ws + L.part[1])};
  u32* pkey[2] = {(u32*)(ws + L.part_key[0]), (u32*)(ws + L.part_key[1])};
  const int c0 = first_chunk(n);
  i64 groups = (n + c0 - 1) / c0;
  launch_level<T, T, VEC, true>(key, pos, n, grad, D, D, c0, limit, scale, out, part[0], L.part_ld, pkey[0], st);
  int at = 0;
  while (groups > 1) {
    const i64 items = 2 * groups;
    groups = (items + NEXT_CHUNK - 1) / NEXT_CHUNK;
    launch_level<float, T, VEC, false>(pkey[at], nullptr, items, part[at], L.part_ld, D, NEXT_CHUNK, limit, scale,
                                       out, part[at ^ 1], L.part_ld, pkey[at ^ 1], st);
    at ^= 1;
  }
}

// elements a thread moves at once: 16 bytes where row width and addresses allow
static int vec_of(const void* a, const void* b, i64 D, i64 ld, int size) {
  const uintptr_t m = (uintptr_t)a | (uintptr_t)b | (uintptr_t)(D * size) | (uintptr_t)(ld * size);
  int bytes = 16;
  while (bytes > size && (m & (uintptr_t)(bytes - 1))) bytes >>= 1;
  return bytes / size;
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
  if (n < 0 || rows < 0 || D < 0 || D > GSB_EMBED_MAX_D || (rows > 1 && ld < D)) return GSB_ERR_INVALID;
  if (n == 0 || D == 0) return GSB_OK;
  if (!idx || !out || (rows > 0 && !weight)) return GSB_ERR_INVALID;
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
  if (!embed_sizes_ok(n, rows, D) || (dtype != GSB_F32 && dtype != GSB_F16 && dtype != GSB_BF16)) return GSB_ERR_INVALID;
  if (rows == 0 || D == 0) return GSB_OK;
  if (!out || (n > 0 && (!grad || !idx))) return GSB_ERR_INVALID;
  cudaStream_t st = (cudaStream_t)cuda_stream;
  GSB_CUDA_OK(cudaMemsetAsync(out, 0, (size_t)rows * D * (dtype == GSB_F32 ? 4 : 2), st));
  if (n == 0) return GSB_OK;
  const EmbedLayout L = embed_layout(n, D, rows);
  if (!workspace || workspace_bytes < L.bytes) return GSB_ERR_WORKSPACE;
  char* ws = (char*)workspace;
  if (n > ST_TILE) GSB_CUDA_OK(cudaMemsetAsync(ws + L.zero_begin, 0, L.zero_bytes, st));
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
  const EmbedLayout L = embed_layout(n, D, rows);
  if (!workspace || workspace_bytes < L.bytes) return GSB_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)cuda_stream;
  char* ws = (char*)workspace;
  GSB_CUDA_OK(cudaMemsetAsync(ws + L.zero_begin, 0, L.zero_bytes, st));
  int which = 0;
  launch_embed_sort((const i64*)idx, n, rows, padding, ws, L, d_err, st, &which);
  u64* status = (u64*)(ws + L.status) + (size_t)sort_plan(rows).passes * L.tiles * 256;
  {
    LaunchScope ls(KID_EMBED_SORT, st);
    // the ranks take the place of the other key buffer
    embed_segments_kernel<<<(int)((n + 2047) / 2048), 256, 0, st>>>(
        (u32*)(ws + L.key[which]), n, (u32)rows, (u32*)(ws + L.key[which ^ 1]), (i64*)ids, (i64*)d_num, status,
        (u32*)(ws + L.ticket) + 4, d_err);
  }
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}

extern "C" int gsb_embedding_grad_rows(const void* grad, int dtype, int64_t D, int64_t n, int64_t rows, int64_t num,
                                       float scale, void* out, void* workspace, size_t workspace_bytes,
                                       void* cuda_stream) {
  if (!embed_sizes_ok(n, rows, D) || num < 0 || num > n || (dtype != GSB_F32 && dtype != GSB_F16 && dtype != GSB_BF16))
    return GSB_ERR_INVALID;
  if (num == 0 || D == 0) return GSB_OK;
  if (!grad || !out) return GSB_ERR_INVALID;
  const EmbedLayout L = embed_layout(n, D, rows);
  if (!workspace || workspace_bytes < L.bytes) return GSB_ERR_WORKSPACE;
  char* ws = (char*)workspace;
  const int which = n <= ST_TILE ? 0 : (sort_plan(rows).passes - 1) & 1;
  segsum_any(dtype, (u32*)(ws + L.key[which ^ 1]), (u32*)(ws + L.pos[which]), n, grad, D, (u32)num, scale, out, ws, L,
             (cudaStream_t)cuda_stream);
  GSB_CUDA_OK(cudaGetLastError());
  return GSB_OK;
}
