// Scaled embedding lookup, and its gradient by sorted tokens.
//
//   y[r, :]      = scale * table[ids[r], :]
//   dtable[v, :] = scale * sum of g[r, :] over the positions r with ids[r] = v, in the order of r
//
// An id outside [0, vocab) gives a row of zeros and no gradient; positions that hold `padding` give no gradient.
//
// The gradient sorts (token, position) pairs with a stable radix sort, so the positions of a token lie together in their
// order and every sum is taken in one fixed order: no atomics, the same bits in every run.  The sorted list is cut in
// tiles of a few positions; a block walks its tile and keeps the running sum of the present token.  Tokens that lie
// inside one tile are written at once.  A token that crosses tiles leaves the sum of each tile as a partial row, and
// join_tokens adds those in order, so a token that fills half of the batch costs no more than its bytes.
// A few hundred positions are not sorted at all, see grad_by_rows.
#include <cuda_runtime.h>
#include <cooperative_groups.h>
#include <stdint.h>

#include "launch.cuh"
#include "scratch.h"
#include "smem_limit.h"

#define TSB_OK 0
#define TSB_ERR_ARG 1
#define TSB_ERR_LAUNCH 3
#define TSB_ERR_OOM 5

namespace {

namespace cg = cooperative_groups;
using tsb_launch::load;

int launch_status(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  else cudaGetLastError();
  return e == cudaSuccess ? TSB_OK : TSB_ERR_LAUNCH | ((int)e << 8);
}

// ------------------------------------------------------------------------------------------------ lookup
// T: float4 where rows are whole 16-byte pieces, float otherwise.  U pieces in flight per thread.
template <class T> __device__ __forceinline__ T zero();
template <> __device__ __forceinline__ float zero<float>() { return 0.f; }
template <> __device__ __forceinline__ float4 zero<float4>() { return make_float4(0.f, 0.f, 0.f, 0.f); }
__device__ __forceinline__ float times(float v, float s) { return v * s; }
__device__ __forceinline__ float4 times(float4 v, float s) { return make_float4(v.x * s, v.y * s, v.z * s, v.w * s); }
__device__ __forceinline__ float plus(float a, float b) { return a + b; }
__device__ __forceinline__ float4 plus(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }

template <class T, int U>
__global__ void __launch_bounds__(256) scaled_lookup(const T* table, const float* ids, T* __restrict__ y, long long pieces,
                                                     long long vocab, unsigned dim, float scale) {
  tsb_launch::enter();
  const long long i = blockIdx.x * (256ll * U) + threadIdx.x;
  T v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long j = i + u * 256;
    v[u] = zero<T>();
    if (j < pieces) {
      const long long r = (pieces >> 32) == 0 ? (long long)((unsigned)j / dim) : j / dim;
      const long long id = (long long)load(ids + r);
      if (id >= 0 && id < vocab) v[u] = times(load(table + id * dim + (j - r * dim)), scale);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (i + u * 256 < pieces) y[i + u * 256] = v[u];
}

// Rows of 32 pieces or more, a warp to each ROWS of them: no piece's place has to be divided by the row's length.  With one row U
// pieces are in flight per thread, with several one of each.
template <class T, int U, int ROWS>
__global__ void __launch_bounds__(256) scaled_lookup_rows(const T* table, const float* ids, T* __restrict__ y, long long n, long long vocab,
                                                          unsigned dim, float scale) {
  tsb_launch::enter();
  const long long r = (blockIdx.x * 8ll + (threadIdx.x >> 5)) * ROWS;
  bool known[ROWS];
  const T* from[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const long long id = r + k < n ? (long long)load(ids + r + k) : -1;
    known[k] = id >= 0 && id < vocab;
    from[k] = table + (known[k] ? id * dim : 0);
  }
  T* const to = y + r * dim;
  if (ROWS == 1) {
    if (r < n)
      tsb_launch::read_then_write<U>(threadIdx.x & 31, dim, 32u, [&](unsigned c) { return known[0] ? times(load(from[0] + c), scale) : zero<T>(); },
                                     [&](unsigned c, T v) { to[c] = v; });
    return;
  }
  for (unsigned c = threadIdx.x & 31; c < dim; c += 32) {
    T v[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) v[k] = known[k] ? times(load(from[k] + c), scale) : zero<T>();
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
      if (r + k < n) to[k * dim + c] = v[k];
  }
}

// ------------------------------------------------------------------------------------------------ sort
// Keys are token ids, `vocab` for positions that give no gradient (they end up last).  What fills the last tile behind
// position n has all bits set, so it stays behind everything in every pass.  Digits of up to 8 bits, the lowest first.  A
// position's rank among equal digits is counted in the order of the positions: lanes by a ballot for each bit, the rounds of
// a warp by a running count, warps and blocks by prefix sums.
constexpr int SORT_THREADS = 1024, SORT_ITEMS = 4, SORT_TILE = SORT_THREADS * SORT_ITEMS, SORT_WARPS = SORT_THREADS / 32;
constexpr int DIGITS = 256, MAX_CLUSTER = 8;
constexpr unsigned FILL = 0xffffffffu;
static_assert(SORT_TILE == 4096, "the launcher and the scratch layout use it");

struct SortShared {
  unsigned counts[SORT_WARPS][DIGITS];       // running counts of each warp, then what lies before it
  unsigned total[DIGITS];                    // of this block (read by the others of the cluster)
  unsigned base[DIGITS];                     // where this block's first position of a digit goes
  unsigned scan[8];
};

__device__ __forceinline__ unsigned key_of(const float* ids, long long r, long long n, unsigned vocab, long long padding) {
  if (r >= n) return FILL;
  const long long id = (long long)load(ids + r);
  return id >= 0 && id < (long long)vocab && id != padding ? (unsigned)id : vocab;
}

// rank[i]: positions of the same digit before item i in this warp (items of a warp lie 32 apart, lane by lane)
template <int ITEMS>
__device__ __forceinline__ void rank_items(const unsigned (&key)[ITEMS], int shift, unsigned mask, unsigned* count, unsigned (&rank)[ITEMS]) {
  const unsigned lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const unsigned d = (key[i] >> shift) & mask;
    unsigned same = 0xffffffffu;             // lanes with this digit
#pragma unroll
    for (int bit = 0; bit < 8; ++bit) {
      const unsigned ones = __ballot_sync(0xffffffffu, d >> bit & 1);
      same &= d >> bit & 1 ? ones : ~ones;
    }
    const unsigned before = __popc(same & ((1u << lane) - 1));
    const unsigned old = count[d];
    __syncwarp();
    if (before == 0) count[d] = old + __popc(same);
    __syncwarp();
    rank[i] = old + before;
  }
}

__device__ __forceinline__ void clear_counts(SortShared& s) {
  for (int i = threadIdx.x; i < SORT_WARPS * DIGITS; i += SORT_THREADS) (&s.counts[0][0])[i] = 0;
}

// Per digit: what lies before each warp, and the block's total.
__device__ __forceinline__ void scan_warps(SortShared& s) {
  if (threadIdx.x < DIGITS) {
    unsigned c[SORT_WARPS], sum = 0;         // (all loads before the first store)
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) c[w] = s.counts[w][threadIdx.x];
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) {
      s.counts[w][threadIdx.x] = sum;
      sum += c[w];
    }
    s.total[threadIdx.x] = sum;
  }
}

// Exclusive prefix sum of one value of each of the first 256 threads (all threads call it).
__device__ __forceinline__ unsigned scan_digits(SortShared& s, unsigned v) {
  const unsigned lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  unsigned sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  if (w < 8 && lane == 31) s.scan[w] = sum;
  __syncthreads();
  unsigned before = 0;
  for (unsigned k = 0; k < w && k < 8; ++k) before += s.scan[k];
  return before + sum - v;
}

// The table's gradient begins as zeros.  What the sort needs of the chip is little, so the blocks behind those of the sort, in
// all of its launches, fill a share of it each: part `part` of `parts`, by `blocks` blocks of SORT_THREADS.
struct Zeros {
  float* at;
  long long cells;
  int part, parts, blocks;
  bool aligned;
};
__device__ __forceinline__ void fill_share(const Zeros& z, unsigned block) {
  const long long all = z.aligned ? z.cells / 4 : z.cells, begin = all / z.parts * z.part;
  const long long end = z.part == z.parts - 1 ? all : all / z.parts * (z.part + 1), step = (long long)z.blocks * SORT_THREADS;
  long long i = begin + (long long)block * SORT_THREADS + threadIdx.x;
  if (z.aligned) {
    for (; i < end; i += step) reinterpret_cast<float4*>(z.at)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (z.part == z.parts - 1 && block == 0 && threadIdx.x < z.cells % 4) z.at[z.cells / 4 * 4 + threadIdx.x] = 0.f;
  } else {
    for (; i < end; i += step) z.at[i] = 0.f;
  }
}

// Up to 32768 positions: one cluster of up to eight blocks keeps them in registers, ITEMS a thread, and trades them through
// distributed shared memory, one launch for all digits.  Counting the ranks is what takes its time, so as many blocks share it
// as there are warps to fill (4099 positions, 10007 x 301: two blocks of four a thread 12.5 us, eight of one 8.9).  The other
// clusters of the grid fill zeros.
template <int ITEMS>
__global__ void __launch_bounds__(SORT_THREADS) sort_cluster(const float* ids, long long n, unsigned vocab, long long padding, int bits,
                                                             int passes, unsigned* __restrict__ out_key, unsigned* __restrict__ out_pos,
                                                             unsigned* __restrict__ joins, const Zeros zeros) {
  tsb_launch::enter();
  if (blockIdx.x == 0 && threadIdx.x == 0) joins[0] = 0;
  extern __shared__ uint4 raw[];
  constexpr unsigned TILE = SORT_THREADS * ITEMS;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned size = cluster.num_blocks(), me = cluster.block_rank();
  if (blockIdx.x >= size) return fill_share(zeros, blockIdx.x - size);
  SortShared& s = *reinterpret_cast<SortShared*>(raw);
  uint2* const items = reinterpret_cast<uint2*>(&s + 1);
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, at = warp * (32 * ITEMS) + lane;
  const int step = (bits + passes - 1) / passes;
  unsigned key[ITEMS], pos[ITEMS], rank[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    pos[i] = me * TILE + at + i * 32;
    key[i] = key_of(ids, pos[i], n, vocab, padding);
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = p * step;
    const unsigned mask = (1u << step) - 1;
    clear_counts(s);
    __syncthreads();
    rank_items(key, shift, mask, s.counts[warp], rank);
    __syncthreads();
    scan_warps(s);
    cluster.sync();                          // totals are there, and every item is in registers
    unsigned all = 0, mine = 0;
    if (threadIdx.x < DIGITS) {
      unsigned c[MAX_CLUSTER];
#pragma unroll
      for (unsigned b = 0; b < MAX_CLUSTER; ++b) c[b] = b < size ? *cluster.map_shared_rank(&s.total[threadIdx.x], b) : 0;
#pragma unroll
      for (unsigned b = 0; b < MAX_CLUSTER; ++b) {
        if (b < me) mine += c[b];
        all += c[b];
      }
    }
    const unsigned before = scan_digits(s, all);
    if (threadIdx.x < DIGITS) s.base[threadIdx.x] = before + mine;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const unsigned d = (key[i] >> shift) & mask;
      const unsigned to = s.base[d] + s.counts[warp][d] + rank[i];
      *cluster.map_shared_rank(&items[to % TILE], to / TILE) = make_uint2(key[i], pos[i]);
    }
    cluster.sync();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint2 v = items[at + i * 32];
      key[i] = v.x;
      pos[i] = v.y;
    }
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const unsigned to = me * TILE + at + i * 32;
    if (to < n) {
      out_key[to] = key[i];
      out_pos[to] = pos[i];
    }
  }
}

// More positions: per digit a histogram of every tile, their prefix sums, and the scatter.
__device__ __forceinline__ void load_items(const float* ids, const unsigned* in_key, const unsigned* in_pos, long long n,
                                           unsigned vocab, long long padding, unsigned (&key)[SORT_ITEMS],
                                           unsigned (&pos)[SORT_ITEMS]) {
  const long long at = blockIdx.x * (long long)SORT_TILE + (threadIdx.x >> 5) * (32 * SORT_ITEMS) + (threadIdx.x & 31);
#pragma unroll
  for (int i = 0; i < SORT_ITEMS; ++i) {
    const long long r = at + i * 32;
    pos[i] = (unsigned)r;
    if (!in_key) key[i] = key_of(ids, r, n, vocab, padding);
    else if (r < n) key[i] = load(in_key + r), pos[i] = load(in_pos + r);
    else key[i] = FILL;
  }
}

__global__ void __launch_bounds__(SORT_THREADS) tile_histogram(const float* ids, const unsigned* in_key, long long n,
                                                               unsigned vocab, long long padding, int shift, unsigned mask,
                                                               unsigned* __restrict__ hist, unsigned tiles, unsigned* __restrict__ joins, const Zeros zeros) {
  tsb_launch::enter();
  if (blockIdx.x == 0 && threadIdx.x == 0) joins[0] = 0;
  if (blockIdx.x >= tiles) return fill_share(zeros, blockIdx.x - tiles);
  __shared__ unsigned count[DIGITS];
  if (threadIdx.x < DIGITS) count[threadIdx.x] = 0;
  __syncthreads();
  const long long at = blockIdx.x * (long long)SORT_TILE;
#pragma unroll
  for (int i = 0; i < SORT_ITEMS; ++i) {
    const long long r = at + i * SORT_THREADS + threadIdx.x;
    const unsigned k = in_key ? (r < n ? load(in_key + r) : FILL) : key_of(ids, r, n, vocab, padding);
    atomicAdd(&count[(k >> shift) & mask], 1u);        // whole numbers: any order gives the same sums
  }
  __syncthreads();
  if (threadIdx.x < DIGITS) hist[(size_t)threadIdx.x * tiles + blockIdx.x] = count[threadIdx.x];
}

__global__ void __launch_bounds__(1024) scan_histogram(unsigned* hist, unsigned entries, const Zeros zeros) {
  tsb_launch::enter();
  if (blockIdx.x) return fill_share(zeros, blockIdx.x - 1);
  __shared__ unsigned sums[32];
  __shared__ unsigned carry;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (unsigned begin = 0; begin < entries; begin += 4096) {          // (a digit has `tiles` entries, 256 digits)
    const unsigned i = begin + threadIdx.x * 4;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (i < entries) v = *reinterpret_cast<const uint4*>(hist + i);   // entries is a multiple of 256
    const unsigned own = v.x + v.y + v.z + v.w;
    unsigned sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) sums[warp] = sum;
    __syncthreads();
    unsigned before = carry, block = 0;
    for (unsigned w = 0; w < 32; ++w) {
      if (w < warp) before += sums[w];
      block += sums[w];
    }
    before += sum - own;
    if (i < entries)
      *reinterpret_cast<uint4*>(hist + i) = make_uint4(before, before + v.x, before + v.x + v.y, before + v.x + v.y + v.z);
    __syncthreads();
    if (threadIdx.x == 0) carry += block;
    __syncthreads();
  }
}

__global__ void __launch_bounds__(SORT_THREADS) scatter_tiles(const float* ids, const unsigned* in_key, const unsigned* in_pos,
                                                              long long n, unsigned vocab, long long padding, int shift,
                                                              unsigned mask, const unsigned* hist, unsigned tiles,
                                                              unsigned* __restrict__ out_key, unsigned* __restrict__ out_pos,
                                                              const Zeros zeros) {
  tsb_launch::enter();
  if (blockIdx.x >= tiles) return fill_share(zeros, blockIdx.x - tiles);
  extern __shared__ uint4 raw[];
  SortShared& s = *reinterpret_cast<SortShared*>(raw);
  unsigned key[SORT_ITEMS], pos[SORT_ITEMS], rank[SORT_ITEMS];
  load_items(ids, in_key, in_pos, n, vocab, padding, key, pos);
  clear_counts(s);
  __syncthreads();
  const unsigned warp = threadIdx.x >> 5;
  rank_items(key, shift, mask, s.counts[warp], rank);
  __syncthreads();
  scan_warps(s);
  if (threadIdx.x < DIGITS) s.base[threadIdx.x] = load(hist + (size_t)threadIdx.x * tiles + blockIdx.x);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SORT_ITEMS; ++i) {
    const unsigned d = (key[i] >> shift) & mask;
    const unsigned to = s.base[d] + s.counts[warp][d] + rank[i];
    if (to < n) {                            // (what fills the last tile is behind all of them)
      out_key[to] = key[i];
      out_pos[to] = pos[i];
    }
  }
}

__global__ void __launch_bounds__(SORT_THREADS) fill_zero(const Zeros zeros) {
  tsb_launch::enter();
  fill_share(zeros, blockIdx.x);
}

// ------------------------------------------------------------------------------------------------ sums
// Block (tile, column slice): positions [tile * size, ...) of the sorted list, one column piece per thread.  BATCH rows in
// flight.  part[2 * tile]: what belongs to a token of an earlier tile; part[2 * tile + 1]: the token that goes on.  joins: how many
// tiles a token begins in and goes on from, then these tiles (in any order: each is a sum of its own).
constexpr int BATCH = 8, SUM_THREADS = 128, MAX_TILE = 64;

template <class T>
__global__ void __launch_bounds__(SUM_THREADS) sum_tiles(const T* g, const unsigned* key, const unsigned* pos, long long n,
                                                         unsigned vocab, unsigned dim, float scale, int size,
                                                         T* __restrict__ dtable, T* __restrict__ part, unsigned* __restrict__ joins) {
  tsb_launch::enter();
  __shared__ unsigned k[MAX_TILE + 2], p[MAX_TILE];
  const long long begin = blockIdx.x * (long long)size;
  const int count = (int)(n - begin < size ? n - begin : size);
  for (int i = threadIdx.x; i < count + 2; i += SUM_THREADS) {
    const long long at = begin + i - 1;
    k[i] = at >= 0 && at < n ? load(key + at) : vocab;
    if (i >= 1 && i <= count) p[i - 1] = load(pos + at);
  }
  __syncthreads();
  if (k[1] == vocab) return;                 // nothing but positions without a gradient from here on
  const unsigned c = blockIdx.y * SUM_THREADS + threadIdx.x;
  if (c >= dim) return;
  const T* row = g + c;
  const bool goes_on = begin + count < n && k[count + 1] == k[count];
  if (c == 0 && goes_on && k[count] != vocab && k[0] != k[count]) joins[1 + atomicAdd(joins, 1u)] = blockIdx.x;
  T acc = zero<T>();
  bool first = k[0] == k[1];                 // the present token began in an earlier tile
  for (int i = 0; i < count; i += BATCH) {
    T v[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (i + u < count && k[i + u + 1] != vocab) v[u] = load(row + (size_t)p[i + u] * dim);
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int j = i + u;
      if (j >= count || k[j + 1] == vocab) break;
      acc = plus(acc, v[u]);
      if (j + 1 < count ? k[j + 2] != k[j + 1] : true) {              // the last one of its token, in this tile at least
        if (first) part[(size_t)(2 * blockIdx.x) * dim + c] = acc;
        else if (j + 1 == count && goes_on) part[(size_t)(2 * blockIdx.x + 1) * dim + c] = acc;
        else dtable[(size_t)k[j + 1] * dim + c] = times(acc, scale);
        acc = zero<T>();
        first = false;
      }
    }
  }
}

// 32 x 8 threads take a token that begins in a tile and goes on, and 32 of its pieces.  Its partial rows are taken by eight groups
// of threads, group j the rows j, j + 8, ..., and the groups are added in their order.
template <class T>
__global__ void __launch_bounds__(256) join_tokens(const T* part, const unsigned* key, const unsigned* joins, unsigned dim, float scale,
                                                   int size, unsigned tiles, T* __restrict__ dtable) {
  tsb_launch::enter();
  __shared__ T sums[8][32];
  const unsigned slices = (dim + 31) / 32;
  const unsigned long long all = (unsigned long long)load(joins) * slices;
  for (unsigned long long work = blockIdx.x; work < all; work += gridDim.x) {
    const unsigned tile = load(joins + 1 + work / slices), slice = (unsigned)(work % slices);
    const unsigned token = load(key + (tile + 1) * (long long)size - 1);
    // the last tile that holds the token: 32 places at a time
    unsigned lo = tile + 1, hi = tiles - 1;
    while (lo < hi) {
      const unsigned step = (hi - lo + 31) / 32, at = min(lo + (threadIdx.x + 1) * step, hi);
      const unsigned more = __popc(__ballot_sync(0xffffffffu, load(key + (long long)at * size) == token));
      // (a place that is hi again counts as often as it is looked at)
      const unsigned next = min(lo + more * step, hi);
      hi = min(next + step - 1, hi);
      lo = next;
    }
    const unsigned rows = lo - tile + 1;                                 // partial rows: its tail, then the heads
    const unsigned c = slice * 32 + threadIdx.x, group = threadIdx.y;
    T acc = zero<T>();
    if (c < dim) {
      for (unsigned r = group; r < rows; r += 8 * BATCH) {
        T v[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          const unsigned q = r + u * 8;
          if (q < rows) v[u] = load(part + (size_t)(q == 0 ? 2 * tile + 1 : 2 * (tile + q)) * dim + c);
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
          if (r + u * 8 < rows) acc = plus(acc, v[u]);
      }
    }
    sums[group][threadIdx.x] = acc;
    __syncthreads();
    if (group == 0 && c < dim) {
#pragma unroll
      for (int j = 1; j < 8; ++j) acc = plus(acc, sums[j][threadIdx.x]);
      dtable[(size_t)token * dim + c] = times(acc, scale);
    }
    __syncthreads();                         // (the next one writes there)
  }
}

// ------------------------------------------------------------------------------------------------ few tokens
// Up to FEW_TOKENS positions need no sort: a block takes every 2^apart-th row of the table (frequent tokens, which are often the
// first ones, go to different blocks) and 32 of its pieces, and looks through all positions for those of its rows.  A warp writes a
// row, zeros or the sum of the row's positions in their order; rows of more than LONG positions are summed by all warps, a run of
// positions each, and joined in the order of the runs.  One launch: 37 x 500 x 128 takes 2.0 us (sorted 9.3), 256 x 10000 x 512 5.9
// (11.8), 512 x 64000 x 1024 44 (51; the zeros alone are 41).  At 1024 positions what one block has to add up can take longer than
// the sort: 1024 x 500 x 128 13.9 us, sorted 11.6.
constexpr int FEW_TOKENS = 512, FEW_ROWS = 1024, LONG = 16;
struct FewShared {
  unsigned list[FEW_TOKENS];               // (row, position) of the block's rows, in the order of the positions
  unsigned first[FEW_ROWS], times[FEW_ROWS];                    // of each row: its first place in the list; how many
  unsigned found[8];
};

// The positions of row r among places [from, to) of the list, added in their order; BATCH rows in flight.  A lane has U columns, 32
// apart, the first `there` of them inside.
template <class T, int U>
__device__ __forceinline__ void sum_of_row(const FewShared& s, unsigned r, unsigned from, unsigned to, const T* column, unsigned dim, int there,
                                           T (&sum)[U]) {
  const unsigned lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < U; ++k) sum[k] = zero<T>();
  for (unsigned i = from; i < to; i += 32) {
    const unsigned item = i + lane < to ? s.list[i + lane] : 0xffffffffu;
    for (unsigned mask = __ballot_sync(0xffffffffu, item >> 16 == r); mask;) {
      T v[BATCH / U][U];
      int count = 0;
#pragma unroll
      for (int u = 0; u < BATCH / U; ++u)
        if (mask) {
          const unsigned at = __shfl_sync(0xffffffffu, item, __ffs(mask) - 1) & 0xffff;
          mask &= mask - 1;
#pragma unroll
          for (int k = 0; k < U; ++k) v[u][k] = k < there ? load(column + (size_t)at * dim + k * 32) : zero<T>();
          count = u + 1;
        }
#pragma unroll
      for (int u = 0; u < BATCH / U; ++u)
        if (u < count)
#pragma unroll
          for (int k = 0; k < U; ++k) sum[k] = plus(sum[k], v[u][k]);
    }
  }
}

template <class T, int U>
__global__ void __launch_bounds__(256) grad_by_rows(const T* g, const float* ids, int n, unsigned vocab, long long padding, unsigned dim,
                                                    int apart, unsigned chunks, float scale, T* __restrict__ dtable) {
  tsb_launch::enter();
  __shared__ FewShared s;
  __shared__ T parts[8][U][32];
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned row0 = blockIdx.x / chunks, count = (vocab - row0 + (1u << apart) - 1) >> apart, c = blockIdx.x % chunks * (32 * U) + lane;
  const int there = c < dim ? min((int)((dim - c + 31) / 32), U) : 0;      // columns of the lane, 32 apart
  constexpr int ITEMS = FEW_TOKENS / 256;
  const int items = (n + 255) / 256;         // 32 positions each that a warp looks at
  unsigned key[ITEMS], mask[ITEMS], own = 0;
  const unsigned at = warp * (32 * items) + lane;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) key[i] = i < items ? key_of(ids, at + i * 32, n, vocab, padding) : vocab;
  for (unsigned r = threadIdx.x; r < count; r += 256) s.first[r] = 0xffffffffu, s.times[r] = 0;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const unsigned token = key[i];           // row row0 + key << apart
    key[i] = token < vocab && (token & ((1u << apart) - 1)) == row0 ? token >> apart : count;
    mask[i] = __ballot_sync(0xffffffffu, key[i] < count);
    own += __popc(mask[i]);
  }
  if (lane == 0) s.found[warp] = own;
  __syncthreads();
  unsigned to = 0, all = 0;
#pragma unroll
  for (unsigned w = 0; w < 8; ++w) {
    if (w < warp) to += s.found[w];
    all += s.found[w];
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if (key[i] < count) {
      const unsigned place = to + __popc(mask[i] & ((1u << lane) - 1));
      s.list[place] = key[i] << 16 | (at + i * 32);
      atomicMin(&s.first[key[i]], place);
      atomicAdd(&s.times[key[i]], 1u);
    }
    to += __popc(mask[i]);
  }
  __syncthreads();
  const T* const column = g + c;
  const size_t step = (size_t)dim << apart;
  T* const out = dtable + (size_t)row0 * dim + c;
  const unsigned run = (all + 255) / 256 * 32;
  for (unsigned i = 0; all > LONG && i < all; ++i) {
    const unsigned r = s.list[i] >> 16;
    if (s.times[r] <= LONG || s.first[r] != i) continue;
    __syncthreads();                         // (the row before has been joined)
    T sum[U];
    sum_of_row(s, r, min(warp * run, all), min(warp * run + run, all), column, dim, there, sum);
#pragma unroll
    for (int k = 0; k < U; ++k) parts[warp][k][lane] = sum[k];
    __syncthreads();
    if (warp == 0)
#pragma unroll
      for (int k = 0; k < U; ++k) {
#pragma unroll
        for (int w = 1; w < 8; ++w) sum[k] = plus(sum[k], parts[w][k][lane]);
        if (k < there) out[r * step + k * 32] = times(sum[k], scale);
      }
  }
  for (unsigned r = warp; r < count; r += 8) {
    const unsigned times_of = s.times[r];
    if (times_of > LONG) continue;
    T sum[U];
    if (times_of) {
      sum_of_row(s, r, s.first[r], all, column, dim, there, sum);
#pragma unroll
      for (int k = 0; k < U; ++k) sum[k] = times(sum[k], scale);
    } else {
#pragma unroll
      for (int k = 0; k < U; ++k) sum[k] = zero<T>();
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (k < there) out[r * step + k * 32] = sum[k];
  }
}

template <class T>
int sums_of_few(const T* g, const float* ids, long long n, long long vocab, long long padding, long long dim, float scale, T* dtable,
                cudaStream_t st) {
  // as many blocks as run at once, eight to an SM, of at most FEW_ROWS rows
  constexpr int U = sizeof(T) == 4 ? 4 : 1;
  const long long chunks = (dim + 32 * U - 1) / (32 * U);
  int apart = 0;
  while ((1ll << apart) * FEW_ROWS < vocab || ((2ll << apart) <= vocab && (2ll << apart) * chunks <= 148 * 8)) ++apart;
  const long long blocks = chunks << apart;
  if (blocks > INT32_MAX) return TSB_ERR_ARG;
  return launch_status(tsb_launch::launch(grad_by_rows<T, U>, dim3((unsigned)blocks), dim3(256), 0, st, g, ids, (int)n, (unsigned)vocab, padding,
                                          (unsigned)dim, apart, (unsigned)chunks, scale, dtable));
}

int bits_of(long long v) {
  int b = 1;
  while (b < 32 && (v >> b)) ++b;
  return b;
}

template <int ITEMS>
cudaError_t sort_in_cluster(const float* ids, long long n, long long vocab, long long padding, int bits, int passes, unsigned* key,
                            unsigned* pos, unsigned* joins, const Zeros& zeros, unsigned blocks, cudaStream_t st) {
  constexpr int smem = (int)sizeof(SortShared) + SORT_THREADS * ITEMS * 8;
  static tsb_launch::SmemLimit limit;
  const cudaError_t e = limit.raise(sort_cluster<ITEMS>, smem);
  if (e != cudaSuccess) return e;
  return tsb_launch::launch_cluster(blocks, sort_cluster<ITEMS>, dim3(blocks + zeros.blocks), dim3(SORT_THREADS), smem, st, ids, n,
                                    (unsigned)vocab, padding, bits, passes, key, pos, joins, zeros);
}

template <class T>
int sums(const T* g, const unsigned* key, const unsigned* pos, long long n, unsigned vocab, unsigned dim, float scale, int size,
         unsigned tiles, T* dtable, T* part, unsigned* joins, cudaStream_t st) {
  cudaError_t e = tsb_launch::launch(sum_tiles<T>, dim3(tiles, (dim + SUM_THREADS - 1) / SUM_THREADS), dim3(SUM_THREADS), 0, st,
                                     g, key, pos, n, vocab, dim, scale, size, dtable, part, joins);
  // (as many blocks as run at once: with one for each tile and slice, most of which find nothing to do, 131072 x 64000 x 1024 takes
  // 174 us in place of 160, 8192 x 32000 x 512 23.4 in place of 22.4)
  const unsigned long long most = (unsigned long long)(tiles - 1) * ((dim + 31) / 32);
  if (e == cudaSuccess && tiles > 1)
    e = tsb_launch::launch(join_tokens<T>, dim3((unsigned)(most < 148 * 4 ? most : 148 * 4)), dim3(32, 8), 0, st, part, key, joins, dim,
                           scale, size, tiles, dtable);
  return launch_status(e);
}

template <class T>
int lookup(const T* table, const float* ids, T* y, long long n, long long vocab, long long dim, float scale, cudaStream_t st) {
  // (8000 x 1023: 7.8 us, piece by piece 18.  Short rows need others beside them, where there are enough: 131072 x 128 16 us by
  // pieces, 25 by single rows)
  const bool rows = dim >= 32;
  const int each = dim < 128 && n >= 148 * 8 * 8 * 4 ? 4 : 1;
  const long long blocks = rows ? (n + 8 * each - 1) / (8 * each) : (n * dim + 1023) / 1024;
  if (blocks > INT32_MAX) return TSB_ERR_ARG;
  const dim3 grid((unsigned)blocks), block(256);
  if (rows && each == 4)
    return launch_status(tsb_launch::launch(scaled_lookup_rows<T, 1, 4>, grid, block, 0, st, table, ids, y, n, vocab, (unsigned)dim, scale));
  if (rows) return launch_status(tsb_launch::launch(scaled_lookup_rows<T, 8, 1>, grid, block, 0, st, table, ids, y, n, vocab, (unsigned)dim, scale));
  return launch_status(tsb_launch::launch(scaled_lookup<T, 4>, grid, block, 0, st, table, ids, y, n * dim, vocab, (unsigned)dim, scale));
}

constexpr long long MAX_TOKENS = 1ll << 30, MAX_VOCAB = 1ll << 24, MAX_DIM = 1ll << 20;     // (ids are whole numbers in fp32)

}  // namespace

extern "C" {

int tsb_embedding_scaled(const float* table, const float* ids, float* y, long long n, long long vocab, long long dim,
                         float scale, void* stream) {
  if (n < 0 || vocab <= 0 || dim <= 0 || dim > MAX_DIM || n > MAX_TOKENS || vocab > MAX_VOCAB) return TSB_ERR_ARG;
  if (n == 0) return TSB_OK;
  if (!table || !ids || !y) return TSB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool v4 = dim % 4 == 0 && ((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  return v4 ? lookup(reinterpret_cast<const float4*>(table), ids, reinterpret_cast<float4*>(y), n, vocab, dim / 4, scale, st)
            : lookup(table, ids, y, n, vocab, dim, scale, st);
}

// Scratch of a gradient: sorted keys and positions (twice, and the histograms, above one cluster's share), partial rows.
int tsb_embedding_sorted_grad(const float* g, const float* ids, float* dtable, long long n, long long vocab, long long dim,
                              float scale, long long padding, void* stream) {
  if (n < 0 || vocab <= 0 || dim <= 0 || dim > MAX_DIM || n > MAX_TOKENS || vocab > MAX_VOCAB) return TSB_ERR_ARG;
  if (!dtable || (n && (!g || !ids))) return TSB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long cells = vocab * dim;
  const bool out16 = (reinterpret_cast<uintptr_t>(dtable) & 15) == 0;
  const bool v4 = dim % 4 == 0 && out16 && (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  const bool one_cluster = n <= (long long)MAX_CLUSTER * SORT_TILE;
  Zeros zeros{dtable, cells, 0, 1, 2 * 148, out16};
  if (n == 0) return launch_status(tsb_launch::launch(fill_zero, dim3(zeros.blocks), dim3(SORT_THREADS), 0, st, zeros));
  if (n <= FEW_TOKENS)
    return v4 ? sums_of_few(reinterpret_cast<const float4*>(g), ids, n, vocab, padding, dim / 4, scale, reinterpret_cast<float4*>(dtable), st)
              : sums_of_few(g, ids, n, vocab, padding, dim, scale, dtable, st);
  const int size = n <= 16384 ? 16 : MAX_TILE;
  const unsigned tiles = (unsigned)((n + size - 1) / size);
  const unsigned sort_tiles = (unsigned)((n + SORT_TILE - 1) / SORT_TILE);
  const size_t list = ((size_t)n * 4 + 255) / 256 * 256;
  const size_t hist_bytes = one_cluster ? 0 : (size_t)DIGITS * sort_tiles * 4;
  const size_t part_bytes = (size_t)2 * tiles * dim * 4;
  const size_t join_bytes = ((size_t)(1 + tiles) * 4 + 255) / 256 * 256;
  char* base = static_cast<char*>(tsb_scratch::get(st, tsb_scratch::EMBED_SORT, list * (one_cluster ? 2 : 4) + hist_bytes + join_bytes + part_bytes));
  if (!base) return TSB_ERR_OOM;
  unsigned* const joins = reinterpret_cast<unsigned*>(base);
  base += join_bytes;
  unsigned* key[2] = {reinterpret_cast<unsigned*>(base), nullptr};
  unsigned* pos[2] = {reinterpret_cast<unsigned*>(base + list), nullptr};
  char* rest = base + 2 * list;
  const int bits = bits_of(vocab), passes = (bits + 7) / 8, step = (bits + passes - 1) / passes;
  int last = 0;
  if (one_cluster) {
    unsigned blocks = 1;
    while (blocks < MAX_CLUSTER && (long long)blocks * SORT_THREADS < n) blocks *= 2;
    // zeros: 64 KB a block, in whole clusters, as many as run at once beside the sort (two to an SM: 8192 x 32000 x 512 takes
    // 16 us so, 20 us with 128)
    const long long fillers = (cells * 4 + 65535) / 65536;
    zeros.blocks = (int)((fillers < 2 * 148 ? fillers : 2 * 148) + blocks - 1) / blocks * blocks;
    const cudaError_t e =
        n <= blocks * SORT_THREADS * 1ll   ? sort_in_cluster<1>(ids, n, vocab, padding, bits, passes, key[0], pos[0], joins, zeros, blocks, st)
        : n <= blocks * SORT_THREADS * 2ll ? sort_in_cluster<2>(ids, n, vocab, padding, bits, passes, key[0], pos[0], joins, zeros, blocks, st)
                                           : sort_in_cluster<4>(ids, n, vocab, padding, bits, passes, key[0], pos[0], joins, zeros, blocks, st);
    if (e != cudaSuccess) return launch_status(e);
  } else {
    key[1] = reinterpret_cast<unsigned*>(rest);
    pos[1] = reinterpret_cast<unsigned*>(rest + list);
    unsigned* hist = reinterpret_cast<unsigned*>(rest + 2 * list);
    rest += 2 * list + hist_bytes;
    const unsigned mask = (1u << step) - 1;
    zeros.parts = 3 * passes;
    for (int p = 0; p < passes; ++p) {
      const unsigned* in_key = p ? key[(p + 1) & 1] : nullptr;
      const unsigned* in_pos = p ? pos[(p + 1) & 1] : nullptr;
      last = p & 1;
      cudaError_t e = tsb_launch::launch(tile_histogram, dim3(sort_tiles + zeros.blocks), dim3(SORT_THREADS), 0, st, ids, in_key, n,
                                         (unsigned)vocab, padding, p * step, mask, hist, sort_tiles, joins, zeros);
      ++zeros.part;
      if (e == cudaSuccess)
        e = tsb_launch::launch(scan_histogram, dim3(1 + zeros.blocks), dim3(SORT_THREADS), 0, st, hist, DIGITS * sort_tiles, zeros);
      ++zeros.part;
      if (e == cudaSuccess)
        e = tsb_launch::launch(scatter_tiles, dim3(sort_tiles + zeros.blocks), dim3(SORT_THREADS), sizeof(SortShared), st, ids, in_key, in_pos,
                               n, (unsigned)vocab, padding, p * step, mask, hist, sort_tiles, key[last], pos[last], zeros);
      ++zeros.part;
      if (e != cudaSuccess) return launch_status(e);
    }
  }
  if (v4)
    return sums(reinterpret_cast<const float4*>(g), key[last], pos[last], n, (unsigned)vocab, (unsigned)(dim / 4), scale, size,
                tiles, reinterpret_cast<float4*>(dtable), reinterpret_cast<float4*>(rest), joins, st);
  return sums(g, key[last], pos[last], n, (unsigned)vocab, (unsigned)dim, scale, size, tiles, dtable,
              reinterpret_cast<float*>(rest), joins, st);
}

}  // extern "C"
