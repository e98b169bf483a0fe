// Log probabilities of given tokens, with the entropy of each row, its log-sum-exp and the `top` likeliest tokens.
//
//   out[r] = [ log p(id_r), H, lse, log p of the top tokens (falling), their ids ],   p = softmax(x[r, :])
//   H = log Z - sum(e^u u) / Z,  log p = u - log Z   with u = x - max, Z = sum e^u
//
// (log p = x - lse would lose what lies below half a step of the maximum, which is all there is of a token that is nearly
// certain.)
// An id outside [0, cols) means no token: 0.  A row of -inf alone has lse = log p = -inf and H = 0, and no gradient.  NaN
// makes the row's results NaN and is no alternative itself (id -1 where fewer than `top` others are left).  Equal logits are
// taken by their column, the lowest first.
//
// One pass over the logits: every thread keeps a running (max, Z, sum e^u u).  Rows of up to 16384 columns, and of up to 32768 where
// there are no more rows than SMs, stay in registers (score_short_rows).  In longer ones (score_rows) the top tokens come from the
// maxima of units of the row (1 KB or more each that a warp reads in one go; in the shares of a cluster that splits a row the 8
// columns that a thread reads in one go).  With W warps, a bound that the ceil(top / W)-th best unit of every warp reaches is
// reached by `top` columns, so by every top token; of the units that reach it the top-th best one is the bound.  Their columns are
// read again (about `top` KB a row); what reaches the bound, some dozens, is collected in shared memory as 64-bit numbers that order
// by logit and then by column, and each one's place is how many are larger.  Where more are found than there is room for (ties,
// many equal units), every warp merges what it finds into a sorted list of the best 32, one per lane, against a rising bound.
// (4096 x 128001, 20 alternatives, without any 310 us: such lists in the first pass 572 us, in the second 497, sorting networks in
// place of counting 415; now 373.)
// What a row's end takes is latency that other rows on the SM have to cover, so it is kept short.
// Few long rows are split over a cluster of blocks that join through distributed shared memory.
#include <cuda_runtime.h>
#include <cooperative_groups.h>
#include <stdint.h>

#include "launch.cuh"

#define TSB_OK 0
#define TSB_ERR_ARG 1
#define TSB_ERR_LAUNCH 3

namespace {

namespace cg = cooperative_groups;
using tsb_launch::load;
typedef unsigned long long u64;

constexpr int MAX_WARPS = 8, MAX_TOP = 32, PENDING = 64, MAX_SPLIT = 8, MAX_UNITS = 1024, FOUND = 512, REACHED = 256;
constexpr unsigned CHUNK = 64;             // 16-byte pieces that a warp reads in one go, two a lane
constexpr float NEG_INF = -__builtin_huge_valf();
constexpr unsigned ALL = 0xffffffffu;

int launch_status(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  else cudaGetLastError();
  return e == cudaSuccess ? TSB_OK : TSB_ERR_LAUNCH | ((int)e << 8);
}

// Larger for a larger logit, then for a lower column; above 0 for every number, 0 stands for "none".  -0 counts as 0.
__device__ __forceinline__ u64 order_of(float x, unsigned col) {
  unsigned b = __float_as_uint(x);
  if ((b << 1) == 0) b = 0;
  b ^= (b >> 31) ? 0xffffffffu : 0x80000000u;
  return ((u64)b << 32) | (ALL - col);
}
__device__ __forceinline__ float logit_of(u64 key) {
  const unsigned b = (unsigned)(key >> 32);
  return __uint_as_float((b >> 31) ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ unsigned col_of(u64 key) { return ALL - (unsigned)key; }

__device__ __forceinline__ u64 larger(u64 a, u64 b) { return a > b ? a : b; }

// One compare-exchange of a bitonic network between lanes `d` apart; `falling`: the larger one to the lower lane.
template <class T> __device__ __forceinline__ T exchange(T v, int d, bool falling) {
  const T o = __shfl_xor_sync(ALL, v, d);
  return (((threadIdx.x & d) == 0) == falling) == (v > o) ? v : o;
}
template <class T> __device__ __forceinline__ T merge_falling(T v) {      // a bitonic sequence of 32 into falling order
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = exchange(v, d, true);
  return v;
}
template <class T> __device__ __forceinline__ T sort_falling(T v) {
#pragma unroll
  for (int size = 2; size < 32; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d > 0; d >>= 1) v = exchange(v, d, (threadIdx.x & size) == 0);
  return merge_falling(v);
}
// The best 32 of two falling lists.
template <class T> __device__ __forceinline__ T best_of(T a, T b) {
  const T o = __shfl_sync(ALL, b, 31 - (threadIdx.x & 31));
  return merge_falling(a > o ? a : o);
}

struct Sums {
  float m, z, t;               // max, sum e^(x - m), sum e^(x - m) (x - m)
};
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float ref = r.m == NEG_INF ? 0.f : r.m;
  const float ua = fmaxf(a.m - ref, -1e4f), ub = fmaxf(b.m - ref, -1e4f);
  const float ea = __expf(ua), eb = __expf(ub);
  r.z = a.z * ea + b.z * eb;
  r.t = ea * (a.t + a.z * ua) + eb * (b.t + b.z * ub);
  return r;
}

// Takes logits of up to N columns into the sums; their maximum.  What is below every real logit by more than e^-10000 counts as
// nothing.
template <int N>
__device__ __forceinline__ float take(Sums& s, const float (&x)[N]) {
  float m = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
  if (m > s.m) s = join(s, Sums{m, 0.f, 0.f});
  const float ref = s.m == NEG_INF ? 0.f : s.m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float u = x[i] - ref;
    const float e = __expf(u);
    s.z += e;
    s.t += e * fmaxf(u, -1e4f);
  }
  return m;
}

__device__ __forceinline__ float log_p(float x, float max, float log_z) { return (x - max) - log_z; }

__device__ __forceinline__ float warp_max(float v) {     // of numbers: a NaN counts as none
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

struct Shared {
  union {
    u64 pending[MAX_WARPS][PENDING];         // of the lists
    u64 found[FOUND];                        // columns that reach the bound
  };
  u64 lists[MAX_WARPS][32];
  u64 best_of_block[32];
  u64 bound;                   // no key below it is among the top of the row
  float maxima[MAX_UNITS];     // of the units, a share for every warp
  float least[MAX_WARPS];      // what each warp has as many units above as it has to
  float reached[REACHED], refined;           // maxima of the units that reach the first bound; the second bound
  unsigned units, count;       // how many these are; columns found
  float lse, max, log_z;       // of the row; NaN-free rows of -inf: lse is -inf
  Sums sums[MAX_WARPS];
  Sums of_block;
};

// A warp's list of the best, and what waits to be merged into it.
struct Chosen {
  u64 best;
  int waiting;
};
__device__ __forceinline__ void merge_waiting(Chosen& c, Shared& s, int top, int count) {
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncwarp();
  const u64 v = (int)lane < count ? s.pending[warp][lane] : 0;
  c.best = best_of(c.best, sort_falling(v));
  const u64 bound = __shfl_sync(ALL, c.best, top - 1);
  if (lane == 0) atomicMax(&s.bound, bound);
  __syncwarp();
  c.waiting -= count;
  if ((int)lane < c.waiting) s.pending[warp][lane] = s.pending[warp][count + lane];
  __syncwarp();
}
// Columns col to col + N - 1 of a lane, those below `limit`.  All lanes of the warp call it.
template <int N>
__device__ __forceinline__ void choose(Chosen& c, Shared& s, int top, const float (&x)[N], unsigned col, unsigned limit) {
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 bound = *(volatile u64*)&s.bound;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const u64 key = order_of(x[i], col + i);
    const bool in = x[i] == x[i] && key > bound && col + i < limit;             // (a NaN is not)
    const unsigned mask = __ballot_sync(ALL, in);
    if (!mask) continue;
    if (in) s.pending[warp][c.waiting + __popc(mask & ((1u << lane) - 1))] = key;
    c.waiting += __popc(mask);
    if (c.waiting >= 32) {
      merge_waiting(c, s, top, 32);
      bound = larger(bound, __shfl_sync(ALL, c.best, top - 1));
    }
  }
}

// Of n keys (0: none) the larger ones each at the place that the number of still larger ones tells: put(place, key).
// Returns how many there are.
template <class Put> __device__ __forceinline__ unsigned place(const u64* keys, unsigned n, Put put) {
  unsigned there = 0;
  for (unsigned t = threadIdx.x; t < n || t == threadIdx.x; t += blockDim.x) {
    const u64 key = t < n ? keys[t] : 0;
    unsigned larger = 0;
    there = 0;
#pragma unroll 4
    for (unsigned j = 0; j < n; ++j) {
      larger += keys[j] > key;
      there += keys[j] != 0;
    }
    if (key) put(larger, key);
  }
  return there;
}

// Grid: (rows * split) blocks in clusters of `split`; a block takes a contiguous part of its row.
template <bool TOP>
__global__ void __launch_bounds__(MAX_WARPS * 32, 6) score_rows(const float* x, const float* ids, float* __restrict__ out,
                                                                long long cols, int top, int split) {
  tsb_launch::enter();
  __shared__ Shared s;
  const long long row = blockIdx.x / split;
  const int part = blockIdx.x % split;
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const float* xr = x + row * cols;
  float* const to = out + row * (3 + 2 * top);
  // whole parts of 4 columns; a part's first columns up to a 16-byte boundary are taken one by one
  const unsigned per = (unsigned)((cols + split - 1) / split + 3) / 4 * 4;
  const unsigned begin = min((long long)part * per, cols), end = min((long long)begin + per, cols);
  const unsigned odd = (unsigned)((-(long long)(reinterpret_cast<uintptr_t>(xr + begin) >> 2)) & 3);
  const unsigned body = min(begin + odd, end), pieces = (end - body) / 4, tail = body + pieces * 4;
  // (the last warp writes the row's numbers: its loads are under way from the start)
  const long long id = (long long)load(ids + row);
  const bool given = id >= 0 && id < cols;
  const float own_x = given && warp == warps - 1 ? load(xr + id) : 0.f;

  Sums a{NEG_INF, 0.f, 0.f};
  const float4* xv = reinterpret_cast<const float4*>(xr + body);
  const float4 none = make_float4(NEG_INF, NEG_INF, NEG_INF, NEG_INF);
  // chunk by chunk, `length` of them a run; a unit is a run, or, in short rows, a lane's part of a chunk
  const unsigned chunks = (pieces + CHUNK - 1) / CHUNK, share = MAX_UNITS / warps;
  const unsigned per_warp = (chunks + warps - 1) / warps;
  const bool lanes_apart = per_warp * 32 <= share;
  const unsigned length = lanes_apart ? 1 : (per_warp + share - 1) / share;
  float* const maxima = s.maxima + warp * share;
  auto get = [&](unsigned chunk, float4& v, float4& w) {
    const unsigned i = chunk * CHUNK + lane;
    v = i < pieces ? load(xv + i) : none;
    w = i + 32 < pieces ? load(xv + i + 32) : none;
  };
  if (TOP && threadIdx.x < 32) {
    s.best_of_block[lane] = 0;
    if (lane == 0) s.count = s.units = 0, s.refined = NEG_INF;
  }
  // this warp's chunks in their order; two are read at a time (it takes some 60 KB under way to an SM to keep memory busy)
  auto chunk_of = [&](unsigned i) { return length == 1 ? warp + i * warps : (i / length * warps + warp) * length + i % length; };
  float most = NEG_INF;
  unsigned units = 0;                        // of this warp
  auto keep = [&](float m, unsigned i) {     // (a NaN is never a maximum here)
    if (lanes_apart) {
      maxima[units + lane] = m;
      units += 32;
      return;
    }
    most = fmaxf(most, m);
    if (length > 1 && (i + 1) % length && chunk_of(i + 1) < chunks) return;
    const float all = warp_max(most);
    if (lane == 0) maxima[units] = all;
    ++units;
    most = NEG_INF;
  };
  for (unsigned i = 0; chunk_of(i) < chunks; i += 2) {
    const bool more = chunk_of(i + 1) < chunks;
    float4 v[4];
    get(chunk_of(i), v[0], v[1]);
    if (more) get(chunk_of(i + 1), v[2], v[3]);
    const float f[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
    const float m = take(a, f);
    if (TOP) keep(m, i);
    if (more) {
      const float h[8] = {v[2].x, v[2].y, v[2].z, v[2].w, v[3].x, v[3].y, v[3].z, v[3].w};
      const float n = take(a, h);
      if (TOP) keep(n, i + 1);
    }
  }
  // up to three columns at either end, a thread of warp 0 each
  const unsigned heads = body - begin, rest = end - tail;
  const unsigned odd_col = threadIdx.x < heads ? begin + threadIdx.x : tail + (threadIdx.x - heads);
  const bool has_odd = threadIdx.x < heads + rest;
  const float odd_x[1] = {has_odd ? load(xr + odd_col) : NEG_INF};
  if (warp == 0) take(a, odd_x);
  {
    const float m = warp_max(a.m);           // one rescaling, then plain sums
    a = join(a, Sums{m, 0.f, 0.f});
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      a.z += __shfl_xor_sync(ALL, a.z, d);
      a.t += __shfl_xor_sync(ALL, a.t, d);
    }
  }
  if (lane == 0) s.sums[warp] = a;
  float least = NEG_INF;
  if (TOP) {
    __syncwarp();
    // the need-th best unit: the best one is taken out that many times less one
    unsigned gone = 0;                       // of the lane's units (bit k: unit 32 k + lane)
    for (int need = (top + warps - 1) / warps; need > 0; --need) {
      float own = NEG_INF;
      unsigned at = 32;
      for (unsigned k = 0; k * 32 + lane < units; ++k)
        if (!(gone >> k & 1) && (at == 32 || maxima[k * 32 + lane] > own)) own = maxima[k * 32 + lane], at = k;
      least = warp_max(own);
      const unsigned holders = __ballot_sync(ALL, own == least && at < 32);
      if (!holders) {                        // fewer units than needed
        least = NEG_INF;
        break;
      }
      if (lane == __ffs(holders) - 1) gone |= 1u << at;
    }
    if (lane == 0) s.least[warp] = least;
  }
  __syncthreads();
  auto finish = [&](Sums r) {                // the row's numbers
    const bool empty = r.m == NEG_INF && r.z == 0.f;                            // (NaN leaves z a NaN)
    const double z = (double)r.z, log_z = log(z);
    const float lse = empty ? NEG_INF : r.m + (float)log_z;
    s.lse = lse, s.max = r.m, s.log_z = (float)log_z;
    to[0] = given ? (empty ? NEG_INF : log_p(own_x, r.m, (float)log_z)) : 0.f;
    to[1] = empty ? 0.f : (float)(log_z - (double)r.t / z);
    to[2] = lse;
  };
  if (warp == warps - 1) {                   // the sums of the block, while the others look for columns
    a = lane < warps ? s.sums[lane] : Sums{NEG_INF, 0.f, 0.f};
#pragma unroll
    for (int d = MAX_WARPS / 2; d > 0; d >>= 1)
      a = join(a, Sums{__shfl_xor_sync(ALL, a.m, d), __shfl_xor_sync(ALL, a.z, d), __shfl_xor_sync(ALL, a.t, d)});
    if (lane == 0) {
      if (split > 1) s.of_block = a;
      else finish(a);
    }
  }
  if (!TOP && split == 1) return;
  auto write = [&](unsigned at, u64 key) {   // an alternative of the row
    if ((int)at >= top) return;
    to[3 + at] = s.lse == NEG_INF ? NEG_INF : log_p(logit_of(key), s.max, s.log_z);
    to[3 + top + at] = (float)col_of(key);
  };
  auto fill = [&](unsigned there) {          // fewer numbers than alternatives
    if (threadIdx.x >= there && (int)threadIdx.x < top) {
      to[3 + threadIdx.x] = __int_as_float(0x7fc00000);
      to[3 + top + threadIdx.x] = -1.f;
    }
  };
  if (TOP) {
    for (unsigned k = 0; k < warps; ++k) least = fminf(least, s.least[k]);
    for (unsigned first = 0; first < units; first += 32) {
      const bool in = first + lane < units && maxima[first + lane] >= least;
      const unsigned mask = __ballot_sync(ALL, in);
      unsigned at = 0;
      if (lane == 0 && mask) at = atomicAdd(&s.units, __popc(mask));            // (their order does not matter)
      at = __shfl_sync(ALL, at, 0) + __popc(mask & ((1u << lane) - 1));
      if (in && at < REACHED) s.reached[at] = maxima[first + lane];
    }
    __syncthreads();
    if (s.units <= REACHED) {
      for (unsigned t = threadIdx.x; t < s.units; t += blockDim.x) {
        const float v = s.reached[t];
        int better = 0;
        for (unsigned j = 0; j < s.units; ++j) better += s.reached[j] > v || (s.reached[j] == v && j < t);
        if (better == top - 1) s.refined = v;
      }
      __syncthreads();
      least = fmaxf(least, s.refined);
    }
    const u64 bound = order_of(least, ALL);  // below every column of that value
    // every warp its own units again, by chunks: f(columns of a lane, first column, limit)
    auto again = [&](auto f) {
      auto both = [&](unsigned chunk, bool mine) {
        float4 v = none, w = none;
        if (mine) get(chunk, v, w);
        const unsigned i = chunk * CHUNK + lane, col = body + i * 4;
        const float p[4] = {v.x, v.y, v.z, v.w}, q[4] = {w.x, w.y, w.z, w.w};
        f(p, col, mine && i < pieces ? end : 0);
        f(q, col + 128, mine && i + 32 < pieces ? end : 0);
      };
      if (lanes_apart) {
        for (unsigned k = 0; k < units; k += 32) {
          const bool mine = maxima[k + lane] >= least;
          if (__any_sync(ALL, mine)) both(chunk_of(k / 32), mine);
        }
      } else {
        for (unsigned first = 0; first < units; first += 32)
          for (unsigned left = __ballot_sync(ALL, first + lane < units && maxima[first + lane] >= least); left; left &= left - 1) {
            const unsigned at = (first + __ffs(left) - 1) * length;
            for (unsigned k = at; k < at + length && chunk_of(k) < chunks; ++k) both(chunk_of(k), true);
          }
      }
      if (warp == 0) f(odd_x, odd_col, has_odd ? end : 0);
    };
    again([&](const auto& x, unsigned col, unsigned limit) {
#pragma unroll
      for (int i = 0; i < (int)(sizeof(x) / sizeof(x[0])); ++i)
        if (x[i] >= least && col + i < limit) {                                    // (a NaN is not)
          const unsigned at = atomicAdd(&s.count, 1u);                          // (their order does not matter)
          if (at < FOUND) s.found[at] = order_of(x[i], col + i);
        }
    });
    __syncthreads();
    unsigned count = s.count;
    const u64* keys = s.found;
    if (count > FOUND) {                     // (the same for all threads)
      __syncthreads();
      if (threadIdx.x == 0) s.bound = bound;
      __syncthreads();
      Chosen c{0, 0};
      again([&](const auto& x, unsigned col, unsigned limit) { choose(c, s, top, x, col, limit); });
      merge_waiting(c, s, top, c.waiting);
      s.lists[warp][lane] = c.best;
      __syncthreads();
      keys = s.lists[0];
      count = warps * 32;
    }
    if (split == 1) {
      fill(place(keys, count, write));
      return;
    }
    place(keys, count, [&](unsigned at, u64 key) {
      if (at < 32) s.best_of_block[at] = key;
    });
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  if (part == 0) {
    if (TOP)
      for (int t = threadIdx.x; t < split * top; t += blockDim.x) s.lists[0][t] = *cluster.map_shared_rank(&s.best_of_block[t % top], t / top);
    if (warp == warps - 1 && lane == 0) {
      for (int k = 1; k < split; ++k) a = join(a, *cluster.map_shared_rank(&s.of_block, k));
      finish(a);
    }
  }
  cluster.sync();
  if (TOP && part == 0) fill(place(s.lists[0], split * top, write));
}

// Short rows stay in registers: WARPS warps take a row of up to 32 N WARPS columns, a warp every WARPS-th 32 of them; with one warp to
// a row a block takes eight rows.  The need-th best of a warp's lane maxima, need = top / WARPS rounded up, is reached by as many
// columns, so the least of these bounds the top columns from below; what reaches it goes to shared memory, where each one's place is
// how many are larger.  Where that is more than there is room for (ties), the best one below the last is looked for `top` times.
// What does not fit one SM's registers with rows to spare goes to score_rows.  (Without alternatives, with five, with twenty: 8192 x
// 1000 5.8, 9.7 and 14 us, by units that are read again 13, 45 and 97; 8192 x 5000 28, 46 and 49, 35, 80 and 114; one row of 32000 3.7,
// 5.8 and 6.2, of which a cluster makes 4, 9 and 14.)
constexpr int SHORT_WARPS = 8, SHORT_FOUND = 128;
template <int N, int WARPS, bool TOP>
__global__ void __launch_bounds__(WARPS > SHORT_WARPS ? WARPS * 32 : SHORT_WARPS * 32)
    score_short_rows(const float* x, const float* ids, float* __restrict__ out, long long rows, int cols, int top) {
  tsb_launch::enter();
  constexpr int ROWS = WARPS == 1 ? SHORT_WARPS : 1, ROOM = WARPS == 1 ? SHORT_FOUND : FOUND;
  __shared__ u64 found[TOP ? ROWS : 1][ROOM], best_of[WARPS];
  __shared__ Sums sums[WARPS];
  __shared__ float leasts[WARPS], lse_of_row, max_of_row, log_z_of_row;
  __shared__ int all;
  const int lane = threadIdx.x & 31, warp = WARPS == 1 ? 0 : threadIdx.x >> 5, own_row = WARPS == 1 ? threadIdx.x >> 5 : 0;
  const long long row = blockIdx.x * (long long)ROWS + own_row;
  if (row >= rows) return;                   // (whole warps, and no block that has barriers)
  auto sync = [] {
    if (WARPS == 1) __syncwarp();
    else __syncthreads();
  };
  const int first = warp * 32 + lane;        // the lane's columns: first + i * 32 WARPS
  const float* const xr = x + row * cols + first;
  float* const to = out + row * (3 + 2 * top);
  float v[N], own = NEG_INF;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = first + i * (32 * WARPS) < cols ? load(xr + i * (32 * WARPS)) : NEG_INF;
  const long long id = (long long)load(ids + row);
  const bool given = id >= 0 && id < cols;
  const float own_x = given ? load(x + row * cols + id) : 0.f;
  if (WARPS > 1 && threadIdx.x == 0) all = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) own = fmaxf(own, v[i]);
  const float most = warp_max(own), ref = most == NEG_INF ? 0.f : most;
  float z[2] = {0.f, 0.f}, t[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float u = v[i] - ref, e = __expf(u);
    z[i & 1] += e;
    t[i & 1] += e * fmaxf(u, -1e4f);
  }
  Sums a{most, z[0] + z[1], t[0] + t[1]};
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    a.z += __shfl_xor_sync(ALL, a.z, d);
    a.t += __shfl_xor_sync(ALL, a.t, d);
  }
  float least = TOP ? __shfl_sync(ALL, sort_falling(own), (top + WARPS - 1) / WARPS - 1) : NEG_INF;
  if (WARPS > 1) {
    if (lane == 0) sums[warp] = a, leasts[warp] = least;
    __syncthreads();
    for (int w = 0; w < WARPS; ++w) least = fminf(least, leasts[w]);
    if (warp == WARPS - 1) {
      a = lane < WARPS ? sums[lane] : Sums{NEG_INF, 0.f, 0.f};
#pragma unroll
      for (int d = WARPS / 2; d > 0; d >>= 1)
        a = join(a, Sums{__shfl_xor_sync(ALL, a.m, d), __shfl_xor_sync(ALL, a.z, d), __shfl_xor_sync(ALL, a.t, d)});
    }
  }
  float lse = 0.f, log_z = 0.f;
  if (warp == WARPS - 1) {
    const bool empty = a.m == NEG_INF && a.z == 0.f;
    const double wide = log((double)a.z);
    log_z = (float)wide;
    lse = empty ? NEG_INF : a.m + log_z;
    if (lane == 0) {
      to[0] = given ? (empty ? NEG_INF : log_p(own_x, a.m, log_z)) : 0.f;
      to[1] = empty ? 0.f : (float)(wide - (double)a.t / (double)a.z);
      to[2] = lse;
      if (WARPS > 1) lse_of_row = lse, max_of_row = a.m, log_z_of_row = log_z;
    }
  }
  if (!TOP) return;
  // which of the lane's columns reach the bound (a NaN does not), and where they go
  u64 bits = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) bits |= (u64)(v[i] >= least) << i;
  const int there = first < cols ? (cols - first + 32 * WARPS - 1) / (32 * WARPS) : 0;
  if (there < 64) bits &= (1ull << there) - 1;
  int count = __popcll(bits), at = count;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(ALL, at, d);
    if (lane >= d) at += o;
  }
  at -= count;
  count = __shfl_sync(ALL, at + count, 31);
  if (WARPS > 1) {
    if (lane == 0 && count) count = atomicAdd(&all, count);                       // (their order does not matter)
    at += __shfl_sync(ALL, count, 0);
  }
  u64* const keys = found[own_row];
  for (; bits && at < ROOM; bits &= bits - 1, ++at) {
    const int i = (__ffsll((long long)bits) - 1) * (32 * WARPS);
    keys[at] = order_of(load(xr + i), first + i);
  }
  sync();
  if (WARPS > 1) count = all, lse = lse_of_row, a.m = max_of_row, log_z = log_z_of_row;
  auto write = [&](int place, u64 key) {
    to[3 + place] = !key ? __int_as_float(0x7fc00000) : lse == NEG_INF ? NEG_INF : log_p(logit_of(key), a.m, log_z);
    to[3 + top + place] = key ? (float)col_of(key) : -1.f;
  };
  if (count <= ROOM) {
    for (int c = first; c < max(count, top); c += 32 * WARPS) {
      const u64 key = c < count ? keys[c] : 0;
      int place = c < count ? 0 : c;
#pragma unroll 4
      for (int j = 0; j < count; ++j) place += c < count && keys[j] > key;
      if (place < top) write(place, key);    // (fewer numbers than alternatives: the places behind them have none)
    }
    return;
  }
  u64 last = ~0ull;
  for (int k = 0; k < top; ++k) {
    u64 best = 0;
#pragma unroll 1
    for (int col = first; col < cols; col += 32 * WARPS) {       // (from memory: the columns' registers are free by now)
      const float y = load(x + row * cols + col);
      const u64 key = y == y ? order_of(y, col) : 0;
      if (key < last) best = larger(best, key);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) best = larger(best, __shfl_xor_sync(ALL, best, d));
    if (WARPS > 1) {
      if (lane == 0) best_of[warp] = best;
      __syncthreads();
      for (int w = 0; w < WARPS; ++w) best = larger(best, best_of[w]);
      __syncthreads();
    }
    if (first == 0) write(k, best);
    last = best;
  }
}
template <int N, int WARPS>
int short_rows(const float* x, const float* ids, float* out, long long rows, int cols, int top, cudaStream_t st) {
  const dim3 grid((unsigned)(WARPS == 1 ? (rows + SHORT_WARPS - 1) / SHORT_WARPS : rows)), block(WARPS == 1 ? SHORT_WARPS * 32 : WARPS * 32);
  if (top) return launch_status(tsb_launch::launch(score_short_rows<N, WARPS, true>, grid, block, 0, st, x, ids, out, rows, cols, top));
  return launch_status(tsb_launch::launch(score_short_rows<N, WARPS, false>, grid, block, 0, st, x, ids, out, rows, cols, top));
}

// dx_c = sum_i w_i (1[c = id_i] - p_c) + w_lse p_c - w_H p_c (log p_c + H), with w the gradient of `out` and the sum over
// the given token and the top ones, of which each lane of a warp has one.  Columns that are an id are computed apart, from the log p
// of `out` and with 1 - p as -expm1(log p), after the rest.  Columns [begin, end) of a row, by `threads` threads that `sync` is for.
template <class Sync>
__device__ __forceinline__ void grad_of_columns(const float* xr, const float* o, const float* w, float* dr, long long id, long long cols, int top,
                                                unsigned begin, unsigned end, unsigned thread, unsigned threads, Sync sync) {
  const int lane = threadIdx.x & 31;
  const bool given = id >= 0 && id < cols;
  const float entropy = load(o + 1), lse = load(o + 2), wh = load(w + 1), w_given = given ? load(w) : 0.f;
  const long long alternative = lane < top ? (long long)load(o + 3 + top + lane) : -1;
  const float w_alternative = alternative >= 0 ? load(w + 3 + lane) : 0.f;
  float weights = w_alternative;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) weights += __shfl_xor_sync(ALL, weights, d);
  weights += w_given;
  const bool empty = lse == NEG_INF;
  const float plain = load(w + 2) - weights;
  // of a column that is no id (w_H log p alone may be beyond fp32 where p is 0: a logit masked by the type's lowest number)
  auto rest = [&](float v) {
    const float lp = v - lse, p = __expf(lp);
    return empty || v == NEG_INF || p == 0.f ? 0.f : p * (plain - wh * (lp + entropy));
  };
  const unsigned odd = (unsigned)((-(long long)(reinterpret_cast<uintptr_t>(xr + begin) >> 2)) & 3);
  const bool same = ((reinterpret_cast<uintptr_t>(xr) ^ reinterpret_cast<uintptr_t>(dr)) & 15) == 0;
  const unsigned body = same ? min(begin + odd, end) : end, pieces = (end - body) / 4, tail = body + pieces * 4;
  const float4* xv = reinterpret_cast<const float4*>(xr + body);
  float4* dv = reinterpret_cast<float4*>(dr + body);
  tsb_launch::read_then_write<4>(thread, pieces, threads, [&](unsigned i) { return load(xv + i); },
                                 [&](unsigned i, float4 v) { dv[i] = make_float4(rest(v.x), rest(v.y), rest(v.z), rest(v.w)); });
  for (unsigned i = begin + thread; i < body; i += threads) dr[i] = rest(load(xr + i));
  for (unsigned i = tail + thread; i < end; i += threads) dr[i] = rest(load(xr + i));
  sync();                                // the columns below are written a second time
  if (thread >= 32 || empty) return;
  auto of_id = [&](long long col, float lp, float own) {
    if (col < (long long)begin || col >= (long long)end) return;
    const float p = expf(lp);
    const float other = p == 0.f ? 0.f : p * (load(w + 2) - (weights - own) - wh * (lp + entropy));
    dr[col] = own * -expm1f(lp) + other;
  };
  of_id(alternative, lane < top ? load(o + 3 + lane) : 0.f, w_alternative + (given && alternative == id ? w_given : 0.f));
  const bool both = __any_sync(ALL, alternative == id);                         // the lane of that one has done it
  if (lane == 0 && given && !both) of_id(id, load(o), w_given);
}

// A block takes a chunk of a row.
__global__ void __launch_bounds__(256) score_grad(const float* x, const float* ids, const float* out, const float* g,
                                                  float* __restrict__ dx, long long cols, int top, unsigned chunk, int chunks) {
  tsb_launch::enter();
  const long long row = blockIdx.x / chunks;
  const unsigned begin = (unsigned)(blockIdx.x % chunks) * chunk, end = (unsigned)min((long long)begin + chunk, cols);
  grad_of_columns(x + row * cols, out + row * (3 + 2 * top), g + row * (3 + 2 * top), dx + row * cols, (long long)load(ids + row), cols, top, begin,
                  end, threadIdx.x, 256u, [] { __syncthreads(); });
}
// A warp takes a row.
__global__ void __launch_bounds__(SHORT_WARPS * 32) score_grad_short(const float* x, const float* ids, const float* out, const float* g,
                                                                     float* __restrict__ dx, long long rows, long long cols, int top) {
  tsb_launch::enter();
  const long long row = blockIdx.x * (long long)SHORT_WARPS + (threadIdx.x >> 5);
  if (row >= rows) return;
  grad_of_columns(x + row * cols, out + row * (3 + 2 * top), g + row * (3 + 2 * top), dx + row * cols, (long long)load(ids + row), cols, top, 0,
                  (unsigned)cols, threadIdx.x & 31, 32u, [] { __syncwarp(); });
}

}  // namespace

extern "C" {

int tsb_token_score(const float* x, const float* ids, float* out, long long rows, long long cols, int top, void* stream) {
  if (rows < 0 || cols <= 0 || cols > (1ll << 24) || rows > (1ll << 27) || top < 0 || top > MAX_TOP || top > cols) return TSB_ERR_ARG;
  if (rows == 0) return TSB_OK;
  if (!x || !ids || !out) return TSB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // short rows: as few warps as hold them (8192 x 5000, five alternatives: four warps of 48 columns a lane 46 us, eight of 32 65); a row
  // of more than 16384 columns takes an SM, so there may be no more of them than SMs (445 x 17000: 13 us by score_rows, 17 so)
  const int c = (int)cols;
  if (cols <= 32) return short_rows<1, 1>(x, ids, out, rows, c, top, st);
  if (cols <= 128) return short_rows<4, 1>(x, ids, out, rows, c, top, st);
  if (cols <= 512) return short_rows<16, 1>(x, ids, out, rows, c, top, st);
  if (cols <= 1024) return short_rows<32, 1>(x, ids, out, rows, c, top, st);
  if (cols <= 2048) return short_rows<32, 2>(x, ids, out, rows, c, top, st);
  if (cols <= 4096) return short_rows<32, 4>(x, ids, out, rows, c, top, st);
  if (cols <= 6144) return short_rows<48, 4>(x, ids, out, rows, c, top, st);
  if (cols <= 8192) return short_rows<64, 4>(x, ids, out, rows, c, top, st);
  if (cols <= 12288) return short_rows<48, 8>(x, ids, out, rows, c, top, st);
  if (cols <= 16384) return short_rows<64, 8>(x, ids, out, rows, c, top, st);
  if (cols <= 32768 && rows <= 148) return short_rows<64, 16>(x, ids, out, rows, c, top, st);
  // a cluster of blocks for a row while the rows leave SMs idle and a block keeps 2048 columns
  int split = 1;
  while (split < MAX_SPLIT && rows * split * 2 <= 148 && cols >= 4096ll * split) split *= 2;
  // eight warps for few rows or long ones only: a row's end is latency, which more rows on an SM cover (4096 rows, 20 alternatives,
  // four warps and eight: 33000 columns 135 and 141 us, 48000 175 and 177, 64000 220 and 219, 96000 315 and 319, 128001 418 and 402)
  const int warps = cols / split >= 65536 || rows * split <= 4 * 148 ? MAX_WARPS : MAX_WARPS / 2;
  const dim3 grid((unsigned)(rows * split)), block(warps * 32);
  const unsigned cluster = split > 1 ? split : 0;
  if (top)
    return launch_status(tsb_launch::launch_cluster(cluster, score_rows<true>, grid, block, 0, st, x, ids, out, cols, top, split));
  return launch_status(tsb_launch::launch_cluster(cluster, score_rows<false>, grid, block, 0, st, x, ids, out, cols, top, split));
}

int tsb_token_score_grad(const float* x, const float* ids, const float* out, const float* g, float* dx, long long rows,
                         long long cols, int top, void* stream) {
  if (rows < 0 || cols <= 0 || cols > (1ll << 24) || rows > (1ll << 27) || top < 0 || top > MAX_TOP || top > cols) return TSB_ERR_ARG;
  if (rows == 0) return TSB_OK;
  if (!x || !ids || !out || !g || !dx) return TSB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // (a block's barrier and the row's numbers are most of a short row: 8192 x 1000, five alternatives, 10 us by warps, 23 by blocks; 300 x
  // 1000 3.3 and 2.2)
  if (cols <= 2048 && rows >= 148 * SHORT_WARPS)
    return launch_status(tsb_launch::launch(score_grad_short, dim3((unsigned)((rows + SHORT_WARPS - 1) / SHORT_WARPS)), dim3(SHORT_WARPS * 32), 0, st,
                                            x, ids, out, g, dx, rows, cols, top));
  // chunks of a row that keep 4 x 4 columns a thread, until there are four blocks for every SM
  long long chunks = 1;
  while (rows * chunks < 148 * 4 && cols >= 8192 * chunks) chunks *= 2;
  const unsigned chunk = (unsigned)((cols + chunks - 1) / chunks + 3) / 4 * 4;
  const int count = (int)((cols + chunk - 1) / chunk);
  if (rows * count > INT32_MAX) return TSB_ERR_ARG;
  return launch_status(tsb_launch::launch(score_grad, dim3((unsigned)(rows * count)), dim3(256), 0, st, x, ids, out, g, dx, cols,
                                          top, chunk, count));
}

}  // extern "C"
