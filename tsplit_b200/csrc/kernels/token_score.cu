// Log probabilities of given tokens, with the entropy of each row, its log-sum-exp and the `top` likeliest tokens.
//
//   out[r] = [ log p(id_r), H, lse, log p of the top tokens (falling), their ids ],   p = softmax(x[r, :])
//   H = log Z - sum(e^u u) / Z   with u = x - max, Z = sum e^u
//
// An id outside [0, cols) means no token: 0.  A row of -inf alone has lse = log p = -inf and H = 0, and no gradient.  NaN
// makes the row's results NaN and is no alternative itself (id -1 where fewer than `top` others are left).  Equal logits are
// taken by their column, the lowest first.
//
// One pass over the logits: every thread keeps a running (max, Z, sum e^u u).  The top tokens: every warp keeps the best 32
// it has seen, one per lane, as 64-bit numbers that order by logit and then by column, and collects what is above its
// bound (the top-th best of any warp of the block) in shared memory until there are 32 of them, which are sorted and merged.
// Few rows are split over a cluster of blocks that join through distributed shared memory.
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

constexpr int MAX_WARPS = 8, MAX_TOP = 32, PENDING = 64, MAX_SPLIT = 8;
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
__device__ __forceinline__ u64 smaller(u64 a, u64 b) { return a < b ? a : b; }

// One compare-exchange of a bitonic network between lanes `d` apart; `falling`: the larger one to the lower lane.
__device__ __forceinline__ u64 exchange(u64 v, int d, bool falling) {
  const u64 o = __shfl_xor_sync(ALL, v, d);
  return (((threadIdx.x & d) == 0) == falling) ? larger(v, o) : smaller(v, o);
}
__device__ __forceinline__ u64 merge_falling(u64 v) {      // a bitonic sequence of 32 into falling order
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = exchange(v, d, true);
  return v;
}
__device__ __forceinline__ u64 sort_falling(u64 v) {
#pragma unroll
  for (int size = 2; size < 32; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d > 0; d >>= 1) v = exchange(v, d, (threadIdx.x & size) == 0);
  return merge_falling(v);
}
// The best 32 of two falling lists.
__device__ __forceinline__ u64 best_of(u64 a, u64 b) { return merge_falling(larger(a, __shfl_sync(ALL, b, 31 - (threadIdx.x & 31)))); }

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

// Takes logits of up to N columns into the sums.  What is below every real logit by more than e^-10000 counts as nothing.
template <int N>
__device__ __forceinline__ void take(Sums& s, const float (&x)[N]) {
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
}

struct Shared {
  u64 pending[MAX_WARPS][PENDING];
  u64 best[MAX_WARPS][32];
  u64 bound;                   // no key below it is among the top of the row
  Sums sums[MAX_WARPS];
  Sums of_block;
  u64 best_of_block[32];
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
// `any`: whether a lane holds something that may be above the bound.  All lanes of the warp call it.
template <int N>
__device__ __forceinline__ void choose(Chosen& c, Shared& s, int top, const float (&x)[N], unsigned col, unsigned limit) {
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 bound = *(volatile u64*)&s.bound;
  const float least = bound ? logit_of(bound) : NEG_INF;
  bool may = false;
#pragma unroll
  for (int i = 0; i < N; ++i) may |= x[i] >= least;
  if (!__any_sync(ALL, may)) return;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const u64 key = order_of(x[i], col + i);
    const bool in = x[i] >= least && key > bound && col + i < limit;          // (a NaN is not)
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

// Grid: (rows * split) blocks in clusters of `split`; a block takes a contiguous part of its row.
template <bool TOP>
__global__ void __launch_bounds__(MAX_WARPS * 32) score_rows(const float* x, const float* ids, float* __restrict__ out,
                                                             long long cols, int top, int split) {
  tsb_launch::enter();
  __shared__ Shared s;
  const long long row = blockIdx.x / split;
  const int part = blockIdx.x % split;
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const float* xr = x + row * cols;
  // whole parts of 4 columns; a part's first columns up to a 16-byte boundary are taken one by one
  const unsigned per = (unsigned)((cols + split - 1) / split + 3) / 4 * 4;
  const unsigned begin = min((long long)part * per, cols), end = min((long long)begin + per, cols);
  const unsigned odd = (unsigned)((-(long long)(reinterpret_cast<uintptr_t>(xr + begin) >> 2)) & 3);
  const unsigned body = min(begin + odd, end), pieces = (end - body) / 4, tail = body + pieces * 4;
  if (TOP && threadIdx.x == 0) s.bound = 0;
  if (TOP) __syncthreads();

  Sums a{NEG_INF, 0.f, 0.f};
  Chosen c{0, 0};
  const float4* xv = reinterpret_cast<const float4*>(xr + body);
  for (unsigned first = 0; first < pieces; first += 2 * blockDim.x) {          // (the same trips for all threads)
    const unsigned i = first + threadIdx.x, j = i + blockDim.x;
    const float4 none = make_float4(NEG_INF, NEG_INF, NEG_INF, NEG_INF);
    const float4 v = i < pieces ? load(xv + i) : none, w = j < pieces ? load(xv + j) : none;
    const float f[8] = {v.x, v.y, v.z, v.w, w.x, w.y, w.z, w.w};
    take(a, f);
    if (TOP) {
      const float g[4] = {v.x, v.y, v.z, v.w}, h[4] = {w.x, w.y, w.z, w.w};
      choose(c, s, top, g, body + i * 4, i < pieces ? end : 0);
      choose(c, s, top, h, body + j * 4, j < pieces ? end : 0);
    }
  }
  {                                                                             // up to three columns at either end
    const unsigned heads = body - begin, rest = end - tail;
    const unsigned col = threadIdx.x < heads ? begin + threadIdx.x : tail + (threadIdx.x - heads);
    const bool in = threadIdx.x < heads + rest;
    const float f[1] = {in ? load(xr + col) : NEG_INF};
    if (warp == 0) {
      take(a, f);
      if (TOP) choose(c, s, top, f, col, in ? end : 0);
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
    a = join(a, Sums{__shfl_xor_sync(ALL, a.m, d), __shfl_xor_sync(ALL, a.z, d), __shfl_xor_sync(ALL, a.t, d)});
  if (lane == 0) s.sums[warp] = a;
  if (TOP) {
    merge_waiting(c, s, top, c.waiting);
    s.best[warp][lane] = c.best;
  }
  __syncthreads();
  if (warp == 0) {
    for (unsigned k = 1; k < warps; ++k) a = join(a, s.sums[k]);
    if (TOP)
      for (unsigned k = 1; k < warps; ++k) c.best = best_of(c.best, s.best[k][lane]);
  }
  if (split > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (warp == 0) {
      if (lane == 0) s.of_block = a;
      if (TOP) s.best_of_block[lane] = c.best;
    }
    cluster.sync();
    if (part == 0 && warp == 0) {
      for (int k = 1; k < split; ++k) {
        a = join(a, *cluster.map_shared_rank(&s.of_block, k));
        if (TOP) c.best = best_of(c.best, *cluster.map_shared_rank(&s.best_of_block[lane], k));
      }
    }
    cluster.sync();
    if (part) return;
  }
  if (warp) return;
  float* to = out + row * (3 + 2 * top);
  const bool empty = a.m == NEG_INF && a.z == 0.f;                              // (NaN leaves z a NaN)
  const float lse = empty ? NEG_INF : a.m + (float)log((double)a.z);
  if (lane == 0) {
    const long long id = (long long)load(ids + row);
    to[0] = id >= 0 && id < cols ? (empty ? NEG_INF : load(xr + id) - lse) : 0.f;
    to[1] = empty ? 0.f : (float)(log((double)a.z) - (double)a.t / (double)a.z);
    to[2] = lse;
  }
  if (TOP && (int)lane < top) {
    const float v = c.best ? logit_of(c.best) : __int_as_float(0x7fc00000);
    to[3 + lane] = empty ? NEG_INF : v - lse;
    to[3 + top + lane] = c.best ? (float)col_of(c.best) : -1.f;
  }
}

// dx_c = sum_i w_i (1[c = id_i] - p_c) + w_lse p_c - w_H p_c (log p_c + H), with w the gradient of `out` and the sum over
// the given token and the top ones.  Columns that are an id are computed apart, with 1 - p as -expm1(log p), after the
// rest; a block takes a chunk of a row.
__global__ void __launch_bounds__(256) score_grad(const float* x, const float* ids, const float* out, const float* g,
                                                  float* __restrict__ dx, long long cols, int top, unsigned chunk, int chunks) {
  tsb_launch::enter();
  const long long row = blockIdx.x / chunks;
  const unsigned begin = (unsigned)(blockIdx.x % chunks) * chunk, end = (unsigned)min((long long)begin + chunk, cols);
  const float* xr = x + row * cols;
  float* dr = dx + row * cols;
  const float* o = out + row * (3 + 2 * top);
  const float* w = g + row * (3 + 2 * top);
  const long long id = (long long)load(ids + row);
  const bool given = id >= 0 && id < cols;
  const float entropy = load(o + 1), lse = load(o + 2), wh = load(w + 1);
  float weights = given ? load(w) : 0.f;
  for (int k = 0; k < top; ++k)
    if (load(o + 3 + top + k) >= 0.f) weights += load(w + 3 + k);
  const bool empty = lse == NEG_INF;
  const float plain = load(w + 2) - weights;
  auto rest = [&](float v) {                                                    // of a column that is no id
    const float lp = v - lse, p = __expf(lp);
    return empty || v == NEG_INF ? 0.f : p * (plain - wh * (lp + entropy));
  };
  const unsigned odd = (unsigned)((-(long long)(reinterpret_cast<uintptr_t>(xr + begin) >> 2)) & 3);
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
  const unsigned body = same ? min(begin + odd, end) : end, pieces = (end - body) / 4, tail = body + pieces * 4;
  const float4* xv = reinterpret_cast<const float4*>(xr + body);
  float4* dv = reinterpret_cast<float4*>(dr + body);
  tsb_launch::read_then_write<4>(threadIdx.x, pieces, 256u, [&](unsigned i) { return load(xv + i); },
                                 [&](unsigned i, float4 v) { dv[i] = make_float4(rest(v.x), rest(v.y), rest(v.z), rest(v.w)); });
  for (unsigned i = begin + threadIdx.x; i < body; i += 256) dr[i] = rest(load(xr + i));
  for (unsigned i = tail + threadIdx.x; i < end; i += 256) dr[i] = rest(load(xr + i));
  __syncthreads();                       // the columns below are written a second time
  const int k = (int)threadIdx.x - 1;    // thread 0: the given token, the others: the top ones
  if (k >= top || empty) return;
  const long long col = k < 0 ? (given ? id : -1) : (long long)load(o + 3 + top + k);
  if (col < (long long)begin || col >= (long long)end) return;
  float own = k < 0 ? load(w) : load(w + 3 + k);
  if (k < 0) {
    for (int j = 0; j < top; ++j)
      if ((long long)load(o + 3 + top + j) == col) return;                      // the thread of that one does it
  } else if (given && id == col) {
    own += load(w);
  }
  const float v = load(xr + col), lp = v - lse, p = expf(lp);
  const float other = v == NEG_INF ? 0.f : p * (load(w + 2) - (weights - own) - wh * (lp + entropy));
  dr[col] = own * -expm1f(lp) + other;
}

}  // namespace

extern "C" {

int tsb_token_score(const float* x, const float* ids, float* out, long long rows, long long cols, int top, void* stream) {
  if (rows < 0 || cols <= 0 || cols > (1ll << 24) || rows > (1ll << 27) || top < 0 || top > MAX_TOP || top > cols) return TSB_ERR_ARG;
  if (rows == 0) return TSB_OK;
  if (!x || !ids || !out) return TSB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // a cluster of blocks for a row while the rows leave SMs idle and a block keeps 2048 columns
  int split = 1;
  while (split < MAX_SPLIT && rows * split * 2 <= 148 && cols >= 4096ll * split) split *= 2;
  int warps = 1;                         // 16 columns a thread, where the row has as many
  while (warps < MAX_WARPS && cols / split >= 512ll * warps * 2) warps *= 2;
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
