// Attention across to an encoder's states, forward and backward.
//
//   q [N, Tq, H, d], kv [N, Tk, 2, G, d] (keys, then values; G heads, each read by H / G query heads), key [N, Tk] (0: out)
//   S = scale q k^T,  P = softmax(S) over the keys that are in,  y = P v
//   dP = dy v^T,  dS = P (dP - rowsum(dy y)),  dq = scale dS k,  dk = scale dS^T q,  dv = P^T dy
//
// A key that is out takes no part, whatever its row holds (it is not read).  A query without any key has y = 0 and no
// gradient.  The scores never leave the chip: the backward kernels compute them again from the rows' log-sum-exp.
//
// Products run on tcgen05 with the accuracy of fp32.  An operand tile is scaled by a power of two that brings its largest
// number to [2^13, 2^14) and split into two fp16 numbers, x = hi + lo, |x - hi - lo| <= 2^-22 |x| (or 2^-38 of the tile's
// largest, where fp16 ends); a product is three: hi hi + hi lo + lo hi.  That takes 1.5 times the tensor time of one TF32
// product, which keeps 2^-11, and the room of fp32, and 16-bit tiles can be read in both directions (K-major and MN-major)
// from one copy in shared memory.  (Two bf16 numbers need no scale but keep 2^-17, three need six products.)  A kernel
// before splits every operand once, in tiles of 128 rows that lie in memory as they will in shared memory, so the kernels
// that multiply load them by bulk copies.  P and dS are split by the threads that compute them and go to tensor memory, from
// where they are the A operand of the next product: P is at most 2^14, dS is scaled by a bound of its own.  What a tile adds
// to y, dq, dk or dv is read from tensor memory and added in registers with the tile's scale.
//
// Scores are kept in units of log 2 (q is scaled by scale * log2(e) as it is loaded), so that an exponential is one ex2.
#include <cuda_runtime.h>
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "launch.cuh"
#include "scratch.h"
#include "smem_limit.h"
#include "tc_common.cuh"

namespace {

namespace cg = cooperative_groups;
using namespace tsb;
using tsb_launch::load;

constexpr float NEG_INF = -__builtin_huge_valf(), LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr unsigned ALL = 0xffffffffu;

// Tiles of pieces, [n][head][tile], and what a number of each tile stands for.
struct Pieces {
  const char* tiles;
  const float* units;
};

struct Problem {
  const float *q, *kv, *key, *dot;
  float *y, *lse, *dq, *dkv;
  Pieces qp, kp, vp, gp;
  int n, tq, tk, heads, shared, d;
  float scale;
  int qtiles, ktiles;
  bool vec;                                  // rows are whole 16-byte pieces on 16-byte boundaries
  int* status;
};

// ------------------------------------------------------------------------------------------------ pieces
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }      // -126 <= e <= 127
// e with |x| 2^e in [2^top, 2^(top+1)), kept where 2^e and 2^-e are normal numbers (0 and tiny x: the largest)
__device__ __forceinline__ int exponent_to(uint32_t bits_of_abs, int top) {
  return min(top + 127 - (int)(bits_of_abs >> 23), 126);
}
constexpr int TOP = 13;                      // of a tile's largest number
constexpr float LARGEST = 16384.f;           // and what that is below, 2^(TOP+1); P is scaled by it too

// A tile of ROWS x D numbers in shared memory: the plane of the hi pieces, then that of the lo pieces; a plane is D / 64
// chunks of [ROWS][64] halves whose rows of 128 bytes are swizzled (16-byte unit u of row r lies at u ^ (r & 7)).
template <int D, int ROWS> struct Tile {
  static constexpr int CHUNK = ROWS * 128, PLANE = ROWS * D * 2, BYTES = 2 * PLANE;
};

// One operand to split: rows of d numbers of [n][t][head].
struct Source {
  const float* x;
  const float* with;                         // an array like x: dots[n, head, t] = sum of x with over a row; or null
  const float* tokens;                       // [n][t], a row whose token is 0 counts as zeros and is not read; or null
  float* dots;
  char* tiles;
  float* units;
  long long batch, row, head;                // strides
  int rows, heads, count;                    // rows of a batch; tiles of a head
  float mult;
};
struct Sources {
  Source s[4];
  int first[5];                              // block where each begins
  int d;
  bool vec;
};

// A block splits a tile of 128 rows.
template <int D>
__global__ void __launch_bounds__(256) split_tiles(const Sources all) {
  tsb_launch::enter();
  using L = Tile<D, 128>;
  constexpr int UNITS = D / 8, TRIPS = 128 * UNITS / 256;
  __shared__ uint32_t largest[8];
  int which = 0;
  while ((int)blockIdx.x >= all.first[which + 1]) ++which;
  const Source& s = all.s[which];
  const int b = blockIdx.x - all.first[which], tile = b % s.count, h = b / s.count % s.heads, n = b / s.count / s.heads;
  const int rows = s.rows - tile * 128, d = all.d;
  const long long at = n * s.batch + (long long)tile * 128 * s.row + h * s.head;
  const float* tokens = s.tokens ? s.tokens + (long long)n * s.rows + tile * 128 : nullptr;
  float v[TRIPS][8];
  auto get = [&](const float* base, int row, int c, bool in, float (&to)[8]) {
    const float* src = base + at + row * s.row + c;
    if (all.vec) {
      float4 w = make_float4(0.f, 0.f, 0.f, 0.f), x = w;
      if (in && c < d) w = load(reinterpret_cast<const float4*>(src));
      if (in && c + 4 < d) x = load(reinterpret_cast<const float4*>(src + 4));
      to[0] = w.x; to[1] = w.y; to[2] = w.z; to[3] = w.w;
      to[4] = x.x; to[5] = x.y; to[6] = x.z; to[7] = x.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) to[k] = in && c + k < d ? load(src + k) : 0.f;
    }
  };
#pragma unroll
  for (int u = 0; u < TRIPS; ++u) {
    const int i = threadIdx.x + u * 256, row = i / UNITS;
    get(s.x, row, i % UNITS * 8, row < rows && (!tokens || load(tokens + row) != 0.f), v[u]);
  }
  if (s.with) {
#pragma unroll
    for (int u = 0; u < TRIPS; ++u) {
      const int i = threadIdx.x + u * 256, row = i / UNITS;
      float w[8], sum = 0.f;
      get(s.with, row, i % UNITS * 8, row < rows, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += v[u][k] * w[k];
#pragma unroll
      for (int o = UNITS / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(ALL, sum, o);
      if (row < rows && i % UNITS == 0) s.dots[((long long)n * s.heads + h) * s.rows + tile * 128 + row] = sum;
    }
  }
  uint32_t most = 0;
#pragma unroll
  for (int u = 0; u < TRIPS; ++u)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[u][k] *= s.mult;
      most = max(most, __float_as_uint(v[u][k]) & 0x7fffffffu);
    }
  most = __reduce_max_sync(ALL, most);
  if ((threadIdx.x & 31) == 0) largest[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) most = max(most, largest[w]);
  const int e = exponent_to(most, TOP);
  const float scale = power_of_two(e);
  if (threadIdx.x == 0) s.units[b] = power_of_two(-e);
  char* out = s.tiles + (size_t)b * L::BYTES;
#pragma unroll
  for (int u = 0; u < TRIPS; ++u) {
    const int i = threadIdx.x + u * 256, row = i / UNITS, c = i % UNITS;
    char* to = out + c / 8 * L::CHUNK + row * 128 + (((c & 7) ^ (row & 7)) << 4);
    uint4 hi, lo;
    split2(v[u][0] * scale, v[u][1] * scale, hi.x, lo.x);
    split2(v[u][2] * scale, v[u][3] * scale, hi.y, lo.y);
    split2(v[u][4] * scale, v[u][5] * scale, hi.z, lo.z);
    split2(v[u][6] * scale, v[u][7] * scale, hi.w, lo.w);
    *reinterpret_cast<uint4*>(to) = hi;
    *reinterpret_cast<uint4*>(to + L::PLANE) = lo;
  }
}

// Copies of tiles into shared memory by the copy engine; `full` gets their bytes.  Both sides are multiples of 16 bytes.
__device__ __forceinline__ void bulk_copy(char* to, const char* from, uint32_t bytes, uint64_t* full) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(to)), "l"(from),
               "r"(bytes), "r"(smem_u32(full))
               : "memory");
}
template <int D>
__device__ __forceinline__ void copy_tile(char* to, const Pieces& p, long long tile, uint64_t* full) {
  mbar_expect_tx(full, Tile<D, 128>::BYTES);
  bulk_copy(to, p.tiles + tile * Tile<D, 128>::BYTES, Tile<D, 128>::BYTES, full);
}
// The first or the last 64 rows of a tile, as a tile of 64 rows.
template <int D>
__device__ __forceinline__ void copy_half(char* to, const Pieces& p, long long tile, int half, uint64_t* full) {
  using L = Tile<D, 128>;
  using H = Tile<D, 64>;
  mbar_expect_tx(full, H::BYTES);
#pragma unroll
  for (int plane = 0; plane < 2; ++plane)
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      bulk_copy(to + plane * H::PLANE + c * H::CHUNK, p.tiles + tile * L::BYTES + plane * L::PLANE + c * L::CHUNK + half * H::CHUNK,
                H::CHUNK, full);
}

// ------------------------------------------------------------------------------------------------ products
__host__ __device__ constexpr uint32_t idesc_f16(int n, int b_mn_major) {      // M = 128, D fp32, A and B fp16, A K-major
  return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
constexpr uint32_t DESC_HI = smem_desc_hi(1024);       // 128-byte swizzle, groups of eight rows 1024 bytes apart

// D [128 x ROWS_B] = A B^T over the D columns of both tiles.
template <int D, int ROWS_A, int ROWS_B>
__device__ __forceinline__ void product_of_rows(uint32_t to, uint32_t a, uint32_t b) {
  using LA = Tile<D, ROWS_A>;
  using LB = Tile<D, ROWS_B>;
  const uint32_t al = smem_desc_lo(a, 16), bl = smem_desc_lo(b, 16);
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
    const uint32_t ao = (k / 4 * LA::CHUNK + k % 4 * 32) >> 4, bo = (k / 4 * LB::CHUNK + k % 4 * 32) >> 4;
    const uint64_t ah = smem_desc_join(DESC_HI, al + ao), bh = smem_desc_join(DESC_HI, bl + bo);
    const uint64_t a2 = smem_desc_join(DESC_HI, al + ao + (LA::PLANE >> 4)), b2 = smem_desc_join(DESC_HI, bl + bo + (LB::PLANE >> 4));
    mma_smem(to, ah, bh, idesc_f16(ROWS_B, 0), k > 0);
    mma_smem(to, ah, b2, idesc_f16(ROWS_B, 0), 1);
    mma_smem(to, a2, bh, idesc_f16(ROWS_B, 0), 1);
  }
}
// D [128 x D] = A B, A [128 x ROWS] in tensor memory: 16 columns for every 16 of its, hi pieces in the first eight.
template <int D, int ROWS>
__device__ __forceinline__ void product_with_columns(uint32_t to, uint32_t a, uint32_t b) {
  using L = Tile<D, ROWS>;
  const uint32_t bl = smem_desc_lo(b, L::CHUNK);
#pragma unroll
  for (int k = 0; k < ROWS / 16; ++k) {
    const uint64_t bh = smem_desc_join(DESC_HI, bl + (k * 2048 >> 4)), b2 = smem_desc_join(DESC_HI, bl + ((k * 2048 + L::PLANE) >> 4));
    mma_tmem(to, a + 16 * k, bh, idesc_f16(D, 1), k > 0);
    mma_tmem(to, a + 16 * k, b2, idesc_f16(D, 1), 1);
    mma_tmem(to, a + 16 * k + 8, bh, idesc_f16(D, 1), 1);
  }
}

__device__ __forceinline__ void tmem_ld16(uint32_t addr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
// 16 numbers of a row as hi pieces in eight columns and lo pieces in the next eight
__device__ __forceinline__ void tmem_st_pieces(uint32_t addr, const float (&v)[16]) {
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) split2(v[2 * i], v[2 * i + 1], r[i], r[8 + i]);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Keys up to the last one that is in, rounded up to what the block looks at in one go.  All threads call it.
__device__ __forceinline__ int keys_in(const float* tokens, int tk) {
  if (!tokens) return tk;
  int end = tk;
  while (end > 0) {
    const int i = end - 1 - (int)threadIdx.x;
    if (__syncthreads_or(i >= 0 && load(tokens + i) != 0.f)) break;
    end -= (int)blockDim.x;
  }
  return end < 0 ? 0 : end;
}
// Bit i: whether key `first + i` is in.
__device__ __forceinline__ unsigned keys_mask(const float* tokens, int first, int tk) {
  const int k = first + (int)(threadIdx.x & 31);
  return __ballot_sync(ALL, k < tk && (!tokens || load(tokens + k) != 0.f));
}

constexpr int TMEM_COLUMNS = 512;

// After a wait that ran out: the products that were issued still use shared and tensor memory.
__device__ __forceinline__ void drain(uint64_t* bar) {
  umma_commit(bar);
  const long long begin = clock64();
  while (!mbar_try_wait(bar, 0) && clock64() - begin < WAIT_LIMIT_CYCLES) {
  }
}

// The tiles begin at a multiple of 1024 bytes, behind the barriers.
template <class Barriers>
__device__ __forceinline__ char* dynamic_tiles(Barriers*& bars) {
  extern __shared__ char raw[];
  static_assert(sizeof(Barriers) <= 1024, "one kilobyte is kept for them");
  char* at = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) / 1024 * 1024);
  bars = reinterpret_cast<Barriers*>(at);
  return at + 1024;
}

// Writes the d first numbers of a row.
template <int COUNT>
__device__ __forceinline__ void store_row(float* to, const float (&v)[COUNT], float mult, int d, bool vec) {
  if (vec) {
#pragma unroll
    for (int c = 0; c < COUNT; c += 4)
      if (c < d) *reinterpret_cast<float4*>(to + c) = make_float4(v[c] * mult, v[c + 1] * mult, v[c + 2] * mult, v[c + 3] * mult);
  } else {
#pragma unroll
    for (int c = 0; c < COUNT; ++c)
      if (c < d) to[c] = v[c] * mult;
  }
}

// ------------------------------------------------------------------------------------------------ forward
// A block takes 128 queries of a head and tiles of 128 keys.  Warps 0 to 3: soft-max, a row per thread; 4: copies; 5 issues
// the products.  Two tiles of scores are in tensor memory, so S of the next tile runs while a thread works on this
// one; P takes the place of its S.  y of a tile is added to the registers (rescaled to the new maximum there) while the next
// tile's P is computed.
template <int D> struct ForwardShape {
  static constexpr int STAGES = D == 64 ? 2 : 1;
  using L = Tile<D, 128>;
  static constexpr int SMEM = 2048 + L::BYTES * (1 + 2 * STAGES);
};
struct ForwardShared {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], drained;
  uint32_t tmem;
};

template <int D>
__global__ void __launch_bounds__(192, 1) attend(const Problem p) {
  using Shape = ForwardShape<D>;
  using L = typename Shape::L;
  constexpr int STAGES = Shape::STAGES;
  ForwardShared* bar;
  char* q_tile = dynamic_tiles(bar);
  char* k_tile = q_tile + L::BYTES;
  char* v_tile = k_tile + STAGES * L::BYTES;
  const int warp = __shfl_sync(ALL, threadIdx.x >> 5, 0);
  if (threadIdx.x == 0) {
    mbar_init(&bar->q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->k_full[i], 1);
      mbar_init(&bar->k_empty[i], 1);
      mbar_init(&bar->v_full[i], 1);
      mbar_init(&bar->v_empty[i], 1);
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->p_full[i], 128);
      mbar_init(&bar->o_full[i], 1);
    }
    mbar_init(&bar->drained, 1);
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(&bar->tmem, TMEM_COLUMNS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem;             // S 0 and 128, y 256 and 384
  tsb_launch::enter();

  const int qt = blockIdx.x % p.qtiles, h = blockIdx.x / p.qtiles % p.heads, n = blockIdx.x / p.qtiles / p.heads;
  const int shared = h / (p.heads / p.shared), q0 = qt * 128;
  const float* tokens = p.key ? p.key + (long long)n * p.tk : nullptr;
  const int tiles = (keys_in(tokens, p.tk) + 127) / 128;
  const long long q_row = (long long)p.heads * p.d;
  const long long q_at = ((long long)n * p.heads + h) * p.qtiles + qt, k_at = ((long long)n * p.shared + shared) * p.ktiles;

  if (warp < 4) {
    float acc[D], m = NEG_INF, l = 0.f, before = 1.f, v_unit = 0.f;
    const float q_unit = load(p.qp.units + q_at);
#pragma unroll
    for (int c = 0; c < D; ++c) acc[c] = 0.f;
    const uint32_t mine = tmem + ((uint32_t)warp << 21);         // this warp's 32 lanes
    bool ok = true;
    auto add_tile = [&](int j, float factor, float unit) {
      if (!mbar_wait(&bar->o_full[j & 1], (j >> 1) & 1, p.status, 0x301)) return false;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < D; c += 16) {
        float o[16];
        tmem_ld16(mine + 256 + (j & 1) * 128 + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c + i] = acc[c + i] * factor + o[i] * unit;
      }
      return true;
    };
    for (int j = 0; j < tiles; ++j) {
      unsigned in[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) in[w] = keys_mask(tokens, j * 128 + w * 32, p.tk);
      const float unit = q_unit * load(p.kp.units + k_at + j), next_unit = load(p.vp.units + k_at + j);
      if (!mbar_wait(&bar->s_full[j & 1], (j >> 1) & 1, p.status, 0x302)) { ok = false; break; }
      tc_fence_after();
      const uint32_t at = mine + (j & 1) * 128;
      float most = NEG_INF;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float s[32];
        tmem_ld_32x32(at + 32 * w, s);
        tmem_ld_wait();
        if (in[w] == ALL) {
#pragma unroll
          for (int i = 0; i < 32; ++i) most = fmaxf(most, s[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) most = fmaxf(most, (in[w] >> i) & 1 ? s[i] : NEG_INF);
        }
      }
      const float top = fmaxf(m, most == NEG_INF ? NEG_INF : most * unit), ref = top == NEG_INF ? 0.f : top;
      const float factor = exp2_fast(m - ref), shift = TOP + 1 - ref;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        float s[16];
        tmem_ld16(at + 16 * w, s);
        tmem_ld_wait();
        const unsigned mask = in[w / 2] >> (w % 2 * 16);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = exp2_fast(s[i] * unit + shift);
          if (in[w / 2] != ALL) s[i] = (mask >> i) & 1 ? s[i] : 0.f;
          sum += s[i];
        }
        tmem_st_pieces(at + 16 * w, s);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bar->p_full[j & 1]);
      l = l * factor + sum;
      m = top;
      if (j > 0 && !(ok = add_tile(j - 1, before, v_unit))) break;
      before = factor;
      v_unit = next_unit;
    }
    if (ok && tiles > 0) ok = add_tile(tiles - 1, before, v_unit);
    const int t = q0 + threadIdx.x;
    if (ok && t < p.tq) {
      store_row(p.y + ((long long)n * p.tq + t) * q_row + (long long)h * p.d, acc, l > 0.f ? 1.f / l : 0.f, p.d, p.vec);
      // (a row without keys: exp2(S - inf) = 0 in the backward pass)
      p.lse[((long long)n * p.heads + h) * p.tq + t] = l > 0.f ? m - (TOP + 1) + log2f(l) : -NEG_INF;
    }
  } else if (warp == 4) {
    if (elect_one() && tiles > 0) {
      copy_tile<D>(q_tile, p.qp, q_at, &bar->q_full);
      for (int j = 0; j < tiles; ++j) {
        const int s = j % STAGES, ph = j / STAGES & 1;
        if (!mbar_wait(&bar->k_empty[s], ph ^ 1, p.status, 0x303)) break;
        copy_tile<D>(k_tile + s * L::BYTES, p.kp, k_at + j, &bar->k_full[s]);
        if (!mbar_wait(&bar->v_empty[s], ph ^ 1, p.status, 0x304)) break;
        copy_tile<D>(v_tile + s * L::BYTES, p.vp, k_at + j, &bar->v_full[s]);
      }
    }
  } else {
    if (elect_one()) {
      const uint32_t qa = smem_u32(q_tile), ka = smem_u32(k_tile), va = smem_u32(v_tile);
      bool ok = tiles == 0 || mbar_wait(&bar->q_full, 0, p.status, 0x305);
      auto scores = [&](int j) {
        const int s = j % STAGES;
        if (!mbar_wait(&bar->k_full[s], j / STAGES & 1, p.status, 0x306)) return false;
        tc_fence_after();
        product_of_rows<D, 128, 128>(tmem + (j & 1) * 128, qa, ka + s * L::BYTES);
        umma_commit(&bar->s_full[j & 1]);
        umma_commit(&bar->k_empty[s]);
        return true;
      };
      for (int j = 0; j < 2 && j < tiles && ok; ++j) ok = scores(j);
      for (int j = 0; j < tiles && ok; ++j) {
        const int s = j % STAGES;
        if (!(ok = mbar_wait(&bar->v_full[s], j / STAGES & 1, p.status, 0x307))) break;
        if (!(ok = mbar_wait(&bar->p_full[j & 1], (j >> 1) & 1, p.status, 0x308))) break;
        tc_fence_after();
        product_with_columns<D, 128>(tmem + 256 + (j & 1) * 128, tmem + (j & 1) * 128, va + s * L::BYTES);
        umma_commit(&bar->o_full[j & 1]);
        umma_commit(&bar->v_empty[s]);
        if (j + 2 < tiles) ok = scores(j + 2);
      }
      if (!ok) drain(&bar->drained);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, TMEM_COLUMNS);
}

// ------------------------------------------------------------------------------------------------ gradients
// A bound of |dP - dot| over a tile: e with (d |g| |v| + |dot|) 2^e below 2^15 (units: what 2^14 of a tile stands for).
__device__ __forceinline__ int exponent_of_ds(int d, float g_unit, float v_unit, float dot) {
  const float most = (float)d * (LARGEST * g_unit) * (LARGEST * v_unit) + fabsf(dot);
  return exponent_to(__float_as_uint(most), TOP + 1);
}

// dq: a block takes 128 queries of a head and tiles of 64 keys; the same roles.  dS takes the place of its S.
template <int D> struct QueryShape {
  static constexpr int K_STAGES = D == 64 ? 3 : 2, V_STAGES = D == 64 ? 3 : 1;
  using LQ = Tile<D, 128>;
  using LK = Tile<D, 64>;
  static constexpr int SMEM = 2048 + 2 * LQ::BYTES + (K_STAGES + V_STAGES) * LK::BYTES;
};
struct QueryShared {
  uint64_t q_full, g_full, k_full[3], k_empty[3], v_full[3], v_empty[3], s_full[2], ds_full[2], dq_full[2], drained;
  uint32_t tmem;
};

template <int D>
__global__ void __launch_bounds__(192, 1) grad_of_queries(const Problem p) {
  using Shape = QueryShape<D>;
  using LQ = typename Shape::LQ;
  using LK = typename Shape::LK;
  constexpr int KS = Shape::K_STAGES, VS = Shape::V_STAGES;
  QueryShared* bar;
  char* q_tile = dynamic_tiles(bar);
  char* g_tile = q_tile + LQ::BYTES;
  char* k_tile = g_tile + LQ::BYTES;
  char* v_tile = k_tile + KS * LK::BYTES;
  const int warp = __shfl_sync(ALL, threadIdx.x >> 5, 0);
  if (threadIdx.x == 0) {
    mbar_init(&bar->q_full, 1);
    mbar_init(&bar->g_full, 1);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&bar->k_full[i], 1);
      mbar_init(&bar->k_empty[i], 1);
      mbar_init(&bar->v_full[i], 1);
      mbar_init(&bar->v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->ds_full[i], 128);
      mbar_init(&bar->dq_full[i], 1);
    }
    mbar_init(&bar->drained, 1);
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(&bar->tmem, TMEM_COLUMNS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem;             // S 0 and 64, dP 128 and 192, dq 256 and 384
  tsb_launch::enter();

  const int qt = blockIdx.x % p.qtiles, h = blockIdx.x / p.qtiles % p.heads, n = blockIdx.x / p.qtiles / p.heads;
  const int shared = h / (p.heads / p.shared), q0 = qt * 128;
  const float* tokens = p.key ? p.key + (long long)n * p.tk : nullptr;
  const int tiles = (keys_in(tokens, p.tk) + 63) / 64;
  const long long q_row = (long long)p.heads * p.d;
  const long long q_at = ((long long)n * p.heads + h) * p.qtiles + qt, k_at = ((long long)n * p.shared + shared) * p.ktiles;

  if (warp < 4) {
    float acc[D], before = 0.f;
#pragma unroll
    for (int c = 0; c < D; ++c) acc[c] = 0.f;
    const uint32_t mine = tmem + ((uint32_t)warp << 21);
    const int t = q0 + threadIdx.x;
    const long long at_row = ((long long)n * p.heads + h) * p.tq + t;
    const float lse = t < p.tq ? load(p.lse + at_row) : -NEG_INF, dot = t < p.tq ? load(p.dot + at_row) : 0.f;
    const float q_unit = load(p.qp.units + q_at), g_unit = load(p.gp.units + q_at);
    bool ok = true;
    auto add_tile = [&](int j, float unit) {
      if (!mbar_wait(&bar->dq_full[j & 1], (j >> 1) & 1, p.status, 0x311)) return false;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < D; c += 16) {
        float o[16];
        tmem_ld16(mine + 256 + (j & 1) * 128 + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c + i] += o[i] * unit;
      }
      return true;
    };
    for (int j = 0; j < tiles; ++j) {
      const unsigned in[2] = {keys_mask(tokens, j * 64, p.tk), keys_mask(tokens, j * 64 + 32, p.tk)};
      const float k_unit = load(p.kp.units + k_at + j / 2), v_unit = load(p.vp.units + k_at + j / 2);
      const int e = exponent_of_ds(p.d, g_unit, v_unit, dot);
      const float s_unit = q_unit * k_unit, dp_unit = g_unit * v_unit, shift = (float)e - lse;
      if (!mbar_wait(&bar->s_full[j & 1], (j >> 1) & 1, p.status, 0x312)) { ok = false; break; }
      tc_fence_after();
      const uint32_t at = mine + (j & 1) * 64;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float s[16], dp[16];
        tmem_ld16(at + 16 * w, s);
        tmem_ld16(at + 128 + 16 * w, dp);
        tmem_ld_wait();
        const unsigned mask = in[w / 2] >> (w % 2 * 16);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = exp2_fast(s[i] * s_unit + shift) * (dp[i] * dp_unit - dot);
          if (in[w / 2] != ALL) s[i] = (mask >> i) & 1 ? s[i] : 0.f;
        }
        tmem_st_pieces(at + 16 * w, s);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bar->ds_full[j & 1]);
      if (j > 0 && !(ok = add_tile(j - 1, before))) break;
      before = k_unit * power_of_two(-e);
    }
    if (ok && tiles > 0) ok = add_tile(tiles - 1, before);
    if (ok && t < p.tq) store_row(p.dq + ((long long)n * p.tq + t) * q_row + (long long)h * p.d, acc, p.scale, p.d, p.vec);
  } else if (warp == 4) {
    if (elect_one() && tiles > 0) {
      copy_tile<D>(q_tile, p.qp, q_at, &bar->q_full);
      copy_tile<D>(g_tile, p.gp, q_at, &bar->g_full);
      for (int j = 0; j < tiles; ++j) {
        const int ks = j % KS, vs = j % VS;
        if (!mbar_wait(&bar->k_empty[ks], (j / KS & 1) ^ 1, p.status, 0x313)) break;
        copy_half<D>(k_tile + ks * LK::BYTES, p.kp, k_at + j / 2, j & 1, &bar->k_full[ks]);
        if (!mbar_wait(&bar->v_empty[vs], (j / VS & 1) ^ 1, p.status, 0x314)) break;
        copy_half<D>(v_tile + vs * LK::BYTES, p.vp, k_at + j / 2, j & 1, &bar->v_full[vs]);
      }
    }
  } else {
    if (elect_one()) {
      const uint32_t qa = smem_u32(q_tile), ga = smem_u32(g_tile), ka = smem_u32(k_tile), va = smem_u32(v_tile);
      bool ok = tiles == 0 || (mbar_wait(&bar->q_full, 0, p.status, 0x315) && mbar_wait(&bar->g_full, 0, p.status, 0x315));
      auto scores = [&](int j) {
        const int ks = j % KS, vs = j % VS;
        if (!mbar_wait(&bar->k_full[ks], j / KS & 1, p.status, 0x316)) return false;
        tc_fence_after();
        product_of_rows<D, 128, 64>(tmem + (j & 1) * 64, qa, ka + ks * LK::BYTES);
        if (!mbar_wait(&bar->v_full[vs], j / VS & 1, p.status, 0x317)) return false;
        tc_fence_after();
        product_of_rows<D, 128, 64>(tmem + 128 + (j & 1) * 64, ga, va + vs * LK::BYTES);
        umma_commit(&bar->s_full[j & 1]);
        umma_commit(&bar->v_empty[vs]);
        return true;
      };
      for (int j = 0; j < 2 && j < tiles && ok; ++j) ok = scores(j);
      for (int j = 0; j < tiles && ok; ++j) {
        if (!(ok = mbar_wait(&bar->ds_full[j & 1], (j >> 1) & 1, p.status, 0x318))) break;
        tc_fence_after();
        product_with_columns<D, 64>(tmem + 256 + (j & 1) * 128, tmem + (j & 1) * 64, ka + j % KS * LK::BYTES);
        umma_commit(&bar->k_empty[j % KS]);
        umma_commit(&bar->dq_full[j & 1]);
        if (j + 2 < tiles) ok = scores(j + 2);
      }
      if (!ok) drain(&bar->drained);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, TMEM_COLUMNS);
}

// dk and dv: a block takes 128 keys of a shared head and tiles of 64 queries of every head that reads it.  S^T and dP^T have
// the keys as rows, so P^T and dS^T are A operands as they lie.  Warps 0 to 3 take the first 32 queries of a tile and add up
// dv, 4 to 7 the others and dk; 8 copies; 9 issues.  Tiles of queries and of gradients share a ring of slots: q, g, q, g.
template <int D> struct StateShape {
  static constexpr int SLOTS = D == 64 ? 6 : 3;
  using LK = Tile<D, 128>;
  using LQ = Tile<D, 64>;
  static constexpr int SMEM = 2048 + 2 * LK::BYTES + SLOTS * LQ::BYTES;
};
struct StateShared {
  uint64_t k_full, v_full, full[6], empty[6], s_full[2], ds_full[2], sum_full, sum_empty, drained;
  uint32_t tmem;
};

template <int D>
__global__ void __launch_bounds__(320, 1) grad_of_states(const Problem p) {
  using Shape = StateShape<D>;
  using LQ = typename Shape::LQ;
  using LK = typename Shape::LK;
  constexpr int SLOTS = Shape::SLOTS;
  StateShared* bar;
  char* k_tile = dynamic_tiles(bar);
  char* v_tile = k_tile + LK::BYTES;
  char* ring = v_tile + LK::BYTES;
  const int warp = __shfl_sync(ALL, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bar->k_full, 1);
    mbar_init(&bar->v_full, 1);
    for (int i = 0; i < 6; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->ds_full[i], 256);
    }
    mbar_init(&bar->sum_full, 1);
    mbar_init(&bar->sum_empty, 256);
    mbar_init(&bar->drained, 1);
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(&bar->tmem, TMEM_COLUMNS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem;             // S^T 0 and 64, dP^T 128 and 192, dv 256, dk 384
  tsb_launch::enter();

  const int kt = blockIdx.x % p.ktiles, shared = blockIdx.x / p.ktiles % p.shared, n = blockIdx.x / p.ktiles / p.shared;
  const int k0 = kt * 128, per = p.heads / p.shared;
  const float* tokens = p.key ? p.key + (long long)n * p.tk : nullptr;
  const long long kv_row = 2ll * p.shared * p.d, k_at = ((long long)n * p.shared + shared) * p.ktiles + kt;
  const bool mine_in = threadIdx.x < 128 && k0 + (int)threadIdx.x < p.tk && (!tokens || load(tokens + k0 + threadIdx.x) != 0.f);
  const int halves = (p.tq + 63) / 64, tiles = __syncthreads_or(mine_in) ? halves * per : 0;

  if (warp < 8) {
    float acc[D];
#pragma unroll
    for (int c = 0; c < D; ++c) acc[c] = 0.f;
    const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21);
    const int half = warp >> 2, row = threadIdx.x & 127;
    const float k_unit = load(p.kp.units + k_at), v_unit = load(p.vp.units + k_at);
    float before = 0.f;
    bool ok = true;
    auto add_tile = [&](int j, float unit) {
      if (!mbar_wait(&bar->sum_full, j & 1, p.status, 0x322)) return false;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < D; c += 16) {
        float o[16];
        tmem_ld16(mine + 256 + half * 128 + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c + i] += o[i] * unit;
      }
      tc_fence_before();
      mbar_arrive(&bar->sum_empty);
      return true;
    };
    for (int j = 0; j < tiles; ++j) {
      // a lane has the log-sum-exp and the dot of one of this half's queries, and the other half's dot for the bound
      const int h = shared * per + j / halves, t0 = j % halves * 64, t = t0 + half * 32 + lane, other = t0 + (half ^ 1) * 32 + lane;
      const long long at_head = ((long long)n * p.heads + h) * p.tq;
      const float lse = t < p.tq ? load(p.lse + at_head + t) : -NEG_INF, dot = t < p.tq ? load(p.dot + at_head + t) : 0.f;
      const float dot2 = other < p.tq ? load(p.dot + at_head + other) : 0.f;
      const float most = __uint_as_float(__reduce_max_sync(ALL, max(__float_as_uint(fabsf(dot)), __float_as_uint(fabsf(dot2)))));
      const long long q_at = ((long long)n * p.heads + h) * p.qtiles + t0 / 128;
      const float q_unit = load(p.qp.units + q_at), g_unit = load(p.gp.units + q_at);
      if (!mbar_wait(&bar->s_full[j & 1], (j >> 1) & 1, p.status, 0x321)) { ok = false; break; }
      tc_fence_after();
      const uint32_t at = mine + (j & 1) * 64 + half * 32;
      const int e = exponent_of_ds(p.d, g_unit, v_unit, most);
      // p = 2^14 P, then dS = p (dP - dot) 2^(e - 14)
      const float s_unit = q_unit * k_unit, f = power_of_two(max(e - TOP - 1, -126)), dp_unit = g_unit * v_unit * f;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        float s[16], dp[16];
        tmem_ld16(at + 16 * w, s);
        tmem_ld16(at + 128 + 16 * w, dp);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = exp2_fast(s[i] * s_unit + (TOP + 1 - __shfl_sync(ALL, lse, 16 * w + i)));
          dp[i] = s[i] * (dp[i] * dp_unit - __shfl_sync(ALL, dot, 16 * w + i) * f);
        }
        tmem_st_pieces(at + 16 * w, s);
        tmem_st_pieces(at + 128 + 16 * w, dp);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bar->ds_full[j & 1]);
      if (j > 0 && !(ok = add_tile(j - 1, before))) break;
      before = half ? q_unit * power_of_two(-e) : g_unit * (1.f / LARGEST);
    }
    if (ok && tiles > 0) ok = add_tile(tiles - 1, before);
    if (ok && k0 + row < p.tk) {
      const bool in = !tokens || load(tokens + k0 + row) != 0.f;
      float* to = p.dkv + ((long long)n * p.tk + k0 + row) * kv_row + (long long)shared * p.d + (half ? 0 : (long long)p.shared * p.d);
      if (!in)
#pragma unroll
        for (int c = 0; c < D; ++c) acc[c] = 0.f;
      store_row(to, acc, half ? LN2 : 1.f, p.d, p.vec);          // (q was loaded times scale * log2(e))
    }
  } else if (warp == 8) {
    if (elect_one() && tiles > 0) {
      copy_tile<D>(k_tile, p.kp, k_at, &bar->k_full);
      copy_tile<D>(v_tile, p.vp, k_at, &bar->v_full);
      for (int i = 0; i < 2 * tiles; ++i) {
        const int s = i % SLOTS, j = i / 2, h = shared * per + j / halves, t0 = j % halves * 64;
        if (!mbar_wait(&bar->empty[s], (i / SLOTS & 1) ^ 1, p.status, 0x323)) break;
        copy_half<D>(ring + s * LQ::BYTES, i & 1 ? p.gp : p.qp, ((long long)n * p.heads + h) * p.qtiles + t0 / 128, t0 / 64 & 1,
                     &bar->full[s]);
      }
    }
  } else {
    if (elect_one()) {
      const uint32_t ra = smem_u32(ring), ka = smem_u32(k_tile), va = smem_u32(v_tile);
      bool ok = tiles == 0 || (mbar_wait(&bar->k_full, 0, p.status, 0x324) && mbar_wait(&bar->v_full, 0, p.status, 0x324));
      // S^T and dP^T of tile j: the second half of it commits
      auto half_of_scores = [&](int j, int half) {
        const int i = 2 * j + half, s = i % SLOTS;
        if (!mbar_wait(&bar->full[s], i / SLOTS & 1, p.status, 0x325)) return false;
        tc_fence_after();
        product_of_rows<D, 128, 64>(tmem + half * 128 + (j & 1) * 64, half ? va : ka, ra + s * LQ::BYTES);
        if (half) {
          umma_commit(&bar->s_full[j & 1]);
        }
        return true;
      };
      // With six slots the scores of two tiles are under way; with three there is room for the next tile's queries only
      constexpr bool WIDE = SLOTS == 6;
      for (int i = 0; i < (WIDE ? 4 : 2) && i < 2 * tiles && ok; ++i) ok = half_of_scores(i / 2, i & 1);
      for (int j = 0; j < tiles && ok; ++j) {
        if (!WIDE && j + 1 < tiles && !(ok = half_of_scores(j + 1, 0))) break;
        if (!(ok = mbar_wait(&bar->ds_full[j & 1], (j >> 1) & 1, p.status, 0x326))) break;
        if (j > 0 && !(ok = mbar_wait(&bar->sum_empty, (j - 1) & 1, p.status, 0x327))) break;
        tc_fence_after();
        const int qs = 2 * j % SLOTS, gs = (2 * j + 1) % SLOTS;
        product_with_columns<D, 64>(tmem + 384, tmem + 128 + (j & 1) * 64, ra + qs * LQ::BYTES);
        umma_commit(&bar->empty[qs]);
        product_with_columns<D, 64>(tmem + 256, tmem + (j & 1) * 64, ra + gs * LQ::BYTES);
        umma_commit(&bar->empty[gs]);
        umma_commit(&bar->sum_full);
        if (WIDE) {
          if (j + 2 < tiles) ok = half_of_scores(j + 2, 0) && half_of_scores(j + 2, 1);
        } else if (j + 1 < tiles) {
          ok = half_of_scores(j + 1, 1);
        }
      }
      if (!ok) drain(&bar->drained);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, TMEM_COLUMNS);
}

// ------------------------------------------------------------------------------------------------ single tokens
// Up to ROWS queries that read one shared head (H / G heads x Tq tokens): bound by reading keys and values once, so plain
// fp32.  LANES threads take a key (four numbers each), so a warp takes 32 / LANES keys at a time and BATCH times that are in
// flight; each such group keeps a soft-max of its own for every row, joined at the end: in the warp by shuffles, in the
// block through shared memory, and over the blocks of a cluster that share a long sentence through distributed shared memory.
constexpr int FEW_WARPS = 8;
template <int LANES, int ROWS> struct FewShared {
  float m[FEW_WARPS][ROWS], l[FEW_WARPS][ROWS];
  float o[FEW_WARPS][ROWS][LANES * 4];
};

template <int LANES, int ROWS, int BATCH>
__global__ void __launch_bounds__(FEW_WARPS * 32) attend_few(const Problem p, int split) {
  tsb_launch::enter();
  __shared__ FewShared<LANES, ROWS> s;
  constexpr int GROUPS = 32 / LANES;
  const int part = blockIdx.x % split, shared = blockIdx.x / split % p.shared, n = blockIdx.x / split / p.shared;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / LANES, c = lane % LANES * 4;
  const int per = p.heads / p.shared, rows = per * p.tq;
  const float* tokens = p.key ? p.key + (long long)n * p.tk : nullptr;
  const long long kv_row = 2ll * p.shared * p.d, q_row = (long long)p.heads * p.d;
  const float* k_base = p.kv + (long long)n * p.tk * kv_row + (long long)shared * p.d + c;
  auto four = [&](const float* at, bool in) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!in || c >= p.d) return v;
    if (p.vec) return load(reinterpret_cast<const float4*>(at));
    v.x = load(at);
    if (c + 1 < p.d) v.y = load(at + 1);
    if (c + 2 < p.d) v.z = load(at + 2);
    if (c + 3 < p.d) v.w = load(at + 3);
    return v;
  };
  float4 q[ROWS], o[ROWS];
  float m[ROWS], l[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {           // row r: query r / per of head r % per
    q[r] = four(p.q + ((long long)n * p.tq + r / per) * q_row + (long long)(shared * per + r % per) * p.d + c, r < rows);
    const float f = p.scale * LOG2E;
    q[r] = make_float4(q[r].x * f, q[r].y * f, q[r].z * f, q[r].w * f);
    o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    m[r] = NEG_INF;
    l[r] = 0.f;
  }
  const int share = (p.tk + split - 1) / split, begin = part * share, end = min(begin + share, p.tk);
  constexpr int STEP = FEW_WARPS * GROUPS;
  for (int first = begin; first < end; first += STEP * BATCH) {
    float4 k[BATCH], v[BATCH];
    bool in[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int t = first + u * STEP + warp * GROUPS + group;
      in[u] = t < end && (!tokens || load(tokens + t) != 0.f);
      k[u] = four(k_base + t * kv_row, in[u]);
      v[u] = four(k_base + t * kv_row + (long long)p.shared * p.d, in[u]);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float x[BATCH], top = m[r];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        float d = q[r].x * k[u].x + q[r].y * k[u].y + q[r].z * k[u].z + q[r].w * k[u].w;
#pragma unroll
        for (int off = LANES / 2; off > 0; off >>= 1) d += __shfl_xor_sync(ALL, d, off);
        x[u] = in[u] ? d : NEG_INF;
        top = fmaxf(top, x[u]);
      }
      const float ref = top == NEG_INF ? 0.f : top, factor = exp2_fast(m[r] - ref);
      m[r] = top;
      l[r] *= factor;
      o[r] = make_float4(o[r].x * factor, o[r].y * factor, o[r].z * factor, o[r].w * factor);
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const float e = in[u] ? exp2_fast(x[u] - ref) : 0.f;
        l[r] += e;
        o[r].x += e * v[u].x; o[r].y += e * v[u].y; o[r].z += e * v[u].z; o[r].w += e * v[u].w;
      }
    }
  }
  // the groups of a warp, then the warps
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
#pragma unroll
    for (int off = LANES; off < 32; off <<= 1) {
      const float m2 = __shfl_xor_sync(ALL, m[r], off), l2 = __shfl_xor_sync(ALL, l[r], off);
      const float4 o2 = make_float4(__shfl_xor_sync(ALL, o[r].x, off), __shfl_xor_sync(ALL, o[r].y, off),
                                    __shfl_xor_sync(ALL, o[r].z, off), __shfl_xor_sync(ALL, o[r].w, off));
      const float top = fmaxf(m[r], m2), ref = top == NEG_INF ? 0.f : top;
      const float a = exp2_fast(m[r] - ref), b = exp2_fast(m2 - ref);
      m[r] = top;
      l[r] = l[r] * a + l2 * b;
      o[r] = make_float4(o[r].x * a + o2.x * b, o[r].y * a + o2.y * b, o[r].z * a + o2.z * b, o[r].w * a + o2.w * b);
    }
    if (group == 0) {
      *reinterpret_cast<float4*>(&s.o[warp][r][c]) = o[r];
      if (lane == 0) s.m[warp][r] = m[r], s.l[warp][r] = l[r];
    }
  }
  __syncthreads();
  constexpr int CELLS = ROWS * LANES * 4;
  for (int i = threadIdx.x; i < CELLS; i += FEW_WARPS * 32) {        // (a thread reads and writes its own cells of o)
    const int r = i / (LANES * 4), col = i % (LANES * 4);
    float top = NEG_INF, lsum = 0.f, sum = 0.f;
    for (int w = 0; w < FEW_WARPS; ++w) top = fmaxf(top, s.m[w][r]);
    const float ref = top == NEG_INF ? 0.f : top;
    for (int w = 0; w < FEW_WARPS; ++w) {
      const float f = exp2_fast(s.m[w][r] - ref);
      lsum += s.l[w][r] * f;
      sum += s.o[w][r][col] * f;
    }
    s.o[0][r][col] = sum;
    if (split == 1) {
      if (r < rows && col < p.d)
        p.y[((long long)n * p.tq + r / per) * q_row + (long long)(shared * per + r % per) * p.d + col] = lsum > 0.f ? sum / lsum : 0.f;
      if (r < rows && col == 0)
        p.lse[((long long)n * p.heads + shared * per + r % per) * p.tq + r / per] = lsum > 0.f ? top + log2f(lsum) : -NEG_INF;
    }
  }
  if (split == 1) return;
  __syncthreads();                                                   // all have read the warps' m and l
  if (threadIdx.x < ROWS) {
    float top = NEG_INF, lsum = 0.f;
    for (int w = 0; w < FEW_WARPS; ++w) top = fmaxf(top, s.m[w][threadIdx.x]);
    const float ref = top == NEG_INF ? 0.f : top;
    for (int w = 0; w < FEW_WARPS; ++w) lsum += s.l[w][threadIdx.x] * exp2_fast(s.m[w][threadIdx.x] - ref);
    s.m[0][threadIdx.x] = top;
    s.l[0][threadIdx.x] = lsum;
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  // every block joins a share of the cells
  for (int i = part * FEW_WARPS * 32 + threadIdx.x; i < CELLS; i += split * FEW_WARPS * 32) {
    const int r = i / (LANES * 4), col = i % (LANES * 4);
    float top = NEG_INF, lsum = 0.f, sum = 0.f;
    for (int b = 0; b < split; ++b) top = fmaxf(top, *cluster.map_shared_rank(&s.m[0][r], b));
    const float ref = top == NEG_INF ? 0.f : top;
    for (int b = 0; b < split; ++b) {
      const float f = exp2_fast(*cluster.map_shared_rank(&s.m[0][r], b) - ref);
      lsum += *cluster.map_shared_rank(&s.l[0][r], b) * f;
      sum += *cluster.map_shared_rank(&s.o[0][r][col], b) * f;
    }
    if (r < rows && col < p.d)
      p.y[((long long)n * p.tq + r / per) * q_row + (long long)(shared * per + r % per) * p.d + col] = lsum > 0.f ? sum / lsum : 0.f;
    if (r < rows && col == 0)
      p.lse[((long long)n * p.heads + shared * per + r % per) * p.tq + r / per] = lsum > 0.f ? top + log2f(lsum) : -NEG_INF;
  }
  cluster.sync();                                                    // nobody leaves while others read its shared memory
}

// ------------------------------------------------------------------------------------------------ host side
int launched(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  else cudaGetLastError();
  if (e != cudaSuccess) return TSB_ERR_LAUNCH | ((int)e << 8);
  const int late = tsb_host::peek_status();
  return late ? TSB_ERR_TIMEOUT | (late << 8) : TSB_OK;
}

constexpr int MAX_DIM = 128, FEW_ROWS = 8;

// False: not a problem that the kernels take.  `vec` holds for all arrays given.
template <class... A>
bool describe(Problem& p, int n, int tq, int tk, int heads, int shared, int d, float scale, const float* q, const float* kv,
              const float* key, A... others) {
  if (n < 0 || tq < 0 || tk < 0 || heads <= 0 || shared <= 0 || heads % shared || d <= 0 || d > MAX_DIM) return false;
  const float* all[] = {q, kv, static_cast<const float*>(others)...};
  uintptr_t bits = 0;
  for (const float* a : all) bits |= reinterpret_cast<uintptr_t>(a);
  p = Problem{};
  p.q = q; p.kv = kv; p.key = key;
  p.n = n; p.tq = tq; p.tk = tk; p.heads = heads; p.shared = shared; p.d = d;
  p.scale = scale;
  p.qtiles = (tq + 127) / 128;
  p.ktiles = (tk + 127) / 128;
  p.vec = d % 4 == 0 && (bits & 15) == 0;
  return true;
}

template <class K>
int run(K kernel, const Problem& p, long long blocks, int threads, int smem, cudaStream_t st, tsb_launch::SmemLimit& limit) {
  if (blocks > INT32_MAX) return TSB_ERR_ARG;
  Problem q = p;
  q.status = tsb_host::status_word(st);
  if (!q.status) return TSB_ERR_LAUNCH;
  cudaError_t e = limit.raise(kernel, smem);
  if (e == cudaSuccess) e = tsb_launch::launch(kernel, dim3((unsigned)blocks), dim3(threads), smem, st, q);
  return launched(e);
}

// Where the pieces of q, k, v and g lie in one buffer, behind them the units and the dots.
struct Layout {
  size_t tiles[4], units[4], dots, bytes;
  Layout(int n, int tq, int tk, int heads, int shared, int d, bool with_g) {
    const size_t tile = d <= 64 ? Tile<64, 128>::BYTES : Tile<128, 128>::BYTES;
    const size_t q = (size_t)n * heads * ((tq + 127) / 128), k = (size_t)n * shared * ((tk + 127) / 128);
    const size_t count[4] = {q, k, k, with_g ? q : 0};
    bytes = 0;
    for (int i = 0; i < 4; ++i) {
      tiles[i] = bytes;
      bytes += count[i] * tile;
    }
    for (int i = 0; i < 4; ++i) {
      units[i] = bytes;
      bytes += count[i] * 4;
    }
    dots = bytes;
    if (with_g) bytes += (size_t)n * heads * tq * 4;
    bytes = (bytes + 15) / 16 * 16;
  }
  Pieces of(const char* base, int i) const { return {base + tiles[i], reinterpret_cast<const float*>(base + units[i])}; }
};
bool fits(const void* prepared, long long have, const Layout& at) {
  return prepared && (reinterpret_cast<uintptr_t>(prepared) & 15) == 0 && have >= (long long)at.bytes;
}
void use(Problem& p, const Layout& at, const char* base) {
  p.qp = at.of(base, 0);
  p.kp = at.of(base, 1);
  p.vp = at.of(base, 2);
  p.gp = at.of(base, 3);
  p.dot = reinterpret_cast<const float*>(base + at.dots);
}

// Splits q, k and v, and g (with the dots) where it is given.
int split(const Problem& p, const float* g, const float* y, const Layout& at, char* base, cudaStream_t st) {
  Sources all = {};
  all.d = p.d;
  all.vec = p.vec;
  const float* from[4] = {p.q, p.kv, p.kv ? p.kv + (long long)p.shared * p.d : nullptr, g};
  long long blocks = 0;
  for (int i = 0; i < 4; ++i) {
    Source& s = all.s[i];
    const bool state = i == 1 || i == 2;
    s.x = from[i];
    s.rows = state ? p.tk : p.tq;
    s.heads = state ? p.shared : p.heads;
    s.count = (s.rows + 127) / 128;
    s.row = state ? 2ll * p.shared * p.d : (long long)p.heads * p.d;
    s.batch = s.rows * s.row;
    s.head = p.d;
    s.mult = i == 0 ? p.scale * LOG2E : 1.f;
    s.tokens = state ? p.key : nullptr;
    s.tiles = base + at.tiles[i];
    s.units = reinterpret_cast<float*>(base + at.units[i]);
    if (i == 3) {
      s.with = y;
      s.dots = reinterpret_cast<float*>(base + at.dots);
    }
    all.first[i] = (int)blocks;
    if (i < 3 || g) blocks += (long long)p.n * s.heads * s.count;
    if (blocks > INT32_MAX) return TSB_ERR_ARG;
  }
  all.first[4] = (int)blocks;
  if (blocks == 0) return TSB_OK;
  return launched(p.d <= 64 ? tsb_launch::launch(split_tiles<64>, dim3((unsigned)blocks), dim3(256), 0, st, all)
                            : tsb_launch::launch(split_tiles<128>, dim3((unsigned)blocks), dim3(256), 0, st, all));
}

template <int LANES, int ROWS> int run_few(const Problem& p, cudaStream_t st) {
  constexpr int BATCH = 4, MAX_SPLIT = 8;
  // a cluster of blocks for a head's keys while SMs are idle and a block keeps four rounds of them
  const long long pairs = (long long)p.n * p.shared;
  int split = 1;
  while (split < MAX_SPLIT && pairs * split * 2 <= 148 * 4 && p.tk >= split * 2 * FEW_WARPS * (32 / LANES) * BATCH) split *= 2;
  if (pairs * split > INT32_MAX) return TSB_ERR_ARG;
  return launched(tsb_launch::launch_cluster(split > 1 ? split : 0, attend_few<LANES, ROWS, BATCH>, dim3((unsigned)(pairs * split)),
                                             dim3(FEW_WARPS * 32), 0, st, p, split));
}
template <int LANES> int few(const Problem& p, int rows, cudaStream_t st) {
  if (rows <= 1) return run_few<LANES, 1>(p, st);
  if (rows <= 2) return run_few<LANES, 2>(p, st);
  if (rows <= 4) return run_few<LANES, 4>(p, st);
  return run_few<LANES, 8>(p, st);
}

}  // namespace

extern "C" {

// y [N, Tq, H, d] and lse [N, H, Tq]: log2 of the sum of the keys' 2^S, +inf for a query without keys.  key may be null.
int tsb_cross_attention(const float* q, const float* kv, const float* key, float* y, float* lse, int n, int tq, int tk, int heads,
                        int shared, int d, float scale, void* stream) {
  Problem p;
  if (!describe(p, n, tq, tk, heads, shared, d, scale, q, kv, key, y)) return TSB_ERR_ARG;
  if (n == 0 || tq == 0) return TSB_OK;
  if (!q || !y || !lse || (tk && !kv)) return TSB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  p.y = y;
  p.lse = lse;
  const long long rows = (long long)(heads / shared) * tq;
  if (rows <= FEW_ROWS) return d <= 32 ? few<8>(p, (int)rows, st) : d <= 64 ? few<16>(p, (int)rows, st) : few<32>(p, (int)rows, st);
  const Layout at(n, tq, tk, heads, shared, d, false);
  char* pieces = static_cast<char*>(tsb_scratch::get(st, tsb_scratch::ATTENTION_PIECES, at.bytes));
  if (!pieces) return TSB_ERR_OOM;
  use(p, at, pieces);
  const int rc = split(p, nullptr, nullptr, at, pieces, st);
  if (rc) return rc;
  const long long blocks = (long long)n * heads * p.qtiles;
  static tsb_launch::SmemLimit limit64, limit128;
  if (d <= 64) return run(attend<64>, p, blocks, 192, ForwardShape<64>::SMEM, st, limit64);
  return run(attend<128>, p, blocks, 192, ForwardShape<128>::SMEM, st, limit128);
}

// The pieces of q, kv and g, and the sums of g y over a head's row, for both gradients.  prepared: `have` bytes on a
// 16-byte boundary, as many as Layout says.
int tsb_cross_attention_prepare(const float* q, const float* kv, const float* key, const float* g, const float* y, void* prepared,
                                long long have, int n, int tq, int tk, int heads, int shared, int d, float scale, void* stream) {
  Problem p;
  if (!describe(p, n, tq, tk, heads, shared, d, scale, q, kv, key, g, y)) return TSB_ERR_ARG;
  if (n == 0) return TSB_OK;
  const Layout at(n, tq, tk, heads, shared, d, true);
  if ((tq && (!q || !g || !y)) || (tk && !kv) || !fits(prepared, have, at)) return TSB_ERR_ARG;
  return split(p, g, y, at, static_cast<char*>(prepared), static_cast<cudaStream_t>(stream));
}

int tsb_cross_attention_grad_q(const void* prepared, long long have, const float* key, const float* lse, float* dq, int n, int tq, int tk, int heads,
                               int shared, int d, float scale, void* stream) {
  Problem p;
  if (!describe(p, n, tq, tk, heads, shared, d, scale, nullptr, nullptr, key, dq)) return TSB_ERR_ARG;
  if (n == 0 || tq == 0) return TSB_OK;
  const Layout at(n, tq, tk, heads, shared, d, true);
  if (!lse || !dq || !fits(prepared, have, at)) return TSB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  use(p, at, static_cast<const char*>(prepared));
  p.lse = const_cast<float*>(lse);
  p.dq = dq;
  const long long blocks = (long long)n * heads * p.qtiles;
  static tsb_launch::SmemLimit limit64, limit128;
  if (d <= 64) return run(grad_of_queries<64>, p, blocks, 192, QueryShape<64>::SMEM, st, limit64);
  return run(grad_of_queries<128>, p, blocks, 192, QueryShape<128>::SMEM, st, limit128);
}

int tsb_cross_attention_grad_kv(const void* prepared, long long have, const float* key, const float* lse, float* dkv, int n, int tq, int tk, int heads,
                                int shared, int d, float scale, void* stream) {
  Problem p;
  if (!describe(p, n, tq, tk, heads, shared, d, scale, nullptr, nullptr, key, dkv)) return TSB_ERR_ARG;
  if (n == 0 || tk == 0) return TSB_OK;
  const Layout at(n, tq, tk, heads, shared, d, true);
  if (!dkv || (tq && !lse) || !fits(prepared, have, at)) return TSB_ERR_ARG;
  if ((long long)((tq + 63) / 64) * (heads / shared) > INT32_MAX / 2) return TSB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  use(p, at, static_cast<const char*>(prepared));
  p.lse = const_cast<float*>(lse);
  p.dkv = dkv;
  const long long blocks = (long long)n * shared * p.ktiles;
  static tsb_launch::SmemLimit limit64, limit128;
  if (d <= 64) return run(grad_of_states<64>, p, blocks, 320, StateShape<64>::SMEM, st, limit64);
  return run(grad_of_states<128>, p, blocks, 320, StateShape<128>::SMEM, st, limit128);
}

}  // extern "C"
