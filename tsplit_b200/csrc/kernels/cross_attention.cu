// Attention across to an encoder's states, forward and backward.
//
//   q [N, Tq, H, d], kv [N, Tk, 2, G, d] (keys, then values; G heads, each read by H / G query heads), key [N, Tk] (0: out)
//   S = scale q k^T,  P = softmax(S) over the keys that are in,  y = P v
//   dP = dy v^T,  dS = P (dP - rowsum(dy y)),  dq = scale dS k,  dk = scale dS^T q,  dv = P^T dy
//
// A key that is out takes no part, whatever its row holds (it is not read).  A query without any key has y = 0 and no
// gradient.  The scores never leave the chip: the backward kernels compute them again from the rows' log-sum-exp.
//
// Products run on tcgen05 with the accuracy of fp32, of numbers that are not too far apart: an operand tile of 128 rows is scaled by
// a power of two that brings its largest number to [2^13, 2^14) and split into two fp16 numbers, x = hi + lo, |x - hi - lo| <= 2^-22
// |x|, or 2^-38 of the tile's largest, where fp16 ends (so a row down to 2^-16 of its tile keeps what fp32 keeps, one at 2^-20 7e-6 of
// itself, at 2^-30 0.9 %); P ends at 2^-39, dS at 2^-39 of its bound.  A product is three: hi hi + hi lo + lo hi.  That takes 1.5
// times the tensor time of one TF32 product, which keeps 2^-11, and the room of fp32, and 16-bit tiles can be read in both directions
// (K-major and MN-major) from one copy in shared memory.  (Two bf16 numbers need no scale but keep 2^-17, three need six products.)
// A kernel before splits every operand once, in tiles of 128 rows that lie in memory as they will in shared memory, so the kernels
// that multiply load them by bulk copies.  P and dS are split by the threads that compute them and go to tensor memory, from where
// they are the A operand of the next product: P is at most 2^14, dS is scaled by a bound of its own.  What a tile adds to y, dq, dk
// or dv is read from tensor memory and added in registers with the tile's scale.
//
// Scores are kept in units of log 2 (q is scaled by scale * log2(e) as it is loaded), so that an exponential is one ex2.
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "launch.cuh"
#include "scratch.h"
#include "smem_limit.h"
#include "tc_common.cuh"

namespace {

using namespace tsb;
using tsb_launch::load;

constexpr float NEG_INF = -__builtin_huge_valf(), LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr unsigned ALL = 0xffffffffu;

// Tiles of pieces, [n][head][tile], and of each tile what a number of it stands for (x) and the length of its longest row (y).
struct Pieces {
  const char* tiles;
  const float2* units;
};

struct Problem {
  const float *q, *kv, *key, *dot, *lengths;
  float *y, *lse, *dq, *dkv;
  Pieces qp, kp, vp, gp;
  int n, tq, tk, heads, shared, d;
  float scale;
  int qtiles, ktiles;
  bool vec;                                  // rows are whole 16-byte pieces on 16-byte boundaries
  int query_blocks;                          // of the gradients: blocks that compute those of queries
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
// e with |x| 2^e in [2^top, 2^(top+1)), kept where 2^e and 2^-e are normal numbers (0 and tiny x: `most`)
__device__ __forceinline__ int exponent_to(uint32_t bits_of_abs, int top, int most = 126) {
  return min(top + 127 - (int)(bits_of_abs >> 23), most);
}
constexpr int TOP = 13;                      // of a tile's largest number
constexpr int LEAST = 112;                   // a tile's unit is 2^-LEAST at the least, and normal when P's scale divides it
constexpr float LARGEST = 16384.f;           // and what that is below, 2^(TOP+1); P is scaled by it too (sums of P v are not)

// A tile of ROWS x D numbers in shared memory: the plane of the hi pieces, then that of the lo pieces; a plane is D / 64
// chunks of [ROWS][64] halves whose rows of 128 bytes are swizzled (16-byte unit u of row r lies at u ^ (r & 7)).
template <int D, int ROWS> struct Tile {
  static constexpr int CHUNK = ROWS * 128, PLANE = ROWS * D * 2, BYTES = 2 * PLANE;
};

// One operand to split: rows of d numbers of [n][t][head].
struct Source {
  const float* x;
  const float* with;                         // an array like x: dots[n, head, tile, row] = sum of x with over a row; or null
  const float* tokens;                       // [n][t], a row whose token is 0 counts as zeros and is not read; or null
  float *dots, *lengths;                     // with `with`: lengths[n, head, tile, row]
  char* tiles;
  float2* units;
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

// A block splits a tile of 128 rows.  Infinities and NaN have no part in the tile's unit, so they stay within their row: its pieces
// are NaN (inf - inf), and so is what is computed with them.
template <int D>
__global__ void __launch_bounds__(256) split_tiles(const Sources all) {
  tsb_launch::enter();
  using L = Tile<D, 128>;
  constexpr int UNITS = D / 8, TRIPS = 128 * UNITS / 256;
  __shared__ uint32_t largest[8], longest[8];
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
      if (i % UNITS == 0) s.dots[(size_t)b * 128 + row] = sum;
    }
  }
  uint32_t most = 0, most_squares = 0;
  float squares[TRIPS];
#pragma unroll
  for (int u = 0; u < TRIPS; ++u) {
    squares[u] = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[u][k] *= s.mult;
      const uint32_t size = __float_as_uint(v[u][k]) & 0x7fffffffu;
      if (size < 0x7f800000u) most = max(most, size);
      squares[u] += v[u][k] * v[u][k];
    }
#pragma unroll
    for (int o = UNITS / 2; o > 0; o >>= 1) squares[u] += __shfl_xor_sync(ALL, squares[u], o);
    most_squares = max(most_squares, __float_as_uint(squares[u]));
  }
  if (s.with && threadIdx.x % UNITS == 0)
#pragma unroll
    for (int u = 0; u < TRIPS; ++u) s.lengths[(size_t)b * 128 + (threadIdx.x + u * 256) / UNITS] = sqrtf(squares[u]);
  most = __reduce_max_sync(ALL, most);
  most_squares = __reduce_max_sync(ALL, most_squares);
  if ((threadIdx.x & 31) == 0) largest[threadIdx.x >> 5] = most, longest[threadIdx.x >> 5] = most_squares;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) most = max(most, largest[w]), most_squares = max(most_squares, longest[w]);
  const int e = exponent_to(most, TOP, LEAST);
  const float scale = power_of_two(e);
  // (a row whose squares overflow, or vanish, or are NaN, has its largest number instead)
  if (threadIdx.x == 0) {
    const float length = sqrtf(__uint_as_float(most_squares)), least = __uint_as_float(most);
    s.units[b] = make_float2(power_of_two(-e), length < 1e15f && length > 1e-15f ? length : least * (float)D);
  }
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
// The first or the last 64 rows of a tile, as a tile of 64 rows; `more` bytes are to come to the same barrier.
template <int D>
__device__ __forceinline__ void copy_half(char* to, const Pieces& p, long long tile, int half, uint64_t* full, int more = 0) {
  using L = Tile<D, 128>;
  using H = Tile<D, 64>;
  mbar_expect_tx(full, H::BYTES + more);
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
// One of the lanes that get here issues: the `leader`.
__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t leader, uint64_t* bar) {
  if (leader) umma_commit(bar);
}
constexpr uint32_t DESC_HI = smem_desc_hi(1024);       // 128-byte swizzle, groups of eight rows 1024 bytes apart

// D [128 x ROWS_B] = A B^T over the D columns of both tiles.  The small products come first: a step of tcgen05 drops what is below
// the last bit of the sum so far, and the sum is at its full size for a third of the steps only (700 x 900, 128 columns: y off by
// 4.9e-7 in place of 1.2e-6, plain fp32 operators 6.7e-7).
template <int D, int ROWS_A, int ROWS_B>
__device__ __forceinline__ void product_of_rows(uint32_t to, uint32_t a, uint32_t b, uint32_t leader) {
  using LA = Tile<D, ROWS_A>;
  using LB = Tile<D, ROWS_B>;
  const uint32_t al = smem_desc_lo(a, 16), bl = smem_desc_lo(b, 16);
  auto at = [&](int k, uint32_t lo, int chunk) { return smem_desc_join(DESC_HI, lo + ((k / 4 * chunk + k % 4 * 32) >> 4)); };
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
    mma_smem(to, at(k, al, LA::CHUNK), at(k, bl + (LB::PLANE >> 4), LB::CHUNK), idesc_f16(ROWS_B, 0), k > 0, leader);
    mma_smem(to, at(k, al + (LA::PLANE >> 4), LA::CHUNK), at(k, bl, LB::CHUNK), idesc_f16(ROWS_B, 0), 1, leader);
  }
#pragma unroll
  for (int k = 0; k < D / 16; ++k) mma_smem(to, at(k, al, LA::CHUNK), at(k, bl, LB::CHUNK), idesc_f16(ROWS_B, 0), 1, leader);
}
// The same with A in tensor memory: its hi pieces in D / 2 columns, two to each, then the lo pieces.
template <int D, int ROWS_B>
__device__ __forceinline__ void product_of_kept_rows(uint32_t to, uint32_t a, uint32_t b, uint32_t leader) {
  using L = Tile<D, ROWS_B>;
  const uint32_t bl = smem_desc_lo(b, 16);
  auto at = [&](int k, int plane) { return smem_desc_join(DESC_HI, bl + ((k / 4 * L::CHUNK + k % 4 * 32 + plane) >> 4)); };
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
    mma_tmem(to, a + 8 * k, at(k, L::PLANE), idesc_f16(ROWS_B, 0), k > 0, leader);
    mma_tmem(to, a + D / 2 + 8 * k, at(k, 0), idesc_f16(ROWS_B, 0), 1, leader);
  }
#pragma unroll
  for (int k = 0; k < D / 16; ++k) mma_tmem(to, a + 8 * k, at(k, 0), idesc_f16(ROWS_B, 0), 1, leader);
}
// The same with A's hi pieces in tensor memory and the lo ones, a plane, in shared memory.
template <int D, int ROWS_A, int ROWS_B>
__device__ __forceinline__ void product_of_half_kept_rows(uint32_t to, uint32_t a_hi, uint32_t a_lo, uint32_t b, uint32_t leader) {
  using LA = Tile<D, ROWS_A>;
  using LB = Tile<D, ROWS_B>;
  const uint32_t al = smem_desc_lo(a_lo, 16), bl = smem_desc_lo(b, 16);
  auto at = [&](int k, uint32_t lo, int chunk) { return smem_desc_join(DESC_HI, lo + ((k / 4 * chunk + k % 4 * 32) >> 4)); };
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
    mma_tmem(to, a_hi + 8 * k, at(k, bl + (LB::PLANE >> 4), LB::CHUNK), idesc_f16(ROWS_B, 0), k > 0, leader);
    mma_smem(to, at(k, al, LA::CHUNK), at(k, bl, LB::CHUNK), idesc_f16(ROWS_B, 0), 1, leader);
  }
#pragma unroll
  for (int k = 0; k < D / 16; ++k) mma_tmem(to, a_hi + 8 * k, at(k, bl, LB::CHUNK), idesc_f16(ROWS_B, 0), 1, leader);
}
// D [128 x D] (+)= A B, A [128 x ROWS] in tensor memory: 16 columns for every 16 of its, hi pieces in the first eight.
template <int D, int ROWS>
__device__ __forceinline__ void product_with_columns(uint32_t to, uint32_t a, uint32_t b, uint32_t leader, bool accumulate = false) {
  using L = Tile<D, ROWS>;
  const uint32_t bl = smem_desc_lo(b, L::CHUNK);
  auto at = [&](int k, int plane) { return smem_desc_join(DESC_HI, bl + ((k * 2048 + plane) >> 4)); };
#pragma unroll
  for (int k = 0; k < ROWS / 16; ++k) {
    mma_tmem(to, a + 16 * k, at(k, L::PLANE), idesc_f16(D, 1), accumulate || k > 0, leader);
    mma_tmem(to, a + 16 * k + 8, at(k, 0), idesc_f16(D, 1), 1, leader);
  }
#pragma unroll
  for (int k = 0; k < ROWS / 16; ++k) mma_tmem(to, a + 16 * k, at(k, 0), idesc_f16(D, 1), 1, leader);
}

// Loads from tensor memory run behind what the thread does until tmem_ld_wait; tmem_arrived then names the registers, so
// that nothing that reads them is moved before the wait.
__device__ __forceinline__ void tmem_begin(uint32_t addr, float (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
               "%14, %15}, [%16];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
                 "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
                 "=f"(v[14]), "=f"(v[15])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void tmem_begin(uint32_t addr, float (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
               "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
                 "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
                 "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]),
                 "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]),
                 "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
               : "r"(addr)
               : "memory");
}
template <int COUNT> __device__ __forceinline__ void tmem_arrived(float (&v)[COUNT]) {
#pragma unroll
  for (int i = 0; i < COUNT; ++i) asm volatile("" : "+f"(v[i]));
}
// Numbers of a row, 16 at a time, as hi pieces in eight columns and lo pieces in the next eight
template <int COUNT> __device__ __forceinline__ void tmem_st_pieces(uint32_t addr, const float (&v)[COUNT]) {
#pragma unroll
  for (int c = 0; c < COUNT; c += 16) {
    uint32_t r[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) split2(v[c + 2 * i], v[c + 2 * i + 1], r[i], r[8 + i]);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
          "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr + c)
        : "memory");
  }
}
// acc = acc times + what the tensor memory holds from addr on, times unit; two loads under way
template <bool TIMES, int COUNT>
__device__ __forceinline__ void add_columns(uint32_t addr, float (&acc)[COUNT], float times, float unit) {
  float v[2][16];
  tmem_begin(addr, v[0]);
#pragma unroll
  for (int c = 0; c < COUNT; c += 16) {
    float(&x)[16] = v[c / 16 & 1];
    tmem_ld_wait();
    tmem_arrived(x);
    if (c + 16 < COUNT) tmem_begin(addr + c + 16, v[(c / 16 + 1) & 1]);
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[c + i] = (TIMES ? acc[c + i] * times : acc[c + i]) + x[i] * unit;
  }
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Keys up to the last one that is in, rounded up to the 256 that a warp looks at in one go.  Every warp finds out for itself.
__device__ __forceinline__ int keys_in(const float* tokens, int tk) {
  if (!tokens) return tk;
  for (int end = tk; end > 0; end -= 256) {
    bool in = false;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = end - 1 - u * 32 - (int)(threadIdx.x & 31);
      in |= i >= 0 && load(tokens + max(i, 0)) != 0.f;
    }
    if (__any_sync(ALL, in)) return end;
  }
  return 0;
}
// The token of key `first` + lane; 0 for a key that is out or that there is not.
__device__ __forceinline__ float token_of(const float* tokens, int first, int tk) {
  const int k = first + (int)(threadIdx.x & 31);
  return k < tk ? (tokens ? load(tokens + k) : 1.f) : 0.f;
}

// After a wait that ran out: the products that were issued still use shared and tensor memory.
__device__ __forceinline__ void drain(uint64_t* bar) {
  umma_commit(bar);
  const long long begin = clock64();
  while (!mbar_try_wait(bar, 0) && clock64() - begin < WAIT_LIMIT_CYCLES) {
  }
}

// Shared memory: tiles from a multiple of 1024 bytes on, and 1024 bytes of barriers behind them.
constexpr int CONTROL = 1024;
extern __shared__ __align__(1024) char tiles_of_block[];
template <class Control> __device__ __forceinline__ Control* control_at(int bytes_of_tiles) {
  static_assert(sizeof(Control) <= CONTROL, "one kilobyte is kept for it");
  return reinterpret_cast<Control*>(tiles_of_block + bytes_of_tiles);
}

// A block has 384 threads: eight warps that compute, and four others of which one copies and one issues the products; the
// registers go to the former.  A row belongs to two threads, in warps w and w + 4.
template <int R> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }

// Half of a row's pieces (columns D / 2 * half on; the hi ones alone with PLANES = 1) of a tile: read from memory, and put into tensor memory as
// product_of_kept_rows takes them.
template <int D, int PLANES = 2> struct KeptRow {
  uint4 v[PLANES][D / 16];
  __device__ __forceinline__ void read(const Pieces& p, long long tile, int row, int half) {
    using L = Tile<D, 128>;
    const char* const from = p.tiles + tile * L::BYTES + row * 128;
#pragma unroll
    for (int plane = 0; plane < PLANES; ++plane)
#pragma unroll
      for (int u = 0; u < D / 16; ++u) {
        const int at = half * (D / 16) + u;
        v[plane][u] = load(reinterpret_cast<const uint4*>(from + plane * L::PLANE + at / 8 * L::CHUNK + (((at & 7) ^ (row & 7)) << 4)));
      }
  }
  __device__ __forceinline__ void keep(uint32_t to, int half) const {
#pragma unroll
    for (int plane = 0; plane < PLANES; ++plane)
#pragma unroll
      for (int u = 0; u < D / 16; u += 4)                            // four pieces of 16 bytes: 16 columns
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
            ::"r"(v[plane][u].x), "r"(v[plane][u].y), "r"(v[plane][u].z), "r"(v[plane][u].w), "r"(v[plane][u + 1].x),
              "r"(v[plane][u + 1].y), "r"(v[plane][u + 1].z), "r"(v[plane][u + 1].w), "r"(v[plane][u + 2].x), "r"(v[plane][u + 2].y),
              "r"(v[plane][u + 2].z), "r"(v[plane][u + 2].w), "r"(v[plane][u + 3].x), "r"(v[plane][u + 3].y), "r"(v[plane][u + 3].z),
              "r"(v[plane][u + 3].w), "r"(to + plane * (D / 2) + half * (D / 4) + u * 4)
            : "memory");
  }
};

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
// A block takes 128 queries of a head, kept in tensor memory, and tiles of 128 keys; keys and values share a ring of slots of
// 32 KB.  Warps 0 to 7: soft-max, w and w + 4 half of the keys of 32 rows each; 8: copies; 9 issues the products.  Two tiles of
// scores are in tensor memory, so S of the next tile runs while the threads work on this one.  P takes the place of its S, and y
// of a tile is added to the registers before the next one's product.
//
// Bound by the tensor cores and by the threads between two products.  With the splitting: 2 x 2000 x 4111, 16 heads of 128 on 4:
// 323 us, 417 TFLOP/s, so 1.25 PFLOP/s of fp16 products; 4 x 2048 x 2048, 16 heads of 64: 222 us; 32 x 255 x 256, 8 heads of 64:
// 49 us.  (A row to a thread and two blocks to an SM, operands in shared memory: 444, 278 and 47 us.  A block's beginning and
// end are not hidden now, which a few key tiles show, but a product with A in tensor memory takes 32 cycles for 16 x 64 numbers
// of B, with A in shared memory 48, and two threads do a row's soft-max in half the time.  Two tiles of queries to a block, sixteen
// soft-max warps: 51 and 258 us for 64 columns, fewer blocks that share the SMs less evenly.)
template <int D> struct ForwardShape {
  static constexpr int PARTS = D / 64, ROWS = 128 / PARTS, SLOTS = 6;              // of a tile in a slot each
  static constexpr int K_SLOTS = PARTS == 1 ? 3 : 2, V_SLOTS = SLOTS - K_SLOTS;
  static constexpr int S_AT = D, Y_AT = S_AT + 2 * 128;                            // behind the queries
  using L = Tile<D, ROWS>;
  static constexpr int TILES = SLOTS * L::BYTES, SMEM = TILES + CONTROL + 2 * 1024;
};
struct ForwardControl {
  uint64_t q_full, full[6], empty[6], s_full[2], p_full[2], y_full, pair[4], drained;
  uint32_t tmem;
};
constexpr int BLOCK = 384, TMEM_COLUMNS = 512;

template <int D>
__global__ void __launch_bounds__(BLOCK, 1) attend(const Problem p) {
  using Shape = ForwardShape<D>;
  using L = typename Shape::L;
  constexpr int SLOTS = Shape::SLOTS, PARTS = Shape::PARTS;
  ForwardControl* bar = control_at<ForwardControl>(Shape::TILES);
  float(*const shared_max)[2][128] = reinterpret_cast<float(*)[2][128]>(tiles_of_block + Shape::TILES + CONTROL);      // [tile & 1][half]
  const int warp = __shfl_sync(ALL, threadIdx.x >> 5, 0);
  if (threadIdx.x == 0) {
    mbar_init(&bar->q_full, 256);
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->p_full[i], 256);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&bar->pair[i], 64);
    mbar_init(&bar->y_full, 1);
    mbar_init(&bar->drained, 1);
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(&bar->tmem, TMEM_COLUMNS);
    tmem_relinquish();
  }
  tsb_launch::enter();
  const int qt = blockIdx.x % p.qtiles, h = blockIdx.x / p.qtiles % p.heads, n = blockIdx.x / p.qtiles / p.heads;
  const int shared = h / (p.heads / p.shared), q0 = qt * 128, half = warp >> 2, row = threadIdx.x & 127;
  const float* tokens = p.key ? p.key + (long long)n * p.tk : nullptr;
  const long long q_row = (long long)p.heads * p.d;
  const long long q_at = ((long long)n * p.heads + h) * p.qtiles + qt, k_at = ((long long)n * p.shared + shared) * p.ktiles;
  KeptRow<D> kept;                             // (under way while the block sets itself up)
  if (warp < 8) kept.read(p.qp, q_at, row, half);
  const int tiles = (keys_in(tokens, p.tk) + 127) / 128;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(ALL, bar->tmem, 0);

  if (warp < 8) {
    more_registers<208>();
    constexpr int OWN = D / 2;                                   // columns of y of a thread
    const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21);   // this warp's 32 lanes
    kept.keep(mine, half);
    tmem_st_wait();
    tc_fence_before();
    mbar_arrive(&bar->q_full);
    float acc[OWN], m = NEG_INF, l = 0.f, before = 1.f, v_unit = 0.f;
    const float q_unit = load(p.qp.units + q_at).x;
#pragma unroll
    for (int c = 0; c < OWN; ++c) acc[c] = 0.f;
    bool ok = true;
    auto add_tile = [&](int j) {                                 // before: from the maximum then to the one that tile j has
      if (!mbar_wait(&bar->y_full, j & 1, p.status, 0x301)) return false;
      tc_fence_after();
      add_columns<true>(mine + Shape::Y_AT + half * OWN, acc, before, v_unit);
      return true;
    };
    // (what a tile needs from memory besides its scores is read a tile ahead)
    float token[2], k_next = 0.f, v_next = 0.f;
    auto look_at = [&](int j) {
#pragma unroll
      for (int w = 0; w < 2; ++w) token[w] = token_of(tokens, j * 128 + half * 64 + w * 32, p.tk);
      k_next = j < tiles ? load(p.kp.units + k_at + j).x : 0.f;
      v_next = j < tiles ? load(p.vp.units + k_at + j).x : 0.f;
    };
    look_at(0);
    for (int j = 0; j < tiles; ++j) {
      const int b = j & 1;
      unsigned in[2];
#pragma unroll
      for (int w = 0; w < 2; ++w) in[w] = __ballot_sync(ALL, token[w] != 0.f);
      // (above 0, so that -inf stays so: tiles of nothing but zeros have the least unit, and scores of 2^-90 are as good as none)
      const float unit = fmaxf(q_unit * k_next, 1.2e-38f), next_unit = v_next;
      look_at(j + 1);
      if (!mbar_wait(&bar->s_full[b], j >> 1 & 1, p.status, 0x302)) { ok = false; break; }
      tc_fence_after();
      const uint32_t at = mine + Shape::S_AT + b * 128 + half * 64;
      float s[2][32], part[4] = {NEG_INF, NEG_INF, NEG_INF, NEG_INF};                // (chains that do not wait for one another)
      tmem_begin(at, s[0]);
      tmem_begin(at + 32, s[1]);
      tmem_ld_wait();
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        tmem_arrived(s[w]);
        if (in[w] != ALL) {
#pragma unroll
          for (int i = 0; i < 32; ++i) s[w][i] = (in[w] >> i) & 1 ? s[w][i] : NEG_INF;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) part[i & 3] = fmaxf(part[i & 3], s[w][i]);
      }
      const float own = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
      shared_max[j & 1][half][row] = own;
      mbar_arrive(&bar->pair[warp & 3]);
      if (!mbar_wait(&bar->pair[warp & 3], j & 1, p.status, 0x309)) { ok = false; break; }
      const float most = fmaxf(own, shared_max[j & 1][half ^ 1][row]);
      const float top = fmaxf(m, most == NEG_INF ? NEG_INF : most * unit), ref = top == NEG_INF ? 0.f : top;
      const float factor = exp2_fast(m - ref), shift = TOP + 1 - ref;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 2; ++w) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          s[w][i] = exp2_fast(s[w][i] * unit + shift);           // (a masked one: 2^-inf)
          sum[i & 3] += s[w][i];
        }
        tmem_st_pieces(at + 32 * w, s[w]);
      }
      tmem_st_wait();
      if (j > 0 && !(ok = add_tile(j - 1))) break;
      tc_fence_before();
      mbar_arrive(&bar->p_full[b]);
      l = l * factor + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
      m = top;
      before = factor;
      v_unit = next_unit * (1.f / LARGEST);
    }
    if (ok && tiles > 0) ok = add_tile(tiles - 1);
    // the halves' sums
    shared_max[tiles & 1][half][row] = l;
    mbar_arrive(&bar->pair[warp & 3]);
    if (ok && mbar_wait(&bar->pair[warp & 3], tiles & 1, p.status, 0x309)) {
      l += shared_max[tiles & 1][half ^ 1][row];
      const int t = q0 + row;
      if (t < p.tq)
        store_row(p.y + ((long long)n * p.tq + t) * q_row + (long long)h * p.d + half * OWN, acc, l != 0.f ? LARGEST / l : 0.f, p.d - half * OWN,
                  p.vec);
      // (a row without keys, or behind the last one: exp2(S - inf) = 0 in the backward pass; l may be NaN)
      if (half == 0) p.lse[q_at * 128 + row] = l != 0.f && t < p.tq ? m - (TOP + 1) + log2f(l) : -NEG_INF;
    }
  } else {
    fewer_registers<88>();
    if (warp == 8 && elect_one()) {
      for (int i = 0; i < 2 * PARTS * tiles; ++i) {
        const int j = i / (2 * PARTS), v = i / PARTS & 1, at = j * PARTS + i % PARTS;
        const int s = v ? Shape::K_SLOTS + at % Shape::V_SLOTS : at % Shape::K_SLOTS;
        const Pieces& from = v ? p.vp : p.kp;
        if (!mbar_wait(&bar->empty[s], (at / (v ? Shape::V_SLOTS : Shape::K_SLOTS) & 1) ^ 1, p.status, 0x303)) break;
        if (PARTS == 1) copy_tile<D>(tiles_of_block + s * L::BYTES, from, k_at + j, &bar->full[s]);
        else copy_half<D>(tiles_of_block + s * L::BYTES, from, k_at + j, i % PARTS, &bar->full[s]);
      }
    }
    if (warp == 9 && tiles > 0) {
      const uint32_t leader = elect_one();      // (all lanes wait and loop, so that descriptors are the warp's: 343 -> 323 us)
      const uint32_t ring = smem_u32(tiles_of_block);
      bool ok = mbar_wait(&bar->q_full, 0, p.status, 0x305);
      tc_fence_after();
      auto scores = [&](int j) {
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const int at = j * PARTS + part, s = at % Shape::K_SLOTS;
          if (!mbar_wait(&bar->full[s], at / Shape::K_SLOTS & 1, p.status, 0x306)) return false;
          tc_fence_after();
          product_of_kept_rows<D, Shape::ROWS>(tmem + Shape::S_AT + (j & 1) * 128 + part * Shape::ROWS, tmem, ring + s * L::BYTES, leader);
          commit_if(leader, &bar->empty[s]);
        }
        commit_if(leader, &bar->s_full[j & 1]);
        return true;
      };
      for (int j = 0; j < 2 && j < tiles && ok; ++j) ok = scores(j);
      for (int j = 0; j < tiles && ok; ++j) {
        const int b = j & 1;
        if (!(ok = mbar_wait(&bar->p_full[b], j >> 1 & 1, p.status, 0x308))) break;
#pragma unroll
        for (int part = 0; part < PARTS && ok; ++part) {
          const int at = j * PARTS + part, s = Shape::K_SLOTS + at % Shape::V_SLOTS;
          if (!(ok = mbar_wait(&bar->full[s], at / Shape::V_SLOTS & 1, p.status, 0x307))) break;
          tc_fence_after();
          product_with_columns<D, Shape::ROWS>(tmem + Shape::Y_AT, tmem + Shape::S_AT + b * 128 + part * Shape::ROWS, ring + s * L::BYTES, leader,
                                               part > 0);
          commit_if(leader, &bar->empty[s]);
        }
        if (!ok) break;
        commit_if(leader, &bar->y_full);
        if (j + 2 < tiles) ok = scores(j + 2);
      }
      if (!ok && leader) drain(&bar->drained);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, TMEM_COLUMNS);
}

// ------------------------------------------------------------------------------------------------ gradients
// A bound of |dP - dot| over rows: e with (|g| |v| + |dot|) 2^e below 2^15, |g| and |v| the lengths of the longest ones.  2^-e times
// `unit`, which what is made of dS is multiplied by, stays a normal number.
__device__ __forceinline__ int exponent_of_ds(float g_length, float v_length, float dot, float unit) {
  const float most = 1.001f * (g_length * v_length) + fabsf(dot);
  return min(exponent_to(__float_as_uint(most), TOP + 1), (int)(__float_as_uint(unit) >> 23) - 1);
}

// dq: a block takes 128 queries of a head and tiles of 64 keys; the same roles.  The queries, and with 64 columns their gradients
// too, are kept in tensor memory, else these lie before the ring.  dS takes the place of its S.  A row's dS is bounded by the length
// of its own g: gradients differ much from row to row (a token that is all but certain has next to none), and each has a row of dq to
// itself.  (100 queries, 130 keys, one row of g 2^20 times its neighbours: bounded by the longest of all rows, dq of these was off by
// 2e-3 of its largest number, and by more the more keys there are; now 1.2e-5, which is what pieces of g keep.  2^16 times: 1.4e-6, as
// without it.)  The cases of attend: 459, 235 and 34 us (a row to a thread, two blocks to an SM, operands in shared memory: 672, 301
// and 32).
template <int D> struct QueryShape {
  static constexpr bool BOTH = D == 64;
  static constexpr int K_SLOTS = BOTH ? 4 : 3, V_SLOTS = BOTH ? 4 : 2, SLOTS = K_SLOTS + V_SLOTS;
  static constexpr int G_AT = D, S_AT = BOTH ? 2 * D : D, DP_AT = S_AT + 2 * 64, DQ_AT = DP_AT + 2 * 64;
  using LQ = Tile<D, 128>;
  using LK = Tile<D, 64>;
  static constexpr int RING_AT = BOTH ? 0 : LQ::BYTES, TILES = RING_AT + SLOTS * LK::BYTES, SMEM = TILES + CONTROL;
};
struct QueryControl {
  uint64_t q_full, g_full, full[8], empty[8], s_full[2], ds_full[2], dq_full, drained;
  uint32_t tmem;
};

template <int D>
__device__ __forceinline__ void grad_of_queries(const Problem& p, const int block) {
  using Shape = QueryShape<D>;
  using LQ = typename Shape::LQ;
  using LK = typename Shape::LK;
  constexpr int SLOTS = Shape::SLOTS;
  char *const g_tile = tiles_of_block, *const ring = tiles_of_block + Shape::RING_AT;
  QueryControl* bar = control_at<QueryControl>(Shape::TILES);
  const int warp = __shfl_sync(ALL, threadIdx.x >> 5, 0);
  if (threadIdx.x == 0) {
    mbar_init(&bar->q_full, 256);
    mbar_init(&bar->g_full, 1);
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->ds_full[i], 256);
    }
    mbar_init(&bar->dq_full, 1);
    mbar_init(&bar->drained, 1);
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(&bar->tmem, TMEM_COLUMNS);
    tmem_relinquish();
  }
  tsb_launch::enter();
  const int qt = block % p.qtiles, h = block / p.qtiles % p.heads, n = block / p.qtiles / p.heads;
  const int shared = h / (p.heads / p.shared), q0 = qt * 128, half = warp >> 2, row = threadIdx.x & 127;
  const float* tokens = p.key ? p.key + (long long)n * p.tk : nullptr;
  const long long q_row = (long long)p.heads * p.d;
  const long long q_at = ((long long)n * p.heads + h) * p.qtiles + qt, k_at = ((long long)n * p.shared + shared) * p.ktiles;
  KeptRow<D> kept;                             // (under way while the block sets itself up)
  KeptRow<Shape::BOTH ? D : 64> kept_g;
  if (warp < 8) {
    kept.read(p.qp, q_at, row, half);
    if (Shape::BOTH) kept_g.read(p.gp, q_at, row, half);
  }
  const int tiles = (keys_in(tokens, p.tk) + 63) / 64;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(ALL, bar->tmem, 0);

  if (warp < 8) {
    more_registers<208>();
    constexpr int OWN = D / 2;
    const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21);
    kept.keep(mine, half);
    if (Shape::BOTH) kept_g.keep(mine + Shape::G_AT, half);
    tmem_st_wait();
    tc_fence_before();
    mbar_arrive(&bar->q_full);
    float acc[OWN], before = 0.f;
#pragma unroll
    for (int c = 0; c < OWN; ++c) acc[c] = 0.f;
    const float lse = load(p.lse + q_at * 128 + row), dot = load(p.dot + q_at * 128 + row);
    const float q_unit = load(p.qp.units + q_at).x;
    const float2 g_unit = load(p.gp.units + q_at);
    // (a length whose squares are below 2^-126 is 0, from 1e-18 on it is too short by a factor of 1.6 at the most, and 2^15 has 2 to go)
    const float own = load(p.lengths + q_at * 128 + row), length = own < 1e15f && own > 1e-18f ? own : g_unit.y;
    bool ok = true;
    auto add_tile = [&](int j) {
      if (!mbar_wait(&bar->dq_full, j & 1, p.status, 0x311)) return false;
      tc_fence_after();
      add_columns<false>(mine + Shape::DQ_AT + half * OWN, acc, 1.f, before);
      return true;
    };
    float token = 0.f, k_next = 0.f;
    float2 v_next = make_float2(0.f, 0.f);
    auto look_at = [&](int j) {
      token = token_of(tokens, j * 64 + half * 32, p.tk);
      if (j < tiles) k_next = load(p.kp.units + k_at + j / 2).x, v_next = load(p.vp.units + k_at + j / 2);
    };
    look_at(0);
    for (int j = 0; j < tiles; ++j) {
      const int b = j & 1;
      const unsigned in = __ballot_sync(ALL, token != 0.f);
      const float k_unit = k_next;
      const float2 v_unit = v_next;
      look_at(j + 1);
      const int e = exponent_of_ds(length, v_unit.y, dot, k_unit);
      // (2^e is not in the exponent, whose rounding it would make coarser)
      const float f = power_of_two(e), s_unit = q_unit * k_unit, dp_unit = g_unit.x * f * v_unit.x, dot_unit = dot * f;
      if (!mbar_wait(&bar->s_full[b], j >> 1 & 1, p.status, 0x312)) { ok = false; break; }
      tc_fence_after();
      const uint32_t at = mine + Shape::S_AT + b * 64 + half * 32, dp_at = mine + Shape::DP_AT + b * 64 + half * 32;
      float s[2][16], dp[2][16];
      tmem_begin(at, s[0]);
      tmem_begin(dp_at, dp[0]);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        float(&v)[16] = s[w];
        float(&x)[16] = dp[w];
        tmem_ld_wait();
        tmem_arrived(v);
        tmem_arrived(x);
        if (w < 1) {
          tmem_begin(at + 16, s[1]);
          tmem_begin(dp_at + 16, dp[1]);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = exp2_fast(v[i] * s_unit - lse) * (x[i] * dp_unit - dot_unit);
        if (in != ALL) {
          const unsigned mask = in >> (w * 16);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = (mask >> i) & 1 ? v[i] : 0.f;
        }
        tmem_st_pieces(at + 16 * w, v);
      }
      tmem_st_wait();
      if (j > 0 && !(ok = add_tile(j - 1))) break;
      tc_fence_before();
      mbar_arrive(&bar->ds_full[b]);
      before = k_unit * power_of_two(-e);
    }
    if (ok && tiles > 0) ok = add_tile(tiles - 1);
    const int t = q0 + row;
    if (ok && t < p.tq)
      store_row(p.dq + ((long long)n * p.tq + t) * q_row + (long long)h * p.d + half * OWN, acc, p.scale, p.d - half * OWN, p.vec);
  } else {
    fewer_registers<88>();
    if (warp == 8 && elect_one()) {
      for (int i = 0; i < 2 * tiles; ++i) {
        const int j = i / 2, of_kind = i & 1 ? Shape::V_SLOTS : Shape::K_SLOTS, s = i & 1 ? Shape::K_SLOTS + j % Shape::V_SLOTS : j % Shape::K_SLOTS;
        if (i == 1 && !Shape::BOTH) copy_tile<D>(g_tile, p.gp, q_at, &bar->g_full);
        if (!mbar_wait(&bar->empty[s], (j / of_kind & 1) ^ 1, p.status, 0x313)) break;
        copy_half<D>(ring + s * LK::BYTES, i & 1 ? p.vp : p.kp, k_at + j / 2, j & 1, &bar->full[s]);
      }
    }
    if (warp == 9 && tiles > 0) {
      const uint32_t leader = elect_one();      // (as in attend: 472 -> 459 us with 128 columns)
      const uint32_t ga = smem_u32(g_tile), ra = smem_u32(ring);
      bool ok = mbar_wait(&bar->q_full, 0, p.status, 0x315);
      tc_fence_after();
      auto scores = [&](int j) {
        const int b = j & 1, ks = j % Shape::K_SLOTS, vs = Shape::K_SLOTS + j % Shape::V_SLOTS;
        if (!mbar_wait(&bar->full[ks], j / Shape::K_SLOTS & 1, p.status, 0x316)) return false;
        tc_fence_after();
        product_of_kept_rows<D, 64>(tmem + Shape::S_AT + b * 64, tmem, ra + ks * LK::BYTES, leader);
        if (!Shape::BOTH && j == 0 && !mbar_wait(&bar->g_full, 0, p.status, 0x315)) return false;
        if (!mbar_wait(&bar->full[vs], j / Shape::V_SLOTS & 1, p.status, 0x317)) return false;
        tc_fence_after();
        if (Shape::BOTH) product_of_kept_rows<D, 64>(tmem + Shape::DP_AT + b * 64, tmem + Shape::G_AT, ra + vs * LK::BYTES, leader);
        else product_of_rows<D, 128, 64>(tmem + Shape::DP_AT + b * 64, ga, ra + vs * LK::BYTES, leader);
        commit_if(leader, &bar->s_full[b]);
        commit_if(leader, &bar->empty[vs]);
        return true;
      };
      // (keys stay in their slot until dq is computed)
      for (int j = 0; j < 2 && j < tiles && ok; ++j) ok = scores(j);
      for (int j = 0; j < tiles && ok; ++j) {
        const int b = j & 1, ks = j % Shape::K_SLOTS;
        if (!(ok = mbar_wait(&bar->ds_full[b], j >> 1 & 1, p.status, 0x318))) break;
        tc_fence_after();
        product_with_columns<D, 64>(tmem + Shape::DQ_AT, tmem + Shape::S_AT + b * 64, ra + ks * LK::BYTES, leader);
        commit_if(leader, &bar->empty[ks]);
        commit_if(leader, &bar->dq_full);
        if (j + 2 < tiles) ok = scores(j + 2);
      }
      if (!ok && leader) drain(&bar->drained);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, TMEM_COLUMNS);
}

// dk and dv: a block takes 128 keys of a shared head and tiles of 64 queries of every head that reads it.  S^T and dP^T have
// the keys as rows, so P^T and dS^T are A operands as they lie.  Halves of the tiles of queries and of gradients share a ring
// of slots (q, g, q, g, ...), each with its rows' log-sum-exps or dots.  Warps 0 to 3 take the first 32 queries of a tile and
// add up dv, 4 to 7 the others and dk; 8: copies; 9 issues.  Two tiles of S^T and dP^T are in tensor memory; with 128 columns one
// of dP^T, and the keys' hi pieces in its place, so that shared memory has room for two tiles of queries and gradients (three
// halves and all pieces of the keys: 855 us in place of 665, a product and a copy more on the way from dS to the next dP).
// 4 x 2048 x 2048, 16 heads of 64: 360 us; 2 x 2000 x 4111, 16 heads of 128 on 4: 665 us, 405 TFLOP/s, so 1.21 PFLOP/s of fp16
// products.  (Two blocks of four such warps to an SM were a third slower, 516 us in place of 397 for the former: the two sums
// leave a thread no registers.  Keys and values of 64 columns in tensor memory: no quicker.)
template <int D> struct StateShape {
  static constexpr bool WIDE = D == 64;
  static constexpr int S_AT = WIDE ? 0 : 64, DP_AT = S_AT + 128, DP_BUFFERS = WIDE ? 2 : 1, DV_AT = 256, DK_AT = 384;
  static constexpr int SLOTS = WIDE ? 6 : 4;
  using LK = Tile<D, 128>;
  using LQ = Tile<D, 64>;
  static constexpr int K_BYTES = WIDE ? LK::BYTES : LK::PLANE, TILES = K_BYTES + LK::BYTES + SLOTS * LQ::BYTES;
  static constexpr int ROWS_AT = 256;            // of the slots' log-sum-exps and dots, behind the barriers
  static constexpr int SMEM = TILES + ROWS_AT + SLOTS * 256;
};
struct StateControl {
  uint64_t k_full, kept, v_full, full[6], empty[6], s_full[2], ds_full[2], sum_full, drained;
  uint32_t tmem;
};
static_assert(sizeof(StateControl) <= StateShape<64>::ROWS_AT, "");

template <int D>
__device__ __forceinline__ void grad_of_states(const Problem& p, const int block) {
  using Shape = StateShape<D>;
  using LQ = typename Shape::LQ;
  using LK = typename Shape::LK;
  constexpr bool WIDE = Shape::WIDE;
  constexpr int SLOTS = Shape::SLOTS;
  char *const k_tile = tiles_of_block, *const v_tile = k_tile + Shape::K_BYTES, *const ring = v_tile + LK::BYTES;
  StateControl* bar = control_at<StateControl>(Shape::TILES);
  float* const rows = reinterpret_cast<float*>(reinterpret_cast<char*>(bar) + Shape::ROWS_AT);        // [SLOTS][64]
  const int warp = __shfl_sync(ALL, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&bar->k_full, 1);
    mbar_init(&bar->kept, 256);
    mbar_init(&bar->v_full, 1);
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&bar->full[i], 1);
      mbar_init(&bar->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->ds_full[i], 256);
    }
    mbar_init(&bar->sum_full, 1);
    mbar_init(&bar->drained, 1);
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(&bar->tmem, 512);
    tmem_relinquish();
  }
  tsb_launch::enter();
  const int kt = block % p.ktiles, shared = block / p.ktiles % p.shared, n = block / p.ktiles / p.shared;
  const int k0 = kt * 128, per = p.heads / p.shared, halves = (p.tq + 63) / 64;
  const float* tokens = p.key ? p.key + (long long)n * p.tk : nullptr;
  const long long kv_row = 2ll * p.shared * p.d, k_at = ((long long)n * p.shared + shared) * p.ktiles + kt;
  const long long q_at = ((long long)n * p.heads + shared * per) * p.qtiles;                // of the first head that reads it
  const bool mine_in = threadIdx.x < 128 && k0 + (int)threadIdx.x < p.tk && (!tokens || load(tokens + k0 + threadIdx.x) != 0.f);
  const int half = warp >> 2, row = threadIdx.x & 127;
  KeptRow<D, 1> kept;                          // (under way while the block sets itself up)
  if (!WIDE && warp < 8) kept.read(p.kp, k_at, row, half);
  tc_fence_before();
  const int tiles = __syncthreads_or(mine_in) ? halves * per : 0;
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(ALL, bar->tmem, 0);
  auto tile_of = [&](int j) { return q_at + (long long)(j / halves) * p.qtiles + j % halves / 2; };

  if (warp < 8) {
    more_registers<208>();
    float acc[D], before = 0.f;
#pragma unroll
    for (int c = 0; c < D; ++c) acc[c] = 0.f;
    const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21);
    if (!WIDE) {
      kept.keep(mine, half);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&bar->kept);
    }
    const float k_unit = load(p.kp.units + k_at).x;
    const float2 v_unit = load(p.vp.units + k_at);
    bool ok = true;
    auto add_tile = [&](int j) {
      if (!mbar_wait(&bar->sum_full, j & 1, p.status, 0x322)) return false;
      tc_fence_after();
      add_columns<false>(mine + (half ? Shape::DK_AT : Shape::DV_AT), acc, 1.f, before);
      return true;
    };
    for (int j = 0; j < tiles; ++j) {
      const int b = j & 1, qs = 2 * j % SLOTS, gs = (2 * j + 1) % SLOTS;
      const long long t = tile_of(j);
      const float q_unit = load(p.qp.units + t).x;
      const float2 g_unit = load(p.gp.units + t);
      if (!mbar_wait(&bar->full[gs], (2 * j + 1) / SLOTS & 1, p.status, 0x321)) { ok = false; break; }
      if (!mbar_wait(&bar->full[qs], 2 * j / SLOTS & 1, p.status, 0x321)) { ok = false; break; }
      const float *const lse = rows + qs * 64, *const dots = rows + gs * 64;
      const uint32_t largest = max(__float_as_uint(fabsf(dots[lane])), __float_as_uint(fabsf(dots[lane + 32])));
      const int e = exponent_of_ds(g_unit.y, v_unit.y, __uint_as_float(__reduce_max_sync(ALL, largest)), q_unit);
      // p = 2^14 P, then dS = p (dP - dot) 2^(e - 14)
      const float s_unit = q_unit * k_unit, f = power_of_two(max(e - TOP - 1, -126)), dp_unit = g_unit.x * f * v_unit.x;
      if (!mbar_wait(&bar->s_full[b], j >> 1 & 1, p.status, 0x321)) { ok = false; break; }
      tc_fence_after();
      const uint32_t at = mine + Shape::S_AT + b * 64 + half * 32, dp_at = mine + Shape::DP_AT + b % Shape::DP_BUFFERS * 64 + half * 32;
      float s[2][16], dp[2][16];
      tmem_begin(at, s[0]);
      tmem_begin(dp_at, dp[0]);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        float(&v)[16] = s[w & 1];
        float(&x)[16] = dp[w & 1];
        tmem_ld_wait();
        tmem_arrived(v);
        tmem_arrived(x);
        if (w + 1 < 2) {
          tmem_begin(at + 16 * w + 16, s[(w + 1) & 1]);
          tmem_begin(dp_at + 16 * w + 16, dp[(w + 1) & 1]);
        }
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 a = *reinterpret_cast<const float4*>(lse + half * 32 + 16 * w + i);
          const float4 c = *reinterpret_cast<const float4*>(dots + half * 32 + 16 * w + i);
          const float as[4] = {a.x, a.y, a.z, a.w}, cs[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[i + k] = exp2_fast(v[i + k] * s_unit + (TOP + 1 - as[k]));
            x[i + k] = v[i + k] * (x[i + k] * dp_unit - cs[k] * f);
          }
        }
        tmem_st_pieces(at + 16 * w, v);
        tmem_st_pieces(dp_at + 16 * w, x);
      }
      tmem_st_wait();
      if (j > 0 && !(ok = add_tile(j - 1))) break;
      tc_fence_before();
      mbar_arrive(&bar->ds_full[b]);                              // (the sums of the tile before are in registers by now)
      before = half ? q_unit * power_of_two(-e) : g_unit.x * (1.f / LARGEST);
    }
    if (ok && tiles > 0) ok = add_tile(tiles - 1);
    if (ok && k0 + row < p.tk) {
      const bool in = !tokens || load(tokens + k0 + row) != 0.f;
      float* to = p.dkv + ((long long)n * p.tk + k0 + row) * kv_row + (long long)shared * p.d;
      if (!in)
#pragma unroll
        for (int c = 0; c < D; ++c) acc[c] = 0.f;
      // (q was scaled by scale * log2(e))
      store_row(half ? to : to + (long long)p.shared * p.d, acc, half ? LN2 : 1.f, p.d, p.vec);
    }
  } else {
    fewer_registers<88>();
    if (warp == 8 && elect_one() && tiles > 0) {
      mbar_expect_tx(&bar->k_full, Shape::K_BYTES);                // (the lo pieces are behind the hi ones)
      bulk_copy(k_tile, p.kp.tiles + (k_at + 1) * LK::BYTES - Shape::K_BYTES, Shape::K_BYTES, &bar->k_full);
      for (int i = 0; i < 2 * tiles; ++i) {
        const int s = i % SLOTS, j = i / 2;
        const long long t = tile_of(j);
        const int h = j % halves % 2;
        if (!mbar_wait(&bar->empty[s], (i / SLOTS & 1) ^ 1, p.status, 0x323)) break;
        copy_half<D>(ring + s * LQ::BYTES, i & 1 ? p.gp : p.qp, t, h, &bar->full[s], 256);
        bulk_copy(reinterpret_cast<char*>(rows + s * 64), reinterpret_cast<const char*>((i & 1 ? p.dot : p.lse) + t * 128 + h * 64), 256,
                  &bar->full[s]);
        if (i == 0) copy_tile<D>(v_tile, p.vp, k_at, &bar->v_full);
      }
    }
    if (warp == 9 && elect_one() && tiles > 0) {
      constexpr uint32_t leader = 1;             // (64 columns: 354 us so, 394 if all lanes take part)
      const uint32_t ra = smem_u32(ring), ka = smem_u32(k_tile), va = smem_u32(v_tile);
      bool ok = mbar_wait(&bar->k_full, 0, p.status, 0x324) && (WIDE || mbar_wait(&bar->kept, 0, p.status, 0x324));
      // S^T or dP^T of tile j; the latter commits both
      auto half_of_scores = [&](int j, int half) {
        const int i = 2 * j + half, s = i % SLOTS, b = j & 1;
        if (i == 1 && !mbar_wait(&bar->v_full, 0, p.status, 0x324)) return false;
        if (!mbar_wait(&bar->full[s], i / SLOTS & 1, p.status, 0x325)) return false;
        tc_fence_after();
        const uint32_t to = tmem + (half ? Shape::DP_AT + b % Shape::DP_BUFFERS * 64 : Shape::S_AT + b * 64), from = ra + s * LQ::BYTES;
        if (!WIDE && !half) product_of_half_kept_rows<D, 128, 64>(to, tmem, ka, from, leader);
        else product_of_rows<D, 128, 64>(to, half ? va : ka, from, leader);
        if (half) commit_if(leader, &bar->s_full[b]);
        return true;
      };
      // (with one buffer of dP^T that of tile 1 waits for dk of tile 0)
      for (int i = 0; i < (WIDE ? 4 : 3) && i < 2 * tiles && ok; ++i) ok = half_of_scores(i / 2, i & 1);
      for (int j = 0; j < tiles && ok; ++j) {
        const int b = j & 1, qs = 2 * j % SLOTS, gs = (2 * j + 1) % SLOTS;
        if (!(ok = mbar_wait(&bar->ds_full[b], j >> 1 & 1, p.status, 0x326))) break;
        tc_fence_after();
        product_with_columns<D, 64>(tmem + Shape::DK_AT, tmem + Shape::DP_AT + b % Shape::DP_BUFFERS * 64, ra + qs * LQ::BYTES, leader);
        commit_if(leader, &bar->empty[qs]);
        if (!WIDE && j + 1 < tiles && !(ok = half_of_scores(j + 1, 1))) break;
        product_with_columns<D, 64>(tmem + Shape::DV_AT, tmem + Shape::S_AT + b * 64, ra + gs * LQ::BYTES, leader);
        commit_if(leader, &bar->empty[gs]);
        commit_if(leader, &bar->sum_full);
        if (j + 2 < tiles) ok = half_of_scores(j + 2, 0) && (!WIDE || half_of_scores(j + 2, 1));
      }
      if (!ok) drain(&bar->drained);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

// The first `query_blocks` blocks compute gradients of queries, the others those of states.  Neither reads what the other writes, so
// in one launch the latter take the SMs that the last of the former leave idle (32 x 255 x 256, 8 heads of 64: 75 us, two
// launches 84; 1 x 512 x 512, 4 heads: 16.5 and 27.7).  Two kernels, the second of which does not wait for the
// first, would need what stands before the first to be visible to a grid that has waited for nobody, which nothing promises.
template <int D> constexpr int gradients_smem() {
  return QueryShape<D>::SMEM > StateShape<D>::SMEM ? QueryShape<D>::SMEM : StateShape<D>::SMEM;
}
template <int D>
__global__ void __launch_bounds__(BLOCK, 1) gradients(const Problem p) {
  const int block = blockIdx.x;
  if (block < p.query_blocks) grad_of_queries<D>(p, block);
  else grad_of_states<D>(p, block - p.query_blocks);
}

// ------------------------------------------------------------------------------------------------ single tokens
// Up to ROWS queries that read one shared head (H / G heads x Tq tokens): bound by reading keys and values once, so plain
// fp32.  A group of D / 4 threads takes four keys at a time, four columns a thread, and keeps a soft-max of its own; a thread
// reads from shared memory only what it had copied there itself, three such steps deep, so nobody waits for anybody until
// the end.  The 4 x ROWS dots of a step are added up over the group by halves: a thread sends half of its sums and keeps the
// other half, until each holds one score, computes one exponential, and hands it to the others.  At the end the groups of a
// block join through shared memory.  A long sentence is shared by as many blocks as leave two to every SM, and join_parts adds
// up what they found (clusters of 8 or 16 that join through distributed shared memory do not spread over all SMs: 97 and 81 us
// for the states below, 16 heads).
// (4 x 16384 x 4 x 128 states, four rows each: registers and an all-reduce for every dot 182 us; tiles that the block shares,
// with three barriers 136, with one 156.)
constexpr int FEW_WARPS = 8, FEW_STAGES = 3, STEP = 4;
template <int D, int ROWS> struct FewShape {
  static constexpr int LANES = D / 4, GROUPS = FEW_WARPS * 32 / LANES, KEYS = GROUPS * STEP;
  static constexpr int HELD = STEP * ROWS > LANES ? STEP * ROWS / LANES : 1;       // scores a thread ends up with, rows of one key
  static constexpr int APART = LANES * HELD / (STEP * ROWS);                       // threads from one of these to the next
  static constexpr int RING = FEW_STAGES * 2 * STEP * FEW_WARPS * 32 * 4;
  // the ring, in its place later y of the groups [GROUPS][ROWS][D]; their maxima and sums
  static constexpr int FLOATS = RING + 2 * GROUPS * ROWS;
  static_assert(GROUPS * ROWS * D <= RING, "the sums of the groups take the place of the ring");
};

// 16 bytes, or zeros where nothing is to be read; `vec`: both sides on 16-byte boundaries
__device__ __forceinline__ void copy_piece(float* to, const float* from, int count, bool vec) {
  if (vec) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(count > 0 ? 16 : 0) : "memory");
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(to + k)), "l"(count > k ? from + k : from), "r"(count > k ? 4 : 0)
                   : "memory");
  }
}

// Cell i of the rows [ROWS][D] that read a shared head: y, and the row's log-sum-exp with its first column.
template <int D> __device__ __forceinline__ void store_cell(const Problem& p, int n, int shared, int i, float top, float total, float sum) {
  const int r = i / D, c = i % D, per = p.heads / p.shared, t = r / per, h = shared * per + r % per;
  if (t >= p.tq) return;
  if (c < p.d) p.y[(((long long)n * p.tq + t) * p.heads + h) * p.d + c] = total != 0.f ? sum / total : 0.f;
  if (c == 0) p.lse[((long long)n * p.heads + h) * 128 + t] = total != 0.f ? top + log2f(total) : -NEG_INF;
}

template <int D, int ROWS>
__global__ void __launch_bounds__(FEW_WARPS * 32, 2) attend_few(const Problem p, int split, float* __restrict__ parts) {
  tsb_launch::enter();
  using S = FewShape<D, ROWS>;
  constexpr int LANES = S::LANES, GROUPS = S::GROUPS, KEYS = S::KEYS, HELD = S::HELD, THREADS = FEW_WARPS * 32;
  float* const ring = reinterpret_cast<float*>(tiles_of_block);
  float *const maxima = ring + S::RING, *const totals = maxima + GROUPS * ROWS;
  const int part = blockIdx.x % split, shared = blockIdx.x / split % p.shared, n = blockIdx.x / split / p.shared;
  const int tid = threadIdx.x, group = tid / LANES, c = tid % LANES * 4, base = tid & 31 & ~(LANES - 1);
  const int per = p.heads / p.shared, rows = per * p.tq;
  const float* tokens = p.key ? p.key + (long long)n * p.tk : nullptr;
  const long long kv_row = 2ll * p.shared * p.d, q_row = (long long)p.heads * p.d, values = (long long)p.shared * p.d;
  const float* k_base = p.kv + (long long)n * p.tk * kv_row + (long long)shared * p.d + c;
  float4 q[ROWS], o[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {                     // row r: query r / per of head r % per
    const float* at = p.q + ((long long)n * p.tq + r / per) * q_row + (long long)(shared * per + r % per) * p.d + c;
    float x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = r < rows && c + k < p.d ? load(at + k) * (p.scale * LOG2E) : 0.f;
    q[r] = make_float4(x[0], x[1], x[2], x[3]);
    o[r] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // (rows behind the last query, of the one tile of each head: see attend)
  for (int i = part * THREADS + tid; i < per * 128; i += split * THREADS)
    if (i % 128 >= p.tq) p.lse[((long long)n * p.heads + shared * per + i / 128) * 128 + i % 128] = -NEG_INF;

  const int share = (p.tk + split - 1) / split, begin = min(part * share, p.tk), end = min(begin + share, p.tk);
  const int count = (end - begin + KEYS - 1) / KEYS;
  float token[STEP];                                   // of the step that is copied next, read a step ahead
  auto read_tokens = [&](int j) {
#pragma unroll
    for (int u = 0; u < STEP; ++u) {
      const int t = begin + j * KEYS + group * STEP + u;
      token[u] = t < end ? (tokens ? load(tokens + t) : 1.f) : 0.f;
    }
  };
  unsigned in[FEW_STAGES] = {};                        // which of the four keys are in, of this step and those behind it
  auto copy = [&](int j) {
    unsigned mask = 0;
    if (j < count) {
      float* const to = ring + (j % FEW_STAGES * 2 * STEP * THREADS + tid) * 4;
      const float* const from = k_base + (begin + j * KEYS + group * STEP) * kv_row;
#pragma unroll
      for (int u = 0; u < STEP; ++u) {
        const bool is = token[u] != 0.f;
        const int numbers = is ? p.d - c : 0;
        mask |= (unsigned)is << u;
        copy_piece(to + u * THREADS * 4, numbers > 0 ? from + u * kv_row : p.kv, numbers, p.vec);
        copy_piece(to + (STEP + u) * THREADS * 4, numbers > 0 ? from + u * kv_row + values : p.kv, numbers, p.vec);
      }
      read_tokens(j + 1);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    return mask;
  };
  read_tokens(0);
#pragma unroll
  for (int j = 0; j < FEW_STAGES - 1; ++j) in[j] = copy(j);
  // This thread's scores: of key `u` of a step, rows r0 to r0 + HELD - 1
  const int place = (tid & (LANES - 1)) / S::APART, u = place / (ROWS / HELD), r0 = place % (ROWS / HELD) * HELD;
  float m[HELD], l[HELD];
#pragma unroll
  for (int i = 0; i < HELD; ++i) m[i] = NEG_INF, l[i] = 0.f;
  for (int j = 0; j < count; ++j) {
    in[FEW_STAGES - 1] = copy(j + FEW_STAGES - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(FEW_STAGES - 1) : "memory");
    const float4* const at = reinterpret_cast<const float4*>(ring) + j % FEW_STAGES * 2 * STEP * THREADS + tid;
    float x[STEP * ROWS];
#pragma unroll
    for (int k = 0; k < STEP; ++k) {
      const float4 v = at[k * THREADS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) x[k * ROWS + r] = q[r].x * v.x + q[r].y * v.y + q[r].z * v.z + q[r].w * v.w;
    }
#pragma unroll
    for (int off = LANES / 2, left = STEP * ROWS; off > 0; off >>= 1) {
      if (left > 1) {
        left /= 2;
#pragma unroll
        for (int i = 0; i < STEP * ROWS / 2; ++i) {
          if (i >= left) break;
          const bool upper = tid & off;
          const float send = upper ? x[i] : x[i + left], keep = upper ? x[i + left] : x[i];
          x[i] = keep + __shfl_xor_sync(ALL, send, off);
        }
      } else {
        x[0] += __shfl_xor_sync(ALL, x[0], off);
      }
    }
    float factor[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      if (!(in[0] >> u & 1)) x[i] = NEG_INF;
      float top = fmaxf(x[i], __shfl_xor_sync(ALL, x[i], LANES / 2));              // (the two highest places tell the key)
      top = fmaxf(m[i], fmaxf(top, __shfl_xor_sync(ALL, top, LANES / 4)));
      const float ref = top == NEG_INF ? 0.f : top;
      factor[i] = exp2_fast(m[i] - ref);
      x[i] = exp2_fast(x[i] - ref);
      l[i] = l[i] * factor[i] + x[i];
      m[i] = top;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float f = __shfl_sync(ALL, factor[r % HELD], base + r / HELD * S::APART);
      o[r] = make_float4(o[r].x * f, o[r].y * f, o[r].z * f, o[r].w * f);
    }
#pragma unroll
    for (int k = 0; k < STEP; ++k) {
      const float4 v = at[(STEP + k) * THREADS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float e = __shfl_sync(ALL, x[r % HELD], base + (k * (ROWS / HELD) + r / HELD) * S::APART);
        o[r].x += e * v.x; o[r].y += e * v.y; o[r].z += e * v.z; o[r].w += e * v.w;
      }
    }
#pragma unroll
    for (int i = 0; i < FEW_STAGES - 1; ++i) in[i] = in[i + 1];
  }
  // the groups of the block
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    l[i] += __shfl_xor_sync(ALL, l[i], LANES / 2);
    l[i] += __shfl_xor_sync(ALL, l[i], LANES / 4);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROWS; ++r) *reinterpret_cast<float4*>(ring + (group * ROWS + r) * D + c) = o[r];
  if (u == 0 && (tid & (LANES - 1)) % S::APART == 0)
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      maxima[group * ROWS + r0 + i] = m[i];
      totals[group * ROWS + r0 + i] = l[i];
    }
  __syncthreads();
  constexpr int CELLS = ROWS * D;
  for (int i = tid; i < CELLS; i += THREADS) {
    const int r = i / D;
    float top = NEG_INF, total = 0.f, sum = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) top = fmaxf(top, maxima[g * ROWS + r]);
    const float ref = top == NEG_INF ? 0.f : top;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const float f = exp2_fast(maxima[g * ROWS + r] - ref);
      total += totals[g * ROWS + r] * f;
      sum += ring[g * CELLS + i] * f;
    }
    if (split == 1) {
      store_cell<D>(p, n, shared, i, top, total, sum);
    } else {
      float* const to = parts + (long long)blockIdx.x * ROWS * (D + 2);
      to[i] = sum;
      if (i % D == 0) to[CELLS + 2 * r] = top, to[CELLS + 2 * r + 1] = total;
    }
  }
}

// 64 cells of the rows that read a shared head: the parts of its keys, in their order.
template <int D, int ROWS>
__global__ void __launch_bounds__(64) join_parts(const Problem p, int split, const float* parts) {
  tsb_launch::enter();
  constexpr int CELLS = ROWS * D, BLOCKS = (CELLS + 63) / 64;
  const int pair = blockIdx.x / BLOCKS, i = blockIdx.x % BLOCKS * 64 + threadIdx.x, r = i / D;
  if (i >= CELLS) return;
  const float* const from = parts + (long long)pair * split * ROWS * (D + 2);
  float top = NEG_INF, total = 0.f, sum = 0.f;
#pragma unroll 8
  for (int b = 0; b < split; ++b) top = fmaxf(top, load(from + b * ROWS * (D + 2) + CELLS + 2 * r));
  const float ref = top == NEG_INF ? 0.f : top;
#pragma unroll 8
  for (int b = 0; b < split; ++b) {
    const float* const at = from + b * ROWS * (D + 2);
    const float f = exp2_fast(load(at + CELLS + 2 * r) - ref);
    total += load(at + CELLS + 2 * r + 1) * f;
    sum += load(at + i) * f;
  }
  store_cell<D>(p, pair / p.shared, pair % p.shared, i, top, total, sum);
}

// ------------------------------------------------------------------------------------------------ host side
int launched(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  else cudaGetLastError();
  if (e != cudaSuccess) return TSB_ERR_LAUNCH | ((int)e << 8);
  const int late = tsb_host::peek_status();
  return late ? TSB_ERR_TIMEOUT | (late << 8) : TSB_OK;
}

constexpr int MAX_DIM = 128, FEW_ROWS = 8, MAX_ROWS = INT32_MAX - 65536;      // (room to round up and look ahead in 32 bits)

// False: not a problem that the kernels take.  `vec` holds for all arrays given.
template <class... A>
bool describe(Problem& p, int n, int tq, int tk, int heads, int shared, int d, float scale, const float* q, const float* kv,
              const float* key, A... others) {
  if (n < 0 || tq < 0 || tk < 0 || heads <= 0 || shared <= 0 || heads % shared || d <= 0 || d > MAX_DIM) return false;
  if (tq > MAX_ROWS || tk > MAX_ROWS) return false;
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
int run(K kernel, const Problem& p, long long blocks, int smem, cudaStream_t st, tsb_launch::SmemLimit& limit) {
  if (blocks > INT32_MAX) return TSB_ERR_ARG;
  Problem q = p;
  q.status = tsb_host::status_word(st);
  if (!q.status) return TSB_ERR_LAUNCH;
  cudaError_t e = limit.raise(kernel, smem);
  if (e == cudaSuccess) e = tsb_launch::launch(kernel, dim3((unsigned)blocks), dim3(BLOCK), smem, st, q);
  return launched(e);
}

// Where the pieces of q, k, v and g lie in one buffer, behind them the units, and the dots and the lengths of the rows of g.
struct Layout {
  size_t tiles[4], units[4], dots, lengths, bytes;             // (units and dots on 16-byte boundaries: they are copied in bulk)
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
      bytes += (count[i] * 8 + 15) / 16 * 16;
    }
    dots = bytes;
    lengths = dots + count[3] * 128 * 4;
    bytes = lengths + count[3] * 128 * 4;
  }
  Pieces of(const char* base, int i) const { return {base + tiles[i], reinterpret_cast<const float2*>(base + units[i])}; }
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
  p.lengths = reinterpret_cast<const float*>(base + at.lengths);
}

// Splits q, k and v where they are given, and g (with the dots).
int split(const Problem& p, const float* g, const float* y, const Layout& at, char* base, cudaStream_t st, bool states = true) {
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
    s.units = reinterpret_cast<float2*>(base + at.units[i]);
    if (i == 3) {
      s.with = y;
      s.dots = reinterpret_cast<float*>(base + at.dots);
      s.lengths = reinterpret_cast<float*>(base + at.lengths);
    }
    all.first[i] = (int)blocks;
    if (i < 3 ? states : g != nullptr) blocks += (long long)p.n * s.heads * s.count;
    if (blocks > INT32_MAX) return TSB_ERR_ARG;
  }
  all.first[4] = (int)blocks;
  if (blocks == 0) return TSB_OK;
  return launched(p.d <= 64 ? tsb_launch::launch(split_tiles<64>, dim3((unsigned)blocks), dim3(256), 0, st, all)
                            : tsb_launch::launch(split_tiles<128>, dim3((unsigned)blocks), dim3(256), 0, st, all));
}

template <int D, int ROWS> int run_few(const Problem& p, cudaStream_t st) {
  using S = FewShape<D, ROWS>;
  constexpr int SMEM = S::FLOATS * 4;
  // two blocks to an SM, of eight steps each at least (a block's beginning and end, and the join, cost about as much)
  const long long pairs = (long long)p.n * p.shared, room = 148 * 2 / pairs, steps = (p.tk + S::KEYS - 1) / S::KEYS;
  int split = (int)(room < steps / 8 ? room : steps / 8);
  if (split < 1) split = 1;
  if (pairs * split > INT32_MAX) return TSB_ERR_ARG;
  float* parts = nullptr;
  if (split > 1) {
    parts = static_cast<float*>(tsb_scratch::get(st, tsb_scratch::ATTENTION_PARTS, (size_t)(pairs * split) * ROWS * (D + 2) * 4));
    if (!parts) return TSB_ERR_OOM;
  }
  static tsb_launch::SmemLimit limit;
  cudaError_t e = limit.raise(attend_few<D, ROWS>, SMEM);
  if (e == cudaSuccess)
    e = tsb_launch::launch(attend_few<D, ROWS>, dim3((unsigned)(pairs * split)), dim3(FEW_WARPS * 32), SMEM, st, p, split, parts);
  if (e == cudaSuccess && split > 1)
    e = tsb_launch::launch(join_parts<D, ROWS>, dim3((unsigned)pairs * ((ROWS * D + 63) / 64)), dim3(64), 0, st, p, split, parts);
  return launched(e);
}
template <int D> int few(const Problem& p, int rows, cudaStream_t st) {
  if (rows <= 1) return run_few<D, 1>(p, st);
  if (rows <= 2) return run_few<D, 2>(p, st);
  if (rows <= 4) return run_few<D, 4>(p, st);
  return run_few<D, 8>(p, st);
}

int forward(const float* q, const float* kv, const float* key, float* y, float* lse, void* prepared, long long have, int n, int tq, int tk, int heads,
            int shared, int d, float scale, void* stream) {
  Problem p;
  if (!describe(p, n, tq, tk, heads, shared, d, scale, q, kv, key, y)) return TSB_ERR_ARG;
  if (n == 0 || tq == 0) return TSB_OK;
  if (!q || !y || !lse || (tk && !kv)) return TSB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  p.y = y;
  p.lse = lse;
  const long long rows = (long long)(heads / shared) * tq;
  const Layout at(n, tq, tk, heads, shared, d, prepared != nullptr);
  char* pieces = static_cast<char*>(prepared);
  if (prepared) {
    if (rows <= FEW_ROWS || !fits(prepared, have, at)) return TSB_ERR_ARG;
  } else {
    if (rows <= FEW_ROWS) return d <= 32 ? few<32>(p, (int)rows, st) : d <= 64 ? few<64>(p, (int)rows, st) : few<128>(p, (int)rows, st);
    pieces = static_cast<char*>(tsb_scratch::get(st, tsb_scratch::ATTENTION_PIECES, at.bytes));
    if (!pieces) return TSB_ERR_OOM;
  }
  use(p, at, pieces);
  const int rc = split(p, nullptr, nullptr, at, pieces, st);
  if (rc) return rc;
  const long long blocks = (long long)n * heads * p.qtiles;
  static tsb_launch::SmemLimit limit64, limit128;
  if (d <= 64) return run(attend<64>, p, blocks, ForwardShape<64>::SMEM, st, limit64);
  return run(attend<128>, p, blocks, ForwardShape<128>::SMEM, st, limit128);
}

// The gradients that are asked for: of the queries (dq), of the states (dkv), or both.
int grads(const void* prepared, long long have, const float* key, const float* lse, float* dq, float* dkv, int n, int tq, int tk, int heads, int shared,
          int d, float scale, void* stream) {
  Problem p;
  if (!describe(p, n, tq, tk, heads, shared, d, scale, nullptr, nullptr, key, dq, dkv)) return TSB_ERR_ARG;
  const long long queries = dq ? (long long)n * heads * p.qtiles : 0, states = dkv ? (long long)n * shared * p.ktiles : 0;
  if (queries + states == 0) return TSB_OK;
  const Layout at(n, tq, tk, heads, shared, d, true);
  if ((tq && !lse) || (reinterpret_cast<uintptr_t>(lse) & 15) || !fits(prepared, have, at)) return TSB_ERR_ARG;
  if ((long long)((tq + 63) / 64) * (heads / shared) > INT32_MAX / 2) return TSB_ERR_ARG;
  if (queries > INT32_MAX || queries + states > INT32_MAX) return TSB_ERR_ARG;
  use(p, at, static_cast<const char*>(prepared));
  p.lse = const_cast<float*>(lse);
  p.dq = dq;
  p.dkv = dkv;
  p.query_blocks = (int)queries;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  static tsb_launch::SmemLimit limit64, limit128;
  if (d <= 64) return run(gradients<64>, p, queries + states, gradients_smem<64>(), st, limit64);
  return run(gradients<128>, p, queries + states, gradients_smem<128>(), st, limit128);
}

}  // namespace

extern "C" {

// y [N, Tq, H, d], and lse [N, H, Tq up to a multiple of 128]: log2 of the sum of the keys' 2^S, +inf for a query without keys
// and behind the last one.  key may be null.
int tsb_cross_attention(const float* q, const float* kv, const float* key, float* y, float* lse, int n, int tq, int tk, int heads,
                        int shared, int d, float scale, void* stream) {
  return forward(q, kv, key, y, lse, nullptr, 0, n, tq, tk, heads, shared, d, scale, stream);
}

// The same where the gradients follow, of more than FEW_ROWS rows to a shared head: the pieces of q, k and v stay in `prepared`, to
// which tsb_cross_attention_prepare_g adds those of g.  (32 x 255 x 256, 8 heads of 64, with the gradients: 149 us a step in place of
// 167.)
int tsb_cross_attention_keep(const float* q, const float* kv, const float* key, float* y, float* lse, void* prepared, long long have, int n, int tq,
                             int tk, int heads, int shared, int d, float scale, void* stream) {
  return prepared ? forward(q, kv, key, y, lse, prepared, have, n, tq, tk, heads, shared, d, scale, stream) : TSB_ERR_ARG;
}

int tsb_cross_attention_prepare_g(const float* g, const float* y, void* prepared, long long have, int n, int tq, int tk, int heads, int shared, int d,
                                  void* stream) {
  Problem p;
  if (!describe(p, n, tq, tk, heads, shared, d, 1.f, nullptr, nullptr, nullptr, g, y)) return TSB_ERR_ARG;
  if (n == 0) return TSB_OK;
  const Layout at(n, tq, tk, heads, shared, d, true);
  if ((tq && (!g || !y)) || !fits(prepared, have, at)) return TSB_ERR_ARG;
  return split(p, g, y, at, static_cast<char*>(prepared), static_cast<cudaStream_t>(stream), false);
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
  if (!dq && n > 0 && tq > 0) return TSB_ERR_ARG;
  return grads(prepared, have, key, lse, dq, nullptr, n, tq, tk, heads, shared, d, scale, stream);
}

int tsb_cross_attention_grad_kv(const void* prepared, long long have, const float* key, const float* lse, float* dkv, int n, int tq, int tk, int heads,
                                int shared, int d, float scale, void* stream) {
  if (!dkv && n > 0 && tk > 0) return TSB_ERR_ARG;
  return grads(prepared, have, key, lse, nullptr, dkv, n, tq, tk, heads, shared, d, scale, stream);
}

// Both, in one launch.
int tsb_cross_attention_grads(const void* prepared, long long have, const float* key, const float* lse, float* dq, float* dkv, int n, int tq, int tk,
                              int heads, int shared, int d, float scale, void* stream) {
  if ((!dq && n > 0 && tq > 0) || (!dkv && n > 0 && tk > 0)) return TSB_ERR_ARG;
  return grads(prepared, have, key, lse, dq, dkv, n, tq, tk, heads, shared, d, scale, stream);
}

}  // extern "C"
