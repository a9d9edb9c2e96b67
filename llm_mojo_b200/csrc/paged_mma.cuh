// paged_mma.cuh -- attention of one new token over a paged cache on the
// tensor cores, split over positions and joined.
//
// One pass over the cache: scores S^T = K Q^T, running maximum M and sum L
// of 2^(s - M), and O^T = V^T P^T, as m16n8k16 products with float32
// accumulators. Positions, and then dimensions, are the 16 rows; the 8
// columns are up to 4 query heads of one kv head, two terms each: a float32
// factor x enters as a sum of 16-bit terms, so that products keep float32's
// accuracy,
//   int8:     x 2^e = f16 + f16 (22 bits; codes are exact in f16),
//   bfloat16: x = bf16 + bf16 + bf16 by truncation (all 24 bits), the third
//             terms as 8 more columns,
//   float32:  both factors in three bf16 terms; of the nine products the
//             cache's second and third term with the other factor's third
//             are left out, 2^-24 of the whole at most (with the former 8 x
//             <=8192, 32 heads on 8 of 128, takes 110 us instead of 98).
// Scores are summed in the product's own accumulators, which truncate: up to
// 8 in a row. What these choices cost stays below float32's own roundings:
// root mean square errors against 64 bits, 64 x 200, 12 heads of 64, are
// 4.7e-8 / 2.8e-8 / 3.5e-8 of the largest output (int8 / bfloat16 / float32;
// 3.2e-8 with that product kept), in plain float32 10.0 / 5.9 / 6.4e-8.
// A lane's accumulators are the terms of one head, so they add up in place,
// and few query heads still fill the columns with what accuracy needs. P goes
// from the accumulators' layout to the operand's by one transposing move per
// 8x8 block.
//
// Both products may take dimensions in any order that their two operands
// share. A warp copies its tiles of 16 rows of K and of V (cp.async, 16-byte
// pieces) into its own ring in shared memory, rows padded by 16 bytes, so
// that ldmatrix reads them without bank conflicts: K as it lies (a lane's 4
// bytes of row lane / 4), V transposed (a pair of rows). For int8 the
// transposed element is a pair of codes, which one byte permute each turns
// into two operands. Copies in flight cost no registers, and warps wait for
// nothing but their own copies. (Rows permuted by exclusive-or instead of
// padded: grouped bfloat16 126 us against 105; 8-byte copies into per-lane
// slots, without ldmatrix: L1 at 77% and 157 us.)
//
// mma.sync, not tcgen05: a new token brings 8 columns to a row of the cache,
// and the tensor pipe is 15-18% busy while memory is the limit; tcgen05 would
// want the rows as 16-bit tiles in shared memory, so int8 codes converted,
// written back and read again.
//
// What bounds it (B200, device times; the copy rate is 6.53 TB/s): bytes in
// long calls, 8 sequences x <=32768 positions, 32 heads on 8 of 128, bfloat16:
// 99 us, 5.3 TB/s (104 with the weights); one sequence x 131071, 12 heads of 64, int8: 48 us, 4.4
// TB/s, of which about 9 us are the start and the join of the chunks (524288
// positions: 164 us, 5.2 TB/s), and 246 instructions per 16 positions, start
// and join among them, fill 57% of the issue slots; latency and those
// instructions (61%) in batches of short sequences, 256 x <=256, 12 heads of
// 64, int8: 18 us, 3.1 TB/s; the latency of one CTA in the smallest, 1 x 200:
// 3.9 us.
#pragma once

#include "paged.cuh"

namespace llmq {

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The first products of a sum.
__device__ __forceinline__ void mma_f16_from0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_bf16_from0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void pm_copy16(unsigned dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void pm_copy4(unsigned dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// Four 8x8 matrices of 16-bit elements; lane 8 m + i gives row i of matrix m.
template <bool TRANS>
__device__ __forceinline__ void pm_ldmatrix(uint32_t *d, unsigned src) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(src)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(src)
                 : "memory");
}
// The transpose of an 8x8 matrix of 16-bit elements, lane (g, t) holding row
// g's elements 2t, 2t + 1.
__device__ __forceinline__ uint32_t pm_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float pm_read1(unsigned src) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(src) : "memory");
  return v;
}

// Two f16 from two biased codes (code ^ 0x80) in bytes i and j of x: 1024 +
// byte, less 1152; all exact. (Keys as subnormals with the bias taken from
// the accumulator's start: 3% faster, 25% less accurate; values that way
// would lose the low bits of sums that nearly cancel.)
__device__ __forceinline__ uint32_t codes_f16(uint32_t x, uint32_t sel) {
  const uint32_t h = __byte_perm(x, 0x64646464u, sel), off = 0x64806480u;
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(off));
  return r;
}

// x, y as two f16 terms each: hi = (f16 x, f16 y), lo = the rest.
__device__ __forceinline__ void split_f16(float x, float y, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *(const uint32_t *)&h;
  lo = *(const uint32_t *)&l;
}

// x, y as three bf16 terms each by truncation, exact: 8 + 8 + 8 bits. t0 =
// (first of x, first of y), and so on.
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t &t0, uint32_t &t1, uint32_t &t2) {
  const uint32_t x0 = __float_as_uint(x) & 0xffff0000u, y0 = __float_as_uint(y) & 0xffff0000u;
  const float xr = x - __uint_as_float(x0), yr = y - __uint_as_float(y0);
  const uint32_t x1 = __float_as_uint(xr) & 0xffff0000u, y1 = __float_as_uint(yr) & 0xffff0000u;
  const float xs = xr - __uint_as_float(x1), ys = yr - __uint_as_float(y1);
  t0 = __byte_perm(x0, y0, 0x7632);
  t1 = __byte_perm(x1, y1, 0x7632);
  t2 = __byte_perm(__float_as_uint(xs), __float_as_uint(ys), 0x7632);
}

// One x: (first, second) and (third, 0).
__device__ __forceinline__ void split_bf16_one(float x, uint32_t &t01, uint32_t &t2) {
  const uint32_t x0 = __float_as_uint(x) & 0xffff0000u;
  const float r = x - __uint_as_float(x0);
  const uint32_t x1 = __float_as_uint(r) & 0xffff0000u;
  t01 = (x0 >> 16) | x1;
  t2 = __float_as_uint(r - __uint_as_float(x1)) >> 16;
}

enum { PM_I8 = 0, PM_BF16 = 1, PM_F32 = 2 };
template <int KIND, int D, int W>
struct PmShape {
  static constexpr int kEs = KIND == PM_I8 ? 1 : KIND == PM_BF16 ? 2 : 4;
  static constexpr int kRow = D * kEs, kNc = kRow / 16;  // bytes and 16-byte pieces of a row
  static constexpr int kPad = kRow + 16;                 // a row in the ring: an odd number of pieces
  static constexpr int kSteps = D / 16;  // steps of the scores; and tiles of dimensions of the output
  // tiles of 16 positions taken together: two while their operands fit in
  // registers (one in the one-warp CTAs, more of which an SM then holds: 3% on
  // 256 x <=256)
  static constexpr int kU = kRow <= 128 && W > 1 ? 2 : 1;
  // a stage of a warp's ring, for each tile: 16 rows of K, 16 of V, and (int8) their scales
  static constexpr int kVat = 16 * kPad, kSat = 32 * kPad, kTile = kSat + (KIND == PM_I8 ? 128 : 0);
  static constexpr int kStage = kU * kTile;
  // stages: one read, the others in flight, 5 KB or more per warp
  static constexpr int kStages = kStage <= 2560 ? 4 : kStage <= 4096 ? 3 : 2;
  static constexpr int kBlock = 16 * kU * W;  // positions that the CTA's warps take together
  static constexpr int kRun = 4096;           // positions whose rows are looked up at a time
  // Dimension of a lane's element u of the operand of step k: where ldmatrix
  // puts 4 codes, a pair of bfloat16 twice, or a float32 four times.
  static __device__ __forceinline__ int kdim(int k, int u, int t) {
    return 16 * k + (KIND == PM_I8 ? 4 * t + u : KIND == PM_BF16 ? (u >> 1) * 8 + 2 * t + (u & 1) : 4 * u + t);
  }
  // Dimension of row g (half 0) or g + 8 (half 1) of output tile j.
  static __device__ __forceinline__ int vdim(int j, int half, int g) {
    return 16 * j + (KIND == PM_I8 ? 2 * g + half : 8 * half + g);
  }
};

// Dynamic shared memory: the rows of a run's tiles (page_size % 16 == 0) or
// of its positions; then the rings, and in their place, at the end, the warps' states, and the join's factors.
constexpr int kPmJoin = 128;  // chunks of a unit at most
template <int KIND, int D, int W>
__host__ __device__ constexpr int pm_rows_bytes(bool fast) {
  return PmShape<KIND, D, W>::kRun / (fast ? 16 : 1) * 4;
}
template <int KIND, int D, int W>
__host__ __device__ constexpr int pm_smem(bool fast) {
  typedef PmShape<KIND, D, W> Sh;
  constexpr int ring = W * Sh::kStages * Sh::kStage, join = W * 8 * (D + 4) * 4;
  constexpr int fac = (8 * kPmJoin + (8 * D > W * 128 ? 8 * D : W * 128)) * 4;
  constexpr int most = ring > join ? ring : join;
  return pm_rows_bytes<KIND, D, W>(fast) + (most > fac ? most : fac);
}

// CTAs of 4 warps per SM that registers are held down for: 96, 128, 168 or
// 255 a thread, as the accumulators and the query need.
constexpr int pm_per_sm(int kind, int D, int HT) {
  return D == 32 ? 5 : D == 64 ? (kind == PM_I8 && HT == 1 ? 5 : 4) : HT == 2 ? 2 : 3;
}

// One CTA: one unit (sequence, kv head, up to 4 HT of its query heads) and
// one chunk of positions, tiles of 16 dealt to the W warps, U at a time.
// FAST: page_size is a multiple of 16, a tile lies in one page. The chunks of
// a unit write their sums to a.part; the last to arrive joins them in chunk
// order (so the bits do not depend on the order of arrival) and leaves its
// ticket zero. grid n_seqs * n_kv_head * head_chunks * splits.
template <int KIND, int D, int HT, bool FAST, int W>
__global__ void __launch_bounds__(W * 32, pm_per_sm(KIND, D, HT) * 4 / W) paged_mma_kernel(AttendArgs a) {
  typedef PmShape<KIND, D, W> Sh;
  constexpr bool I8 = KIND == PM_I8;
  constexpr int NT = Sh::kSteps, S = Sh::kStages, NC = Sh::kNc, U = Sh::kU, NH = 4 * HT;
  extern __shared__ __align__(16) char smem[];
  __shared__ int s_last;
  __shared__ float s_stat[8][2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
  const int hc = unit % a.head_chunks, kh = unit / a.head_chunks % a.c.n_kv_head;
  const int b = unit / a.head_chunks / a.c.n_kv_head;
  const int G = a.n_head / a.c.n_kv_head, ps = a.c.page_size;
  const int h0 = kh * G + hc * NH, nh = min(NH, G - hc * NH);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // the query's rows, as they are: column g of the operand is a term of head g / 2
  float xq[HT][NT][4];
#pragma unroll
  for (int ht = 0; ht < HT; ht++) {
    const int h = ht * 4 + (g >> 1);
    const float *q = a.q + (size_t)b * a.q_stride + (size_t)(h0 + h) * D;
#pragma unroll
    for (int k = 0; k < NT; k++) {
      float(&x)[4] = xq[ht][k];
      // int8: 4 dimensions in a row, bfloat16: 2 and 2
      if (KIND != PM_F32 && a.q_vec) {
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (h < nh) {
          if constexpr (I8) {
            y = *(const float4 *)(q + Sh::kdim(k, 0, t));
          } else {
            const float2 y0 = *(const float2 *)(q + Sh::kdim(k, 0, t)), y1 = *(const float2 *)(q + Sh::kdim(k, 2, t));
            y = make_float4(y0.x, y0.y, y1.x, y1.y);
          }
        }
        x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = h < nh ? q[Sh::kdim(k, e, t)] : 0.0f;
      }
    }
  }

  const int len = paged_len(a, b), ns = max(1, (len + a.chunk - 1) / a.chunk);
  if (split >= ns) return;
  const int p0 = split * a.chunk, p1 = min(len, p0 + a.chunk);  // the chunk's positions
  int *rows = (int *)smem;
  char *pool = smem + pm_rows_bytes<KIND, D, W>(FAST);
  auto sync = [] {
    if constexpr (W > 1)
      __syncthreads();
    else
      __syncwarp();
  };

  const unsigned ring = (unsigned)__cvta_generic_to_shared(pool) + warp * (S * Sh::kStage);
  // of a tile: the lane's scores are positions g and g + 8 of head t, its
  // operands of V positions 2t, 2t + 1, 8 + 2t and 9 + 2t
  auto vpos = [&](int i) { return (i >> 1) * 8 + 2 * t + (i & 1); };
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  // Where the lane's i-th piece of a tile's K (or V) goes: piece 32 i + lane.
  const int piece0 = lane / NC * Sh::kPad + lane % NC * 16;
  auto piece_at = [&](int i) {
    if constexpr (32 % NC == 0) return piece0 + i * (32 / NC) * Sh::kPad;
    const int p = 32 * i + lane;
    return p / NC * Sh::kPad + p % NC * 16;
  };
  // ldmatrix: lane 8 m + i names row i of matrix m. K: matrix = (n-tile, piece), V: (half of the rows, piece)
  const int matrix0 = (NC == 2 ? (lane >> 4) * 8 + (lane & 7) : lane & 7) * Sh::kPad + (NC == 2 ? lane >> 3 & 1 : lane >> 3) * 16;
  auto matrix_at = [&](int i) {
    if constexpr (NC == 2) return matrix0;
    if constexpr (NC % 4 == 0) return matrix0 + 4 * i / NC * 8 * Sh::kPad + 4 * i % NC * 16;
    const int mt = 4 * i + (lane >> 3);
    return (mt / NC * 8 + (lane & 7)) * Sh::kPad + mt % NC * 16;
  };
  // V, the four matrices of one product's tile: int8 (piece, half of the rows), bfloat16 (half of the rows, piece)
  const int half = I8 ? lane >> 3 & 1 : lane >> 4, vpiece = I8 ? lane >> 4 : lane >> 3 & 1;
  const int vmatrix0 = Sh::kVat + (half * 8 + (lane & 7)) * Sh::kPad + vpiece * 16;

  const size_t first = a.c.row(a.layer, 0, kh, 0);
  const char *kl = (const char *)a.c.k + first * Sh::kRow + (FAST ? lane * 16 : 0);
  const char *vl = (const char *)a.c.v + first * Sh::kRow + (FAST ? lane * 16 : 0);
  // int8 scales: a lane's piece of a tile's 16 + 16 (FAST), or of its positions
  const float *scl = I8 ? (FAST ? (lane < 4 ? a.c.ks : a.c.vs) + first + (lane & 3) * 4
                                : (lane < 16 ? a.c.ks : a.c.vs) + first)
                        : nullptr;
  int c0 = p0, n, ntiles;  // the run of positions whose rows are at hand
  bool hole;               // whether any of them has no page
  auto issue = [&](int tile0, int stage) {  // tiles tile0 .. tile0 + U - 1, as far as there are
#pragma unroll
    for (int v = 0; v < U; v++) {
      const int tile = U == 1 ? tile0 : min(tile0 + v, ntiles - 1);
      const unsigned d = ring + stage * Sh::kStage + v * Sh::kTile;
      const size_t at0 = FAST ? (size_t)max(rows[tile], 0) : 0;
      const char *kt = kl + at0 * Sh::kRow, *vt = vl + at0 * Sh::kRow;
#pragma unroll
      for (int i = 0; i < NC / 2; i++) {  // 16 NC pieces of K, and of V, 32 at a time
        if constexpr (FAST) {
          pm_copy16(d + piece_at(i), kt + i * 512);
          pm_copy16(d + piece_at(i) + Sh::kVat, vt + i * 512);
        } else {
          const int p = 32 * i + lane;
          const size_t off = (size_t)max(rows[tile * 16 + p / NC], 0) * Sh::kRow + p % NC * 16;
          pm_copy16(d + piece_at(i), kl + off);
          pm_copy16(d + piece_at(i) + Sh::kVat, vl + off);
        }
      }
      if constexpr (I8) {
        if constexpr (FAST) {
          if (lane < 8) pm_copy16(d + Sh::kSat + lane * 16, scl + at0);
        } else {
          pm_copy4(d + Sh::kSat + lane * 4, scl + max(rows[tile * 16 + (lane & 15)], 0));
        }
      }
    }
  };
  // the run from c0 on: its rows, relative to this layer's and kv head's
  // first, -1: no page; and the first copies
  auto open_run = [&] {
    n = min(p1 - c0, Sh::kRun), ntiles = (n + 15) / 16;
    hole = false;
    for (int i = tid; i < (FAST ? ntiles : ntiles * 16); i += W * 32) {
      const int j = FAST ? i * 16 : i;
      int row = -1;
      if (j < n) {
        const int pi = (c0 + j) / ps, page = a.t.page(b, pi);
        if (page >= 0 && page < a.c.n_pages)
          row = page * (a.c.n_kv_head * ps) + (c0 + j - pi * ps);
        else
          hole = true;
      }
      rows[i] = row;
    }
    if constexpr (W > 1) {
      hole = __syncthreads_or(hole);
    } else {
      hole = __any_sync(0xffffffffu, hole);
      __syncwarp();  // the vote alone does not order the other lanes' rows before the copies below
    }
#pragma unroll
    for (int i = 0; i < S - 1; i++) {
      if ((warp + i * W) * U < ntiles) issue((warp + i * W) * U, i);
      commit();
    }
  };
  open_run();

  // the query's operand, kept for the whole chunk: the first or the second
  // term (int8, bfloat16), qb the third of bfloat16 in the even columns
  uint32_t qa[HT][NT][2], qb[HT][I8 ? 1 : NT][2];
  float fs[HT];  // the scores' factor of the lane's own head t
#pragma unroll
  for (int ht = 0; ht < HT; ht++) {
    fs[ht] = a.scale2;
    if constexpr (I8) {
      // the largest |q| of the head to [2^13, 2^14): the second terms reach 2^-38 of it
      float mx = 0.0f;
#pragma unroll
      for (int k = 0; k < NT; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) mx = fmaxf(mx, fabsf(xq[ht][k][i]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const int e = min(max((int)(__float_as_uint(mx) >> 23), 1), 254) - 127;
      const float up = pow2i(min(13 - e, 126)), down = a.scale2 * pow2i(max(e - 13, -126));
#pragma unroll
      for (int k = 0; k < NT; k++)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          uint32_t hi, lo;
          split_f16(xq[ht][k][i] * up, xq[ht][k][i + 1] * up, hi, lo);
          qa[ht][k][i / 2] = g & 1 ? lo : hi;
        }
      fs[ht] = __shfl_sync(0xffffffffu, down, 8 * t);
    } else {
#pragma unroll
      for (int k = 0; k < NT; k++)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          uint32_t t0, t1, t2;
          split_bf16(xq[ht][k][i], xq[ht][k][i + 1], t0, t1, t2);
          qa[ht][k][i / 2] = g & 1 ? t1 : t0;
          qb[ht][k][i / 2] = g & 1 ? 0u : t2;
        }
    }
  }

  {
    float acc[HT][NT][4], m[HT], l[HT], vlim = 0x1p-100f, vinv = 0x1p115f;
#pragma unroll
    for (int ht = 0; ht < HT; ht++) {
      m[ht] = -INFINITY;
      l[ht] = 0.0f;
#pragma unroll
      for (int j = 0; j < NT; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[ht][j][i] = 0.0f;
    }

    for (;;) {
      int stage = 0;
      for (int tile = warp * U; tile < ntiles; tile += W * U) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        __syncwarp();  // every lane's copies of this tile; and every lane is done with the stage that is filled next
        if (tile + (S - 1) * W * U < ntiles) issue(tile + (S - 1) * W * U, stage == 0 ? S - 1 : stage - 1);
        commit();
        const unsigned src = ring + stage * Sh::kStage;
        stage = stage == S - 1 ? 0 : stage + 1;
        float s[HT][U][2], sv[U][2];
#pragma unroll
        for (int v = 0; v < U; v++) {
          uint32_t kr[2 * NC];  // [rows 0-7, 8-15][piece]
#pragma unroll
          for (int i = 0; i < NC / 2; i++) pm_ldmatrix<false>(kr + 4 * i, src + v * Sh::kTile + matrix_at(i));
          float c[HT][4], c2[HT][4];
#pragma unroll
          for (int k = 0; k < NT; k++) {
            if constexpr (I8) {
              const uint32_t x = kr[k] ^ 0x80808080u, y = kr[NC + k] ^ 0x80808080u;
              const uint32_t f[4] = {codes_f16(x, 0x4140), codes_f16(y, 0x4140), codes_f16(x, 0x4342), codes_f16(y, 0x4342)};
#pragma unroll
              for (int ht = 0; ht < HT; ht++) {
                if (k == 0)
                  mma_f16_from0(c[ht], f, qa[ht][k][0], qa[ht][k][1]);
                else
                  mma_f16(c[ht], f, qa[ht][k][0], qa[ht][k][1]);
              }
            } else if constexpr (KIND == PM_BF16) {
              const uint32_t f[4] = {kr[2 * k], kr[NC + 2 * k], kr[2 * k + 1], kr[NC + 2 * k + 1]};
#pragma unroll
              for (int ht = 0; ht < HT; ht++) {
                if (k == 0) {
                  mma_bf16_from0(c[ht], f, qa[ht][k][0], qa[ht][k][1]);
                  mma_bf16_from0(c2[ht], f, qb[ht][k][0], qb[ht][k][1]);
                } else {
                  mma_bf16(c[ht], f, qa[ht][k][0], qa[ht][k][1]);
                  mma_bf16(c2[ht], f, qb[ht][k][0], qb[ht][k][1]);
                }
              }
            } else {
              uint32_t f[3][4];
#pragma unroll
              for (int i = 0; i < 4; i++) {  // operand register i: rows 8 (i & 1) on, elements 2 (i / 2), + 1
                const uint32_t *x = kr + (i & 1) * NC + 4 * k + (i >> 1) * 2;
                split_bf16(__uint_as_float(x[0]), __uint_as_float(x[1]), f[0][i], f[1][i], f[2][i]);
              }
#pragma unroll
              for (int ht = 0; ht < HT; ht++) {
                if (k == 0) {
                  mma_bf16_from0(c2[ht], f[2], qa[ht][k][0], qa[ht][k][1]);
                  mma_bf16_from0(c[ht], f[0], qa[ht][k][0], qa[ht][k][1]);
                } else {
                  mma_bf16(c2[ht], f[2], qa[ht][k][0], qa[ht][k][1]);
                  mma_bf16(c[ht], f[0], qa[ht][k][0], qa[ht][k][1]);
                }
                mma_bf16(c2[ht], f[1], qa[ht][k][0], qa[ht][k][1]);
                mma_bf16(c2[ht], f[0], qb[ht][k][0], qb[ht][k][1]);
              }
            }
          }
          float ks[2] = {1.0f, 1.0f};
          if constexpr (I8) {
            const unsigned at = src + v * Sh::kTile + Sh::kSat + g * 4;
            ks[0] = pm_read1(at), ks[1] = pm_read1(at + 32);
            sv[v][0] = pm_read1(at + 64), sv[v][1] = pm_read1(at + 96);
          }
#pragma unroll
          for (int ht = 0; ht < HT; ht++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
              float y = c[ht][2 * i] + c[ht][2 * i + 1];
              if constexpr (!I8) y = c[ht][2 * i] + (c[ht][2 * i + 1] + (c2[ht][2 * i] + c2[ht][2 * i + 1]));
              s[ht][v][i] = y * fs[ht];
              if constexpr (I8) s[ht][v][i] *= ks[i];
            }
        }
        // positions past the end or without a page: no score, and a zero value
        // (0 times what is there might be NaN)
        const bool part_live = hole || (tile + U) * 16 > n;
        if (part_live) {
#pragma unroll
          for (int v = 0; v < U; v++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const int j = (tile + v) * 16 + g + 8 * i;
              if (j >= n || rows[FAST ? tile + v : j] < 0) {
                sv[v][i] = 0.0f;
#pragma unroll
                for (int ht = 0; ht < HT; ht++) s[ht][v][i] = -INFINITY;
              }
            }
        }
        if (a.scores) {
#pragma unroll
          for (int ht = 0; ht < HT; ht++)
            if (ht * 4 + t < nh) {
              float *out = a.scores + ((size_t)b * a.n_head + h0 + ht * 4 + t) * a.score_stride + c0 + tile * 16 + g;
#pragma unroll
              for (int v = 0; v < U; v++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                  if ((tile + v) * 16 + g + 8 * i < n) out[v * 16 + 8 * i] = s[ht][v][i];
            }
        }
        float mx[HT], vm = 0.0f;
        bool grow = false;
#pragma unroll
        for (int ht = 0; ht < HT; ht++) {
          mx[ht] = s[ht][0][0];
#pragma unroll
          for (int v = 0; v < U; v++)
#pragma unroll
            for (int i = 0; i < 2; i++) mx[ht] = fmaxf(mx[ht], s[ht][v][i]);
          grow = grow || mx[ht] > m[ht];
        }
        if constexpr (I8) {
#pragma unroll
          for (int v = 0; v < U; v++) vm = fmaxf(vm, fmaxf(sv[v][0], sv[v][1]));
          grow = grow || vm > vlim;
        }
        if (__any_sync(0xffffffffu, grow)) {
          float fv = 1.0f;
          if constexpr (I8) {
            // vlim: a power of two not below any value scale so far
            for (int o = 16; o > 2; o >>= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, o));
            if (vm > vlim) {
              const float up = __uint_as_float(min((__float_as_uint(vm) & 0x7f800000u) + 0x800000u, 254u << 23));
              fv = vlim / up;
              vlim = up;
              vinv = 0x1p15f / up;
            }
          }
#pragma unroll
          for (int ht = 0; ht < HT; ht++) {
            for (int o = 16; o > 2; o >>= 1) mx[ht] = fmaxf(mx[ht], __shfl_xor_sync(0xffffffffu, mx[ht], o));
            const float mn = fmaxf(m[ht], mx[ht]);
            const float f = m[ht] == -INFINITY ? 0.0f : exp2_approx(m[ht] - mn);
            l[ht] *= f;
            m[ht] = mn;
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
              for (int i = 0; i < 4; i++) acc[ht][j][i] *= f * fv;
          }
        }
#pragma unroll
        for (int v = 0; v < U; v++) {
          uint32_t pa[HT][2], pb[HT][2];  // P's operands: positions 2t, 2t + 1, and 8 more; the third terms
#pragma unroll
          for (int ht = 0; ht < HT; ht++) {
            const float mu = m[ht] == -INFINITY ? 0.0f : m[ht];
            float p[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
              p[i] = exp2_approx(s[ht][v][i] - mu);
              l[ht] += p[i];
            }
            if constexpr (I8) {
              uint32_t hi, lo;
              split_f16(p[0] * (sv[v][0] * vinv), p[1] * (sv[v][1] * vinv), hi, lo);
              pa[ht][0] = pm_transpose(__byte_perm(hi, lo, 0x5410));
              pa[ht][1] = pm_transpose(__byte_perm(hi, lo, 0x7632));
            } else {
#pragma unroll
              for (int i = 0; i < 2; i++) {
                split_bf16_one(p[i], pa[ht][i], pb[ht][i]);
                pa[ht][i] = pm_transpose(pa[ht][i]);
                pb[ht][i] = pm_transpose(pb[ht][i]);
              }
            }
          }
          // The products join the running sums by rounded additions: their own truncates, which adds up along a
          // chunk (20000 positions of one sign in one: int8 2.1e-5 too little, three times the error in bfloat16)
          bool ok[4] = {true, true, true, true};  // the lane's operand positions of V
          if (!I8 && part_live) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const int j = (tile + v) * 16 + vpos(i);
              ok[i] = j < n && rows[FAST ? tile + v : j] >= 0;
            }
          }
          if constexpr (I8) {
#pragma unroll
            for (int j = 0; j < NT; j += 2) {
              uint32_t w[4];  // piece j: rows 0-7, 8-15; piece j + 1: rows 0-7, 8-15
              pm_ldmatrix<true>(w, src + v * Sh::kTile + vmatrix0 + 16 * j);
#pragma unroll
              for (int e = 0; e < 2; e++) {
                const uint32_t x = w[2 * e] ^ 0x80808080u, y = w[2 * e + 1] ^ 0x80808080u;
                const uint32_t f[4] = {codes_f16(x, 0x4240), codes_f16(x, 0x4341), codes_f16(y, 0x4240), codes_f16(y, 0x4341)};
#pragma unroll
                for (int ht = 0; ht < HT; ht++) {
                  float o[4];
                  mma_f16_from0(o, f, pa[ht][0], pa[ht][1]);
#pragma unroll
                  for (int i = 0; i < 4; i++) acc[ht][j + e][i] += o[i];
                }
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < NT; j++) {
              if constexpr (KIND == PM_BF16) {
                uint32_t w[4];  // rows 0-7 of pieces 2 j, 2 j + 1; rows 8-15
                pm_ldmatrix<true>(w, src + v * Sh::kTile + vmatrix0 + 32 * j);
                if (part_live) {
                  const uint32_t z0 = (ok[0] ? 0xffffu : 0u) | (ok[1] ? 0xffff0000u : 0u);
                  const uint32_t z1 = (ok[2] ? 0xffffu : 0u) | (ok[3] ? 0xffff0000u : 0u);
                  w[0] &= z0, w[1] &= z0, w[2] &= z1, w[3] &= z1;
                }
#pragma unroll
                for (int ht = 0; ht < HT; ht++) {
                  float o[4];
                  mma_bf16_from0(o, w, pb[ht][0], pb[ht][1]);
                  mma_bf16(o, w, pa[ht][0], pa[ht][1]);
#pragma unroll
                  for (int i = 0; i < 4; i++) acc[ht][j][i] += o[i];
                }
              } else {
                uint32_t f[3][4];
#pragma unroll
                for (int i = 0; i < 4; i++) {  // operand register i: dimensions 8 (i & 1) on, positions 8 (i / 2) on
                  float y[2];
#pragma unroll
                  for (int e = 0; e < 2; e++) {
                    const int r = (i >> 1) * 2 + e;
                    y[e] = pm_read1(src + v * Sh::kTile + Sh::kVat + vpos(r) * Sh::kPad + (16 * j + 8 * (i & 1) + g) * 4);
                    if (!ok[r]) y[e] = 0.0f;
                  }
                  split_bf16(y[0], y[1], f[0][i], f[1][i], f[2][i]);
                }
#pragma unroll
                for (int ht = 0; ht < HT; ht++) {
                  float o[4];
                  mma_bf16_from0(o, f[0], pb[ht][0], pb[ht][1]);
#pragma unroll
                  for (int k = 2; k >= 0; k--) mma_bf16(o, f[k], pa[ht][0], pa[ht][1]);
#pragma unroll
                  for (int i = 0; i < 4; i++) acc[ht][j][i] += o[i];
                }
              }
            }
          }
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      c0 += Sh::kRun;
      if (c0 >= p1) break;
      sync();
      open_run();
    }

    // join the warps: [warp][head][D sums, M, L, -, -] in the rings' place
    constexpr int kJ = D + 4;
    float *join = (float *)pool;
    sync();
#pragma unroll
    for (int ht = 0; ht < HT; ht++) {
      for (int o = 4; o < 32; o <<= 1) l[ht] += __shfl_xor_sync(0xffffffffu, l[ht], o);
      if (ht * 4 + t >= nh) continue;
      float *o = join + (warp * NH + ht * 4 + t) * kJ;
      const float f = I8 ? vlim * 0x1p-15f : 1.0f;
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const float x = (acc[ht][j][0] + acc[ht][j][1]) * f, y = (acc[ht][j][2] + acc[ht][j][3]) * f;
        if constexpr (I8) {
          *(float2 *)(o + Sh::vdim(j, 0, g)) = make_float2(x, y);
        } else {
          o[Sh::vdim(j, 0, g)] = x;
          o[Sh::vdim(j, 1, g)] = y;
        }
      }
      if (g == 0) {
        o[D] = m[ht];
        o[D + 1] = l[ht];
      }
    }
    sync();
    constexpr int kStep = NH * kJ;  // floats of a partial result, laid out the same
    for (int i = tid; i < nh * D; i += W * 32) {
      const int h = i / D, d = i % D;
      const float *o = join + h * kJ;
      float M = -INFINITY, L = 0.0f, x = 0.0f;
      if constexpr (W == 1) {
        M = o[D], L = o[D + 1], x = o[d];
      } else {
#pragma unroll
        for (int w = 0; w < W; w++) M = fmaxf(M, o[w * NH * kJ + D]);
        const float mu = M == -INFINITY ? 0.0f : M;
#pragma unroll
        for (int w = 0; w < W; w++) {
          const float f = exp2_approx(o[w * NH * kJ + D] - mu);
          L = fmaf(o[w * NH * kJ + D + 1], f, L);
          x = fmaf(o[w * NH * kJ + d], f, x);
        }
      }
      if (ns == 1) {
        a.out[(size_t)b * a.out_stride + (size_t)(h0 + h) * D + d] = L == 0.0f ? 0.0f : x / L;
        if (a.stat && d == 0) {
          a.stat[2 * ((size_t)b * a.n_head + h0 + h)] = M;
          a.stat[2 * ((size_t)b * a.n_head + h0 + h) + 1] = L;
        }
      } else {
        float *part = a.part + ((size_t)unit * a.splits + split) * kStep + h * kJ;
        part[d] = x;
        if (d == 0) {
          part[D] = M;
          part[D + 1] = L;
        }
      }
    }
    if (ns == 1) return;
    __threadfence();
    sync();
    if (tid == 0) s_last = atomicAdd(&a.tickets[unit], 1) == ns - 1;
    sync();
    if (!s_last) return;
    __threadfence();
    // M, L and the parts' factors 2^(M_k - M) of each head; then the sums, the
    // parts dealt to as many groups of threads as there are, joined in order
    const float *part = a.part + (size_t)unit * a.splits * kStep;
    float *fac = (float *)pool, *sums = fac + 8 * kPmJoin;  // [head][kPmJoin]; [group][nh * D]
    for (int h = warp; h < nh; h += W) {
      constexpr int kN = kPmJoin / 32;
      float mk[kN], lk[kN], M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int i = 0; i < kN; i++) {
        const int k = i * 32 + lane;
        const float *o = part + (size_t)k * kStep + h * kJ + D;
        mk[i] = k < ns ? __ldcg(o) : -INFINITY;
        lk[i] = k < ns ? __ldcg(o + 1) : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < kN; i++) M = fmaxf(M, mk[i]);
      for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      const float mu = M == -INFINITY ? 0.0f : M;
#pragma unroll
      for (int i = 0; i < kN; i++) {
        const float f = exp2_approx(mk[i] - mu);
        L = fmaf(lk[i], f, L);
        fac[h * kPmJoin + i * 32 + lane] = f;
      }
      for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
      if (lane == 0) {
        s_stat[h][0] = M;
        s_stat[h][1] = L;
      }
    }
    sync();
    const int no = nh * D / 4, groups = max(1, W * 32 / no);  // four dimensions a thread
    for (int i = tid; i < no * groups; i += W * 32) {
      const int grp = i / no, o = i % no * 4, h = o / D;
      const float *src = part + h * kJ + o % D, *f = fac + h * kPmJoin;
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int k0 = grp; k0 < ns; k0 += 8 * groups) {
        float4 y[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (k0 + j * groups < ns) y[j] = __ldcg((const float4 *)(src + (size_t)(k0 + j * groups) * kStep));
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (k0 + j * groups < ns) {
            const float w = f[k0 + j * groups];
            x.x = fmaf(y[j].x, w, x.x), x.y = fmaf(y[j].y, w, x.y), x.z = fmaf(y[j].z, w, x.z), x.w = fmaf(y[j].w, w, x.w);
          }
      }
      *(float4 *)(sums + grp * nh * D + o) = x;
    }
    sync();
    for (int i = tid; i < nh * D; i += W * 32) {
      const int h = i / D, d = i % D;
      float x = sums[i];
      for (int grp = 1; grp < groups; grp++) x += sums[grp * nh * D + i];
      const float L = s_stat[h][1];
      a.out[(size_t)b * a.out_stride + (size_t)(h0 + h) * D + d] = L == 0.0f ? 0.0f : x / L;
      if (a.stat && d == 0) {
        a.stat[2 * ((size_t)b * a.n_head + h0 + h)] = s_stat[h][0];
        a.stat[2 * ((size_t)b * a.n_head + h0 + h) + 1] = L;
      }
    }
    if (tid == 0) a.tickets[unit] = 0;
  }
}

}  // namespace llmq
