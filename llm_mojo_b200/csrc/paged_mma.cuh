// paged_mma.cuh -- attention of one new token over a paged cache on the
// tensor cores, split over positions and joined.
//
// One pass over the cache: scores S = Q K^T, running maximum M and sum L of
// 2^(s - M), and O = P V, as m16n8k16 products with float32 accumulators,
// from registers to registers: the score tile's accumulator layout is the
// operand layout of P. The rows of the 16-row operand hold up to 8 query
// heads of one kv head, twice: a float32 factor x enters as a sum of 16-bit
// terms, so that products keep float32's accuracy,
//   int8:     x 2^e = f16 + f16: rows 0-7 the first term, rows 8-15 the
//             second (22 bits; codes are exact in f16),
//   bfloat16: x = bf16 + bf16 + bf16 by truncation (all 24 bits): rows 0-7
//             and 8-15 the first two, a second product the third,
//   float32:  both factors in three bf16 terms, the products of weight
//             2^-24 and above,
// and a head's result is the sum of its rows. The terms sit in rows that one
// query head or a few would leave idle.
//
// Both products may take dimensions and positions in any order that their
// two operands share, so a lane reads contiguous bytes of a row as its
// operand: of K, rows (lane / 4) and + 8, pieces of every run; of V, the
// four rows whose weights the lane holds, an eighth each. A lane copies
// (cp.async) the bytes that it will read itself into its own slots of a ring
// in shared memory, [piece][lane], so that reads have no bank conflicts,
// nothing waits for another lane, and the copies in flight cost no
// registers.
#pragma once

#include "paged.cuh"

namespace llmq {

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// BYTES (4, 8 or 16) into the lane's slot; 16 bypass L1: the cache is read once.
template <int BYTES>
__device__ __forceinline__ void pm_copy(unsigned dst, const void *src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void pm_read(uint32_t *d, unsigned src) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(src)
                 : "memory");
  else if constexpr (BYTES == 8)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(d[0]), "=r"(d[1]) : "r"(src) : "memory");
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(d[0]) : "r"(src) : "memory");
}

// Two f16 from two biased codes (code ^ 0x80) in bytes i and j of x: 1024 +
// byte, less 1152; all exact.
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

// x, y as three bf16 terms each by truncation, exact: 8 + 8 + 8 bits.
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t &t0, uint32_t &t1, uint32_t &t2) {
  const uint32_t x0 = __float_as_uint(x) & 0xffff0000u, y0 = __float_as_uint(y) & 0xffff0000u;
  const float xr = x - __uint_as_float(x0), yr = y - __uint_as_float(y0);
  const uint32_t x1 = __float_as_uint(xr) & 0xffff0000u, y1 = __float_as_uint(yr) & 0xffff0000u;
  const float xs = xr - __uint_as_float(x1), ys = yr - __uint_as_float(y1);
  t0 = __byte_perm(x0, y0, 0x7632);
  t1 = __byte_perm(x1, y1, 0x7632);
  t2 = __byte_perm(__float_as_uint(xs), __float_as_uint(ys), 0x7632);
}

// How a lane's bytes of a row map to dimensions. K: runs of 4 kCk bytes, a
// lane's piece t; V: runs of 8 kCv bytes, piece g.
enum { PM_I8 = 0, PM_BF16 = 1, PM_F32 = 2 };
template <int KIND, int D>
struct PmShape {
  static constexpr int kEs = KIND == PM_I8 ? 1 : KIND == PM_BF16 ? 2 : 4;
  static constexpr int kRow = D * kEs;
  static constexpr int kKb = kRow / 4, kVb = kRow / 8;  // a lane's bytes of a K / V row
  static constexpr int kCk = kKb % 16 == 0 ? 16 : 8;
  static constexpr int kCv = kVb % 16 == 0 ? 16 : (kVb % 8 == 0 ? 8 : 4);
  static constexpr int kNk = kKb / kCk, kNv = kVb / kCv;  // pieces
  static constexpr int kSteps = D / 16;
  // a stage of a warp's ring: two K rows, four V rows and (int8) the scales
  // of four positions for keys and values, of each lane
  static constexpr int kStage = 32 * (2 * kKb + 4 * kVb + (KIND == PM_I8 ? 32 : 0));
  // stages: about 3 KB or more in flight per warp
  static constexpr int kStages = kStage <= 2048 ? 4 : kStage <= 4096 ? 3 : 2;
  static __device__ __forceinline__ int kdim(int x, int t) {  // dimension of a lane's x-th K element
    constexpr int E = kCk / kEs;
    return (x / E * 4 + t) * E + x % E;
  }
  static __device__ __forceinline__ int vdim(int x, int g) {
    constexpr int E = kCv / kEs;
    return (x / E * 8 + g) * E + x % E;
  }
};

// Dynamic shared memory: the rows of the tiles (page_size % 16 == 0) or of
// every position of a chunk; then the rings, and in their place, at the end,
// the warps' states.
__host__ __device__ inline int pm_rows_bytes(int chunk, bool fast) { return ((fast ? chunk / 16 : chunk) * 4 + 15) / 16 * 16; }
template <int KIND, int D, int W>
__host__ __device__ inline size_t pm_smem(int chunk, bool fast) {
  typedef PmShape<KIND, D> Sh;
  const size_t ring = (size_t)W * Sh::kStages * Sh::kStage, join = (size_t)W * 8 * (D + 2) * 4;
  return pm_rows_bytes(chunk, fast) + (ring > join ? ring : join);
}

// One CTA: one unit (sequence, kv head, up to 8 of its query heads) and one
// chunk of positions, tiles of 16 dealt to the W warps. FAST: page_size is a
// multiple of 16, a tile lies in one page. The chunks of a unit write their
// sums to a.part; the last to arrive joins them in chunk order (so the bits
// do not depend on the order of arrival) and leaves its ticket zero.
// grid n_seqs * n_kv_head * head_chunks * splits.
template <int KIND, int D, bool FAST, int W>
__global__ void __launch_bounds__(W * 32) paged_mma_kernel(AttendArgs a) {
  typedef PmShape<KIND, D> Sh;
  constexpr bool I8 = KIND == PM_I8;
  constexpr int NT = D / 8, S = Sh::kStages;
  extern __shared__ __align__(16) char smem[];
  __shared__ int s_last;
  const int split = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
  const int hc = unit % a.head_chunks, kh = unit / a.head_chunks % a.c.n_kv_head;
  const int b = unit / a.head_chunks / a.c.n_kv_head;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = a.n_head / a.c.n_kv_head, h0 = kh * G + hc * 8, nh = min(8, G - hc * 8);
  const int len = paged_len(a, b), ps = a.c.page_size;
  const int ns = max(1, (len + a.chunk - 1) / a.chunk);
  if (split >= ns) return;
  const int c0 = split * a.chunk, n = min(len - c0, a.chunk);  // the chunk's positions
  const int ntiles = (n + 15) / 16;
  int *rows = (int *)smem;
  char *pool = smem + pm_rows_bytes(a.chunk, FAST);

  // rows of the chunk, relative to this layer's and kv head's first; -1: no page
  for (int i = tid; i < (FAST ? ntiles : ntiles * 16); i += W * 32) {
    const int j = FAST ? i * 16 : i;
    int row = -1;
    if (j < n) {
      const int pi = (c0 + j) / ps, page = a.t.page(b, pi);
      if (page >= 0 && page < a.c.n_pages) row = page * (a.c.n_kv_head * ps) + (c0 + j - pi * ps);
    }
    rows[i] = row;
  }

  // the query's operand, kept for the whole chunk
  uint32_t qa[Sh::kSteps][4], qb[I8 ? 1 : Sh::kSteps][2];
  float fs = a.scale2;
  {
    float x[D / 4];
    const float *q = a.q + (size_t)b * a.q_stride + (size_t)(h0 + g) * D;
    float mx = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 4; i++) {
      x[i] = g < nh ? q[Sh::kdim(i, t)] : 0.0f;
      mx = fmaxf(mx, fabsf(x[i]));
    }
    if constexpr (I8) {
      // the largest |q| of the head to [2^13, 2^14): the second terms reach 2^-38 of it
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const int e = min(max((int)(__float_as_uint(mx) >> 23), 1), 254) - 127;
      const float up = pow2i(min(13 - e, 126));
#pragma unroll
      for (int i = 0; i < D / 4; i++) x[i] *= up;
      fs = a.scale2 * pow2i(max(e - 13, -126));
    }
#pragma unroll
    for (int k = 0; k < Sh::kSteps; k++) {
      if constexpr (I8) {
        split_f16(x[4 * k], x[4 * k + 1], qa[k][0], qa[k][1]);
        split_f16(x[4 * k + 2], x[4 * k + 3], qa[k][2], qa[k][3]);
      } else {
        split_bf16(x[4 * k], x[4 * k + 1], qa[k][0], qa[k][1], qb[k][0]);
        split_bf16(x[4 * k + 2], x[4 * k + 3], qa[k][2], qa[k][3], qb[k][1]);
      }
    }
  }
  if constexpr (W > 1)
    __syncthreads();
  else
    __syncwarp();

  // the lane's first bytes in the pool, and its slots
  const size_t first = a.c.row(a.layer, 0, kh, 0);
  const char *kl = (const char *)a.c.k + first * Sh::kRow + t * Sh::kCk + (FAST ? g * Sh::kRow : 0);
  const char *vl = (const char *)a.c.v + first * Sh::kRow + g * Sh::kCv + (FAST ? 2 * t * Sh::kRow : 0);
  const float *ksl = I8 ? a.c.ks + first + (FAST ? 2 * t : 0) : nullptr;
  const float *vsl = I8 ? a.c.vs + first + (FAST ? 2 * t : 0) : nullptr;
  const unsigned ring = (unsigned)__cvta_generic_to_shared(pool) + warp * (S * Sh::kStage);
  constexpr int kVat = 64 * Sh::kKb, kSat = kVat + 128 * Sh::kVb;  // a stage: K, V, scales
  auto pos_of = [&](int i) { return (i >> 1) * 8 + 2 * t + (i & 1); };  // the lane's position i of a tile
  auto issue = [&](int tile, int stage) {
    const unsigned d = ring + stage * Sh::kStage;
    const int base = FAST ? max(rows[tile], 0) : 0;
#pragma unroll
    for (int r = 0; r < 2; r++) {
      const char *p = FAST ? kl + (size_t)base * Sh::kRow + r * 8 * Sh::kRow
                           : kl + (size_t)max(rows[tile * 16 + 8 * r + g], 0) * Sh::kRow;
#pragma unroll
      for (int i = 0; i < Sh::kNk; i++)
        pm_copy<Sh::kCk>(d + (r * Sh::kNk + i) * 32 * Sh::kCk + lane * Sh::kCk, p + i * 4 * Sh::kCk);
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int row = FAST ? base : max(rows[tile * 16 + pos_of(r)], 0);
      const char *p = vl + (size_t)row * Sh::kRow + (FAST ? ((r >> 1) * 8 + (r & 1)) * Sh::kRow : 0);
#pragma unroll
      for (int i = 0; i < Sh::kNv; i++)
        pm_copy<Sh::kCv>(d + kVat + (r * Sh::kNv + i) * 32 * Sh::kCv + lane * Sh::kCv, p + i * 8 * Sh::kCv);
      if constexpr (I8) {
        const unsigned sd = d + kSat + lane * 8 + (r >> 1) * 256;
        if constexpr (FAST) {
          if (r % 2 == 0) {
            pm_copy<8>(sd, ksl + (size_t)row + (r >> 1) * 8);
            pm_copy<8>(sd + 512, vsl + (size_t)row + (r >> 1) * 8);
          }
        } else {
          pm_copy<4>(sd + (r & 1) * 4, ksl + row);
          pm_copy<4>(sd + 512 + (r & 1) * 4, vsl + row);
        }
      }
    }
  };
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };

  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; j++)
#pragma unroll
    for (int i = 0; i < 4; i++) acc[j][i] = 0.0f;
  float m = -INFINITY, l = 0.0f, vlim = 0x1p-100f, vinv = 0x1p115f;

#pragma unroll
  for (int i = 0; i < S - 1; i++) {
    if (warp + i * W < ntiles) issue(warp + i * W, i);
    commit();
  }
  int stage = 0;
  for (int tile = warp; tile < ntiles; tile += W) {
    asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
    if (tile + (S - 1) * W < ntiles) issue(tile + (S - 1) * W, stage == 0 ? S - 1 : stage - 1);
    commit();
    const unsigned src = ring + stage * Sh::kStage;
    stage = stage == S - 1 ? 0 : stage + 1;
    // scores of 16 positions: two n-tiles of 8
    float c[2][4];
#pragma unroll
    for (int r = 0; r < 2; r++) {
#pragma unroll
      for (int i = 0; i < 4; i++) c[r][i] = 0.0f;
      uint32_t kr[Sh::kKb / 4];
#pragma unroll
      for (int i = 0; i < Sh::kNk; i++)
        pm_read<Sh::kCk>(kr + i * (Sh::kCk / 4), src + (r * Sh::kNk + i) * 32 * Sh::kCk + lane * Sh::kCk);
#pragma unroll
      for (int k = 0; k < Sh::kSteps; k++) {
        if constexpr (KIND == PM_I8) {
          const uint32_t x = kr[k] ^ 0x80808080u;
          mma_f16(c[r], qa[k], codes_f16(x, 0x4140), codes_f16(x, 0x4342));
        } else {
          const uint32_t q2[4] = {qb[k][0], 0u, qb[k][1], 0u};
          if constexpr (KIND == PM_BF16) {
            mma_bf16(c[r], qa[k], kr[2 * k], kr[2 * k + 1]);
            mma_bf16(c[r], q2, kr[2 * k], kr[2 * k + 1]);
          } else {
            uint32_t x[3], y[3];
            split_bf16(__uint_as_float(kr[4 * k]), __uint_as_float(kr[4 * k + 1]), x[0], x[1], x[2]);
            split_bf16(__uint_as_float(kr[4 * k + 2]), __uint_as_float(kr[4 * k + 3]), y[0], y[1], y[2]);
            mma_bf16(c[r], q2, x[0], y[0]);
#pragma unroll
            for (int i = 2; i >= 0; i--) mma_bf16(c[r], qa[k], x[i], y[i]);
          }
        }
      }
    }
    float s[4], sv[4];
    if constexpr (I8) {
      uint32_t ks[4], vs[4];
      pm_read<8>(ks, src + kSat + lane * 8);
      pm_read<8>(ks + 2, src + kSat + 256 + lane * 8);
      pm_read<8>(vs, src + kSat + 512 + lane * 8);
      pm_read<8>(vs + 2, src + kSat + 768 + lane * 8);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        s[i] = (c[i >> 1][i & 1] + c[i >> 1][2 + (i & 1)]) * fs * __uint_as_float(ks[i]);
        sv[i] = __uint_as_float(vs[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) s[i] = (c[i >> 1][i & 1] + c[i >> 1][2 + (i & 1)]) * fs;
    }
    // positions past the end or without a page: no score, and a zero value
    // (0 times what is there might be NaN)
    unsigned masked = 0;
    if (!FAST || tile * 16 + 16 > n || rows[tile] < 0) {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (tile * 16 + pos_of(i) >= n || rows[FAST ? tile : tile * 16 + pos_of(i)] < 0) {
          masked |= 1u << i;
          s[i] = -INFINITY;
          sv[i] = 0.0f;
        }
    }
    if (a.scores && g < nh) {
      float *out = a.scores + ((size_t)b * a.n_head + h0 + g) * a.max_len + c0 + tile * 16;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (tile * 16 + pos_of(i) < n) out[pos_of(i)] = s[i];
    }
    float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    bool grow = mx > m;
    float vm = 0.0f;
    if constexpr (I8) {
      vm = fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]));
      grow = grow || vm > vlim;
    }
    if (__any_sync(0xffffffffu, grow)) {
      const float mn = fmaxf(m, mx);
      float f = m == -INFINITY ? 0.0f : exp2_approx(m - mn);
      l *= f;
      m = mn;
      if constexpr (I8) {
        // vlim: a power of two not below any value scale so far
        for (int o = 16; o > 0; o >>= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, o));
        if (vm > vlim) {
          const float up = __uint_as_float(min((__float_as_uint(vm) & 0x7f800000u) + 0x800000u, 254u << 23));
          f *= vlim / up;
          vlim = up;
          vinv = 0x1p15f / up;
        }
      }
#pragma unroll
      for (int j = 0; j < NT; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[j][i] *= f;
    }
    const float mu = m == -INFINITY ? 0.0f : m;
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      p[i] = exp2_approx(s[i] - mu);
      l += p[i];
    }
    uint32_t pa[4], pb[4] = {0u, 0u, 0u, 0u};
    if constexpr (I8) {
#pragma unroll
      for (int i = 0; i < 4; i++) p[i] *= sv[i] * vinv;
      split_f16(p[0], p[1], pa[0], pa[1]);
      split_f16(p[2], p[3], pa[2], pa[3]);
    } else {
      split_bf16(p[0], p[1], pa[0], pa[1], pb[0]);
      split_bf16(p[2], p[3], pa[2], pa[3], pb[2]);
    }
#pragma unroll
    for (int i = 0; i < Sh::kNv; i++) {
      constexpr int kW = Sh::kCv / 4;
      uint32_t vr[4][kW];
#pragma unroll
      for (int r = 0; r < 4; r++)
        pm_read<Sh::kCv>(vr[r], src + kVat + (r * Sh::kNv + i) * 32 * Sh::kCv + lane * Sh::kCv);
      if constexpr (!I8) {
        if (masked) {
#pragma unroll
          for (int r = 0; r < 4; r++)
#pragma unroll
            for (int w = 0; w < kW; w++)
              if (masked >> r & 1u) vr[r][w] = 0u;
        }
      }
#pragma unroll
      for (int w = 0; w < kW; w++) {
        if constexpr (KIND == PM_I8) {
          float (*o)[4] = acc + 4 * (i * kW + w);
          const uint32_t v0 = vr[0][w] ^ 0x80808080u, v1 = vr[1][w] ^ 0x80808080u, v2 = vr[2][w] ^ 0x80808080u,
                         v3 = vr[3][w] ^ 0x80808080u;
          const uint32_t x = __byte_perm(v0, v1, 0x5140), y = __byte_perm(v2, v3, 0x5140);
          const uint32_t z = __byte_perm(v0, v1, 0x7362), u = __byte_perm(v2, v3, 0x7362);
          mma_f16(o[0], pa, codes_f16(x, 0x4140), codes_f16(y, 0x4140));
          mma_f16(o[1], pa, codes_f16(x, 0x4342), codes_f16(y, 0x4342));
          mma_f16(o[2], pa, codes_f16(z, 0x4140), codes_f16(u, 0x4140));
          mma_f16(o[3], pa, codes_f16(z, 0x4342), codes_f16(u, 0x4342));
        } else if constexpr (KIND == PM_BF16) {
          float (*o)[4] = acc + 2 * (i * kW + w);
          const uint32_t x0 = __byte_perm(vr[0][w], vr[1][w], 0x5410), x1 = __byte_perm(vr[2][w], vr[3][w], 0x5410);
          const uint32_t y0 = __byte_perm(vr[0][w], vr[1][w], 0x7632), y1 = __byte_perm(vr[2][w], vr[3][w], 0x7632);
          mma_bf16(o[0], pa, x0, x1);
          mma_bf16(o[1], pa, y0, y1);
          mma_bf16(o[0], pb, x0, x1);
          mma_bf16(o[1], pb, y0, y1);
        } else {
          float (&o)[4] = acc[i * kW + w];
          uint32_t x[3], y[3];
          split_bf16(__uint_as_float(vr[0][w]), __uint_as_float(vr[1][w]), x[0], x[1], x[2]);
          split_bf16(__uint_as_float(vr[2][w]), __uint_as_float(vr[3][w]), y[0], y[1], y[2]);
          mma_bf16(o, pb, x[0], y[0]);
#pragma unroll
          for (int k = 2; k >= 0; k--) mma_bf16(o, pa, x[k], y[k]);
        }
      }
    }
  }

  // join the warps: [warp][head][D sums, M, L] in the rings' place
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  float *join = (float *)pool;
  if constexpr (W > 1) __syncthreads();
  else __syncwarp();
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  if (g < nh) {
    float *o = join + (warp * 8 + g) * (D + 2);
    const float f = I8 ? vlim * 0x1p-15f : 1.0f;
#pragma unroll
    for (int j = 0; j < NT; j++) {
      o[Sh::vdim(j, 2 * t)] = (acc[j][0] + acc[j][2]) * f;
      o[Sh::vdim(j, 2 * t + 1)] = (acc[j][1] + acc[j][3]) * f;
    }
    if (t == 0) {
      o[D] = m;
      o[D + 1] = l;
    }
  }
  if constexpr (W > 1)
    __syncthreads();
  else
    __syncwarp();
  for (int i = tid; i < nh * D; i += W * 32) {
    const int h = i / D, d = i % D;
    const float *o = join + h * (D + 2);
    float M = -INFINITY, L = 0.0f, x = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) M = fmaxf(M, o[w * 8 * (D + 2) + D]);
    const float mu = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int w = 0; w < W; w++) {
      const float f = exp2_approx(o[w * 8 * (D + 2) + D] - mu);
      L = fmaf(o[w * 8 * (D + 2) + D + 1], f, L);
      x = fmaf(o[w * 8 * (D + 2) + d], f, x);
    }
    if (ns == 1) {
      a.out[(size_t)b * a.out_stride + (size_t)(h0 + h) * D + d] = L == 0.0f ? 0.0f : x / L;
      if (a.stat && d == 0) {
        a.stat[2 * ((size_t)b * a.n_head + h0 + h)] = M;
        a.stat[2 * ((size_t)b * a.n_head + h0 + h) + 1] = L;
      }
    } else {
      float *part = a.part + (((size_t)unit * a.splits + split) * 8 + h) * (D + 2);
      part[d] = x;
      if (d == 0) {
        part[D] = M;
        part[D + 1] = L;
      }
    }
  }
  if (ns == 1) return;
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(&a.tickets[unit], 1) == ns - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  for (int i = tid; i < nh * D; i += W * 32) {
    const int h = i / D, d = i % D;
    const float *part = a.part + ((size_t)unit * a.splits * 8 + h) * (D + 2);
    float M = -INFINITY, L = 0.0f, x = 0.0f;
    for (int k = 0; k < ns; k++) M = fmaxf(M, __ldcg(part + (size_t)k * 8 * (D + 2) + D));
    const float mu = M == -INFINITY ? 0.0f : M;
    for (int k = 0; k < ns; k++) {
      const float *o = part + (size_t)k * 8 * (D + 2);
      const float f = exp2_approx(__ldcg(o + D) - mu);
      L = fmaf(__ldcg(o + D + 1), f, L);
      x = fmaf(__ldcg(o + d), f, x);
    }
    a.out[(size_t)b * a.out_stride + (size_t)(h0 + h) * D + d] = L == 0.0f ? 0.0f : x / L;
    if (a.stat && d == 0) {
      a.stat[2 * ((size_t)b * a.n_head + h0 + h)] = M;
      a.stat[2 * ((size_t)b * a.n_head + h0 + h) + 1] = L;
    }
  }
  if (tid == 0) a.tickets[unit] = 0;
}

}  // namespace llmq
