// paged_mma.cuh -- attention of one new token over a paged int8 or bfloat16
// cache on the tensor cores, split over positions and joined.
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
// and a head's result is the sum of its rows. One pass with the terms in
// otherwise idle rows costs no more issue slots than a half-empty tile would.
//
// Both products may take dimensions and positions in any order that their
// two operands share, so a lane loads contiguous bytes of a row straight
// from memory into operand registers: of K, rows (lane / 4) and + 8, bytes
// of the lane's quarter of each run; of V, the four rows whose weights the
// lane holds, an eighth each.
#pragma once

#include "paged.cuh"

namespace llmq {

constexpr int kPmWarps = 4;

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

// BYTES (4, 8 or 16) of the cache into registers; read once, so not kept in L1.
template <int BYTES>
__device__ __forceinline__ void pm_load(uint32_t *d, const char *p) {
  if constexpr (BYTES == 16)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "l"(p));
  else if constexpr (BYTES == 8)
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(d[0]), "=r"(d[1]) : "l"(p));
  else
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(d[0]) : "l"(p));
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
template <bool I8, int D>
struct PmShape {
  static constexpr int kEs = I8 ? 1 : 2;
  static constexpr int kKb = D / 4 * kEs, kVb = D / 8 * kEs;  // a lane's bytes of a K / V row
  static constexpr int kCk = kKb % 16 == 0 ? 16 : 8;
  static constexpr int kCv = kVb % 16 == 0 ? 16 : (kVb % 8 == 0 ? 8 : 4);
  static constexpr int kSteps = D / 16;
  static __device__ __forceinline__ int kdim(int x, int t) {  // dimension of a lane's x-th K element
    constexpr int E = kCk / kEs;
    return (x / E * 4 + t) * E + x % E;
  }
  static __device__ __forceinline__ int vdim(int x, int g) {
    constexpr int E = kCv / kEs;
    return (x / E * 8 + g) * E + x % E;
  }
};

__host__ __device__ inline size_t pm_smem(int chunk, int D, bool fast) {
  // the tiles' first rows (page_size % 16 == 0) or every position's row; then the warps' states
  const size_t rows = ((size_t)(fast ? chunk / 16 : chunk) * 4 + 15) / 16 * 16;
  const size_t join = (size_t)kPmWarps * 8 * (D + 2) * 4;
  return rows + join;
}

// One CTA: one unit (sequence, kv head, up to 8 of its query heads) and one
// chunk of positions, tiles of 16 dealt to the 4 warps. FAST: page_size is a
// multiple of 16, a tile lies in one page. The chunks of a unit write their
// sums to a.part; the last to arrive joins them in chunk order (so the bits
// do not depend on the order of arrival) and leaves its ticket zero.
// grid n_seqs * n_kv_head * head_chunks * splits.
template <bool I8, int D, bool FAST>
__global__ void __launch_bounds__(kPmWarps * 32) paged_mma_kernel(AttendArgs a) {
  typedef PmShape<I8, D> Sh;
  constexpr int kKw = Sh::kKb / 4, kVw = Sh::kVb / 4, NT = D / 8;
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
  const int c0 = split * a.chunk, c1 = min(len, c0 + a.chunk);
  const int ntiles = (c1 - c0 + 15) / 16;
  int *rows = (int *)smem;
  float *join = (float *)(smem + ((size_t)(FAST ? a.chunk / 16 : a.chunk) * 4 + 15) / 16 * 16);

  // rows of the chunk, relative to this layer's and kv head's first; -1: no page
  for (int i = tid; i < (FAST ? ntiles : ntiles * 16); i += kPmWarps * 32) {
    const int pos = c0 + (FAST ? i * 16 : i);
    int row = -1;
    if (pos < c1) {
      const int pi = pos / ps, page = a.t.page(b, pi);
      if (page >= 0 && page < a.c.n_pages) row = page * (a.c.n_kv_head * ps) + (pos - pi * ps);
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
  __syncthreads();

  const size_t first = a.c.row(a.layer, 0, kh, 0);
  const char *kb = (const char *)a.c.k + first * (D * Sh::kEs), *vb = (const char *)a.c.v + first * (D * Sh::kEs);
  uint32_t kr[2][kKw], vr[4][kVw];
  float ksc[4], vsc[4];  // the scales of the lane's positions 2t, 2t + 1, 8 + 2t, 9 + 2t
  auto pos_of = [&](int i) { return (i >> 1) * 8 + 2 * t + (i & 1); };
  auto row_of = [&](int tile, int i) { return max(FAST ? rows[tile] + i : rows[tile * 16 + i], 0); };
  auto load_k = [&](int tile) {
#pragma unroll
    for (int r = 0; r < 2; r++) {
      const char *p = kb + (size_t)row_of(tile, 8 * r + g) * (D * Sh::kEs);
#pragma unroll
      for (int i = 0; i < Sh::kKb / Sh::kCk; i++) pm_load<Sh::kCk>(&kr[r][i * (Sh::kCk / 4)], p + (i * 4 + t) * Sh::kCk);
    }
    if constexpr (I8) {
#pragma unroll
      for (int i = 0; i < 4; i++) ksc[i] = a.c.ks[first + row_of(tile, pos_of(i))];
    }
  };
  auto load_v = [&](int tile) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const char *p = vb + (size_t)row_of(tile, pos_of(r)) * (D * Sh::kEs);
#pragma unroll
      for (int i = 0; i < Sh::kVb / Sh::kCv; i++) pm_load<Sh::kCv>(&vr[r][i * (Sh::kCv / 4)], p + (i * 8 + g) * Sh::kCv);
    }
    if constexpr (I8) {
#pragma unroll
      for (int i = 0; i < 4; i++) vsc[i] = a.c.vs[first + row_of(tile, pos_of(i))];
    }
  };

  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; j++)
#pragma unroll
    for (int i = 0; i < 4; i++) acc[j][i] = 0.0f;
  float m = -INFINITY, l = 0.0f, vlim = 0x1p-100f;

  if (warp < ntiles) {
    load_k(warp);
    load_v(warp);
  }
  for (int tile = warp; tile < ntiles; tile += kPmWarps) {
    const bool more = tile + kPmWarps < ntiles;
    // scores of 16 positions: two n-tiles of 8
    float c[2][4];
#pragma unroll
    for (int r = 0; r < 2; r++) {
#pragma unroll
      for (int i = 0; i < 4; i++) c[r][i] = 0.0f;
#pragma unroll
      for (int k = 0; k < Sh::kSteps; k++) {
        if constexpr (I8) {
          const uint32_t x = kr[r][k] ^ 0x80808080u;
          mma_f16(c[r], qa[k], codes_f16(x, 0x4140), codes_f16(x, 0x4342));
        } else {
          mma_bf16(c[r], qa[k], kr[r][2 * k], kr[r][2 * k + 1]);
          const uint32_t q2[4] = {qb[k][0], 0u, qb[k][1], 0u};
          mma_bf16(c[r], q2, kr[r][2 * k], kr[r][2 * k + 1]);
        }
      }
    }
    float s[4], sv[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      s[i] = (c[i >> 1][i & 1] + c[i >> 1][2 + (i & 1)]) * fs;
      if constexpr (I8) {
        s[i] *= ksc[i];
        sv[i] = vsc[i];
      }
    }
    // positions past the end or without a page
    bool ok[4];
    bool whole = c0 + tile * 16 + 16 <= c1;
    if constexpr (FAST)
      whole = whole && rows[tile] >= 0;
    else
      whole = false;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        ok[i] = c0 + tile * 16 + pos_of(i) < c1 && rows[FAST ? tile : tile * 16 + pos_of(i)] >= 0;
        if (!ok[i]) {
          s[i] = -INFINITY;
          sv[i] = 0.0f;
          // 0 times what is there might be NaN
#pragma unroll
          for (int w = 0; w < kVw; w++) vr[i][w] = 0;
        }
      }
    }
    if (more) load_k(tile + kPmWarps);
    if (a.scores && g < nh) {
      float *out = a.scores + ((size_t)b * a.n_head + h0 + g) * a.max_len;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int pos = c0 + tile * 16 + pos_of(i);
        if (pos < c1) out[pos] = s[i];
      }
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
      const float f = 0x1p15f / vlim;
#pragma unroll
      for (int i = 0; i < 4; i++) p[i] *= sv[i] * f;
      split_f16(p[0], p[1], pa[0], pa[1]);
      split_f16(p[2], p[3], pa[2], pa[3]);
    } else {
      split_bf16(p[0], p[1], pa[0], pa[1], pb[0]);
      split_bf16(p[2], p[3], pa[2], pa[3], pb[2]);
    }
#pragma unroll
    for (int w = 0; w < kVw; w++) {
      if constexpr (I8) {
        const uint32_t v0 = vr[0][w] ^ 0x80808080u, v1 = vr[1][w] ^ 0x80808080u, v2 = vr[2][w] ^ 0x80808080u,
                       v3 = vr[3][w] ^ 0x80808080u;
        const uint32_t x = __byte_perm(v0, v1, 0x5140), y = __byte_perm(v2, v3, 0x5140);
        const uint32_t z = __byte_perm(v0, v1, 0x7362), u = __byte_perm(v2, v3, 0x7362);
        mma_f16(acc[4 * w], pa, codes_f16(x, 0x4140), codes_f16(y, 0x4140));
        mma_f16(acc[4 * w + 1], pa, codes_f16(x, 0x4342), codes_f16(y, 0x4342));
        mma_f16(acc[4 * w + 2], pa, codes_f16(z, 0x4140), codes_f16(u, 0x4140));
        mma_f16(acc[4 * w + 3], pa, codes_f16(z, 0x4342), codes_f16(u, 0x4342));
      } else {
        const uint32_t x0 = __byte_perm(vr[0][w], vr[1][w], 0x5410), x1 = __byte_perm(vr[2][w], vr[3][w], 0x5410);
        const uint32_t y0 = __byte_perm(vr[0][w], vr[1][w], 0x7632), y1 = __byte_perm(vr[2][w], vr[3][w], 0x7632);
        mma_bf16(acc[2 * w], pa, x0, x1);
        mma_bf16(acc[2 * w + 1], pa, y0, y1);
        mma_bf16(acc[2 * w], pb, x0, x1);
        mma_bf16(acc[2 * w + 1], pb, y0, y1);
      }
    }
    if (more) load_v(tile + kPmWarps);
  }

  // join the warps: [warp][head][D sums, M, L]
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
  __syncthreads();
  for (int i = tid; i < nh * D; i += kPmWarps * 32) {
    const int h = i / D, d = i % D;
    const float *o = join + h * (D + 2);
    float M = -INFINITY, L = 0.0f, x = 0.0f;
#pragma unroll
    for (int w = 0; w < kPmWarps; w++) M = fmaxf(M, o[w * 8 * (D + 2) + D]);
    const float mu = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int w = 0; w < kPmWarps; w++) {
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
  for (int i = tid; i < nh * D; i += kPmWarps * 32) {
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
