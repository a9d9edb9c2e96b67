// paged.cuh -- a KV cache in pages and the attention of one new token per
// sequence over it.
//
// The pool holds keys and values as [layer][page][kv_head][slot][dim] in
// int8 (with a float32 scale per [layer][page][kv_head][slot], QuantKV[8]'s
// rule), bfloat16 or float32. A page of one key head is contiguous, so a
// tile of positions is one run of memory. Position j of sequence b is slot
// j % page_size of page table[b][j / page_size]; an entry outside
// [0, n_pages) is no page: nothing is stored there and its positions are
// masked.
#pragma once

#include "common.cuh"

namespace llmq {

struct PagedView {
  void *k, *v;
  float *ks, *vs;  // int8 only
  int kind, n_layer, n_pages, page_size, n_kv_head, head_dim;

  // Index of (layer, page, kv head, slot) in rows of head_dim elements.
  __host__ __device__ size_t row(int layer, int page, int h, int slot) const {
    return (((size_t)layer * n_pages + page) * n_kv_head + h) * page_size + slot;
  }
};

struct PageTable {
  const int *ids;  // [n_seqs] rows of cols entries
  long long stride;
  int cols, n_seqs;

  __device__ int page(int seq, int i) const { return ids[seq * stride + i]; }
};

// The element types of the pool.
struct PgInt8 {
  typedef int8_t T;
  static constexpr bool kScaled = true;
};
struct PgBf16 {
  typedef uint16_t T;
  static constexpr bool kScaled = false;
};
struct PgF32 {
  typedef float T;
  static constexpr bool kScaled = false;
};

struct StoreArgs {
  PagedView c;
  PageTable t;
  int layer, n_rows;
  const float *k, *v;
  long long k_stride, v_stride;
  const int *seq, *pos;
};

// Elements as the pool keeps them, four at a time.
template <typename E>
__device__ __forceinline__ void pack_store(typename E::T *dst, const float4 &x, float inv) {
  if constexpr (E::kScaled) {
    const int c0 = (int)roundf(x.x * inv) & 255, c1 = (int)roundf(x.y * inv) & 255, c2 = (int)roundf(x.z * inv) & 255,
              c3 = (int)roundf(x.w * inv) & 255;
    *(unsigned *)dst = c0 | c1 << 8 | c2 << 16 | c3 << 24;
  } else if constexpr (sizeof(typename E::T) == 2) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
    *(uint2 *)dst = make_uint2(*(const unsigned *)&a, *(const unsigned *)&b);
  } else {
    *(float4 *)dst = x;
  }
}

// A warp has one row and up to kStoreHeads heads per group of LG lanes (D / 4,
// and 8 of 32 idle at D = 96), key and value, four elements a lane: the row's
// page is looked up once, and 2 kStoreHeads loads are in flight a lane.
// int8: s = max|x| / 127 (1 when 0), codes round(x * (1 / s)), half away from
// zero, as QuantKV.quantize (kvcache.mojo:319-331). VEC: 16-byte loads
// (aligned rows). Memory bounds it: 16387 rows of 8 x 128 to bfloat16 take 33
// us at 6.2 TB/s (with the lookup in every head's lanes, 41). grid of 256
// threads over (row, block of heads).
constexpr int kStoreHeads = 4;

template <typename E, int D, bool VEC>
__global__ void __launch_bounds__(256) paged_store_kernel(StoreArgs a) {
  constexpr int LG = D == 96 ? 32 : D / 4, kG = 32 / LG, kH = kG * kStoreHeads;  // kH: heads of a warp
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x % LG, grp = threadIdx.x % 32 / LG, nh = a.c.n_kv_head, blocks = (nh + kH - 1) / kH;
  const unsigned w = blockIdx.x * 8 + threadIdx.x / 32, r = w / (unsigned)blocks;
  if (r >= (unsigned)a.n_rows) return;
  const int h0 = (int)(w - r * blocks) * kH + grp;
  const bool on = lane * 4 < D;
  const float *src[2] = {a.k + r * a.k_stride + h0 * D + lane * 4, a.v + r * a.v_stride + h0 * D + lane * 4};
  float4 x[kStoreHeads][2];
#pragma unroll
  for (int j = 0; j < kStoreHeads; j++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      x[j][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (!on || h0 + j * kG >= nh) continue;
      const float *p = src[i] + j * kG * D;
      if constexpr (VEC)
        x[j][i] = __ldcs((const float4 *)p);
      else
        x[j][i] = make_float4(p[0], p[1], p[2], p[3]);
    }
  const int pos = a.pos[r], sq = a.seq ? a.seq[r] : (int)r;
  if (pos < 0 || sq < 0 || sq >= a.t.n_seqs) return;
  const int pi = pos / a.c.page_size;
  if (pi >= a.t.cols) return;
  const int page = a.t.page(sq, pi);
  if (page < 0 || page >= a.c.n_pages) return;
  const size_t row0 = a.c.row(a.layer, page, h0, pos - pi * a.c.page_size);
#pragma unroll
  for (int j = 0; j < kStoreHeads; j++) {
    const size_t row = row0 + (size_t)(j * kG) * a.c.page_size;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      float inv = 0.0f, s = 1.0f;
      if constexpr (E::kScaled) {
        const float4 &y = x[j][i];
        float m = fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)));
#pragma unroll
        for (int o = LG / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        s = m / 127.0f;
        if (s == 0.0f) s = 1.0f;
        inv = 1.0f / s;
      }
      if (h0 + j * kG >= nh) continue;
      if (E::kScaled && lane == 0) (i ? a.c.vs : a.c.ks)[row] = s;
      if (on) pack_store<E>((typename E::T *)(i ? a.c.v : a.c.k) + row * D + lane * 4, x[j][i], inv);
    }
  }
}

struct AttendArgs {
  PagedView c;
  PageTable t;
  int layer, n_head, max_len;
  const float *q;
  float *out;
  long long q_stride, out_stride;
  bool q_vec;  // rows of q are 16-byte aligned
  const int *lens;
  float scale2;   // scale * log2(e): scores are exponents of two
  float *scores;  // [n_seqs][n_head][score_stride], for the weights; else null
  int score_stride;  // max_len to a multiple of 4
  float *stat;    // [n_seqs][n_head][2]: the maximum score M and the sum of 2^(score - M)
  // the split over positions (paged_mma.cuh)
  int chunk, splits, head_chunks, unit_heads;
  float *part;   // [unit][split][unit_heads][D + 4]: sums, then M and L of each head
  int *tickets;  // [unit], zero between launches
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The positions sequence b attends to.
__device__ __forceinline__ int paged_len(const AttendArgs &a, int b) {
  const long long cap = (long long)a.t.cols * a.c.page_size;
  return max(0, min(min(a.lens[b], a.max_len), (int)min(cap, (long long)INT_MAX)));
}

// Four floats from j on, of a row of n; VEC: aligned rows.
template <bool VEC>
__device__ __forceinline__ float4 row_load4(const float *p, int j, int n) {
  if (VEC && j + 3 < n) return *(const float4 *)(p + j);
  return make_float4(p[j], j + 1 < n ? p[j + 1] : 0.0f, j + 2 < n ? p[j + 2] : 0.0f, j + 3 < n ? p[j + 3] : 0.0f);
}

// weights_out[b][kv head][j] = weights[b][kv head][j] + sum over the kv
// head's query heads of their softmax weight of position j (0 past the
// length) for j < n: four positions a thread, the heads' scores (which the
// attention left in L2) in head order. Launched to overlap the attention's
// end. Latency and L2 bound it: about 6 us after 8 sequences x <=32768 with 4
// heads to a kv head (12 alone, with cold caches). grid (ceil(n / 1024), n_seqs * n_kv_head), 256 threads.
template <bool VEC>
__global__ void __launch_bounds__(256) paged_weights_kernel(AttendArgs a, int n, const float *win, float *wout,
                                                            long long stride) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int j = (blockIdx.x * 256 + threadIdx.x) * 4, G = a.n_head / a.c.n_kv_head;
  if (j >= n) return;
  for (int u = blockIdx.y; u < a.t.n_seqs * a.c.n_kv_head; u += gridDim.y) {
    const int b = u / a.c.n_kv_head, kh = u % a.c.n_kv_head, len = paged_len(a, b);
    if (j >= len && win == wout) continue;
    float4 w = win ? row_load4<VEC>(win + (size_t)u * stride, j, n) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (j < len) {
      const size_t r0 = (size_t)b * a.n_head + kh * G;
      float4 p = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // the heads' sum, rounded into w once
#pragma unroll 4
      for (int g = 0; g < G; g++) {
        const float4 s = *(const float4 *)(a.scores + (r0 + g) * a.score_stride + j);
        const float2 st = *(const float2 *)(a.stat + 2 * (r0 + g));
        const float M = st.x == -INFINITY ? 0.0f : st.x, inv = st.y > 0.0f ? 1.0f / st.y : st.y;
        p.x = fmaf(exp2_approx(s.x - M), inv, p.x);
        if (j + 1 < len) p.y = fmaf(exp2_approx(s.y - M), inv, p.y);
        if (j + 2 < len) p.z = fmaf(exp2_approx(s.z - M), inv, p.z);
        if (j + 3 < len) p.w = fmaf(exp2_approx(s.w - M), inv, p.w);
      }
      w.x += p.x, w.y += p.y, w.z += p.z, w.w += p.w;
    }
    float *o = wout + (size_t)u * stride + j;
    if (VEC && j + 3 < n) {
      *(float4 *)o = w;
    } else {
      o[0] = w.x;
      if (j + 1 < n) o[1] = w.y;
      if (j + 2 < n) o[2] = w.z;
      if (j + 3 < n) o[3] = w.w;
    }
  }
}

}  // namespace llmq
