// evict.cuh -- bounding a paged cache by accumulated attention weight.
//
// Of a row (layer, sequence, kv head) with more positions than the budget,
// the first `sinks` and the last `recent` stay, and of the others those with
// the largest weights (equal weights: the lower position first), `budget` in
// all. The kept positions move in their order to the pages of a second
// table, so the source pages, which other sequences may share, are only
// read.
#pragma once

#include "paged.cuh"

namespace llmq {

struct EvictArgs {
  PagedView c;
  PageTable src, dst;
  int layer0, n_layers, max_len, budget, sinks, recent;
  const int *lens;
  const float *w;
  long long w_stride;
  int *kept;  // [n_layers][n_seqs][n_kv_head][budget]
  float *wout;
  long long wout_stride;
  int *lens_out;
};

__device__ __forceinline__ int evict_len(const EvictArgs &a, int b) {
  const long long cap = (long long)a.src.cols * a.c.page_size;
  return max(0, min(min(a.lens[b], a.max_len), (int)min(cap, (long long)INT_MAX)));
}

// An unsigned key in the order of the floats; NaN is below every number and
// -0 equals 0.
__device__ __forceinline__ unsigned evict_key(float x) {
  if (x != x) return 0u;
  const unsigned u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kEvThreads = 1024;

// A thread's four weights from position j on, j a multiple of 4 (positions
// past the row's end: unspecified).
template <bool VEC>
__device__ __forceinline__ float4 evict_load(const float *w, int j, int len) {
  if (j >= len) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (VEC && j + 3 < len) return *(const float4 *)(w + j);
  return make_float4(w[j], j + 1 < len ? w[j + 1] : 0.0f, j + 2 < len ? w[j + 2] : 0.0f, j + 3 < len ? w[j + 3] : 0.0f);
}

// One CTA per row. The need-th largest key of the positions between the
// sinks and the recent ones by radix select: digits of 11, 11 and 10 bits
// from the top, each a histogram of the keys that agree with the digits
// found so far, in shared memory (integer atomics: exact). Then the kept
// positions in order: one prefix sum of (above the threshold or always kept,
// equal to it) per 4096 positions, of the equal ones the first `ties`. The
// row is read four times, but for the first time from L2.
// grid (n_layers * n_seqs * n_kv_head), 1024 threads.
template <bool VEC>
__global__ void __launch_bounds__(kEvThreads) evict_select_kernel(EvictArgs a) {
  __shared__ int hist[2048];
  __shared__ int wsum[32];
  __shared__ int s_bin, s_need;
  const int row = blockIdx.x, b = row / a.c.n_kv_head % a.src.n_seqs, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int len = evict_len(a, b), n = min(len, a.budget);
  const float *w = a.w + row * a.w_stride;
  float *wout = a.wout + row * a.wout_stride;
  int *kept = a.kept + (size_t)row * a.budget;
  if (row < a.src.n_seqs * a.c.n_kv_head && row % a.c.n_kv_head == 0 && tid == 0) a.lens_out[b] = n;
  for (long long j = n + tid; j < a.wout_stride; j += kEvThreads) wout[j] = 0.0f;
  for (int j = n + tid; j < a.budget; j += kEvThreads) kept[j] = -1;
  if (len <= a.budget) {
    for (int j = tid; j < len; j += kEvThreads) {
      kept[j] = j;
      wout[j] = w[j];
    }
    return;
  }
  const int lo = a.sinks, hi = len - a.recent;
  int need = a.budget - a.sinks - a.recent;
  unsigned thr = 0;  // the digits found, from the top
  if (need > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
      const unsigned known = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u;
      for (int i = tid; i < 2048; i += kEvThreads) hist[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (int j = tid * 4; j < hi; j += kEvThreads * 4) {
        const float4 x = evict_load<VEC>(w, j, hi);
        const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const unsigned key = evict_key(y[i]);
          if (j + i >= lo && j + i < hi && ((key ^ thr) & known) == 0) atomicAdd(&hist[key >> shift & (bins - 1)], 1);
        }
      }
      __syncthreads();
      // the bin of the need-th largest: bins from the top, two a thread
      const int b1 = 2047 - 2 * tid, h1 = hist[b1], h0 = hist[b1 - 1];
      int s = h1 + h0;
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
      }
      if (lane == 31) wsum[wid] = s;
      __syncthreads();
      if (wid == 0) {
        int t = wsum[lane];
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, t, o);
          if (lane >= o) t += u;
        }
        wsum[lane] = t;
      }
      __syncthreads();
      s += wid ? wsum[wid - 1] : 0;  // keys in this thread's bins and above
      const int above = s - h1 - h0;
      if (above < need && need <= s) {
        const bool first = need <= above + h1;
        s_bin = first ? b1 : b1 - 1;
        s_need = need - above - (first ? 0 : h1);
      }
      __syncthreads();
      thr |= (unsigned)s_bin << shift;
      need = s_need;
      __syncthreads();
    }
  } else {
    thr = 0xffffffffu;  // no key reaches it (NaN of any kind maps to 0)
  }
  // need is now how many of the keys equal to thr stay
  int base = 0, tbase = 0;
  for (int j0 = 0; j0 < len; j0 += kEvThreads * 4) {
    const int j = j0 + tid * 4;
    const float4 x = evict_load<VEC>(w, j, len);
    const float y[4] = {x.x, x.y, x.z, x.w};
    int flag[4], mine = 0;  // low half: kept whatever the ties; high half: equal to the threshold
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const unsigned key = evict_key(y[i]);
      const bool mid = j + i >= lo && j + i < hi;
      flag[i] = j + i >= len ? 0 : (!mid || key > thr) ? 1 : key == thr ? 0x10000 : 0;
      mine += flag[i];
    }
    int s = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += t;
    }
    if (lane == 31) wsum[wid] = s;
    __syncthreads();
    int t = wsum[lane];
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += u;
    }
    const int all = __shfl_sync(0xffffffffu, t, 31), before = wid ? __shfl_sync(0xffffffffu, t, max(wid - 1, 0)) : 0;
    s += before - mine;
    int sure = base + (s & 0xffff), ties = tbase + (s >> 16);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (flag[i] == 1 || (flag[i] && ties < need)) {
        const int at = sure + min(ties, need);
        kept[at] = j + i;
        wout[at] = y[i];
      }
      sure += flag[i] & 1;
      ties += flag[i] >> 16;
    }
    base += all & 0xffff;
    tbase += all >> 16;
    __syncthreads();
  }
}

constexpr int kEvPos = 64;  // kept positions that a CTA moves

// Moves the kept rows, key and value (and scales), of kEvPos positions of one
// row (layer, sequence, kv head) per CTA: 16-byte pieces, 8 in flight a
// thread. NV: pieces of a cache row.
template <int NV>
__global__ void __launch_bounds__(256) evict_move_kernel(EvictArgs a, int tiles) {
  __shared__ long long from[kEvPos], to[kEvPos];  // rows; from < 0: nothing to move
  const int row = blockIdx.x / tiles, j0 = blockIdx.x % tiles * kEvPos, tid = threadIdx.x;
  const int h = row % a.c.n_kv_head, b = row / a.c.n_kv_head % a.src.n_seqs;
  const int layer = a.layer0 + row / a.c.n_kv_head / a.src.n_seqs, ps = a.c.page_size;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the selection
  if (tid < kEvPos) {
    const int j = j0 + tid, s = j < a.budget ? a.kept[(size_t)row * a.budget + j] : -1;
    from[tid] = -1;
    if (s >= 0 && j / ps < a.dst.cols) {
      const int sp = a.src.page(b, s / ps), dp = a.dst.page(b, j / ps);
      if (sp >= 0 && sp < a.c.n_pages && dp >= 0 && dp < a.c.n_pages) {
        from[tid] = (long long)a.c.row(layer, sp, h, s % ps);
        to[tid] = (long long)a.c.row(layer, dp, h, j % ps);
        if (a.c.ks) {
          a.c.ks[to[tid]] = a.c.ks[from[tid]];
          a.c.vs[to[tid]] = a.c.vs[from[tid]];
        }
      }
    }
  }
  __syncthreads();
  constexpr int kAll = 2 * kEvPos * NV, kU = 8;
  for (int i0 = tid; i0 < kAll; i0 += 256 * kU) {
    uint4 x[kU];
#pragma unroll
    for (int u = 0; u < kU; u++) {
      const int i = i0 + u * 256, p = i / NV % kEvPos;
      if (i < kAll && from[p] >= 0)
        x[u] = __ldcs((const uint4 *)(i < kAll / 2 ? a.c.k : a.c.v) + from[p] * NV + i % NV);
    }
#pragma unroll
    for (int u = 0; u < kU; u++) {
      const int i = i0 + u * 256, p = i / NV % kEvPos;
      if (i < kAll && from[p] >= 0) ((uint4 *)(i < kAll / 2 ? a.c.k : a.c.v))[to[p] * NV + i % NV] = x[u];
    }
  }
}

}  // namespace llmq
