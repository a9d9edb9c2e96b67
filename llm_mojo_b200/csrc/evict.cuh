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

// One CTA per row: the need-th largest key of the middle positions by
// bisection over its bits (32 counts of the row), then the kept positions by
// prefix sums in order. grid (n_layers * n_seqs * n_kv_head), 1024 threads.
__global__ void __launch_bounds__(1024) evict_select_kernel(EvictArgs a) {
  __shared__ int part[33], part2[33];
  const int row = blockIdx.x, b = row / a.c.n_kv_head % a.src.n_seqs, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int len = evict_len(a, b), n = min(len, a.budget);
  const float *w = a.w + row * a.w_stride;
  float *wout = a.wout + row * a.wout_stride;
  int *kept = a.kept + (size_t)row * a.budget;
  if (row < a.src.n_seqs * a.c.n_kv_head && row % a.c.n_kv_head == 0 && tid == 0) a.lens_out[b] = n;
  for (long long j = n + tid; j < a.wout_stride; j += 1024) wout[j] = 0.0f;
  for (int j = n + tid; j < a.budget; j += 1024) kept[j] = -1;
  if (len <= a.budget) {
    for (int j = tid; j < len; j += 1024) {
      kept[j] = j;
      wout[j] = w[j];
    }
    return;
  }
  const int lo = a.sinks, hi = len - a.recent, need = a.budget - a.sinks - a.recent;
  auto block_sum = [&](int v) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) part[wid] = v;
    __syncthreads();
    int t = 0;
    for (int i = 0; i < 32; i++) t += part[i];
    return t;
  };
  // the largest key that at least `need` positions reach
  unsigned thr = 0;
  for (int bit = 31; bit >= 0; bit--) {
    const unsigned t = thr | (1u << bit);
    int c = 0;
    for (int j = lo + tid; j < hi; j += 1024) c += evict_key(w[j]) >= t;
    if (block_sum(c) >= need) thr = t;
  }
  int above = 0;
  for (int j = lo + tid; j < hi; j += 1024) above += evict_key(w[j]) > thr;
  const int ties = need - block_sum(above);  // how many of the equal ones stay
  int base = 0, tbase = 0;
  for (int j0 = 0; j0 < len; j0 += 1024) {
    const int j = j0 + tid;
    const bool mid = j >= lo && j < hi;
    const unsigned key = mid ? evict_key(w[j]) : 0u;
    const bool eq = mid && key == thr;
    const unsigned eb = __ballot_sync(0xffffffffu, eq);
    __syncthreads();
    if (lane == 0) part2[wid] = __popc(eb);
    __syncthreads();
    int before = tbase + __popc(eb & ((1u << lane) - 1)), tall = 0;
    for (int i = 0; i < 32; i++) {
      if (i < wid) before += part2[i];
      tall += part2[i];
    }
    const bool keep = j < len && (!mid || key > thr || (eq && before < ties));
    const unsigned kb = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) part[wid] = __popc(kb);
    __syncthreads();
    int at = base + __popc(kb & ((1u << lane) - 1)), all = 0;
    for (int i = 0; i < 32; i++) {
      if (i < wid) at += part[i];
      all += part[i];
    }
    if (keep) {
      kept[at] = j;
      wout[at] = w[j];
    }
    base += all;
    tbase += tall;
  }
}

// Moves the kept rows: one warp per (row, kept position), key and value (and
// scales). grid over warps, 256 threads.
__global__ void __launch_bounds__(256) evict_move_kernel(EvictArgs a, int row_bytes) {
  const long long gw = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long long row = gw / a.budget;
  const int j = (int)(gw % a.budget);
  if (row >= (long long)a.n_layers * a.src.n_seqs * a.c.n_kv_head) return;
  const int h = row % a.c.n_kv_head, b = (int)(row / a.c.n_kv_head % a.src.n_seqs);
  const int layer = a.layer0 + (int)(row / a.c.n_kv_head / a.src.n_seqs);
  const int s = a.kept[row * a.budget + j], ps = a.c.page_size;
  if (s < 0 || j / ps >= a.dst.cols) return;
  const int sp = a.src.page(b, s / ps), dp = a.dst.page(b, j / ps);
  if (sp < 0 || sp >= a.c.n_pages || dp < 0 || dp >= a.c.n_pages) return;
  const size_t from = a.c.row(layer, sp, h, s % ps), to = a.c.row(layer, dp, h, j % ps);
  for (int i = lane * 4; i < row_bytes; i += 128) {
    *(uint32_t *)((char *)a.c.k + to * row_bytes + i) = *(const uint32_t *)((const char *)a.c.k + from * row_bytes + i);
    *(uint32_t *)((char *)a.c.v + to * row_bytes + i) = *(const uint32_t *)((const char *)a.c.v + from * row_bytes + i);
  }
  if (a.c.ks && lane == 0) {
    a.c.ks[to] = a.c.ks[from];
    a.c.vs[to] = a.c.vs[from];
  }
}

}  // namespace llmq
