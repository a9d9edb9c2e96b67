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
  const int u = __float_as_int(x + 0.0f);
  const unsigned k = (unsigned)u ^ ((unsigned)(u >> 31) | 0x80000000u);
  return x != x ? 0u : k;
}

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
// found so far, in shared memory (integer atomics: exact). The second pass
// also lists the keys that agree, a few percent of a spread row, so that the
// third reads the list where it fits. Then the kept positions in order: one
// prefix sum of (above the threshold or always kept, equal to it) per 4 NTH
// positions, of the equal ones the first `ties`. The row is read three or
// four times, but for the first time from L2; instructions bound it, and, in
// short rows, barriers and latency: NTH 256 up to 2048 positions (144 rows of
// 1024, profiled alone: 9.5 us, 10.1 with 1024 threads and three times the
// instructions), 1024 beyond (256 rows of <=16384: 28 us).
// grid (n_layers * n_seqs * n_kv_head), NTH threads.
constexpr int kEvList = 4096;

template <bool VEC, int NTH>
__global__ void __launch_bounds__(NTH) evict_select_kernel(EvictArgs a) {
  constexpr int kBins = 2048, kPer = kBins / NTH, kW = NTH / 32;
  __shared__ int hist[kBins];
  __shared__ unsigned list[kEvList];
  __shared__ int wsum[kW];
  __shared__ int s_bin, s_need, s_listed;
  const int row = blockIdx.x, b = row / a.c.n_kv_head % a.src.n_seqs, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int len = evict_len(a, b), n = min(len, a.budget);
  const float *w = a.w + row * a.w_stride;
  float *wout = a.wout + row * a.wout_stride;
  int *kept = a.kept + (size_t)row * a.budget;
  if (row < a.src.n_seqs * a.c.n_kv_head && row % a.c.n_kv_head == 0 && tid == 0) a.lens_out[b] = n;
  for (int j = n + tid; j < a.budget; j += NTH) {
    kept[j] = -1;
    wout[j] = 0.0f;
  }
  if (len <= a.budget) {
    for (int j = tid; j < len; j += NTH) {
      kept[j] = j;
      wout[j] = w[j];
    }
    return;
  }
  // the sum of v over the threads up to and with this one; all: over all of them
  auto scan = [&](int v, int &all) {
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += t;
    }
    if (lane == 31) wsum[wid] = v;
    __syncthreads();
    int t = lane < kW ? wsum[lane] : 0;
    for (int o = 1; o < kW; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += u;
    }
    all = __shfl_sync(0xffffffffu, t, kW - 1);
    const int before = __shfl_sync(0xffffffffu, t, max(wid - 1, 0));
    return v + (wid ? before : 0);
  };
  const int lo = a.sinks, hi = len - a.recent;
  int need = a.budget - a.sinks - a.recent;
  unsigned thr = 0;  // the digits found, from the top
  if (need > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const unsigned mask = pass == 2 ? 1023u : 2047u;
      const unsigned known = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u;
      for (int i = tid; i < kBins; i += NTH) hist[i] = 0;
      if (tid == 0 && pass < 2) s_listed = 0;
      __syncthreads();
      auto count = [&](unsigned key) {
        if ((key ^ thr) & known) return;
        atomicAdd(&hist[key >> shift & mask], 1);
        if (pass == 1) {
          const int at = atomicAdd(&s_listed, 1);
          if (at < kEvList) list[at] = key;
        }
      };
      if (pass == 2 && s_listed <= kEvList) {
        for (int i = tid; i < s_listed; i += NTH) count(list[i]);
      } else {
#pragma unroll 2
        for (int j = tid * 4; j < hi; j += NTH * 4) {
          const float4 x = evict_load<VEC>(w, j, hi);
          const unsigned key[4] = {evict_key(x.x), evict_key(x.y), evict_key(x.z), evict_key(x.w)};
          if (j >= lo && j + 3 < hi) {
#pragma unroll
            for (int i = 0; i < 4; i++) count(key[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (j + i >= lo && j + i < hi) count(key[i]);
          }
        }
      }
      __syncthreads();
      // the bin of the need-th largest: bins from the top, kPer a thread
      const int top = kBins - 1 - kPer * tid;
      int mine = 0;
#pragma unroll
      for (int i = 0; i < kPer; i++) mine += hist[top - i];
      int all;
      const int upto = scan(mine, all), above = upto - mine;
      if (above < need && need <= upto) {
        int s = above, i = 0;
        while (s + hist[top - i] < need) s += hist[top - i++];
        s_bin = top - i;
        s_need = need - s;
      }
      __syncthreads();
      thr |= (unsigned)s_bin << shift;
      need = s_need;
    }
  } else {
    thr = 0xffffffffu;  // no key reaches it (NaN of any kind maps to 0)
  }
  // need is now how many of the keys equal to thr stay
  int base = 0, tbase = 0;
  for (int j0 = 0; j0 < len; j0 += NTH * 4) {
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
    __syncthreads();
    int all;
    const int before = scan(mine, all) - mine;
    int sure = base + (before & 0xffff), ties = tbase + (before >> 16);
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
  }
}

constexpr int kEvPos = 64;  // kept positions that a CTA moves

// Moves the kept rows, key and value (and scales), of kEvPos positions of one
// row (layer, sequence, kv head) per CTA: 16-byte pieces, 8 in flight a
// thread. A sequence of which a kept position has no page gets length -1
// (every CTA that sees one writes the same). NV: pieces of a cache row. Memory bounds it: 4 layers x 8 sequences
// x 8 heads, <=4096 rows of 256 bytes kept in each: 139 us at 6.1 TB/s; 144
// rows of 512 x 256 bytes, one and a half waves of CTAs: 15 us, 5.1 TB/s.
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
    if (s >= 0) {
      const int sp = a.src.page(b, s / ps), dp = j / ps < a.dst.cols ? a.dst.page(b, j / ps) : -1;
      const bool there = sp >= 0 && sp < a.c.n_pages;
      // nothing to move: slot j would hold what lay there before, and be attended to
      if (!there) a.lens_out[b] = -1;
      if (there && dp >= 0 && dp < a.c.n_pages) {
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
