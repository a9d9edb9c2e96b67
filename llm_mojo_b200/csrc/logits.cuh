// logits.cuh -- the rules between the head and the sampler: penalties for
// repeated tokens, biases and a mask of the allowed tokens.
//
// Each logit is read and written once, so memory bounds the call; the history
// touches a few percent of a row's tokens. Two ways, by size:
//  - small calls, one launch: each CTA counts its tile's tokens of the
//    history in shared memory beside its logits (logit_rules_kernel);
//  - large calls: the history and the biases scatter into per-token cells and
//    a bitmap of the touched tokens (logit_count_kernel); one pass streams the
//    others without waiting for anything (logit_stream_kernel); the touched
//    ones follow, each claimed through its bit by one of its occurrences
//    (logit_touch_kernel). Cells and bits are zero again afterwards.
#pragma once

#include "common.cuh"

namespace llmq {

struct RuleArgs {
  const float *x;
  float *out;
  long long x_stride, out_stride;
  int n, V, tiles;
  const float *repetition, *presence, *frequency;
  const int *ids, *n_ids, *n_prompt;
  long long ids_stride;
  int max_ids, n_bias;
  const int *bias_off, *bias_ids;
  const float *bias_val;
  const uint32_t *mask;
  long long mask_stride;
  unsigned long long *best;  // small calls: [n][tiles] each tile's largest key; large ones: [n], zero between calls
  int *tickets;              // [n], zero between calls
  int *argmax;               // or null
  // large calls, rows r0 on; zero between calls
  unsigned *bits;  // [n][words] touched tokens
  uint2 *cells;    // [n][V]: x as the counts below, y the bias
  int words, parts;  // parts: CTAs of a row's history and biases
};

// (ordered value, ~id): the largest key is the first of the largest logits;
// 0 for a logit that nothing picks (-inf and NaN).
__device__ __forceinline__ unsigned long long rule_key(float x, int id) {
  if (!(x > -INFINITY)) return 0ull;
  const unsigned u = __float_as_uint(x + 0.0f);
  const unsigned asc = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)asc << 32) | (unsigned)~id;
}

// The tile of one item, as a thread holds it.
template <int NG>
struct RuleTile {
  int r, t0, lo, hi;  // row; tokens: of the tile's first slot, of its first and past its last
  unsigned mine;      // bits of the tokens 32 lane .. of the warp's run: allowed and in the row
  float4 x[NG];
};

// The 32 bits of row's tokens v .. v + 31 (v from -3), those outside [0, V) 0.
__device__ __forceinline__ unsigned rule_bits(const uint32_t *row, int v, int V) {
  const uint32_t w0 = row[max(v, 0) >> 5], w1 = row[min(v + 31, V - 1) >> 5];
  return v >= 0 ? __funnelshift_r(w0, w1, v & 31) : w0 << -v;
}

// Each warp has a run of 32 VPT logits, a lane VPT / 4 groups of four,
// aligned to 16 bytes whatever the row's start (a row of odd length starts
// anywhere: the first group may begin before it).
template <int NTH, int VPT>
__device__ __forceinline__ void rule_open(const RuleArgs &a, int item, RuleTile<VPT / 4> &w) {
  const int lane = threadIdx.x & 31, tile = item % a.tiles;
  w.r = item / a.tiles;
  const float *xr = a.x + w.r * a.x_stride;
  const int lead = (int)(((uintptr_t)xr >> 2) & 3);  // logits between the 16-byte boundary and the row's start
  w.t0 = tile * NTH * VPT - lead;
  w.lo = max(w.t0, 0);
  w.hi = min(w.t0 + NTH * VPT, a.V);
  w.mine = 0;
  const int v = w.t0 + (threadIdx.x >> 5) * 32 * VPT + lane * 32;
  if (lane < VPT && v < w.hi && v + 32 > w.lo) {
    w.mine = 0xffffffffu;
    if (a.mask) w.mine = rule_bits(a.mask + w.r * a.mask_stride, v, a.V);
    if (v < 0) w.mine &= 0xffffffffu << -v;
    if (v + 32 > w.hi) w.mine &= 0xffffffffu >> (v + 32 - w.hi);
  }
}

// The allowed ones of group i's four tokens.
__device__ __forceinline__ unsigned rule_keep(unsigned mine, int i) {
  return __shfl_sync(0xffffffffu, mine, i * 4 + ((threadIdx.x & 31) >> 3)) >> (threadIdx.x & 7) * 4 & 15u;
}

template <int VPT>
__device__ __forceinline__ void rule_load(const RuleArgs &a, RuleTile<VPT / 4> &w) {
  const float *xr = a.x + w.r * a.x_stride;
  const int v0 = w.t0 + (threadIdx.x >> 5) * 32 * VPT + (threadIdx.x & 31) * 4;
#pragma unroll
  for (int i = 0; i < VPT / 4; i++) {
    const unsigned keep = rule_keep(w.mine, i);
    const int v = v0 + i * 128;
    w.x[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (!keep) continue;
    if (v >= 0 && v + 3 < a.V) {
      w.x[i] = *(const float4 *)(xr + v);
    } else {
      if (keep & 1u) w.x[i].x = xr[v];
      if (keep & 2u) w.x[i].y = xr[v + 1];
      if (keep & 4u) w.x[i].z = xr[v + 2];
      if (keep & 8u) w.x[i].w = xr[v + 3];
    }
  }
}

// One CTA per (row, tile of NTH VPT logits). The mask is read first, a word
// per lane, and only groups that it leaves something of are loaded: a
// grammar's mask spares most of the read. While those loads are in flight
// the history is counted in shared memory (integer atomics: any order gives
// the same counts; each CTA reads the whole history and keeps its tile's
// tokens) and the biases are laid out; then every rule is applied in
// registers. The row's last CTA joins the tiles' argmax (exact in any
// order).
// Dynamic shared memory: 4 bytes per logit of the tile for a history, and
// for a bias.
template <int NTH, int VPT>
__global__ void __launch_bounds__(NTH) logit_rules_kernel(RuleArgs a) {
  constexpr int T = NTH * VPT, NG = VPT / 4;
  extern __shared__ __align__(16) unsigned rsm[];
  __shared__ unsigned long long red[NTH / 32];
  unsigned *cnt = rsm;                             // bit 31: in the prompt; the rest: times in the answer
  float *bias = (float *)(rsm + (a.ids ? T : 0));  // of the tile
  const int tid = threadIdx.x, lane = tid & 31, r = blockIdx.x / a.tiles;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // the first quads of each thread's history, on their way with the logits
  const int *ids = a.ids ? a.ids + r * a.ids_stride : nullptr;
  const int first = (int)((4 - (((uintptr_t)ids >> 2) & 3)) & 3);  // ids before a 16-byte boundary
  const int quads = a.ids ? max(a.max_ids - first, 0) / 4 : 0;
  const int4 *q4 = (const int4 *)(ids + first);
  int4 early[2];
#pragma unroll
  for (int j = 0; j < 2; j++)
    if (tid + j * NTH < quads) early[j] = q4[tid + j * NTH];
  RuleTile<NG> w;
  rule_open<NTH, VPT>(a, blockIdx.x, w);
  rule_load<VPT>(a, w);
  if (a.ids || a.bias_off) {
    uint4 *z = (uint4 *)rsm;
    const int n = ((a.ids ? T : 0) + (a.bias_off ? T : 0)) / 4;
#pragma unroll 4
    for (int i = tid; i < n; i += NTH) z[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  if (a.ids) {
    const int H = min(max(0, a.n_ids[r]), a.max_ids), P = a.n_prompt ? a.n_prompt[r] : 0;
    const unsigned span = w.hi - w.lo;
    unsigned *c0 = cnt + (w.lo - w.t0);
    auto count = [&](int i, int id) {
      const unsigned k = (unsigned)id - (unsigned)w.lo;
      if (k < span && i < H) {
        if (i >= P)
          atomicAdd(&c0[k], 1u);
        else
          atomicOr(&c0[k], 0x80000000u);
      }
    };
    auto count4 = [&](int q, const int4 &v) {
      const int i = first + 4 * q;
      count(i, v.x);
      count(i + 1, v.y);
      count(i + 2, v.z);
      count(i + 3, v.w);
    };
    if (tid < min(first, H)) count(tid, ids[tid]);
#pragma unroll
    for (int j = 0; j < 2; j++)
      if (tid + j * NTH < quads) count4(tid + j * NTH, early[j]);
    const int end = min(quads, (max(H - first, 0) + 3) / 4);
    for (int q = tid + 2 * NTH; q < end; q += 4 * NTH) {
      int4 v[4];
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = q4[min(q + j * NTH, end - 1)];
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (q + j * NTH < end) count4(q + j * NTH, v[j]);
    }
    const int rest = first + quads * 4 + tid;
    if (rest < H) count(rest, ids[rest]);
  }
  if (a.bias_off) {
    const int b0 = max(a.bias_off[r], 0), b1 = min(a.bias_off[r + 1], a.n_bias);
    for (int i = b0 + tid; i < b1; i += NTH) {
      const int id = a.bias_ids[i];
      if (id < w.lo || id >= w.hi || (i > b0 && a.bias_ids[i - 1] == id)) continue;
      float s = a.bias_val[i];
      for (int e = i + 1; e < b1 && a.bias_ids[e] == id; e++) s += a.bias_val[e];
      bias[id - w.t0] = s;
    }
  }
  if (a.ids || a.bias_off) __syncthreads();
  const float rep = a.repetition ? a.repetition[r] : 1.0f, fr = a.frequency ? a.frequency[r] : 0.0f,
              pr = a.presence ? a.presence[r] : 0.0f;
  float *outr = a.out + r * a.out_stride;
  const bool vec_out = (((uintptr_t)(outr + w.t0) >> 2) & 3) == 0;
  const int at0 = (tid >> 5) * 32 * VPT + lane * 4;  // the thread's group i: at0 + 128 i
  float bv = -INFINITY;                              // the thread's largest logit and its token, first of equals
  int bt = -1;
#pragma unroll
  for (int i = 0; i < NG; i++) {
    const unsigned keep = rule_keep(w.mine, i);
    const int at = at0 + i * 128, v = w.t0 + at;
    if (v >= w.hi || v + 3 < w.lo) continue;
    float y[4] = {w.x[i].x, w.x[i].y, w.x[i].z, w.x[i].w};
    if (a.ids) {
      const uint4 c4 = *(const uint4 *)(cnt + at);
      const unsigned c[4] = {c4.x, c4.y, c4.z, c4.w};
      if (c4.x | c4.y | c4.z | c4.w) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const unsigned co = c[j] & 0x7fffffffu;
          if (c[j]) y[j] = y[j] > 0.0f ? y[j] / rep : y[j] * rep;
          if (co) y[j] = (y[j] - fr * (float)co) - pr;
        }
      }
    }
    if (a.bias_off) {
      const float4 b4 = *(const float4 *)(bias + at);
      y[0] += b4.x;
      y[1] += b4.y;
      y[2] += b4.z;
      y[3] += b4.w;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (!(keep >> j & 1u)) y[j] = -INFINITY;
      if (y[j] > bv) {
        bv = y[j];
        bt = v + j;
      }
    }
    if (vec_out && v >= w.lo && v + 3 < w.hi) {
      *(float4 *)(outr + v) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (v + j >= w.lo && v + j < w.hi) outr[v + j] = y[j];
    }
  }
  if (!a.argmax) return;
  unsigned long long k = rule_key(bv, bt);
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  if (lane == 0) red[tid >> 5] = k;
  __syncthreads();
  if (tid >= 32) return;
  k = lane < NTH / 32 ? red[lane] : 0ull;
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  int last = a.tiles == 1;
  if (!last) {
    unsigned long long *best = a.best + (size_t)r * a.tiles;
    if (lane == 0) {
      best[blockIdx.x % a.tiles] = k;
      __threadfence();
      last = atomicAdd(&a.tickets[r], 1) == a.tiles - 1;
      if (last) __threadfence();
    }
    last = __shfl_sync(0xffffffffu, last, 0);
    if (last) {
      for (int i = lane; i < a.tiles; i += 32) k = max(k, __ldcg(best + i));
      for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
      if (lane == 0) a.tickets[r] = 0;
    }
  }
  if (last && lane == 0) a.argmax[r] = k ? (int)~(unsigned)k : -1;
}

// ---- large calls -------------------------------------------------------------

constexpr int kTouchThreads = 512, kTouchPer = 2048;  // history ids and biases of a CTA

// A row's entry i: history ids, then biases. Returns the token, or -1.
__device__ __forceinline__ int rule_entry(const RuleArgs &a, int r, int i, int H, int b0) {
  const int id = i < H ? a.ids[r * a.ids_stride + i] : a.bias_ids[b0 + i - H];
  return id >= 0 && id < a.V ? id : -1;
}
// How many entries row r has; of them H are history, and its biases start at b0.
__device__ __forceinline__ int rule_entries(const RuleArgs &a, int r, int &H, int &b0) {
  H = a.ids ? min(max(0, a.n_ids[r]), a.max_ids) : 0;
  b0 = a.bias_off ? max(a.bias_off[r], 0) : 0;
  return H + (a.bias_off ? max(min(a.bias_off[r + 1], a.n_bias) - b0, 0) : 0);
}

// grid n * parts
__global__ void __launch_bounds__(kTouchThreads) logit_count_kernel(RuleArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int r = blockIdx.x / a.parts;
  int H, b0;
  const int total = rule_entries(a, r, H, b0), P = a.n_prompt ? a.n_prompt[r] : 0;
  for (int i = blockIdx.x % a.parts * kTouchThreads + threadIdx.x; i < total; i += a.parts * kTouchThreads) {
    const int id = rule_entry(a, r, i, H, b0);
    if (id < 0) continue;
    uint2 *cell = a.cells + (size_t)r * a.V + id;
    if (i < H) {
      if (i >= P)
        atomicAdd(&cell->x, 1u);
      else
        atomicOr(&cell->x, 0x80000000u);
    } else {
      // the first of equal ids adds them up, in order
      const int j = b0 + i - H, end = b0 + total - H;
      if (j > b0 && a.bias_ids[j - 1] == id) continue;
      float s = a.bias_val[j];
      for (int e = j + 1; e < end && a.bias_ids[e] == id; e++) s += a.bias_val[e];
      cell->y = __float_as_uint(s);
    }
    atomicOr(&a.bits[(size_t)r * a.words + (id >> 5)], 1u << (id & 31));
  }
}

// Every token that nothing touched: allowed ones as they are, others
// -infinity. One CTA per (row, tile of 4096), as in logit_rules_kernel but
// for a thread's own groups only: no barrier, no shared memory. The largest
// logit goes to the row's key by one atomic maximum a warp.
__global__ void __launch_bounds__(256) logit_stream_kernel(RuleArgs a) {
  constexpr int VPT = 16, NG = VPT / 4;
  const int lane = threadIdx.x & 31;
  RuleTile<NG> w;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  rule_open<256, VPT>(a, blockIdx.x, w);
  unsigned touched = 0;
  const int v0 = w.t0 + (threadIdx.x >> 5) * 32 * VPT;
  if (a.bits && lane < VPT && v0 + lane * 32 < w.hi && v0 + lane * 32 + 32 > w.lo)
    touched = rule_bits(a.bits + (size_t)w.r * a.words, v0 + lane * 32, a.V);
  w.mine &= ~touched;
  rule_load<VPT>(a, w);
  float *outr = a.out + w.r * a.out_stride;
  const bool vec_out = (((uintptr_t)(outr + w.t0) >> 2) & 3) == 0;
  float bv = -INFINITY;
  int bt = INT_MAX;
#pragma unroll
  for (int i = 0; i < NG; i++) {
    const int v = v0 + i * 128 + lane * 4;
    const unsigned skip = __shfl_sync(0xffffffffu, touched, i * 4 + (lane >> 3)) >> (lane & 7) * 4 & 15u;
    const unsigned keep = rule_keep(w.mine, i);
    if (v >= w.hi || v + 3 < w.lo) continue;
    float y[4] = {w.x[i].x, w.x[i].y, w.x[i].z, w.x[i].w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (!(keep >> j & 1u)) y[j] = -INFINITY;
      if (y[j] > bv) {
        bv = y[j];
        bt = v + j;
      }
    }
    if (vec_out && v >= w.lo && v + 3 < w.hi && !skip) {
      *(float4 *)(outr + v) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (v + j >= w.lo && v + j < w.hi && !(skip >> j & 1u)) outr[v + j] = y[j];
    }
  }
  if (!a.argmax) return;
  const unsigned long long k = rule_key(bv, bt);
  const unsigned top = __reduce_max_sync(0xffffffffu, (unsigned)(k >> 32));
  if (!top) return;
  const unsigned first = __reduce_max_sync(0xffffffffu, (unsigned)(k >> 32) == top ? (unsigned)k : 0u);
  if (lane == 0) atomicMax(&a.best[w.r], ((unsigned long long)top << 32) | first);
}

// The touched tokens, and the row's argmax. grid n * parts; the row's last
// part finishes it.
__global__ void __launch_bounds__(kTouchThreads) logit_touch_kernel(RuleArgs a) {
  __shared__ unsigned long long red[kTouchThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int r = blockIdx.x / a.parts, lane = threadIdx.x & 31;
  int H, b0;
  const int total = rule_entries(a, r, H, b0);
  const float rep = a.repetition ? a.repetition[r] : 1.0f, fr = a.frequency ? a.frequency[r] : 0.0f,
              pr = a.presence ? a.presence[r] : 0.0f;
  unsigned long long best = 0;
  for (int i = blockIdx.x % a.parts * kTouchThreads + threadIdx.x; i < total; i += a.parts * kTouchThreads) {
    const int id = rule_entry(a, r, i, H, b0);
    if (id < 0) continue;
    unsigned *word = &a.bits[(size_t)r * a.words + (id >> 5)];
    if (!(*(volatile unsigned *)word >> (id & 31) & 1u)) continue;  // done by another occurrence
    if (!(atomicAnd(word, ~(1u << (id & 31))) >> (id & 31) & 1u)) continue;
    uint2 *cell = a.cells + (size_t)r * a.V + id;
    const uint2 c = __ldcg(cell);
    float y = a.x[r * a.x_stride + id];
    const unsigned co = c.x & 0x7fffffffu;
    if (c.x) y = y > 0.0f ? y / rep : y * rep;
    if (co) y = (y - fr * (float)co) - pr;
    y += __uint_as_float(c.y);
    if (a.mask && !(a.mask[r * a.mask_stride + (id >> 5)] >> (id & 31) & 1u)) y = -INFINITY;
    a.out[r * a.out_stride + id] = y;
    *cell = make_uint2(0u, 0u);
    best = max(best, rule_key(y, id));
  }
  if (!a.argmax) return;
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) red[threadIdx.x >> 5] = best;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < kTouchThreads / 32; i++) best = max(best, red[i]);
  if (a.parts > 1) {
    atomicMax(&a.best[r], best);
    __threadfence();
    if (atomicAdd(&a.tickets[r], 1) != a.parts - 1) return;
    __threadfence();
    a.tickets[r] = 0;
  }
  best = max(best, __ldcg(&a.best[r]));
  a.best[r] = 0;
  a.argmax[r] = best ? (int)~(unsigned)best : -1;
}

}  // namespace llmq
