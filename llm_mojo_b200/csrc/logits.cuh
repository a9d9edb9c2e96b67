// logits.cuh -- the rules between the head and the sampler: penalties for
// repeated tokens, biases and a mask of the allowed tokens.
//
// Each logit is read and written once, so memory bounds a call in the end:
// 256 x 50257 without rules takes 20 us, 5.2 TB/s (torch.mul from the same
// rows to others 16.6 us). With every rule 33 us, 3.2 TB/s: 830
// instructions a warp per 512 logits, 440 of them without rules, fill 73% of
// the issue slots, and CTAs wait at their barriers for the history. Tried and
// slower: persistent CTAs with the next tile's loads ahead (66 us), counts
// scattered into per-token cells in global memory before one streaming pass
// (67), the touched tokens listed and worked out by a thread each (35.5) or
// dealt to each warp's lanes (35.6), tiles of 8192 (38). One row: 5 us, the
// latency of a CTA and of the tickets.
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
  unsigned long long *best;  // [n][tiles * warps] keys of the warps' largest logits
  int *tickets;              // [n], zero between launches; null: logit_argmax_kernel follows
  int *argmax;               // or null
};

// (ordered value, ~id): the largest key is the first of the largest logits;
// 0 for a logit that nothing picks (-inf and NaN).
__device__ __forceinline__ unsigned long long rule_key(float x, int id) {
  if (!(x > -INFINITY)) return 0ull;
  const unsigned u = __float_as_uint(x + 0.0f);
  const unsigned asc = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)asc << 32) | (unsigned)~id;
}

// The 32 bits of row's tokens v .. v + 31 (v from -3), those outside [0, V) 0.
__device__ __forceinline__ unsigned rule_bits(const uint32_t *row, int v, int V) {
  const uint32_t w0 = row[max(v, 0) >> 5], w1 = row[min(v + 31, V - 1) >> 5];
  return v >= 0 ? __funnelshift_r(w0, w1, v & 31) : w0 << -v;
}

// The largest of a row's keys: argmax[r] = its token, -1 when there is none.
__device__ __forceinline__ void rule_finish(const unsigned long long *best, int n, int *argmax) {
  unsigned long long k = 0;
  for (int i = threadIdx.x & 31; i < n; i += 32) k = max(k, __ldcg(best + i));
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  if ((threadIdx.x & 31) == 0) *argmax = k ? (int)~(unsigned)k : -1;
}

// One CTA per (row, tile of NTH VPT logits). Each warp has a run of 32 VPT
// logits, a lane VPT / 4 groups of four, aligned to 16 bytes whatever the
// row's start (a row of odd length starts anywhere: the first group may begin
// before it). The mask is read first, a word per lane, and only groups that
// it leaves something of are loaded: a grammar's mask spares most of the
// read. While those loads are in flight the history is counted in shared
// memory (integer atomics: any order gives the same counts; each CTA reads
// the whole history and keeps its tile's tokens) and the biases are laid out,
// marked in a bitmap; then every rule is applied in registers. A thread keeps
// the largest value only; its token is looked up by the lanes that hold the
// warp's largest (the first of equals, in any order of the warps).
// Dynamic shared memory: 4 bytes per logit of the tile for a history, and
// for a bias.
template <int NTH, int VPT>
__global__ void __launch_bounds__(NTH) logit_rules_kernel(RuleArgs a) {
  constexpr int T = NTH * VPT, NG = VPT / 4;
  extern __shared__ __align__(16) unsigned rsm[];
  __shared__ unsigned biased[T / 32];  // bit of a slot: it has a bias
  unsigned *cnt = rsm;                 // bit 31: in the prompt; the rest: times in the answer
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x / a.tiles, tile = blockIdx.x - r * a.tiles;
  float *bias = (float *)(rsm + (a.ids ? T : 0));  // of the tile, where there is one
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float *xr = a.x + r * a.x_stride;
  const int lead = (int)(((uintptr_t)xr >> 2) & 3);  // logits between the 16-byte boundary and the row's start
  // the tile's tokens: [lo, hi), none in a last tile that only a row of a larger lead has tokens in
  const int t0 = tile * T - lead, lo = max(t0, 0), hi = max(lo, min(t0 + T, a.V));
  const bool inner = t0 >= 0 && t0 + T <= a.V;
  const int at0 = warp * 32 * VPT + lane * 4;  // the thread's group i: slots at0 + 128 i on
  // the first quads of each thread's history, on their way with the logits
  const int *ids = a.ids ? a.ids + r * a.ids_stride : nullptr;
  const int first = (int)((4 - (((uintptr_t)ids >> 2) & 3)) & 3);  // ids before a 16-byte boundary
  const int quads = a.ids ? max(a.max_ids - first, 0) / 4 : 0;
  const int4 *q4 = (const int4 *)(ids + first);
  int4 early[2];
#pragma unroll
  for (int j = 0; j < 2; j++)
    if (tid + j * NTH < quads) early[j] = q4[tid + j * NTH];
  const int H = a.ids ? min(max(0, a.n_ids[r]), a.max_ids) : 0, P = a.n_prompt ? a.n_prompt[r] : 0;
  const int b0 = a.bias_off ? max(a.bias_off[r], 0) : 0, b1 = a.bias_off ? min(a.bias_off[r + 1], a.n_bias) : 0;
  // bits of the slots 32 lane .. 32 lane + 31 of the warp's run: in the row, and allowed
  unsigned mine = 0xffffffffu;
  if ((a.mask || !inner) && lane < VPT) {
    const int v = t0 + warp * 32 * VPT + lane * 32;
    if (v < hi && v + 32 > lo) {
      if (a.mask) mine = rule_bits(a.mask + r * a.mask_stride, v, a.V);
      if (v < 0) mine &= 0xffffffffu << -v;
      if (v + 32 > hi) mine &= 0xffffffffu >> (v + 32 - hi);
    } else {
      mine = 0;
    }
  }
  float4 x[NG];
  unsigned keep = 0;  // four bits a group
  if (a.mask || !inner) {
#pragma unroll
    for (int i = 0; i < NG; i++) {
      const unsigned k = __shfl_sync(0xffffffffu, mine, i * 4 + (lane >> 3)) >> (lane & 7) * 4 & 15u;
      const int v = t0 + at0 + i * 128;
      keep |= k << (4 * i);
      x[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (!k) continue;
      if (v >= 0 && v + 3 < a.V) {
        x[i] = *(const float4 *)(xr + v);
      } else {
        if (k & 1u) x[i].x = xr[v];
        if (k & 2u) x[i].y = xr[v + 1];
        if (k & 4u) x[i].z = xr[v + 2];
        if (k & 8u) x[i].w = xr[v + 3];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NG; i++) x[i] = *(const float4 *)(xr + t0 + at0 + i * 128);
  }
  if (H || b1 > b0) {
    if (H) {
#pragma unroll
      for (int i = 0; i < NG; i++) ((uint4 *)cnt)[tid + i * NTH] = make_uint4(0, 0, 0, 0);
    }
    if (b1 > b0 && tid < T / 32) biased[tid] = 0;
    __syncthreads();
    const unsigned span = hi - lo;
    unsigned *c0 = cnt + (lo - t0);
    auto count = [&](int i, int id) {
      const unsigned k = (unsigned)id - (unsigned)lo;
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
    const int end = min(quads, (max(H - first, 0) + 3) / 4);
    if (tid < min(first, H)) count(tid, ids[tid]);
#pragma unroll
    for (int j = 0; j < 2; j++)
      if (tid + j * NTH < end) count4(tid + j * NTH, early[j]);
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
    for (int i = b0 + tid; i < b1; i += NTH) {
      const int id = a.bias_ids[i];
      if (id < lo || id >= hi || (i > b0 && a.bias_ids[i - 1] == id)) continue;
      float s = a.bias_val[i];  // the first of equal ids adds them up, in order
      for (int e = i + 1; e < b1 && a.bias_ids[e] == id; e++) s += a.bias_val[e];
      bias[id - t0] = s;
      atomicOr(&biased[(id - t0) >> 5], 1u << ((id - t0) & 31));
    }
    __syncthreads();
  }
  const float rep = a.repetition ? a.repetition[r] : 1.0f, fr = a.frequency ? a.frequency[r] : 0.0f,
              pr = a.presence ? a.presence[r] : 0.0f;
  const unsigned bword = b1 > b0 && lane < VPT ? biased[warp * VPT + lane] : 0u;
  const bool anyb = __any_sync(0xffffffffu, bword != 0u);
  float *outr = a.out + r * a.out_stride + t0;
  const bool vec_out = ((uintptr_t)outr & 15) == 0;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NG; i++) {
    const int at = at0 + i * 128;
    float y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    if (H) {
      const uint4 c4 = *(const uint4 *)(cnt + at);
      if (c4.x | c4.y | c4.z | c4.w) {
        const unsigned c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const unsigned co = c[j] & 0x7fffffffu;
          if (c[j]) y[j] = y[j] > 0.0f ? y[j] / rep : y[j] * rep;
          if (co) y[j] = (y[j] - fr * (float)co) - pr;
        }
      }
    }
    if (anyb) {
      const unsigned bb = __shfl_sync(0xffffffffu, bword, i * 4 + (lane >> 3)) >> (lane & 7) * 4 & 15u;
      if (bb) {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (bb >> j & 1u) y[j] += bias[at + j];
      }
    }
    if (a.mask || !inner) {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (!(keep >> (4 * i + j) & 1u)) y[j] = -INFINITY;
    }
    top = fmaxf(fmaxf(fmaxf(top, y[0]), fmaxf(y[1], y[2])), y[3]);
    x[i] = make_float4(y[0], y[1], y[2], y[3]);
    if (vec_out && (inner || (t0 + at >= lo && t0 + at + 3 < hi))) {
      *(float4 *)(outr + at) = x[i];
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (t0 + at + j >= lo && t0 + at + j < hi) outr[at + j] = y[j];
    }
  }
  if (!a.argmax) return;
  const unsigned value = (unsigned)(rule_key(top, 0) >> 32), most = __reduce_max_sync(0xffffffffu, value);
  unsigned token = 0xffffffffu;
  if (most && value == most) {
#pragma unroll
    for (int i = NG - 1; i >= 0; i--) {
      const float y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int j = 3; j >= 0; j--)
        if (y[j] == top) token = t0 + at0 + i * 128 + j;
    }
  }
  token = __reduce_min_sync(0xffffffffu, token);
  unsigned long long *best = a.best + (size_t)r * a.tiles * (NTH / 32);
  if (lane == 0) best[tile * (NTH / 32) + warp] = most ? ((unsigned long long)most << 32) | (unsigned)~token : 0ull;
  if (!a.tickets) return;
  __threadfence();
  __syncthreads();
  if (tid >= 32) return;
  int last = 0;
  if (lane == 0) {
    last = atomicAdd(&a.tickets[r], 1) == a.tiles - 1;
    __threadfence();
    if (last) a.tickets[r] = 0;
  }
  if (__shfl_sync(0xffffffffu, last, 0)) rule_finish(best, a.tiles * (NTH / 32), a.argmax + r);
}

// grid ceil(n / 4), 128 threads: a warp per row of `keys` keys.
__global__ void __launch_bounds__(128) logit_argmax_kernel(const unsigned long long *best, int keys, int *argmax, int n) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 5);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (r < n) rule_finish(best + (size_t)r * keys, keys, argmax + r);
}

}  // namespace llmq
