// logits.cuh -- the rules between the head and the sampler: penalties for
// repeated tokens, biases and a mask of the allowed tokens.
#pragma once

#include "common.cuh"

namespace llmq {

constexpr int kRuleTile = 4096;  // logits of one CTA

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
  unsigned long long *best;  // [n][tiles] (ordered value, ~id) of each tile's largest logit; or null
};

// 0 for a logit that nothing picks (-inf and NaN).
__device__ __forceinline__ unsigned long long rule_key(float x, int id) {
  if (!(x > -INFINITY)) return 0ull;
  const unsigned u = __float_as_uint(x + 0.0f);
  const unsigned asc = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)asc << 32) | (unsigned)~id;
}

// One CTA per (row, tile): the history's counts of the tile's tokens in
// shared memory (integer atomics: any order gives the same counts), then the
// biases, then one pass over the logits.
__global__ void __launch_bounds__(256) logit_rules_kernel(RuleArgs a) {
  __shared__ unsigned cnt[kRuleTile];  // bit 31: seen; the rest: times in the answer
  __shared__ float bias[kRuleTile];
  __shared__ unsigned long long red[8];
  const int r = blockIdx.x / a.tiles, t0 = blockIdx.x % a.tiles * kRuleTile, tid = threadIdx.x;
  const int nv = min(kRuleTile, a.V - t0);
  for (int i = tid; i < nv; i += 256) {
    cnt[i] = 0;
    bias[i] = 0.0f;
  }
  __syncthreads();
  const int H = a.ids ? min(max(0, a.n_ids[r]), a.max_ids) : 0, P = a.n_prompt ? a.n_prompt[r] : 0;
  for (int i = tid; i < H; i += 256) {
    const int id = a.ids[r * a.ids_stride + i] - t0;
    if (id >= 0 && id < nv) {
      atomicOr(&cnt[id], 0x80000000u);
      if (i >= P) atomicAdd(&cnt[id], 1u);
    }
  }
  if (a.bias_off) {
    const int b0 = max(a.bias_off[r], 0), b1 = min(a.bias_off[r + 1], a.n_bias);
    for (int i = b0 + tid; i < b1; i += 256) {
      const int id = a.bias_ids[i];
      if (id < t0 || id >= t0 + nv || (i > b0 && a.bias_ids[i - 1] == id)) continue;
      float s = a.bias_val[i];
      for (int e = i + 1; e < b1 && a.bias_ids[e] == id; e++) s += a.bias_val[e];
      bias[id - t0] = s;
    }
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[r] : 1.0f, fr = a.frequency ? a.frequency[r] : 0.0f,
              pr = a.presence ? a.presence[r] : 0.0f;
  unsigned long long best = 0;
  for (int i = tid; i < nv; i += 256) {
    float x = a.x[r * a.x_stride + t0 + i];
    const unsigned c = cnt[i], co = c & 0x7fffffffu;
    if (c) x = x > 0.0f ? x / rep : x * rep;
    if (co) x = (x - fr * (float)co) - pr;
    if (a.bias_off) x += bias[i];
    if (a.mask && !(a.mask[r * a.mask_stride + ((t0 + i) >> 5)] >> ((t0 + i) & 31) & 1u)) x = -INFINITY;
    a.out[r * a.out_stride + t0 + i] = x;
    best = max(best, rule_key(x, t0 + i));
  }
  if (!a.best) return;
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) red[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < 8; i++) best = max(best, red[i]);
    a.best[blockIdx.x] = best;
  }
}

// argmax[r] from the tiles' best; -1 when no logit is above -inf. One warp a row.
__global__ void logit_argmax_kernel(const unsigned long long *best, int tiles, int *argmax) {
  unsigned long long k = 0;
  for (int i = threadIdx.x; i < tiles; i += 32) k = max(k, best[(size_t)blockIdx.x * tiles + i]);
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
  if (threadIdx.x == 0) argmax[blockIdx.x] = k ? (int)~(unsigned)k : -1;
}

}  // namespace llmq
