// C entry points of the serving operators: the paged cache's store, attention
// and eviction, and the rules on logits (include/llmq.h).
#include <algorithm>
#include <climits>
#include <mutex>

#include "context.cuh"
#include "evict.cuh"
#include "logits.cuh"
#include "paged.cuh"
#include "paged_mma.cuh"

using namespace llmq;

struct llmq_paged {
  int device = 0;
  bool owned = false;  // whether the buffers are the handle's
  PagedView v{};
};

namespace {

// Grows one of the workspace's buffers. The old one stays for calls in flight
// and graphs captured with it.
llmq_status serve_grow(llmq_ctx *ctx, ServeWs &w, void **buf, size_t *have, size_t bytes, bool zero) {
  if (*have >= bytes) return LLMQ_OK;
  cudaStreamCaptureStatus cap;
  CK(cudaStreamIsCapturing(ctx->stream, &cap));
  if (cap != cudaStreamCaptureStatusNone)
    return fail(ctx, LLMQ_ERR_INVALID, "the serving workspace grows on first use: run the call once before capturing it");
  void *grown = nullptr;
  size_t size = std::max(bytes, 2 * *have);
  cudaError_t e = cudaMalloc(&grown, size);
  if (e != cudaSuccess && size > bytes) {
    cudaGetLastError();
    size = bytes;
    e = cudaMalloc(&grown, size);
  }
  if (e == cudaSuccess && zero && (e = cudaMemsetAsync(grown, 0, size, ctx->stream)) != cudaSuccess) cudaFree(grown);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(ctx, e == cudaErrorMemoryAllocation ? LLMQ_ERR_NOMEM : LLMQ_ERR_CUDA,
                "serving workspace of " + std::to_string(bytes) + " bytes: " + cudaGetErrorString(e));
  }
  if (*buf) w.retired.push_back(*buf);
  *buf = grown;
  *have = size;
  return LLMQ_OK;
}

// The stream's workspace with at least `bytes` of buffer and `zeros` bytes
// that are zero.
llmq_status serve_ws(llmq_ctx *ctx, size_t bytes, size_t zeros, ServeWs **out) {
  ServeWs &w = ctx->serve_ws[ctx->stream];
  llmq_status st = serve_grow(ctx, w, &w.buf, &w.bytes, bytes, false);
  if (st == LLMQ_OK) st = serve_grow(ctx, w, &w.zeros, &w.zero_bytes, zeros, true);
  *out = &w;
  return st;
}

constexpr int kMaxDevices = 64;

int elem_bytes(int kind) { return kind == LLMQ_KV_F32 ? 4 : kind == LLMQ_KV_BF16 ? 2 : 1; }

// What store, attend and evict all check.
llmq_status paged_check(llmq_ctx *ctx, const llmq_paged *p, int layer0, int n_layers, const int *table,
                        long long table_stride, int table_cols, int n_seqs) {
  if (!ctx || !p || !table) return fail(ctx, LLMQ_ERR_INVALID, "null argument");
  if (p->device != ctx->device) return fail(ctx, LLMQ_ERR_INVALID, "the cache is on another device");
  if (layer0 < 0 || n_layers <= 0 || layer0 > p->v.n_layer - n_layers) return fail(ctx, LLMQ_ERR_INVALID, "bad layer");
  if (n_seqs <= 0 || table_cols <= 0 || table_stride < 0) return fail(ctx, LLMQ_ERR_INVALID, "bad page table shape");
  return LLMQ_OK;
}

llmq_status max_len_check(llmq_ctx *ctx, int max_len) {
  return max_len > 0 && max_len <= 1 << 30 ? LLMQ_OK : fail(ctx, LLMQ_ERR_INVALID, "bad max_len");
}

// A launch that may begin while the kernel before it on the stream ends; its
// own first step waits for that kernel (griddepcontrol.wait).
template <typename... P, typename... A>
cudaError_t launch_after(void (*k)(P...), dim3 grid, unsigned threads, cudaStream_t s, size_t smem, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, static_cast<P>(args)...);
}

// A kernel with its shared memory and how many of its CTAs an SM holds
// (asked for once per device).
struct AttendKernel {
  void (*fn)(AttendArgs) = nullptr;
  int threads = 0, smem = 0, block = 0, per_sm[kMaxDevices] = {};
};
template <int KIND, int D, int HT, bool FAST, int W>
AttendKernel *attend_kernel_w() {
  static AttendKernel k = [] {
    AttendKernel x;
    x.fn = paged_mma_kernel<KIND, D, HT, FAST, W>;
    x.threads = W * 32;
    x.smem = pm_smem<KIND, D, W>(FAST);
    x.block = PmShape<KIND, D, W>::kBlock;
    return x;
  }();
  return &k;
}
template <int KIND, int D, int HT>
AttendKernel *attend_kernel_h(bool fast, int warps) {
  if (warps == 1) return fast ? attend_kernel_w<KIND, D, HT, true, 1>() : attend_kernel_w<KIND, D, HT, false, 1>();
  if (warps == 2) return fast ? attend_kernel_w<KIND, D, HT, true, 2>() : attend_kernel_w<KIND, D, HT, false, 2>();
  return fast ? attend_kernel_w<KIND, D, HT, true, 4>() : attend_kernel_w<KIND, D, HT, false, 4>();
}
template <int KIND, int D>
AttendKernel *attend_kernel_d(int heads, bool fast, int warps) {
  return heads == 4 ? attend_kernel_h<KIND, D, 1>(fast, warps) : attend_kernel_h<KIND, D, 2>(fast, warps);
}
template <int KIND>
AttendKernel *attend_kernel_k(int D, int heads, bool fast, int warps) {
  switch (D) {
    case 32: return attend_kernel_d<KIND, 32>(heads, fast, warps);
    case 64: return attend_kernel_d<KIND, 64>(heads, fast, warps);
    case 96: return attend_kernel_d<KIND, 96>(heads, fast, warps);
    default: return attend_kernel_d<KIND, 128>(heads, fast, warps);
  }
}
// The kernel for a call, ready to launch on ctx's device.
llmq_status attend_kernel(llmq_ctx *ctx, const AttendArgs &a, int warps, AttendKernel **out) {
  const bool fast = a.c.page_size % 16 == 0;
  AttendKernel *k = a.c.kind == LLMQ_KV_QUANT8 ? attend_kernel_k<PM_I8>(a.c.head_dim, a.unit_heads, fast, warps)
                    : a.c.kind == LLMQ_KV_BF16 ? attend_kernel_k<PM_BF16>(a.c.head_dim, a.unit_heads, fast, warps)
                                               : attend_kernel_k<PM_F32>(a.c.head_dim, a.unit_heads, fast, warps);
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  int &n = k->per_sm[ctx->device % kMaxDevices];
  if (!n) {
    CK(cudaFuncSetAttribute((const void *)k->fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k->smem));
    CK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k->fn, k->threads, k->smem));
    if (n <= 0) return fail(ctx, LLMQ_ERR_UNSUPPORTED, "the attention kernel does not fit on this device");
  }
  *out = k;
  return LLMQ_OK;
}

template <typename E, int D>
cudaError_t launch_store_d(const StoreArgs &a, bool vec, unsigned grid, cudaStream_t s) {
  return launch_after(vec ? paged_store_kernel<E, D, true> : paged_store_kernel<E, D, false>, dim3(grid), 256, s, 0, a);
}
template <typename E>
cudaError_t launch_store_e(const StoreArgs &a, bool vec, unsigned grid, cudaStream_t s) {
  switch (a.c.head_dim) {
    case 32: return launch_store_d<E, 32>(a, vec, grid, s);
    case 64: return launch_store_d<E, 64>(a, vec, grid, s);
    case 96: return launch_store_d<E, 96>(a, vec, grid, s);
    default: return launch_store_d<E, 128>(a, vec, grid, s);
  }
}
cudaError_t launch_store(const StoreArgs &a, bool vec, unsigned grid, cudaStream_t s) {
  if (a.c.kind == LLMQ_KV_QUANT8) return launch_store_e<PgInt8>(a, vec, grid, s);
  if (a.c.kind == LLMQ_KV_BF16) return launch_store_e<PgBf16>(a, vec, grid, s);
  return launch_store_e<PgF32>(a, vec, grid, s);
}

cudaError_t launch_move(const EvictArgs &a, int tiles, unsigned grid, cudaStream_t s) {
  auto go = [&](void (*k)(EvictArgs, int)) { return launch_after(k, dim3(grid), 256, s, 0, a, tiles); };
  switch (a.c.head_dim * elem_bytes(a.c.kind) / 16) {
    case 2: return go(evict_move_kernel<2>);
    case 4: return go(evict_move_kernel<4>);
    case 6: return go(evict_move_kernel<6>);
    case 8: return go(evict_move_kernel<8>);
    case 12: return go(evict_move_kernel<12>);
    case 16: return go(evict_move_kernel<16>);
    case 24: return go(evict_move_kernel<24>);
    default: return go(evict_move_kernel<32>);
  }
}

// Blocks of a one-dimensional grid, or 0 when there would be too many.
unsigned grid1(long long n) { return n > 0 && n <= INT_MAX ? (unsigned)n : 0u; }

llmq_status paged_shape_check(llmq_ctx *ctx, int kind, int n_layer, int n_pages, int page_size, int n_kv_head,
                              int head_dim) {
  if (kind != LLMQ_KV_QUANT8 && kind != LLMQ_KV_F32 && kind != LLMQ_KV_BF16)
    return fail(ctx, LLMQ_ERR_UNSUPPORTED, "a paged cache holds int8, float32 or bfloat16");
  if (n_layer <= 0 || n_pages <= 0 || page_size <= 0 || n_kv_head <= 0 || head_dim <= 0 || head_dim % 32 ||
      head_dim > 128)
    return fail(ctx, LLMQ_ERR_INVALID, "bad paged cache shape (head_dim: 32, 64, 96 or 128)");
  const double rows = (double)n_pages * n_kv_head * page_size;
  if (rows * n_layer * head_dim * 4 > 4e12) return fail(ctx, LLMQ_ERR_NOMEM, "paged cache larger than any device");
  if (rows > INT_MAX) return fail(ctx, LLMQ_ERR_INVALID, "more than 2^31 - 1 rows in a layer");
  return LLMQ_OK;
}

}  // namespace

llmq_status llmq::paged_step_check(llmq_ctx *ctx, const llmq_paged *p, int n_layers, const int *table,
                                   long long table_stride, int table_cols, int n_seqs, int max_len) {
  const llmq_status st = paged_check(ctx, p, 0, n_layers, table, table_stride, table_cols, n_seqs);
  return st != LLMQ_OK ? st : max_len_check(ctx, max_len);
}

extern "C" {

llmq_status llmq_paged_create_in(llmq_ctx *ctx, int kind, int n_layer, int n_pages, int page_size, int n_kv_head,
                                 int head_dim, void *k, void *v, float *ks, float *vs, llmq_paged **out) {
  if (!ctx || !out) return fail(ctx, LLMQ_ERR_INVALID, "null argument");
  *out = nullptr;
  const llmq_status st = paged_shape_check(ctx, kind, n_layer, n_pages, page_size, n_kv_head, head_dim);
  if (st != LLMQ_OK) return st;
  const bool scaled = kind == LLMQ_KV_QUANT8;
  if (!k || !v || (scaled && (!ks || !vs))) return fail(ctx, LLMQ_ERR_INVALID, "null buffer");
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)ks | (uintptr_t)vs) % 16)
    return fail(ctx, LLMQ_ERR_INVALID, "buffers must be 16-byte aligned");
  llmq_paged *p = new llmq_paged();
  p->device = ctx->device;
  p->v = PagedView{k, v, scaled ? ks : nullptr, scaled ? vs : nullptr, kind, n_layer, n_pages, page_size, n_kv_head, head_dim};
  *out = p;
  return LLMQ_OK;
}

llmq_status llmq_paged_create(llmq_ctx *ctx, int kind, int n_layer, int n_pages, int page_size, int n_kv_head,
                              int head_dim, llmq_paged **out) {
  if (!ctx || !out) return fail(ctx, LLMQ_ERR_INVALID, "null argument");
  *out = nullptr;
  llmq_status st = paged_shape_check(ctx, kind, n_layer, n_pages, page_size, n_kv_head, head_dim);
  if (st != LLMQ_OK) return st;
  CK(cudaSetDevice(ctx->device));
  const size_t rows = (size_t)n_layer * n_pages * n_kv_head * page_size;
  const size_t bytes[4] = {rows * head_dim * elem_bytes(kind), rows * head_dim * elem_bytes(kind), rows * 4, rows * 4};
  void *buf[4] = {};
  cudaError_t e = cudaSuccess;
  for (int i = 0; i < (kind == LLMQ_KV_QUANT8 ? 4 : 2) && e == cudaSuccess; i++) {
    e = cudaMalloc(&buf[i], bytes[i]);
    if (e == cudaSuccess) e = cudaMemsetAsync(buf[i], 0, bytes[i], ctx->stream);
  }
  if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);
  if (e == cudaSuccess) {
    st = llmq_paged_create_in(ctx, kind, n_layer, n_pages, page_size, n_kv_head, head_dim, buf[0], buf[1],
                              (float *)buf[2], (float *)buf[3], out);
  } else {
    cudaGetLastError();
    st = fail(ctx, e == cudaErrorMemoryAllocation ? LLMQ_ERR_NOMEM : LLMQ_ERR_CUDA,
              std::string("paged cache: ") + cudaGetErrorString(e));
  }
  if (st != LLMQ_OK) {
    for (void *q : buf)
      if (q) cudaFree(q);
    return st;
  }
  (*out)->owned = true;
  return LLMQ_OK;
}

llmq_status llmq_paged_free(llmq_paged *p) {
  if (!p) return LLMQ_ERR_INVALID;
  if (p->owned) {
    cudaSetDevice(p->device);
    for (void *q : {p->v.k, p->v.v, (void *)p->v.ks, (void *)p->v.vs})
      if (q) cudaFree(q);
  }
  delete p;
  return LLMQ_OK;
}

llmq_status llmq_paged_shape(const llmq_paged *p, int *kind, int *n_layer, int *n_pages, int *page_size, int *n_kv_head,
                             int *head_dim) {
  if (!p) return LLMQ_ERR_INVALID;
  int *out[6] = {kind, n_layer, n_pages, page_size, n_kv_head, head_dim};
  const int val[6] = {p->v.kind, p->v.n_layer, p->v.n_pages, p->v.page_size, p->v.n_kv_head, p->v.head_dim};
  for (int i = 0; i < 6; i++)
    if (out[i]) *out[i] = val[i];
  return LLMQ_OK;
}

llmq_status llmq_paged_buffers(const llmq_paged *p, void **k, void **v, float **ks, float **vs) {
  if (!p) return LLMQ_ERR_INVALID;
  if (k) *k = p->v.k;
  if (v) *v = p->v.v;
  if (ks) *ks = p->v.ks;
  if (vs) *vs = p->v.vs;
  return LLMQ_OK;
}

llmq_status llmq_paged_store(llmq_ctx *ctx, llmq_paged *p, int layer, const float *k, long long k_stride,
                             const float *v, long long v_stride, const int *seq, const int *pos, int n_rows,
                             const int *table, long long table_stride, int table_cols, int n_seqs) {
  llmq_status st = paged_check(ctx, p, layer, 1, table, table_stride, table_cols, n_seqs);
  if (st != LLMQ_OK) return st;
  if (!k || !v || !pos) return fail(ctx, LLMQ_ERR_INVALID, "null argument");
  if (n_rows <= 0 || (!seq && n_rows > n_seqs)) return fail(ctx, LLMQ_ERR_INVALID, "bad row count");
  if (k_stride < 0 || v_stride < 0) return fail(ctx, LLMQ_ERR_INVALID, "negative stride");
  CK(cudaSetDevice(ctx->device));
  const StoreArgs a{p->v, PageTable{table, table_stride, table_cols, n_seqs}, layer, n_rows, k, v, k_stride, v_stride,
                    seq, pos};
  const int per = kStoreHeads * (p->v.head_dim == 96 ? 1 : 128 / p->v.head_dim);  // heads of a warp
  const long long warps = (long long)n_rows * ((p->v.n_kv_head + per - 1) / per);
  const unsigned g = warps <= INT_MAX ? grid1((warps + 7) / 8) : 0;
  if (!g) return fail(ctx, LLMQ_ERR_INVALID, "too many rows for one call");
  const bool vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && (n_rows == 1 || (k_stride % 4 == 0 && v_stride % 4 == 0));
  CK(launch_store(a, vec, g, ctx->stream));
  return LLMQ_OK;
}

llmq_status llmq_paged_attend(llmq_ctx *ctx, const llmq_paged *p, int layer, const float *q, long long q_stride,
                              float *out, long long out_stride, int n_seqs, int n_head, const int *table,
                              long long table_stride, int table_cols, const int *lens, int max_len, float scale,
                              const float *weights, float *weights_out, long long weights_stride) {
  llmq_status st = paged_check(ctx, p, layer, 1, table, table_stride, table_cols, n_seqs);
  if (st != LLMQ_OK) return st;
  if (!q || !out || !lens) return fail(ctx, LLMQ_ERR_INVALID, "null argument");
  if (n_head <= 0 || n_head % p->v.n_kv_head) return fail(ctx, LLMQ_ERR_INVALID, "n_head must be a multiple of n_kv_head");
  const long long C = (long long)n_head * p->v.head_dim;
  if (q_stride < 0 || (n_seqs > 1 && out_stride < C)) return fail(ctx, LLMQ_ERR_INVALID, "rows overlap");
  if ((st = max_len_check(ctx, max_len)) != LLMQ_OK) return st;
  if (weights && !weights_out) return fail(ctx, LLMQ_ERR_INVALID, "weights without weights_out");
  if (weights_out && weights_stride < max_len) return fail(ctx, LLMQ_ERR_INVALID, "weights_stride below max_len");
  CK(cudaSetDevice(ctx->device));
  AttendArgs a{};
  a.c = p->v;
  a.t = PageTable{table, table_stride, table_cols, n_seqs};
  a.layer = layer;
  a.n_head = n_head;
  a.max_len = (int)std::min((long long)max_len, (long long)table_cols * p->v.page_size);
  a.score_stride = (int)(((long long)a.max_len + 3) / 4 * 4);
  a.q = q;
  a.out = out;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.q_vec = (uintptr_t)q % 16 == 0 && q_stride % 4 == 0;
  a.lens = lens;
  a.scale2 = (float)(scale * 1.4426950408889634);
  const size_t rows = (size_t)n_seqs * n_head;
  const int D = p->v.head_dim, G = n_head / p->v.n_kv_head;
  a.unit_heads = G <= 4 ? 4 : 8;
  a.head_chunks = (G + a.unit_heads - 1) / a.unit_heads;
  const long long units = (long long)n_seqs * p->v.n_kv_head * a.head_chunks;
  // Fewer warps a CTA for many units of short sequences, whose prologues and
  // joins then cost less than idle warps do. 64 dimensions, us with 1 / 2 / 4
  // warps:
  //                    int8 x <=256        x <=320             x <=384             bfloat16 x <=256    x <=320
  //   3072 units       18.6/20.3/24.5      21.3/23.2/27.0      25.9/25.2/28.6      26.5/27.3/34.2      32.2/31.0/37.8
  //   2448             20.3/17.2/20.8      24.1/19.5/23.0      26.1/21.6/24.0      19.9/22.4/27.6      24.7/25.6/30.7
  //   1344             16.4/10.8/12.8      19.1/13.4/14.7      19.3/14.2/15.1      18.1/14.0/16.8      21.6/16.5/19.0
  //   768              14.0/11.3/9.7       15.1/14.1/9.1       14.8/15.0/9.4       16.4/10.9/12.0      16.6/10.5/12.6
  // (int8's 2448 units leave room for two one-warp chunks each, which have to
  // be joined: there two warps would do better)
  int warps = units >= ctx->num_sms * 16 && a.max_len <= 256 ? 1 : units >= ctx->num_sms * 8 ? 2 : 4;
  AttendKernel *k;
  if ((st = attend_kernel(ctx, a, warps, &k)) != LLMQ_OK) return st;
  // Chunks, in whole blocks, two at least (1 x 200 positions: 3.9 us, 6.2 in
  // single blocks, which have to be joined), at most kPmJoin of a unit: twice
  // as many as the GPU holds CTAs at once, since only the longest sequences
  // fill theirs (8 ragged sequences x <=32768: 105 us, 126 with once as many;
  // one sequence x 131071: 48 us with either)
  const long long wave = (long long)ctx->num_sms * k->per_sm[ctx->device % kMaxDevices];
  const long long fit = std::min((long long)kPmJoin, std::max(1LL, 2 * wave / units));
  const long long blocks = (a.max_len + k->block - 1) / k->block;
  a.chunk = (int)std::max(2LL, (blocks + fit - 1) / fit) * k->block;
  a.splits = (a.max_len + a.chunk - 1) / a.chunk;
  const unsigned g = grid1(units * a.splits);
  if (!g) return fail(ctx, LLMQ_ERR_INVALID, "too many sequences for one call");
  ServeWs *ws;
  const size_t parts = a.splits > 1 ? (size_t)g * a.unit_heads * (D + 4) : 0;
  const size_t floats = parts + (weights_out ? rows * (a.score_stride + 2) + 4 : 0);
  if ((st = serve_ws(ctx, floats * 4, a.splits > 1 ? (size_t)units * 4 : 0, &ws)) != LLMQ_OK) return st;
  a.part = (float *)ws->buf;
  a.tickets = (int *)ws->zeros;
  if (weights_out) {
    a.scores = a.part + (parts + 3) / 4 * 4;  // 16-byte aligned rows
    a.stat = a.scores + rows * a.score_stride;
  }
  CK(launch_after(k->fn, dim3(g), k->threads, ctx->stream, k->smem, a));
  if (weights_out) {
    const dim3 wg((max_len + 1023) / 1024, (unsigned)std::min((long long)n_seqs * p->v.n_kv_head, 65535LL));
    const bool vec = ((uintptr_t)weights | (uintptr_t)weights_out) % 16 == 0 && weights_stride % 4 == 0;
    CK(launch_after(vec ? paged_weights_kernel<true> : paged_weights_kernel<false>, wg, 256, ctx->stream, 0, a, max_len,
                    weights, weights_out, weights_stride));
  }
  return LLMQ_OK;
}

llmq_status llmq_paged_evict(llmq_ctx *ctx, llmq_paged *p, int layer0, int n_layers, int n_seqs, const int *table,
                             long long table_stride, int table_cols, const int *lens, int max_len, const float *weights,
                             long long weights_stride, int budget, int sinks, int recent, const int *dst_table,
                             long long dst_stride, int dst_cols, int *kept, float *weights_out, long long weights_out_stride,
                             int *lens_out) {
  llmq_status st = paged_check(ctx, p, layer0, n_layers, table, table_stride, table_cols, n_seqs);
  if (st != LLMQ_OK) return st;
  if (!lens || !weights || !dst_table || !kept || !weights_out || !lens_out)
    return fail(ctx, LLMQ_ERR_INVALID, "null argument");
  if (max_len <= 0 || max_len > 1 << 30 || budget <= 0 || sinks < 0 || recent < 0 || sinks > budget || recent > budget - sinks)
    return fail(ctx, LLMQ_ERR_INVALID, "sinks and recent must fit in a positive budget");
  if (weights_stride < max_len || weights_out_stride < budget || weights_out_stride > INT_MAX)
    return fail(ctx, LLMQ_ERR_INVALID, "bad weights stride");
  if (dst_cols <= 0 || dst_stride < 0 || (long long)dst_cols * p->v.page_size < std::min(budget, max_len))
    return fail(ctx, LLMQ_ERR_INVALID, "dst_table holds fewer positions than the budget");
  CK(cudaSetDevice(ctx->device));
  EvictArgs a{p->v, PageTable{table, table_stride, table_cols, n_seqs}, PageTable{dst_table, dst_stride, dst_cols, n_seqs}, layer0, n_layers,
              max_len, budget, sinks, recent, lens, weights, weights_stride, kept, weights_out, weights_out_stride,
              lens_out};
  const long long rows = (long long)n_layers * n_seqs * p->v.n_kv_head;
  const int tiles = (std::min(budget, max_len) + kEvPos - 1) / kEvPos;
  const unsigned g = grid1(rows), gm = g ? grid1(rows * tiles) : 0;
  if (!g || !gm) return fail(ctx, LLMQ_ERR_INVALID, "too many rows for one call");
  const bool vec = (uintptr_t)weights % 16 == 0 && weights_stride % 4 == 0;
  if (max_len <= 2048)
    CK(launch_after(vec ? evict_select_kernel<true, 256> : evict_select_kernel<false, 256>, dim3(g), 256, ctx->stream, 0, a));
  else
    CK(launch_after(vec ? evict_select_kernel<true, 1024> : evict_select_kernel<false, 1024>, dim3(g), 1024, ctx->stream, 0,
                    a));
  CK(launch_move(a, tiles, gm, ctx->stream));
  return LLMQ_OK;
}

llmq_status llmq_process_logits(llmq_ctx *ctx, const float *logits, long long logits_stride, float *out,
                                long long out_stride, int n, int V, const llmq_logit_rules *rules, int *argmax) {
  if (!ctx || !logits || !out || !rules) return fail(ctx, LLMQ_ERR_INVALID, "null argument");
  if (n <= 0 || V <= 0 || V > (1 << 24)) return fail(ctx, LLMQ_ERR_INVALID, "bad logits shape");
  if (n > 1 && (logits_stride < 0 || out_stride < V)) return fail(ctx, LLMQ_ERR_INVALID, "rows overlap");
  const llmq_logit_rules &u = *rules;
  if ((u.ids != nullptr) != (u.n_ids != nullptr) || (u.n_prompt && !u.ids) || (u.ids && (u.ids_stride < 0 || u.max_ids < 0)))
    return fail(ctx, LLMQ_ERR_INVALID, "a history needs ids and n_ids");
  if ((u.repetition || u.presence || u.frequency) && !u.ids)
    return fail(ctx, LLMQ_ERR_INVALID, "a penalty needs a history");
  if ((u.bias_offsets != nullptr) != (u.bias_ids != nullptr) || (u.bias_ids != nullptr) != (u.bias_values != nullptr))
    return fail(ctx, LLMQ_ERR_INVALID, "a bias needs offsets, ids and values");
  if ((u.bias_ids && u.n_bias < 0) || (u.mask && u.mask_stride < 0)) return fail(ctx, LLMQ_ERR_INVALID, "negative size");
  if (!grid1((long long)n * ((V + 1026) / 1024))) return fail(ctx, LLMQ_ERR_INVALID, "too many rows for one call");
  CK(cudaSetDevice(ctx->device));
  RuleArgs a{};
  a.x = logits, a.x_stride = logits_stride, a.out = out, a.out_stride = out_stride, a.n = n, a.V = V;
  a.repetition = u.repetition, a.presence = u.presence, a.frequency = u.frequency;
  a.ids = u.ids, a.n_ids = u.n_ids, a.n_prompt = u.n_prompt, a.ids_stride = u.ids_stride, a.max_ids = u.max_ids;
  a.bias_off = u.bias_offsets, a.bias_ids = u.bias_ids, a.bias_val = u.bias_values, a.n_bias = u.n_bias;
  a.mask = u.mask, a.mask_stride = u.mask_stride, a.argmax = argmax;
  // Tiles of 4096 logits, or smaller ones while the call has fewer CTAs than
  // two per SM (256 x 50257: 33 us with 4096, 39 with 2048, whose CTAs read
  // the history twice as often)
  int vpt = 16;
  constexpr int nth = 256;
  while (vpt > 4 && (long long)n * ((V + 3 + nth * vpt - 1) / (nth * vpt)) < 2 * ctx->num_sms) vpt /= 2;
  const int T = nth * vpt;
  a.tiles = (V + 3 + T - 1) / T;  // a row may start 3 logits past a 16-byte boundary
  const int keys = a.tiles * (nth / 32);
  // A second launch joins the argmax from two CTAs per SM on, where waiting
  // for each CTA's stores before its ticket costs more (256 x 50257: 33 us
  // against 38; 1 x 50257, with tickets, 5.0 us)
  const bool follow = argmax && (long long)n * a.tiles >= 2 * ctx->num_sms;
  if (argmax) {
    ServeWs *ws;
    const llmq_status st = serve_ws(ctx, (size_t)n * keys * 8, follow ? 0 : (size_t)n * 4, &ws);
    if (st != LLMQ_OK) return st;
    a.best = (unsigned long long *)ws->buf;
    a.tickets = follow ? nullptr : (int *)ws->zeros;
  }
  const size_t sm = (size_t)T * 4 * ((a.ids ? 1 : 0) + (a.bias_off ? 1 : 0));
  CK(launch_after(vpt == 16 ? logit_rules_kernel<nth, 16> : vpt == 8 ? logit_rules_kernel<nth, 8> : logit_rules_kernel<nth, 4>,
                  dim3(n * a.tiles), nth, ctx->stream, sm, a));
  if (follow) CK(launch_after(logit_argmax_kernel, dim3((n + 3) / 4), 128, ctx->stream, 0, a.best, keys, argmax, n));
  return LLMQ_OK;
}

}  // extern "C"
