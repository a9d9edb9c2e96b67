// The context behind llmq_ctx and the error helpers of the C entry points,
// shared by the files that implement include/llmq.h.
#pragma once

#include <cuda_runtime.h>

#include <map>
#include <string>
#include <vector>

#include "../../include/llmq.h"

namespace llmq {
struct DecodeState;
}

// The serving operators' device workspace on one stream: buf holds partial
// results within a call, zeros (tickets, counts) is all zero between calls.
// A buffer that became too small is kept with the context, for the graphs
// captured with it; each is at least twice the one before where memory
// allows, so that together they are no larger than the last.
struct ServeWs {
  void *buf = nullptr;
  size_t bytes = 0;
  void *zeros = nullptr;
  size_t zero_bytes = 0;
  std::vector<void *> retired;
};

struct llmq_ctx {
  int device = 0;
  int num_sms = 148;
  cudaStream_t own = nullptr;
  cudaStream_t stream = nullptr;
  std::string err;
  // scratch owned by the context (grown on demand)
  void *scratch = nullptr;
  size_t scratch_bytes = 0;
  llmq::DecodeState *state = nullptr;  // device, for llmq_head_argmax
  int dense_parts = 4;           // gemv's parts: the reference team of 4 threads (gpt2t.mojo:281 on 4 cores)
  int prefill_kernel = LLMQ_PREFILL_AUTO;
  long long wait_cycles = 4000000000LL;  // limit of a persistent kernel's or a row GEMV's device-side wait
  int *tc_err = nullptr;         // device error code of the tcgen05 GEMM (a wait that gave up)
  bool tc_used = false;          // a tcgen05 GEMM ran since the last check
  // sampling scratch (device, grown on demand): sort keys, chunk candidates,
  // the Rng state of llmq_generate_sampled
  unsigned long long *samp_keys = nullptr;
  unsigned long long *samp_cand = nullptr;
  unsigned long long *samp_rng = nullptr;
  int *samp_done = nullptr;  // set by topk_fast_kernel when it finished the draw
  int samp_n = 0;
  // workspaces of the serving operators (serving.cu), one per stream that
  // they ran on, so that calls on two streams share nothing
  std::map<cudaStream_t, ServeWs> serve_ws;
};

namespace llmq {

inline llmq_status fail(llmq_ctx *ctx, llmq_status st, const std::string &msg) {
  if (ctx) ctx->err = msg;
  return st;
}

#define CK(call)                                                                                 \
  do {                                                                                           \
    cudaError_t e_ = (call);                                                                     \
    if (e_ != cudaSuccess)                                                                       \
      return fail(ctx, LLMQ_ERR_CUDA, std::string(#call) + ": " + cudaGetErrorString(e_));     \
  } while (0)

#define CKL()                                                                                    \
  do {                                                                                           \
    cudaError_t e_ = cudaGetLastError();                                                         \
    if (e_ != cudaSuccess) return fail(ctx, LLMQ_ERR_CUDA, std::string("launch: ") + cudaGetErrorString(e_)); \
  } while (0)

// Whether llmq_paged_store and llmq_paged_attend would refuse a step over
// n_layers layers of p with these arguments (serving.cu).
llmq_status paged_step_check(llmq_ctx *ctx, const llmq_paged *p, int n_layers, const int *table, long long table_stride,
                             int table_cols, int n_seqs, int max_len);

}  // namespace llmq
