// Arguments of the scoring kernels (ms_scores.cu): log-probabilities with
// entropy and top alternatives, their gradient, and distillation.
#pragma once
#include "ms_device.cuh"
#include "ms_scores_args.h"

namespace ms {

// The teacher's mass outside its list counts as none below this: the fp32
// log-probabilities of a list sum to 1 only up to about H * 2^-24.
constexpr double kNoTail = 1.0 / (1 << 20);

struct ScoreArgs {
  const void* x;          // [B, ld] logits
  int64_t B, ld;
  int32_t V;
  double T, rT;           // temperature, fp64(1 / T)
  float a;                // fp32(log2(e) / T)
  const int32_t* tokens;  // [B, n_tok] (null: n_tok 0)
  int32_t n_tok, top_n;
  ms_scores out;          // forward: each pointer may be null
  // backward
  const double* row_max;
  const double* row_sum;
  const float* entropy;
  const float* g_lp;      // [B, n_tok] or null
  const float* g_ent;     // [B] or null
  void* dx;               // [B, dld]
  int64_t dld;
};

struct DistillArgs {
  const void* x;          // [B, ld] logits
  int64_t B, ld;
  int32_t V;
  double rT;              // fp64(1 / T)
  float a;                // fp32(log2(e) / T)
  const int32_t* ids;     // [B, K]
  const float* values;    // [B, K]
  int32_t K, kind;
  const float* weight;    // [B] or null (1)
  float* loss;            // [B] or null
  void* dx;               // [B, dld] or null
  int64_t dld;
};

cudaError_t launch_logprobs(const ScoreArgs& A, int dtype, cudaStream_t stream);
int64_t logprobs_backward_blocks(int64_t B, int32_t V, int dtype);
cudaError_t launch_logprobs_backward(const ScoreArgs& A, int dtype, cudaStream_t stream);
cudaError_t launch_distill(const DistillArgs& A, int dtype, cudaStream_t stream);

}  // namespace ms
