// Argument checks of the scoring calls, without CUDA: each returns NULL or what
// is wrong with the call.
#pragma once
#include <cstddef>
#include <cstdint>

#include "../../include/minisample.h"

namespace ms {

constexpr int kScoreMax = 256;                      // largest n_tokens, top_n and teacher list
constexpr int64_t kScoreVMax = (int64_t)65535 * 16384;  // ms_sample's limit

inline int64_t elem_bytes(int dtype) { return dtype == MS_F32 ? 4 : 2; }

inline bool misaligned(const void* p, size_t bytes) { return (uintptr_t)p % bytes != 0; }

inline const char* bad_block(const void* logits, int dtype, int64_t B, int64_t V, int64_t ld, double temperature) {
  if (dtype != MS_F32 && dtype != MS_BF16 && dtype != MS_F16) return "dtype is not MS_F32, MS_BF16 or MS_F16";
  if (B < 0 || B > INT32_MAX) return "B out of range";
  if (V < 1 || V > kScoreVMax) return "V out of range";
  if (B > 1 && ld < V) return "ld < V";
  if (B > 1 && ld > INT64_MAX / 8 / B) return "B * ld too large";
  if (!(temperature > 0.0001 && temperature <= 10000.0)) return "temperature must be in (0.0001, 10000]";
  if (B > 0 && !logits) return "logits is NULL";
  if ((uintptr_t)logits % elem_bytes(dtype)) return "logits is not aligned to an element";
  return nullptr;
}

// A gradient block: the logits themselves, or apart from them.
inline const char* bad_grad(const void* logits, int dtype, int64_t B, int64_t V, int64_t ld, const void* dx,
                            int64_t dld) {
  if (!dx) return "dlogits is NULL";
  if (B > 1 && dld < V) return "dld < V";
  if (B > 1 && dld > INT64_MAX / 8 / B) return "B * dld too large";
  const uintptr_t es = (uintptr_t)elem_bytes(dtype);
  if ((uintptr_t)dx % es) return "dlogits is not aligned to an element";
  if (dx == logits && (B == 1 || dld == ld)) return nullptr;
  const uintptr_t x0 = (uintptr_t)logits, x1 = x0 + ((uintptr_t)(B - 1) * (B > 1 ? ld : 0) + V) * es;
  const uintptr_t d0 = (uintptr_t)dx, d1 = d0 + ((uintptr_t)(B - 1) * (B > 1 ? dld : 0) + V) * es;
  if (x0 < d1 && d0 < x1) return "dlogits overlaps logits without being them";
  return nullptr;
}

inline const char* bad_logprobs(const void* logits, int dtype, int64_t B, int64_t V, int64_t ld, double temperature,
                                const int32_t* tokens, int32_t n_tokens, int32_t top_n, const ms_scores* out) {
  if (const char* e = bad_block(logits, dtype, B, V, ld, temperature)) return e;
  if (n_tokens < 0 || n_tokens > kScoreMax) return "n_tokens must be in [0, 256]";
  if (top_n < 0 || top_n > kScoreMax) return "top_n must be in [0, 256]";
  if (!out) return "out is NULL";
  if (B > 0 && n_tokens > 0 && !tokens) return "tokens is NULL";
  if (misaligned(tokens, 4)) return "tokens is not aligned to an element";
  return nullptr;
}

inline const char* bad_scores(const ms_scores& o) {
  if (misaligned(o.logprobs, 4) || misaligned(o.entropy, 4) || misaligned(o.top_ids, 4) ||
      misaligned(o.top_logprobs, 4) || misaligned(o.row_max, 8) || misaligned(o.row_sum, 8))
    return "an output is not aligned to an element";
  return nullptr;
}

inline const char* bad_logprobs_backward(const void* logits, int dtype, int64_t B, int64_t V, int64_t ld,
                                         double temperature, const int32_t* tokens, int32_t n_tokens,
                                         const double* row_max, const double* row_sum, const float* entropy,
                                         const float* g_logprobs, const float* g_entropy, const void* dlogits,
                                         int64_t dld) {
  if (const char* e = bad_block(logits, dtype, B, V, ld, temperature)) return e;
  if (n_tokens < 0 || n_tokens > kScoreMax) return "n_tokens must be in [0, 256]";
  if (B == 0) return nullptr;
  if (n_tokens > 0 && !tokens) return "tokens is NULL";
  if (n_tokens == 0 && g_logprobs) return "g_logprobs without tokens";
  if (!row_max || !row_sum) return "row_max/row_sum is NULL";
  if (g_entropy && !entropy) return "g_entropy without entropy";
  if (misaligned(tokens, 4) || misaligned(row_max, 8) || misaligned(row_sum, 8) || misaligned(entropy, 4) ||
      misaligned(g_logprobs, 4) || misaligned(g_entropy, 4))
    return "an input is not aligned to an element";
  return bad_grad(logits, dtype, B, V, ld, dlogits, dld);
}

inline const char* bad_distill(const void* logits, int dtype, int64_t B, int64_t V, int64_t ld, double temperature,
                               const int32_t* ids, const float* values, int32_t K, int kind, const float* loss,
                               const void* dlogits, int64_t dld, const float* weight = nullptr) {
  if (const char* e = bad_block(logits, dtype, B, V, ld, temperature)) return e;
  if (K < 1 || K > kScoreMax) return "K must be in [1, 256]";
  if (kind != MS_TEACHER_LOGITS && kind != MS_TEACHER_LOGPROBS)
    return "kind is not MS_TEACHER_LOGITS or MS_TEACHER_LOGPROBS";
  if (B == 0) return nullptr;
  if (!ids || !values) return "ids/values is NULL";
  if (!loss && !dlogits) return "loss and dlogits are both NULL";
  if (misaligned(ids, 4) || misaligned(values, 4) || misaligned(loss, 4) || misaligned(weight, 4))
    return "ids, values, weight or loss is not aligned to an element";
  return dlogits ? bad_grad(logits, dtype, B, V, ld, dlogits, dld) : nullptr;
}

}  // namespace ms
