// Host-side interface of the token log-probability kernels (wb_logprobs.cu).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

#include "wb_common.h"

namespace wb {

constexpr int kLogprobMaxTop = 32;
constexpr uint32_t kLogprobMaxColumns = 1u << 30;      // column numbers fit 32 signed bits, a tile past the end too
constexpr uint32_t kLogprobMaxTopVocab = 1u << 21;     // columns with alternatives: the tiles' maxima fit 32 KiB of shared memory

// Rows of logits: row r = (r / inner, r % inner) starts at element (r / inner) * stride_outer +
// (r % inner) * stride_inner; its columns are contiguous.  The same split addresses the tokens.
struct LogprobRows {
  const void* logits;
  const void* tokens;          // int64, or int32 with tokens_i32
  int64_t stride_outer, stride_inner;
  int64_t tok_outer, tok_inner;
  uint32_t rows, inner;
  uint32_t vocab;              // valid columns
  uint32_t dtype;              // DT_BF16 / DT_F16 / DT_F32
  int32_t tokens_i32;
  float inv_temp;
  int64_t ignore_index;
};

struct LogprobOut {
  float* logprobs;             // [rows]
  float* entropy;              // [rows]
  float* stats;                // [rows, 2]: max logit and log2 of the sum (+inf: an empty row), or null
  float* top_logprobs;         // [rows, top_k] or null
  int64_t* top_ids;
  int top_k;                   // 0 .. kLogprobMaxTop
};

struct LogprobGrad {
  const float* stats;
  const float* entropy;
  const float* g_logprobs;     // null: zero
  const float* g_entropy;
  int64_t g_logprobs_stride, g_entropy_stride;
  void* grad;                  // [rows, cols], contiguous, the logits' type
  uint32_t cols;               // >= vocab; columns past the vocabulary get zeros
};

cudaError_t launch_token_logprobs(const LogprobRows& in, const LogprobOut& out, int sms, cudaStream_t stream);
cudaError_t launch_token_logprobs_grad(const LogprobRows& in, const LogprobGrad& g, cudaStream_t stream);

}  // namespace wb
