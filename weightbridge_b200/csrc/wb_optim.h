// Host-side interface of the optimizer kernels (wb_optim.cu): the AdamW step over many tensors and
// the sum of squares of many tensors.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

#include "wb_common.h"

namespace wb {

constexpr uint32_t kStateBlock = 128;     // elements that share a scale in the 8-bit states
constexpr uint32_t kAdamTile = 4096;      // a work item of the step is a multiple of this; a CTA takes 2048 or 4096 at once
constexpr uint32_t kNormChunk = 16384;    // elements of one work item of the norm

// One parameter tensor (resident on the GPU).
struct alignas(16) AdamTensor {
  uint64_t param;
  uint64_t numel;
  uint64_t state;          // first element of its slice of the flat state buffers, a multiple of 128
  uint32_t dtype;          // DT_BF16 / DT_F16 / DT_F32
  float weight_decay;
};
static_assert(sizeof(AdamTensor) == 32, "AdamTensor layout");

struct AdamChunk {
  uint32_t tensor;
  uint32_t chunk;          // elements [chunk * AdamArgs::chunk, ...)
};

// The device's own record of the steps taken, so that a captured step can be replayed.
struct AdamClock {
  int64_t step;
  double b1t, b2t;         // beta^step
  uint32_t done;           // CTAs of the running launch that finished
  uint32_t reserved;
};
static_assert(sizeof(AdamClock) == 32, "AdamClock layout");

struct AdamArgs {
  const AdamTensor* tensors;
  const AdamChunk* chunks;
  uint32_t n_tensors;
  uint32_t chunk;          // elements of a work item
  float* master;           // flat, or null
  void* m;                 // flat fp32, or e4m3
  void* v;                 // flat fp32 second moment, or e4m3 of its root
  float* m_scale;          // one per 128 elements (8-bit states)
  float* v_scale;
  AdamClock* clock;
  double beta1, beta2;
  double lr;
  const void* lr_ptr;      // device scalar instead of lr, or null
  int lr_f64;
  double eps;
  const double* partial;   // the squared gradient norm is the sum of these; null: no clipping
  uint32_t n_partial;
  double max_norm;
  float* norm;             // receives the norm (with partial)
};

// Gradients travel as launch arguments: their addresses change from step to step, and arguments
// need no staging buffer that a later step could overwrite.  Bit 0: an fp32 gradient of a 16-bit
// parameter.  0: the tensor is left alone in this step.
constexpr uint32_t kGradsPerLaunch = 3800;

// chunk_start[t]: first work item of tensor t (n_tensors + 1 values, host).
cudaError_t launch_adamw(const AdamArgs& a, const uint64_t* grads, const uint32_t* chunk_start, int sms, cudaStream_t stream);

struct NormTensor {
  uint64_t ptr;
  uint64_t numel;
  uint32_t dtype;
  uint32_t first_chunk;    // filled in by the launcher
};
static_assert(sizeof(NormTensor) == 24, "NormTensor layout");
constexpr uint32_t kNormTensorsPerLaunch = 1300;

// Partial sums of squares that launch_partial_sums writes over all tensors, at most.
uint64_t partial_sums_size(uint32_t n, int sms);
// Writes partial sums (a fixed split of the work, so the same bits every time); *n_partial of them.
cudaError_t launch_partial_sums(NormTensor* t, uint32_t n, double* partial, uint32_t* n_partial, int sms, cudaStream_t stream);
// sum_sq[0] = the sum of the partial sums, norm[0] = its root.
cudaError_t launch_norm(const double* partial, uint32_t n_partial, double* sum_sq, float* norm, cudaStream_t stream);

}  // namespace wb
