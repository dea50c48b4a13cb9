// dlr_losses.h -- launchers of the softmax-loss kernels (dlr_losses.hip).
// Arguments are checked by the C entries (dlr_losses.cpp); a launcher only
// picks the kernel and its grid.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstdint>

#include "distlr_losses.h"

namespace dlr {

// Bytes of scratch memory of launch_token_logprob and launch_policy_loss.
int64_t logits_workspace(int64_t rows, int64_t vocab, int32_t dtype);
hipError_t launch_token_logprob(hipStream_t st, const dlr_logits &x, void *workspace, float *logprob, float *lse);
hipError_t launch_token_logprob_grad(hipStream_t st, const dlr_logits &x, const float *lse, const float *grad,
                                     void *out, int64_t out_stride);
hipError_t launch_policy_loss(hipStream_t st, const dlr_logits &x, const dlr_policy &p, void *workspace, float *loss,
                              float *logprob, float *kl, uint8_t *clipped, void *out, int64_t out_stride);
hipError_t launch_preference_loss(hipStream_t st, const dlr_preference &p, float *loss, float *chosen,
                                  float *rejected, float *grad);

// Bytes of launch_head_logprob's workspace.
int64_t head_workspace(int64_t rows, int64_t vocab, int64_t dim);
hipError_t launch_head_logprob(hipStream_t st, const dlr_head &h, void *workspace, float *logprob, float *lse);

}  // namespace dlr
