// Launchers behind the entry points of mamba3_b200_lm.h.
#pragma once

#include <cuda_runtime.h>

#include "mamba3_b200_lm.h"

namespace m3 {

// Products with 4-bit weights (m3_w4.cu); arguments already validated.
cudaError_t launch_linear_w4(const m3_w4_args &a, cudaStream_t stream);

// Logit adjustments and the choice of the next token (m3_logits.cu);
// arguments already validated.
cudaError_t launch_process_logits(const m3_logits_args &a, cudaStream_t stream);
cudaError_t launch_next_tokens(const m3_logits_args &a, cudaStream_t stream);

}  // namespace m3
