// Host-side launchers of the kernels of attention with rules on its scores.
#pragma once
#include <cuda_runtime.h>
#include "score_rules.cuh"

namespace et {

// Any head width and alignment: a warp to a query of a head.
cudaError_t attention_rules_rows_launch(const RuleParams& p, cudaStream_t st);

}  // namespace et
