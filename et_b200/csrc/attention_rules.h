// Host-side launchers of the kernels of attention with rules on its scores.
#pragma once
#include <cuda_runtime.h>
#include "score_rules.cuh"

namespace et {

// Any head width and alignment: a warp to a query of a head.
cudaError_t attention_rules_rows_launch(const RuleParams& p, cudaStream_t st);

// A few queries over keys kept from before: heads of a multiple of 16 up to 128, rows that start on 16 bytes.
bool attention_rules_token_takes(const RuleParams& p);
int attention_rules_token_launch(const RuleParams& p, cudaStream_t st);
// Heads of a multiple of 16 up to 128 in rows that start on 16 bytes; scratch: documents' summary, or NULL without documents.
bool attention_rules_tc_takes(const RuleParams& p);
int attention_rules_tc_launch(const RuleParams& p, void* scratch, cudaStream_t st);

}  // namespace et
