// Host-side launchers of the kernels for drafted tokens over a cache in int8.
#pragma once
#include <cuda_runtime.h>
#include "attention_tree.cuh"

namespace et {

int attention_tree_launch(const TreeParams& p, cudaStream_t st);
// tcgen05 kernel for many rows (attention_tree_tc.cu).
bool attention_tree_tc_takes(const TreeParams& p);
int attention_tree_tc_launch(const TreeParams& p, cudaStream_t st);

}  // namespace et
