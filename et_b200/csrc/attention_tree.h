// Host-side launchers of the kernels for drafted tokens over a cache in int8.
#pragma once
#include <cuda_runtime.h>
#include "attention_tree.cuh"

namespace et {

int attention_tree_launch(const TreeParams& p, cudaStream_t st);

}  // namespace et
