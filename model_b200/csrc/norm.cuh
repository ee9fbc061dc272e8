// Layer norm with a fused residual add, and its gradient (norm.cu).
#pragma once

#include "common.cuh"

namespace ml {

constexpr int kNormMaxWidth = 16384;   // 1024 threads x 16 values in registers

// Most blocks of the gradient's row pass (its column partials: blocks x 2 x d floats).
int norm_backward_blocks(int64_t rows, int d, int dtype);

cudaError_t launch_layer_norm(const memlayer_norm_config& c, const memlayer_norm_args& a, cudaStream_t s);
cudaError_t launch_layer_norm_backward(const memlayer_norm_config& c, const memlayer_norm_grads& g, float* part,
                                       int* err, cudaStream_t s);

}  // namespace ml
