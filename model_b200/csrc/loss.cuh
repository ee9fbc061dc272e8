// Softmax cross entropy of hidden states against a vocabulary matrix, and its
// gradient, without the [tokens, vocabulary] logits (loss.cu).
#pragma once

#include "common.cuh"

namespace ml {

// Workspace bytes of a call; false: the sizes are out of range.
bool loss_workspace(const memlayer_loss_config& c, bool backward, size_t* bytes);

cudaError_t launch_loss_forward(const memlayer_loss_config& c, const memlayer_loss_args& a, char* ws, cudaStream_t s);
cudaError_t launch_loss_backward(const memlayer_loss_config& c, const memlayer_loss_args& a,
                                 const memlayer_loss_grads& g, char* ws, cudaStream_t s);

}  // namespace ml
