// Orthogonalised update of Dense kernels by Newton-Schulz products (orth.cu).
#pragma once

#include "common.cuh"

namespace ml {

bool orth_workspace(const memlayer_orth_config& c, size_t* bytes);
// The iteration stays inside the range its 16-bit pieces have.
bool orth_coefficients_ok(const memlayer_orth_config& c);
cudaError_t launch_orthogonalize(const memlayer_orth_config& c, const void* update, void* out, char* ws,
                                 cudaStream_t s);

}  // namespace ml
