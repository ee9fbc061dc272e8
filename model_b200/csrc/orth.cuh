// Orthogonalised update of Dense kernels by Newton-Schulz products (orth.cu;
// orth_chain.cu: small matrices in one launch).
#pragma once

#include "common.cuh"

namespace ml {

// Scale of the iteration's f16 pieces.
constexpr float kOrthScale = 4096.f;

bool orth_workspace(const memlayer_orth_config& c, size_t* bytes);
// The iteration stays inside the range its 16-bit pieces have.
bool orth_coefficients_ok(const memlayer_orth_config& c);
cudaError_t launch_orthogonalize(const memlayer_orth_config& c, const void* update, void* out, char* ws,
                                 cudaStream_t s);

// Matrices that a cluster's shared memory holds, and their iteration in one launch.
bool orth_in_cluster(const memlayer_orth_config& c);
cudaError_t launch_orth_chain(const memlayer_orth_config& c, const void* update, void* out, int* err, cudaStream_t s);

}  // namespace ml
