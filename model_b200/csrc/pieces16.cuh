// 16-bit forms of matrices for the GEMM of gemm16.cuh (gemm16.cu).
#pragma once

#include "common.cuh"

namespace ml {

namespace g16 {

// (a, b) as f16 hi + lo.
__device__ __forceinline__ void split2(float a, float b, __half2& hi, __half2& lo) {
  hi = __floats2half2_rn(a, b);
  const float2 f = __half22float2(hi);
  lo = __floats2half2_rn(a - f.x, b - f.y);
}

}  // namespace g16

struct AmaxMat {
  const float* x;
  int64_t rows, cols, pitch;
  unsigned* out;               // zeroed by the caller
  int blocks;                  // set by the launcher
};
struct AmaxArgs { AmaxMat m[4]; };

struct PiecesMat {
  const void* x;               // rows x cols, row pitch `pitch`
  int64_t rows, cols, pitch;
  void *hi, *lo;               // rows x ld (ld a multiple of 8); lo: float32 sources only
  int64_t ld;
  const unsigned* amax;        // float32 sources: the scale's maximum
  int blocks;
};
struct PiecesArgs { PiecesMat m[2]; };

// Largest finite magnitudes of up to four float32 matrices (rows 0: none).
cudaError_t launch_amax(AmaxArgs A, cudaStream_t s);
// Pieces (float32) or padded copies (16-bit) of up to two matrices.
cudaError_t launch_pieces(PiecesArgs A, int dtype, cudaStream_t s);

}  // namespace ml
