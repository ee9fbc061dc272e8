// 16-bit forms of matrices for the GEMM of gemm16.cuh (gemm16.cu).
#pragma once

#include "common.cuh"

namespace ml {

namespace g16 {

int device_sms();

// (a, b) as f16 hi + lo.
__device__ __forceinline__ void split2(float a, float b, __half2& hi, __half2& lo) {
  hi = __floats2half2_rn(a, b);
  const float2 f = __half22float2(hi);
  lo = __floats2half2_rn(a - f.x, b - f.y);
}

}  // namespace g16

constexpr int PIECE_THREADS = 256;

// Blocks of PIECE_THREADS for so many items.
inline int piece_blocks(int64_t items, int per_thread) {
  const int64_t per = (int64_t)PIECE_THREADS * per_thread, b = (items + per - 1) / per, cap = 8 * g16::device_sms();
  return (int)(b < 1 ? 1 : b < cap ? b : cap);
}

// Bits of |x| where x is finite, else 0 (the order of non-negative floats is that of their bits).
__device__ __forceinline__ unsigned finite_bits(float x) {
  const unsigned u = __float_as_uint(x) & 0x7FFFFFFFu;
  return u < 0x7F800000u ? u : 0u;
}

struct AmaxMat {
  const float* x;
  int64_t rows, cols, pitch;
  unsigned* out;               // zeroed by the caller
  int blocks;
};

// Block b of the search for the largest finite magnitude of a float32 matrix.
__device__ __forceinline__ void amax_block(const AmaxMat& M, int b) {
  __shared__ unsigned red[PIECE_THREADS / 32];
  unsigned mx = 0;
  const int64_t step = (int64_t)M.blocks * PIECE_THREADS, at = (int64_t)b * PIECE_THREADS + threadIdx.x;
  if (M.pitch == M.cols && (reinterpret_cast<uintptr_t>(M.x) & 15) == 0) {
    const int64_t n = M.rows * M.cols, n4 = n >> 2;
    const float4* x4 = reinterpret_cast<const float4*>(M.x);
    auto take4 = [&](float4 v) {
      mx = max(max(mx, max(finite_bits(v.x), finite_bits(v.y))), max(finite_bits(v.z), finite_bits(v.w)));
    };
    int64_t e = at;
    for (; e + 3 * step < n4; e += 4 * step) {     // four loads in flight
      float4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = x4[e + j * step];
#pragma unroll
      for (int j = 0; j < 4; ++j) take4(v[j]);
    }
    for (; e < n4; e += step) take4(x4[e]);
    if (at < (n & 3)) mx = max(mx, finite_bits(M.x[(n4 << 2) + at]));
  } else {
    const int64_t n = M.rows * M.cols;
    for (int64_t e = at; e < n; e += step) mx = max(mx, finite_bits(M.x[(e / M.cols) * M.pitch + e % M.cols]));
  }
  mx = __reduce_max_sync(FULL, mx);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mx;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < PIECE_THREADS / 32; ++w) mx = max(mx, red[w]);
    if (mx) atomicMax(M.out, mx);                  // a maximum: the order does not matter
  }
}

struct PiecesMat {
  const void* x;               // rows x cols, row pitch `pitch`
  int64_t rows, cols, pitch;
  void *hi, *lo;               // rows x ld (ld a multiple of 8); lo: float32 sources only
  int64_t ld;
  const unsigned* amax;        // float32 sources: the largest magnitude, for a scale of the matrix; or
  const int* row_tgt;          // by row: PIECE_SKIP leaves it out (zeros),
  const int* row_exp;          // else it goes by piece_exp(*peak) - row_exp (float32 and f16; null: unscaled)
  const unsigned* peak;
  int blocks;
};
constexpr int PIECE_SKIP = -2;
// The largest exponent of a row less its row_exp, as a word for atomicMax (0:
// no row), and the power of two that brings it to 2^14.
__device__ __forceinline__ unsigned piece_peak(int e) { return (unsigned)(e + 1024); }
__device__ __forceinline__ int piece_exp(unsigned peak) { return peak ? 14 - ((int)peak - 1024) : 0; }
struct PiecesArgs { PiecesMat m[3]; };

// Pieces (float32) or padded copies (16-bit) of up to three matrices.
cudaError_t launch_pieces(PiecesArgs A, int dtype, cudaStream_t s);

}  // namespace ml
