// Layer norm of the language model's blocks (memory_pool_model/model.py:87,
// 96,124) as an operator of its own, with its gradient:
//
//   s = x + residual (rounded to the storage type: the stream as stored)
//   y = (s - mean) rstd scale + bias,  rstd = 1 / sqrt(var + eps)
//   gy = dy scale,  c1 = mean(gy),  c2 = mean(gy xhat)
//   dx = rstd (gy - c1 - xhat c2) + dresidual
//   dscale = sum over rows of dy xhat,  dbias = sum over rows of dy
//
// Both passes are bound by HBM: every tensor crosses it once.  A row is held
// in the registers of `tpr` threads, 16 values each (16-byte accesses when
// width, row strides and addresses allow, single elements otherwise), so the
// variance is the centred one from registers -- E[x^2] - E[x]^2 loses the
// variance of a row whose mean is large -- and the gradient recomputes mean
// and rstd from the row it reads anyway instead of reading them back.
// Statistics and sums are float32 whatever the storage type.
//
// The parameter gradients: a block keeps dscale / dbias of its columns in
// registers over all of its rows, adds its row groups in shared memory and
// writes one partial row; a second kernel adds the partials in block order,
// so the result does not depend on timing (no atomics).
#include "norm.cuh"

namespace ml {

namespace {

constexpr int VALS = 16;          // values of a row per thread
constexpr int NT = 256;           // threads per block for rows of up to a warp

template <typename E> struct Elem;
template <> struct Elem<float> {
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};
template <> struct Elem<__half> {
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
};
template <> struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};

// The thread's share of a row: vector i holds columns (i tpr + t) VEC .. + VEC.
template <typename E, int VEC>
struct RowPart {
  static constexpr int NV = VALS / VEC;
  struct alignas(VEC * sizeof(E)) Vec { E e[VEC]; };
  Vec v[NV];
  __device__ __forceinline__ void load(const E* row, int t, int tpr, int d) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * tpr + t) * VEC;
      if (j < d) v[i] = *reinterpret_cast<const Vec*>(row + j);
    }
  }
  __device__ __forceinline__ void store(E* row, int t, int tpr, int d) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * tpr + t) * VEC;
      if (j < d) *reinterpret_cast<Vec*>(row + j) = v[i];
    }
  }
  __device__ __forceinline__ float get(int k) const { return Elem<E>::up(v[k / VEC].e[k % VEC]); }
  __device__ __forceinline__ void set(int k, float x) { v[k / VEC].e[k % VEC] = Elem<E>::down(x); }
};

template <int VEC>
__device__ __forceinline__ int col_of(int k, int t, int tpr) {
  return ((k / VEC) * tpr + t) * VEC + k % VEC;
}

// Sum over the tpr threads of a row.  Up to a warp: shuffles inside the
// group.  WIDE: one row per block, warp sums through `red` (one slot per
// warp; the leading barrier lets the slots be used again).
template <bool WIDE>
__device__ __forceinline__ float row_sum(float x, int tpr, float* red) {
  if constexpr (!WIDE) {
    for (int o = tpr >> 1; o > 0; o >>= 1) x += __shfl_xor_sync(FULL, x, o);
    return x;
  } else {
    x = warp_sum(x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
    __syncthreads();
    float t = (threadIdx.x & 31) < (tpr >> 5) ? red[threadIdx.x & 31] : 0.f;
    return warp_sum(t);
  }
}

struct NormArgs {
  int64_t rows;
  int d, tpr;
  float eps, inv_d;
  const void *x, *r, *dy, *dr;
  int64_t ldx, ldr, lddy, lddr;
  const float *scale, *bias;
  void *y, *sum, *dx;
  float* part;
};

template <typename E, int VEC, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 1024 : NT) layer_norm_kernel(NormArgs A) {
  __shared__ float red[32];
  using Part = RowPart<E, VEC>;
  const int tpr = A.tpr, d = A.d;
  const int t = threadIdx.x & (tpr - 1), g = threadIdx.x / tpr, groups = blockDim.x / tpr;
  const int64_t step = (int64_t)gridDim.x * groups;
  // whole warps run the same number of passes (the shuffles need every lane)
  for (int64_t base = (int64_t)blockIdx.x * groups; base < A.rows; base += step) {
    const int64_t row = base + g;
    const bool on = row < A.rows;
    const int64_t at = on ? row : 0;
    Part p;
    p.load(reinterpret_cast<const E*>(A.x) + at * A.ldx, t, tpr, d);
    if (A.r) {
      Part q;
      q.load(reinterpret_cast<const E*>(A.r) + at * A.ldr, t, tpr, d);
#pragma unroll
      for (int k = 0; k < VALS; ++k)
        if (col_of<VEC>(k, t, tpr) < d) p.set(k, p.get(k) + q.get(k));
      if (A.sum && on) p.store(reinterpret_cast<E*>(A.sum) + row * (int64_t)d, t, tpr, d);
    }
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < VALS; ++k)
      if (col_of<VEC>(k, t, tpr) < d) s += p.get(k);
    const float mean = row_sum<WIDE>(s, tpr, red) * A.inv_d;
    float s2 = 0.f;
#pragma unroll
    for (int k = 0; k < VALS; ++k)
      if (col_of<VEC>(k, t, tpr) < d) {
        const float c = p.get(k) - mean;
        s2 = fmaf(c, c, s2);
      }
    const float rstd = 1.0f / sqrtf(row_sum<WIDE>(s2, tpr, red) * A.inv_d + A.eps);
#pragma unroll
    for (int k = 0; k < VALS; ++k) {
      const int j = col_of<VEC>(k, t, tpr);
      if (j < d) p.set(k, fmaf((p.get(k) - mean) * rstd, A.scale[j], A.bias[j]));
    }
    if (on) p.store(reinterpret_cast<E*>(A.y) + row * (int64_t)d, t, tpr, d);
  }
}

template <typename E, int VEC, bool WIDE>
__global__ void __launch_bounds__(WIDE ? 1024 : NT) layer_norm_backward_kernel(NormArgs A) {
  __shared__ float red[32];
  extern __shared__ float cols[];          // !WIDE: [groups][VALS * tpr]
  using Part = RowPart<E, VEC>;
  const int tpr = A.tpr, d = A.d;
  const int t = threadIdx.x & (tpr - 1), g = threadIdx.x / tpr, groups = blockDim.x / tpr;
  const int64_t step = (int64_t)gridDim.x * groups;
  float ag[VALS], ab[VALS];
#pragma unroll
  for (int k = 0; k < VALS; ++k) ag[k] = ab[k] = 0.f;
  for (int64_t base = (int64_t)blockIdx.x * groups; base < A.rows; base += step) {
    const int64_t row = base + g;
    const bool on = row < A.rows;
    const int64_t at = on ? row : 0;
    Part p, q, r;
    p.load(reinterpret_cast<const E*>(A.x) + at * A.ldx, t, tpr, d);
    q.load(reinterpret_cast<const E*>(A.dy) + at * A.lddy, t, tpr, d);
    if (A.dr) r.load(reinterpret_cast<const E*>(A.dr) + at * A.lddr, t, tpr, d);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < VALS; ++k)
      if (col_of<VEC>(k, t, tpr) < d) s += p.get(k);
    const float mean = row_sum<WIDE>(s, tpr, red) * A.inv_d;
    float s2 = 0.f;
#pragma unroll
    for (int k = 0; k < VALS; ++k)
      if (col_of<VEC>(k, t, tpr) < d) {
        const float c = p.get(k) - mean;
        s2 = fmaf(c, c, s2);
      }
    const float rstd = 1.0f / sqrtf(row_sum<WIDE>(s2, tpr, red) * A.inv_d + A.eps);
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int k = 0; k < VALS; ++k) {
      const int j = col_of<VEC>(k, t, tpr);
      if (j < d) {
        const float xh = (p.get(k) - mean) * rstd, dy = q.get(k), gy = __fmul_rn(dy, A.scale[j]);
        c1 += gy;
        c2 = fmaf(gy, xh, c2);
        if (on) {
          ag[k] = fmaf(dy, xh, ag[k]);
          ab[k] += dy;
        }
      }
    }
    c1 = row_sum<WIDE>(c1, tpr, red) * A.inv_d;
    c2 = row_sum<WIDE>(c2, tpr, red) * A.inv_d;
#pragma unroll
    for (int k = 0; k < VALS; ++k) {
      const int j = col_of<VEC>(k, t, tpr);
      if (j < d) {
        const float xh = (p.get(k) - mean) * rstd;
        // the same rounded product as in c1: a constant row cancels exactly
        float x = rstd * (__fmul_rn(q.get(k), A.scale[j]) - c1 - xh * c2);
        if (A.dr) x += r.get(k);
        p.set(k, x);
      }
    }
    if (on) p.store(reinterpret_cast<E*>(A.dx) + row * (int64_t)d, t, tpr, d);
  }
  // the block's partial row: [dscale | dbias]
  float* out = A.part + (int64_t)blockIdx.x * 2 * d;
  if constexpr (WIDE) {
#pragma unroll
    for (int k = 0; k < VALS; ++k) {
      const int j = col_of<VEC>(k, t, tpr);
      if (j < d) {
        out[j] = ag[k];
        out[d + j] = ab[k];
      }
    }
  } else {
    const int w = VALS * tpr;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < VALS; ++k) cols[g * w + col_of<VEC>(k, t, tpr)] = which ? ab[k] : ag[k];
      __syncthreads();
      for (int j = threadIdx.x; j < d; j += blockDim.x) {
        float x = 0.f;
        for (int i = 0; i < groups; ++i) x += cols[i * w + j];
        out[which * d + j] = x;
      }
    }
  }
}

// dscale | dbias = the blocks' partial rows added in block order: 8 groups of
// blocks per column, then the groups in order.
__global__ void __launch_bounds__(256) layer_norm_params_kernel(const float* __restrict__ part, int blocks, int d,
                                                                float* __restrict__ dscale,
                                                                float* __restrict__ dbias) {
  __shared__ float red[8][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + c;
  float x = 0.f;
  if (j < 2 * d) {
    const float* p = part + j;
    int b = g;
    for (; b + 56 < blocks; b += 64) {      // eight loads in flight
      float a[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = p[(int64_t)(b + 8 * i) * 2 * d];
#pragma unroll
      for (int i = 0; i < 8; ++i) x += a[i];
    }
    for (; b < blocks; b += 8) x += p[(int64_t)b * 2 * d];
  }
  red[g][c] = x;
  __syncthreads();
  if (g == 0 && j < 2 * d) {
    float t = red[0][c];
#pragma unroll
    for (int i = 1; i < 8; ++i) t += red[i][c];
    (j < d ? dscale[j] : dbias[j - d]) = t;
  }
}

// Threads of a row: the power of two that holds its width at 16 values each.
int norm_tpr(int d) {
  int t = 4;
  while (t * VALS < d) t *= 2;
  return t;
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename E>
cudaError_t norm_forward_t(NormArgs& A, bool vec, cudaStream_t s) {
  constexpr int V = 16 / sizeof(E);
  const bool wide = A.tpr > 32;
  const int nt = wide ? A.tpr : NT;
  const int64_t need = (A.rows + nt / A.tpr - 1) / (nt / A.tpr);
  const int grid = (int)(need < (1 << 20) ? need : (1 << 20));
  if (vec)
    wide ? layer_norm_kernel<E, V, true><<<grid, nt, 0, s>>>(A) : layer_norm_kernel<E, V, false><<<grid, nt, 0, s>>>(A);
  else
    wide ? layer_norm_kernel<E, 1, true><<<grid, nt, 0, s>>>(A) : layer_norm_kernel<E, 1, false><<<grid, nt, 0, s>>>(A);
  count_launch();
  return cudaGetLastError();
}

template <typename E>
cudaError_t norm_backward_t(NormArgs& A, bool vec, int grid, cudaStream_t s) {
  constexpr int V = 16 / sizeof(E);
  const bool wide = A.tpr > 32;
  const int nt = wide ? A.tpr : NT;
  const size_t sm = wide ? 0 : (size_t)nt * VALS * sizeof(float);   // 16 KB
  if (vec)
    wide ? layer_norm_backward_kernel<E, V, true><<<grid, nt, sm, s>>>(A)
         : layer_norm_backward_kernel<E, V, false><<<grid, nt, sm, s>>>(A);
  else
    wide ? layer_norm_backward_kernel<E, 1, true><<<grid, nt, sm, s>>>(A)
         : layer_norm_backward_kernel<E, 1, false><<<grid, nt, sm, s>>>(A);
  count_launch();
  return cudaGetLastError();
}

}  // namespace

int norm_backward_blocks(int64_t rows, int d) {
  const int tpr = norm_tpr(d), nt = tpr > 32 ? tpr : NT;
  const int64_t need = (rows + nt / tpr - 1) / (nt / tpr);
  const int64_t cap = (int64_t)sm_count() * (nt >= 1024 ? 1 : nt >= 512 ? 1 : 512 / nt);
  return (int)(need < cap ? need : cap);
}

cudaError_t launch_layer_norm(const memlayer_norm_config& c, const memlayer_norm_args& a, cudaStream_t s) {
  if (c.rows == 0) return cudaSuccess;
  NormArgs A{};
  A.rows = c.rows;
  A.d = c.d_model;
  A.tpr = norm_tpr(c.d_model);
  A.eps = c.epsilon;
  A.inv_d = 1.0f / (float)c.d_model;
  A.x = a.x;
  A.r = a.residual;
  A.ldx = a.x_stride;
  A.ldr = a.residual_stride;
  A.scale = a.scale;
  A.bias = a.bias;
  A.y = a.y;
  A.sum = a.sum;
  const int v = c.dtype == MEMLAYER_F32 ? 4 : 8;
  const bool vec = c.d_model % v == 0 && a.x_stride % v == 0 && (!a.residual || a.residual_stride % v == 0) &&
                   al16(a.x) && al16(a.residual) && al16(a.y) && al16(a.sum);
  switch (c.dtype) {
    case MEMLAYER_F16: return norm_forward_t<__half>(A, vec, s);
    case MEMLAYER_BF16: return norm_forward_t<__nv_bfloat16>(A, vec, s);
    default: return norm_forward_t<float>(A, vec, s);
  }
}

cudaError_t launch_layer_norm_backward(const memlayer_norm_config& c, const memlayer_norm_grads& g, float* part,
                                       cudaStream_t s) {
  NormArgs A{};
  A.rows = c.rows;
  A.d = c.d_model;
  A.tpr = norm_tpr(c.d_model);
  A.eps = c.epsilon;
  A.inv_d = 1.0f / (float)c.d_model;
  A.x = g.x;
  A.dy = g.dy;
  A.dr = g.dresidual;
  A.ldx = g.x_stride;
  A.lddy = g.dy_stride;
  A.lddr = g.dresidual_stride;
  A.scale = g.scale;
  A.dx = g.dx;
  A.part = part;
  const int v = c.dtype == MEMLAYER_F32 ? 4 : 8;
  const bool vec = c.d_model % v == 0 && g.x_stride % v == 0 && g.dy_stride % v == 0 &&
                   (!g.dresidual || g.dresidual_stride % v == 0) && al16(g.x) && al16(g.dy) && al16(g.dresidual) &&
                   al16(g.dx);
  const int grid = norm_backward_blocks(c.rows, c.d_model);
  cudaError_t e = cudaSuccess;
  if (grid > 0) switch (c.dtype) {
      case MEMLAYER_F16: e = norm_backward_t<__half>(A, vec, grid, s); break;
      case MEMLAYER_BF16: e = norm_backward_t<__nv_bfloat16>(A, vec, grid, s); break;
      default: e = norm_backward_t<float>(A, vec, grid, s); break;
    }
  if (e != cudaSuccess) return e;
  layer_norm_params_kernel<<<(2 * c.d_model + 31) / 32, 256, 0, s>>>(part, grid, c.d_model, g.dscale, g.dbias);
  count_launch();
  return cudaGetLastError();
}

}  // namespace ml
