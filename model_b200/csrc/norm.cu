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
// in registers, so the variance is the centred one -- E[x^2] - E[x]^2 loses
// the variance of a row whose mean is large -- and the gradient recomputes
// mean and rstd from the row it reads anyway instead of reading them back.
// A float32 mean is off by some units of its last place, which is the whole of
// a centred value where the row is (nearly) constant: its xhat came to 1
// instead of 0 at values of 1e4.  So the centred values are summed beside their
// squares; their mean is what the first one was off by, and is taken out.
// Statistics and sums are float32 whatever the storage type.  Three layouts:
//
//   group   a row in a power of two of threads, 16 values each; up to a warp
//           (512 columns) its sums are shuffles.  Also every width whose rows
//           16-byte accesses cannot reach, with single elements;
//   warp    the forward up to 512 vectors, the gradient up to 2048 columns: a
//           row in a warp, no barriers.  The gradient keeps its columns'
//           parameter sums in registers (64 columns a lane), so few warps fit
//           an SM; a ring of rows in shared memory, filled by bulk copies,
//           keeps HBM busy beside them.  In a block per row its reductions
//           took four times the instructions (16384 x 2048 bf16: 113 us for
//           the 66 of the ring);
//   wide    beyond, a block per row.  Also packed rows of more than 512
//           columns whose width is no multiple of a vector, by vectors that
//           the rows begin inside of (forward and gradient of 9557 x 2498
//           bf16 68 + 130 us, by single elements 211 + 304).
//
// The parameter gradients: dscale / dbias of the columns stay in registers over
// all of a block's rows; it adds its row groups in shared memory and writes one
// partial row; a second kernel adds the partials, 32 groups of blocks in block
// order and the groups in a fixed tree, so the result does not depend on timing
// (no atomics).
//
// Launches are dependent ones: a kernel's start hides behind the end of the
// one before it (8192 x 256 float32, forward and gradient: 22.3 us for 24.6).
#include "norm.cuh"

#include <algorithm>
#include <numeric>

#include "gemm16.cuh"

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

// The variance from the mean square around a mean that is `off` from the row's.
__device__ __forceinline__ float variance(float mean_square, float off) {
  return fmaxf(fmaf(-off, off, mean_square), 0.f);
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
  int* err;             // status word (gradient), cleared by the first block
};

// MAXT > 0: a row in the whole block (at most MAXT threads).
template <typename E, int VEC, int MAXT>
__global__ void __launch_bounds__(MAXT ? MAXT : NT, MAXT ? 1 : 2) layer_norm_kernel(NormArgs A) {
  constexpr bool WIDE = MAXT > 0;
  __shared__ float red[32];
  allow_next();
  wait_previous();
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
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < VALS; ++k)
      if (col_of<VEC>(k, t, tpr) < d) {
        const float c = p.get(k) - mean;
        s1 += c;
        s2 = fmaf(c, c, s2);
      }
    const float off = row_sum<WIDE>(s1, tpr, red) * A.inv_d;
    const float rstd = 1.0f / sqrtf(variance(row_sum<WIDE>(s2, tpr, red) * A.inv_d, off) + A.eps);
#pragma unroll
    for (int k = 0; k < VALS; ++k) {
      const int j = col_of<VEC>(k, t, tpr);
      if (j < d) p.set(k, fmaf((p.get(k) - mean - off) * rstd, A.scale[j], A.bias[j]));
    }
    if (on) p.store(reinterpret_cast<E*>(A.y) + row * (int64_t)d, t, tpr, d);
  }
}

template <typename E, int VEC, int MAXT>
__global__ void __launch_bounds__(MAXT ? MAXT : NT, MAXT ? 1 : 2) layer_norm_backward_kernel(NormArgs A) {
  constexpr bool WIDE = MAXT > 0;
  __shared__ float red[32];
  allow_next();
  wait_previous();
  extern __shared__ float cols[];          // !WIDE: [groups][VALS * tpr]
  using Part = RowPart<E, VEC>;
  const int tpr = A.tpr, d = A.d;
  const int t = threadIdx.x & (tpr - 1), g = threadIdx.x / tpr, groups = blockDim.x / tpr;
  const int64_t step = (int64_t)gridDim.x * groups;
  if (blockIdx.x == 0 && threadIdx.x == 0) *A.err = 0;
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
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < VALS; ++k)
      if (col_of<VEC>(k, t, tpr) < d) {
        const float c = p.get(k) - mean;
        s1 += c;
        s2 = fmaf(c, c, s2);
      }
    const float off = row_sum<WIDE>(s1, tpr, red) * A.inv_d;
    const float rstd = 1.0f / sqrtf(variance(row_sum<WIDE>(s2, tpr, red) * A.inv_d, off) + A.eps);
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int k = 0; k < VALS; ++k) {
      const int j = col_of<VEC>(k, t, tpr);
      if (j < d) {
        const float xh = (p.get(k) - mean - off) * rstd, dy = q.get(k), gy = __fmul_rn(dy, A.scale[j]);
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
        const float xh = (p.get(k) - mean - off) * rstd;
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

// ---- wide rows ---------------------------------------------------------------------
template <typename E, int V>
struct alignas(V * sizeof(E)) Vec16 { E e[V]; };

// Sums of N values over the block, the same in every thread: warp sums in
// `red` (32 slots a value, those without a warp zero), added in warp order.
// One barrier: callers alternate two buffers.
template <int N>
__device__ __forceinline__ void block_sums(float (&x)[N], float* red) {
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = warp_sum(x[i]);
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[i * 32 + warp] = x[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float4* r4 = reinterpret_cast<const float4*>(red + i * 32);
    float t = 0.f;
    for (int w = 0; w < warps; w += 4) {
      const float4 r = r4[w >> 2];
      t += (r.x + r.y) + (r.z + r.w);
    }
    x[i] = t;
  }
}

// Two float32 at once (the packed forms of add, multiply and fused
// multiply-add: half the instructions, the same roundings).
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ void split(F2 x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float sum(F2 x) {
  float a, b;
  split(x, a, b);
  return a + b;
}

__device__ __forceinline__ void unpack2(const Vec16<float, 4>& v, F2 (&x)[2]) {
  x[0] = f2(v.e[0], v.e[1]);
  x[1] = f2(v.e[2], v.e[3]);
}
__device__ __forceinline__ void unpack2(const Vec16<__half, 8>& v, F2 (&x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(v.e + 2 * k));
    x[k] = f2(t.x, t.y);
  }
}
__device__ __forceinline__ void unpack2(const Vec16<__nv_bfloat16, 8>& v, F2 (&x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const unsigned u = *reinterpret_cast<const unsigned*>(v.e + 2 * k);
    x[k] = f2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  }
}

template <typename E, int V>
__device__ __forceinline__ void unpack(const Vec16<E, V>& v, float (&x)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) x[k] = Elem<E>::up(v.e[k]);
}

template <int V>
__device__ __forceinline__ void load_f32(const float* p, float (&x)[V]) {
  if constexpr (V == 1) x[0] = __ldg(p);
#pragma unroll
  for (int k = 0; k + 4 <= V; k += 4) {
    const float4 t = __ldg(reinterpret_cast<const float4*>(p + k));
    x[k] = t.x;
    x[k + 1] = t.y;
    x[k + 2] = t.z;
    x[k + 3] = t.w;
  }
}

template <typename E>
__device__ __forceinline__ void pack(Vec16<E, 1>& v, const float (&x)[1]) {
  v.e[0] = Elem<E>::down(x[0]);
}
__device__ __forceinline__ void pack(Vec16<float, 4>& v, const float (&x)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) v.e[k] = x[k];
}
__device__ __forceinline__ void pack(Vec16<__half, 8>& v, const float (&x)[8]) {
#pragma unroll
  for (int k = 0; k < 8; k += 2) *reinterpret_cast<__half2*>(v.e + k) = __floats2half2_rn(x[k], x[k + 1]);
}
__device__ __forceinline__ void pack(Vec16<__nv_bfloat16, 8>& v, const float (&x)[8]) {
#pragma unroll
  for (int k = 0; k < 8; k += 2) *reinterpret_cast<__nv_bfloat162*>(v.e + k) = __floats2bfloat162_rn(x[k], x[k + 1]);
}

// A row in a warp: vector i of lane t is columns (32 i + t) V .. + V.  No
// barrier, and 12 to 24 warps an SM with 8 KB of loads in flight each.
template <typename E, int V, int NV>
__global__ void __launch_bounds__(128) layer_norm_warp_kernel(NormArgs A) {
  using Vec = Vec16<E, V>;
  allow_next();
  wait_previous();
  const int d = A.d, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= A.rows) return;
  Vec p[NV];
  const E* x = reinterpret_cast<const E*>(A.x) + row * A.ldx;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (i * 32 + lane) * V;
    if (j < d) p[i] = *reinterpret_cast<const Vec*>(x + j);
  }
  if (A.r) {
    Vec q[NV];
    const E* r = reinterpret_cast<const E*>(A.r) + row * A.ldr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * 32 + lane) * V;
      if (j < d) q[i] = *reinterpret_cast<const Vec*>(r + j);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * 32 + lane) * V;
      if (j >= d) continue;
      float a[V], b[V];
      unpack(p[i], a);
      unpack(q[i], b);
#pragma unroll
      for (int k = 0; k < V; ++k) a[k] += b[k];
      pack(p[i], a);
      if (A.sum) *reinterpret_cast<Vec*>(reinterpret_cast<E*>(A.sum) + row * (int64_t)d + j) = p[i];
    }
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * 32 + lane) * V < d) {
      float a[V];
      unpack(p[i], a);
#pragma unroll
      for (int k = 0; k < V; ++k) s += a[k];
    }
  const float mean = warp_sum(s) * A.inv_d;
  float s1 = 0.f, s2 = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * 32 + lane) * V < d) {
      float a[V];
      unpack(p[i], a);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float c = a[k] - mean;
        s1 += c;
        s2 = fmaf(c, c, s2);
      }
    }
  const float off = warp_sum(s1) * A.inv_d;
  const float rstd = 1.0f / sqrtf(variance(warp_sum(s2) * A.inv_d, off) + A.eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (i * 32 + lane) * V;
    if (j >= d) continue;
    float a[V], sc[V], bi[V];
    unpack(p[i], a);
    load_f32(A.scale + j, sc);
    load_f32(A.bias + j, bi);
#pragma unroll
    for (int k = 0; k < V; ++k) a[k] = fmaf((a[k] - mean - off) * rstd, sc[k], bi[k]);
    pack(p[i], a);
    *reinterpret_cast<Vec*>(reinterpret_cast<E*>(A.y) + row * (int64_t)d + j) = p[i];
  }
}

// Rows one after another in memory whose width is no multiple of a vector
// (SHIFT): row r starts r d mod V entries into one.  A block takes rows of
// the same start, so its columns keep their threads; the vectors at a row's
// ends hold entries of the rows beside it, which are loaded with them (but
// not past the last row), count for nothing and are not stored.
template <int V>
__device__ __forceinline__ bool at_edge(int j, int d) { return j < 0 || j + V > d; }
template <int V>
__device__ __forceinline__ bool in_row(int j, int k, int d) { return (unsigned)(j + k) < (unsigned)d; }

template <typename E, int V, bool SHIFT>
__device__ __forceinline__ Vec16<E, V> load_part(const E* row, int j, int d, bool last) {
  if (SHIFT && last && j + V > d) {
    Vec16<E, V> v;
#pragma unroll
    for (int k = 0; k < V; ++k) v.e[k] = j + k < d ? row[j + k] : Elem<E>::down(0.f);
    return v;
  }
  return *reinterpret_cast<const Vec16<E, V>*>(row + j);
}
template <typename E, int V, bool SHIFT>
__device__ __forceinline__ void store_part(E* row, int j, int d, const Vec16<E, V>& v) {
  if (SHIFT && at_edge<V>(j, d)) {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (in_row<V>(j, k, d)) row[j + k] = v.e[k];
  } else {
    *reinterpret_cast<Vec16<E, V>*>(row + j) = v;
  }
}
// The entries of other rows replaced.
template <int V, bool SHIFT>
__device__ __forceinline__ void keep_row(float (&x)[V], int j, int d, float other) {
  if (SHIFT && at_edge<V>(j, d)) {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (!in_row<V>(j, k, d)) x[k] = other;
  }
}
template <int V, bool SHIFT>
__device__ __forceinline__ void keep_row(F2 (&x)[V / 2], int j, int d, float other) {
  if (SHIFT && at_edge<V>(j, d)) {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      float a, b;
      split(x[k], a, b);
      x[k] = f2(in_row<V>(j, 2 * k, d) ? a : other, in_row<V>(j, 2 * k + 1, d) ? b : other);
    }
  }
}
// The parameters of a thread's columns: aligned, or entry by entry, zeros outside.
template <int V, bool SHIFT>
__device__ __forceinline__ void load_columns(const float* p, int j, int d, float (&x)[V]) {
  if constexpr (SHIFT) {
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = in_row<V>(j, k, d) ? p[j + k] : 0.f;
  } else {
    load_f32(p + j, x);
  }
}
template <int V, bool SHIFT>
__device__ __forceinline__ int block_shift(int d) { return SHIFT ? (int)((blockIdx.x * (unsigned)d) & (V - 1)) : 0; }

// A row in a block, for rows that a warp does not hold: thread t has columns
// (i blockDim + t) V .. + V, i < NV (less the shift).
template <typename E, int NV, int MAXT, int MINB, bool SHIFT>
__global__ void __launch_bounds__(MAXT, MINB) layer_norm_wide_kernel(NormArgs A) {
  constexpr int V = 16 / sizeof(E);
  using Vec = Vec16<E, V>;
  __shared__ alignas(16) float red[2][2 * 32];
  const int d = A.d, t = threadIdx.x, nt = blockDim.x, o = block_shift<V, SHIFT>(d);
  allow_next();
  wait_previous();
  for (int i = t; i < 2 * 2 * 32; i += nt) (&red[0][0])[i] = 0.f;       // slots without a warp
  __syncthreads();
  float scale[NV][V], bias[NV][V];       // SHIFT: kept over the block's rows
  if constexpr (SHIFT) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * nt + t) * V - o;
      if (j >= d) continue;
      load_columns<V, true>(A.scale, j, d, scale[i]);
      load_columns<V, true>(A.bias, j, d, bias[i]);
    }
  }
  for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
    const bool last = row + 1 == A.rows;
    Vec p[NV], q[NV];
    float s[1] = {0.f}, s2[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * nt + t) * V - o;
      if (j >= d) continue;
      p[i] = load_part<E, V, SHIFT>(reinterpret_cast<const E*>(A.x) + row * A.ldx, j, d, last);
      if (A.r) q[i] = load_part<E, V, SHIFT>(reinterpret_cast<const E*>(A.r) + row * A.ldr, j, d, last);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * nt + t) * V - o;
      if (j >= d) continue;
      float a[V];
      unpack(p[i], a);
      if (A.r) {
        float b[V];
        unpack(q[i], b);
#pragma unroll
        for (int k = 0; k < V; ++k) a[k] += b[k];
        pack(p[i], a);
        unpack(p[i], a);
        if (A.sum) store_part<E, V, SHIFT>(reinterpret_cast<E*>(A.sum) + row * (int64_t)d, j, d, p[i]);
      }
      keep_row<V, SHIFT>(a, j, d, 0.f);
#pragma unroll
      for (int k = 0; k < V; ++k) s[0] += a[k];
    }
    block_sums(s, red[0]);
    const float mean = s[0] * A.inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * nt + t) * V - o;
      if (j >= d) continue;
      float a[V];
      unpack(p[i], a);
      keep_row<V, SHIFT>(a, j, d, mean);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float c = a[k] - mean;
        s2[0] = fmaf(c, c, s2[0]);
        s2[1] += c;
      }
    }
    block_sums(s2, red[1]);
    const float off = s2[1] * A.inv_d;
    const float rstd = 1.0f / sqrtf(variance(s2[0] * A.inv_d, off) + A.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * nt + t) * V - o;
      if (j >= d) continue;
      float a[V], sc[V], bi[V];
      unpack(p[i], a);
      if constexpr (SHIFT) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          sc[k] = scale[i][k];
          bi[k] = bias[i][k];
        }
      } else {
        load_f32(A.scale + j, sc);
        load_f32(A.bias + j, bi);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) a[k] = fmaf((a[k] - mean - off) * rstd, sc[k], bi[k]);
      pack(p[i], a);
      store_part<E, V, SHIFT>(reinterpret_cast<E*>(A.y) + row * (int64_t)d, j, d, p[i]);
    }
  }
}

// A block's row, as loaded.
template <typename E, int NV, bool SHIFT>
struct WideRow {
  static constexpr int V = 16 / sizeof(E);
  Vec16<E, V> p[NV], q[NV], e[NV];
  __device__ __forceinline__ void load(const NormArgs& A, int64_t row, int o) {
    if (row >= A.rows) return;
    const int t = threadIdx.x, nt = blockDim.x;
    const bool last = row + 1 == A.rows;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * nt + t) * V - o;
      if (j >= A.d) continue;
      p[i] = load_part<E, V, SHIFT>(reinterpret_cast<const E*>(A.x) + row * A.ldx, j, A.d, last);
      q[i] = load_part<E, V, SHIFT>(reinterpret_cast<const E*>(A.dy) + row * A.lddy, j, A.d, last);
      if (A.dr) e[i] = load_part<E, V, SHIFT>(reinterpret_cast<const E*>(A.dr) + row * A.lddr, j, A.d, last);
    }
  }
};

// AHEAD: the next row's loads are issued before this one's sums, so HBM is
// busy during the barriers (where the registers allow it: shifted 16-bit rows
// would spill, 155 us for 130 at 9557 x 2498).
template <typename E, int NV, int MAXT, int MINB, bool AHEAD, bool SHIFT>
__global__ void __launch_bounds__(MAXT, MINB) layer_norm_wide_backward_kernel(NormArgs A) {
  constexpr int V = 16 / sizeof(E), H = V / 2;
  using Vec = Vec16<E, V>;
  allow_next();
  wait_previous();
  __shared__ alignas(16) float red[2][4 * 32];
  const int d = A.d, t = threadIdx.x, nt = blockDim.x, o = block_shift<V, SHIFT>(d);
  for (int i = t; i < 2 * 4 * 32; i += nt) (&red[0][0])[i] = 0.f;       // slots without a warp
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) *A.err = 0;
  F2 ag[NV][H], ab[NV][H], sc[NV][H];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (i * nt + t) * V - o;
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = 0.f;
    if (j < d) load_columns<V, SHIFT>(A.scale, j, d, f);
#pragma unroll
    for (int k = 0; k < H; ++k) {
      ag[i][k] = ab[i][k] = f2(0.f);
      sc[i][k] = f2(f[2 * k], f[2 * k + 1]);
    }
  }
  WideRow<E, NV, SHIFT> next;
  if constexpr (AHEAD) next.load(A, blockIdx.x, o);
  for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
    WideRow<E, NV, SHIFT> b;
    if constexpr (AHEAD) {
      b = next;
      next.load(A, row + gridDim.x, o);
    } else {
      b.load(A, row, o);
    }
    float s[1];
    {
      F2 acc = f2(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (const int j = (i * nt + t) * V - o; j < d) {
          F2 a[H];
          unpack2(b.p[i], a);
          keep_row<V, SHIFT>(a, j, d, 0.f);
#pragma unroll
          for (int k = 0; k < H; ++k) acc = acc + a[k];
        }
      s[0] = sum(acc);
    }
    block_sums(s, red[0]);
    // around the mean: sum c^2, sum gy, sum gy c (c2 = rstd times it), sum c
    const float mean_f = s[0] * A.inv_d;
    const F2 mean = f2(-mean_f);
    float m[4];
    {
      F2 s1 = f2(0.f), s2 = f2(0.f), sg = f2(0.f), sgc = f2(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (const int j = (i * nt + t) * V - o; j < d) {
          F2 a[H], g[H];
          unpack2(b.p[i], a);
          unpack2(b.q[i], g);
          keep_row<V, SHIFT>(a, j, d, mean_f);
          keep_row<V, SHIFT>(g, j, d, 0.f);
#pragma unroll
          for (int k = 0; k < H; ++k) {
            const F2 c = a[k] + mean, gy = g[k] * sc[i][k];
            s1 = s1 + c;
            s2 = fma2(c, c, s2);
            sg = sg + gy;
            sgc = fma2(gy, c, sgc);
          }
        }
      m[0] = sum(s2);
      m[1] = sum(sg);
      m[2] = sum(sgc);
      m[3] = sum(s1);
    }
    block_sums(m, red[1]);
    // rsqrtf: within 2 units of the last place
    const float off = m[3] * A.inv_d, rstd_f = rsqrtf(variance(m[0] * A.inv_d, off) + A.eps);
    const F2 rstd = f2(rstd_f), c1 = f2(-(m[1] * A.inv_d)), c2 = f2(-(fmaf(-off, m[1], m[2]) * rstd_f * A.inv_d)),
             noff = f2(-off);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * nt + t) * V - o;
      if (j >= d) continue;
      F2 a[H], g[H];
      float x[V];
      unpack2(b.p[i], a);
      unpack2(b.q[i], g);
#pragma unroll
      for (int k = 0; k < H; ++k) {
        const F2 xh = (a[k] + mean + noff) * rstd;
        ag[i][k] = fma2(g[k], xh, ag[i][k]);
        ab[i][k] = ab[i][k] + g[k];
        a[k] = rstd * fma2(xh, c2, g[k] * sc[i][k] + c1);
      }
      if (A.dr) {
        unpack2(b.e[i], g);
#pragma unroll
        for (int k = 0; k < H; ++k) a[k] = a[k] + g[k];
      }
#pragma unroll
      for (int k = 0; k < H; ++k) split(a[k], x[2 * k], x[2 * k + 1]);
      Vec v;
      pack(v, x);
      store_part<E, V, SHIFT>(reinterpret_cast<E*>(A.dx) + row * (int64_t)d, j, d, v);
    }
  }
  float* out = A.part + (int64_t)blockIdx.x * 2 * d;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (i * nt + t) * V - o;
    if (j >= d) continue;
#pragma unroll
    for (int k = 0; k < H; ++k) {
      float a, c;
      split(ag[i][k], a, c);
      if (!SHIFT || in_row<V>(j, 2 * k, d)) out[j + 2 * k] = a;
      if (!SHIFT || in_row<V>(j, 2 * k + 1, d)) out[j + 2 * k + 1] = c;
      split(ab[i][k], a, c);
      if (!SHIFT || in_row<V>(j, 2 * k, d)) out[d + j + 2 * k] = a;
      if (!SHIFT || in_row<V>(j, 2 * k + 1, d)) out[d + j + 2 * k + 1] = c;
    }
  }
}

// The gradient of rows that a warp holds: a warp per row, without a barrier.
// Each warp streams its rows of x and dy through a ring of its own in shared
// memory (bulk copies, signalled by mbarriers) and reads them from there: the
// mean, the four sums around it, dx.  The columns' parameter sums stay in its
// registers over all of its rows; the block adds its warps' at the end.
template <typename E, int NV, int MAXW>
__global__ void __launch_bounds__(MAXW * 32, 1) layer_norm_ring_backward_kernel(NormArgs A, int stages) {
  constexpr int V = 16 / sizeof(E), H = V / 2;
  using Vec = Vec16<E, V>;
  extern __shared__ uint8_t smem_raw[];
  allow_next();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int d = A.d, rb = d * (int)sizeof(E);
  constexpr int tensors = 2;                 // x and dy
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem) + warp * 4;              // 4 stages at most
  volatile int* abort = reinterpret_cast<int*>(smem + 12 * 32);
  float* scale_s = reinterpret_cast<float*>(smem + 512);
  uint8_t* rings = smem + 512 + (((size_t)d * 4 + 127) & ~size_t(127));
  const int rbp = (rb + 127) & ~127;                                           // a row's pitch in the ring
  uint8_t* ring = rings + (size_t)warp * stages * tensors * rbp;
  if (lane == 0)
    for (int i = 0; i < stages; ++i) tc::mbar_init(&full[i], 1);
  if (threadIdx.x == 0) *abort = 0;
  tc::fence_mbar_init();
  wait_previous();
  if (blockIdx.x == 0 && threadIdx.x == 0) *A.err = 0;
  for (int j = threadIdx.x; j < d; j += blockDim.x) scale_s[j] = A.scale[j];
  __syncthreads();

  const int64_t first = (int64_t)blockIdx.x * warps + warp, step = (int64_t)gridDim.x * warps;
  auto fetch = [&](int64_t row, int st) {   // lane 0
    tc::mbar_expect_tx(&full[st], (uint32_t)(tensors * rb));
    uint8_t* at = ring + (size_t)st * tensors * rbp;
    auto copy = [&](uint8_t* dst, const void* src) {
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                       tc::smem_u32(dst)),
                   "l"(src), "r"(rb), "r"(tc::smem_u32(&full[st]))
                   : "memory");
    };
    copy(at, reinterpret_cast<const E*>(A.x) + row * A.ldx);
    copy(at + rbp, reinterpret_cast<const E*>(A.dy) + row * A.lddy);
  };
  F2 ag[NV][H], ab[NV][H];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < H; ++k) ag[i][k] = ab[i][k] = f2(0.f);
  if (lane == 0)
    for (int i = 0; i < stages; ++i)
      if (first + i * step < A.rows) fetch(first + i * step, i);
  int st = 0;
  uint32_t ph = 0;
  for (int64_t row = first; row < A.rows; row += step) {
    Vec e[NV];                               // used last: loaded straight into registers meanwhile
    if (A.dr) {
      const Vec* es = reinterpret_cast<const Vec*>(reinterpret_cast<const E*>(A.dr) + row * A.lddr);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if ((i * 32 + lane) * V < d) e[i] = es[i * 32 + lane];
    }
    if (!__all_sync(FULL, tc::mbar_wait(&full[st], ph, abort, A.err, 11))) {
      const long long t0 = clock64();        // time for the copies in flight to land
      while (clock64() - t0 < 2000000) {}    // about a millisecond
      break;
    }
    const uint8_t* at = ring + (size_t)st * tensors * rbp;
    const Vec* xs = reinterpret_cast<const Vec*>(at);
    const Vec* gs = reinterpret_cast<const Vec*>(at + rbp);
    F2 acc = f2(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * 32 + lane) * V < d) {
        F2 a[H];
        unpack2(xs[i * 32 + lane], a);
#pragma unroll
        for (int k = 0; k < H; ++k) acc = acc + a[k];
      }
    const F2 mean = f2(-(warp_sum(sum(acc)) * A.inv_d));
    F2 s1 = f2(0.f), s2 = f2(0.f), sg = f2(0.f), sgc = f2(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * 32 + lane) * V < d) {
        F2 a[H], g[H];
        unpack2(xs[i * 32 + lane], a);
        unpack2(gs[i * 32 + lane], g);
        const F2* sc = reinterpret_cast<const F2*>(scale_s + (i * 32 + lane) * V);
#pragma unroll
        for (int k = 0; k < H; ++k) {
          const F2 c = a[k] + mean, gy = g[k] * sc[k];
          s1 = s1 + c;
          s2 = fma2(c, c, s2);
          sg = sg + gy;
          sgc = fma2(gy, c, sgc);
        }
      }
    const float off = warp_sum(sum(s1)) * A.inv_d, gsum = warp_sum(sum(sg));
    const float rstd_f = rsqrtf(variance(warp_sum(sum(s2)) * A.inv_d, off) + A.eps);
    const F2 rstd = f2(rstd_f), c1 = f2(-(gsum * A.inv_d)),
             c2 = f2(-(fmaf(-off, gsum, warp_sum(sum(sgc))) * rstd_f * A.inv_d)), noff = f2(-off);
    Vec* out = reinterpret_cast<Vec*>(reinterpret_cast<E*>(A.dx) + row * (int64_t)d);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * 32 + lane) * V < d) {
        F2 a[H], g[H];
        float x[V];
        unpack2(xs[i * 32 + lane], a);
        unpack2(gs[i * 32 + lane], g);
        const F2* sc = reinterpret_cast<const F2*>(scale_s + (i * 32 + lane) * V);
#pragma unroll
        for (int k = 0; k < H; ++k) {
          const F2 xh = (a[k] + mean + noff) * rstd;
          ag[i][k] = fma2(g[k], xh, ag[i][k]);
          ab[i][k] = ab[i][k] + g[k];
          a[k] = rstd * fma2(xh, c2, g[k] * sc[k] + c1);
        }
        if (A.dr) {
          unpack2(e[i], g);
#pragma unroll
          for (int k = 0; k < H; ++k) a[k] = a[k] + g[k];
        }
#pragma unroll
        for (int k = 0; k < H; ++k) split(a[k], x[2 * k], x[2 * k + 1]);
        Vec o;
        pack(o, x);
        out[i * 32 + lane] = o;
      }
    __syncwarp();                            // every lane has read the stage
    if (lane == 0 && row + stages * step < A.rows) fetch(row + stages * step, st);
    if (++st == stages) {
      st = 0;
      ph ^= 1;
    }
  }
  // the warps' sums, in warp order, through the rings' memory
  __syncthreads();
  float* all = reinterpret_cast<float*>(rings);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (i * 32 + lane) * V;
    if (j >= d) continue;
#pragma unroll
    for (int k = 0; k < H; ++k) {
      *reinterpret_cast<F2*>(all + (size_t)warp * 2 * d + j + 2 * k) = ag[i][k];
      *reinterpret_cast<F2*>(all + (size_t)warp * 2 * d + d + j + 2 * k) = ab[i][k];
    }
  }
  __syncthreads();
  float* part = A.part + (int64_t)blockIdx.x * 2 * d;
  for (int j = threadIdx.x; j < 2 * d; j += blockDim.x) {
    float x = 0.f;
    for (int w = 0; w < warps; ++w) x += all[(size_t)w * 2 * d + j];
    part[j] = x;
  }
}

// dscale | dbias = the blocks' partial rows: 32 groups of blocks a column, each
// added in block order, then the groups in a fixed tree.
__global__ void __launch_bounds__(1024) layer_norm_params_kernel(const float* __restrict__ part, int blocks, int d,
                                                                 float* __restrict__ dscale,
                                                                 float* __restrict__ dbias, int* err) {
  wait_previous();
  if (blocks == 0 && blockIdx.x == 0 && threadIdx.x == 0) *err = 0;
  __shared__ float red[32][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + c;
  float x = 0.f;
  if (j < 2 * d) {
    const float* p = part + j;
    int b = g;
    for (; b + 7 * 32 < blocks; b += 8 * 32) {      // eight loads in flight
      float a[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = p[(int64_t)(b + 32 * i) * 2 * d];
#pragma unroll
      for (int i = 0; i < 8; ++i) x += a[i];
    }
    float a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = b + 32 * i < blocks ? p[(int64_t)(b + 32 * i) * 2 * d] : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x += a[i];
  }
  red[g][c] = x;
  __syncthreads();
  // warp g: column g of this block's 32
  const float t = warp_sum(red[c][g]);
  const int k = blockIdx.x * 32 + g;
  if (c == 0 && k < 2 * d) (k < d ? dscale[k] : dbias[k - d]) = t;
}

// Threads of a row: the power of two that holds its width at 16 values each.
int norm_tpr(int d) {
  int t = 4;
  while (t * VALS < d) t *= 2;
  return t;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The block-per-row layouts: threads a row, vectors a thread, rows at a time.
struct Wide {
  int nt, nv;
  // Blocks of an SM where `most` of 256 threads fit, more of smaller ones.
  int per_sm(int most) const { return nt <= 256 ? most * 256 / nt : 1; }
};

bool wide_rows(int d, int v) { return d > 32 * VALS && d % v == 0; }

// Up to 4096 columns in blocks of at most 256 threads, several on an SM
// (gradient of 4096 x 4096 float32 56 us, in one block of 1024 105); beyond in
// one of up to 1024.
Wide wide_for(int d, int v) {
  const int vecs = (d + v - 1) / v;
  int nv = 1;
  if (vecs * v <= 4096)
    while (vecs > 256 * nv) nv *= 2;
  else
    nv = vecs <= 1024 ? 1 : vecs <= 2048 ? 2 : 4;
  return {((vecs + nv - 1) / nv + 31) / 32 * 32, nv};
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a call's rows are read: by entries, by 16-byte vectors, or by vectors
// that rows packed one after another start inside of (SHIFT).
enum Access { ENTRIES, VECTORS, SHIFTED };

bool shifted_rows(int d, int v) { return wide_rows(d, 1) && wide_for(d + v - 1, v).nt <= 1024; }

// Blocks for shifted rows: at most `most`, and then a multiple of the rows
// after which starts repeat.
int shifted_grid(int64_t rows, int d, int v, int64_t most) {
  if (rows <= most) return (int)rows;
  const int period = v / std::gcd(d, v);
  return (int)(most / period * period);
}

// The ring layout of the gradient: rows of up to 256 vectors (16-bit) or 512
// (float32), 64 columns a lane; as many warps as the rings leave room for.
struct Ring {
  int warps, stages;
  size_t smem;
};

bool ring_rows(int d, int v) { return wide_rows(d, v) && d <= 2048; }

Ring ring_for(int d, int esize) {
  const size_t rbp = ((size_t)d * esize + 127) / 128 * 128, head = 128 + 512 + ((size_t)d * 4 + 127) / 128 * 128;
  const size_t room = 227 * 1024 - head, row = rbp * 2;
  const size_t most = d > 1024 ? 8 : 12;                     // 128 sums a lane leave registers for 8 warps
  Ring r{};
  r.stages = 3 * row * most <= room ? 3 : 2;
  const size_t w = room / (row * r.stages);
  r.warps = (int)(w < most ? w : most);
  r.smem = head + row * r.stages * r.warps;
  return r;
}

template <typename E>
cudaError_t norm_forward_t(NormArgs& A, Access how, cudaStream_t s) {
  constexpr int V = 16 / sizeof(E);
  constexpr int64_t MOST = 1 << 20;
  const int vecs = A.d / V;
  const bool vec = how == VECTORS;
  if (how == SHIFTED) {
    // 16-bit rows of up to 4096 columns: a vector a thread in blocks of up to
    // 512 (9557 x 2498 68 us, two vectors in blocks of 160 82)
    Wide w = wide_for(A.d + V - 1, V);
    if (V == 8 && w.nv == 2 && w.nt <= 256) w = {(int)ceil_div(A.d + V - 1, V * 32) * 32, 1};
    const int most = w.nt > 256 ? 1024 / w.nt : w.per_sm(w.nv * V > 8 ? 3 : 4);
    const int grid = shifted_grid(A.rows, A.d, V, (int64_t)most * g16::device_sms());
    count_launch();
    if (w.nt > 256) {
      if constexpr (V == 8)
        if (w.nv == 1)
          return launch_dependent(layer_norm_wide_kernel<E, 1, 1024, 1, true>, dim3(grid), w.nt, 0, s, A);
      if (w.nv == 2) return launch_dependent(layer_norm_wide_kernel<E, 2, 1024, 1, true>, dim3(grid), w.nt, 0, s, A);
      if (w.nv == 4) return launch_dependent(layer_norm_wide_kernel<E, 4, 1024, 1, true>, dim3(grid), w.nt, 0, s, A);
    } else {
      if (w.nv == 1) return launch_dependent(layer_norm_wide_kernel<E, 1, 256, 4, true>, dim3(grid), w.nt, 0, s, A);
      if constexpr (V == 4) {
        if (w.nv == 2) return launch_dependent(layer_norm_wide_kernel<E, 2, 256, 4, true>, dim3(grid), w.nt, 0, s, A);
        if (w.nv == 4) return launch_dependent(layer_norm_wide_kernel<E, 4, 256, 3, true>, dim3(grid), w.nt, 0, s, A);
      }
    }
    return cudaErrorInvalidConfiguration;                 // no such width
  }
  const bool warp = A.d > 32 * VALS && (vec ? vecs <= 512 : A.d <= 2048);
  if (warp) {
    const int64_t grid = ceil_div(A.rows, 4);
    if (grid >= (1ll << 31)) return cudaErrorInvalidValue;
    const unsigned g = (unsigned)grid;
    if (!vec)
      A.d <= 1024 ? launch_dependent(layer_norm_warp_kernel<E, 1, 32>, dim3(g), 128, 0, s, A)
                  : launch_dependent(layer_norm_warp_kernel<E, 1, 64>, dim3(g), 128, 0, s, A);
    else if (vecs <= 128)
      launch_dependent(layer_norm_warp_kernel<E, V, 4>, dim3(g), 128, 0, s, A);
    else if (vecs <= 256)
      launch_dependent(layer_norm_warp_kernel<E, V, 8>, dim3(g), 128, 0, s, A);
    else
      launch_dependent(layer_norm_warp_kernel<E, V, 16>, dim3(g), 128, 0, s, A);
  } else if (vec && vecs > 512) {
    const Wide w = wide_for(A.d, V);
    const int grid = (int)(A.rows < MOST ? A.rows : MOST);
    count_launch();
    if constexpr (V == 8)                // float32 rows begin at two vectors, 16-bit ones end there
      if (w.nv == 1) return launch_dependent(layer_norm_wide_kernel<E, 1, 1024, 1, false>, dim3(grid), w.nt, 0, s, A);
    if (w.nv == 2) return launch_dependent(layer_norm_wide_kernel<E, 2, 1024, 1, false>, dim3(grid), w.nt, 0, s, A);
    if constexpr (V == 4)
      if (w.nv == 4) return launch_dependent(layer_norm_wide_kernel<E, 4, 1024, 1, false>, dim3(grid), w.nt, 0, s, A);
    return cudaErrorInvalidConfiguration;                 // no such width
  } else {
    const bool wide = A.tpr > 32;
    const int nt = wide ? A.tpr : NT;
    const int64_t need = ceil_div(A.rows, nt / A.tpr);
    const int grid = (int)(need < MOST ? need : MOST);
    if (vec)
      launch_dependent(layer_norm_kernel<E, V, 0>, dim3(grid), nt, 0, s, A);
    else if (wide)
      launch_dependent(layer_norm_kernel<E, 1, 1024>, dim3(grid), nt, 0, s, A);
    else
      launch_dependent(layer_norm_kernel<E, 1, 0>, dim3(grid), nt, 0, s, A);
  }
  count_launch();
  return cudaGetLastError();
}

template <typename E, int NV, int MAXW>
cudaError_t launch_ring(const NormArgs& A, const Ring& r, int grid, cudaStream_t s) {
  auto kern = layer_norm_ring_backward_kernel<E, NV, MAXW>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = g16::allow_smem(reinterpret_cast<const void*>(kern), &done);
  if (e != cudaSuccess) return e;
  launch_dependent(kern, dim3(grid), r.warps * 32, r.smem, s, A, r.stages);
  return cudaSuccess;
}

// Blocks of 256 threads an SM holds with the gradient's registers: by columns a thread.
int backward_resident(int cols) { return cols <= 4 ? 4 : cols <= 8 ? 3 : 2; }

// Aligned rows come here from 2049 columns on and shifted ones from 513 on,
// so a type has some of the shapes only.
template <typename E, bool SHIFT>
cudaError_t launch_wide_backward(const NormArgs& A, const Wide& w, int grid, cudaStream_t s) {
  constexpr int V = 16 / sizeof(E);
  constexpr bool F = V == 4;           // float32
  if (w.nt > 256) {
    if constexpr (!F)
      if (w.nv == 1)
        return launch_dependent(layer_norm_wide_backward_kernel<E, 1, 1024, 1, false, SHIFT>, dim3(grid), w.nt, 0, s, A);
    if (w.nv == 2)
      return launch_dependent(layer_norm_wide_backward_kernel<E, 2, 1024, 1, false, SHIFT>, dim3(grid), w.nt, 0, s, A);
    if constexpr (F || SHIFT)
      if (w.nv == 4)
        return launch_dependent(layer_norm_wide_backward_kernel<E, 4, 1024, 1, false, SHIFT>, dim3(grid), w.nt, 0, s, A);
  } else {
    constexpr bool AHEAD = F || !SHIFT;
    if constexpr (SHIFT)
      if (w.nv == 1)
        return launch_dependent(layer_norm_wide_backward_kernel<E, 1, 256, F ? 4 : 3, AHEAD, SHIFT>, dim3(grid), w.nt, 0,
                                s, A);
    if constexpr (!F || SHIFT)
      if (w.nv == 2)
        return launch_dependent(layer_norm_wide_backward_kernel<E, 2, 256, F ? 3 : 2, AHEAD, SHIFT>, dim3(grid), w.nt, 0,
                                s, A);
    if constexpr (F)
      if (w.nv == 4)
        return launch_dependent(layer_norm_wide_backward_kernel<E, 4, 256, 2, false, SHIFT>, dim3(grid), w.nt, 0, s, A);
  }
  return cudaErrorInvalidConfiguration;                   // no such width
}

template <typename E>
cudaError_t norm_backward_t(NormArgs& A, Access how, int grid, cudaStream_t s) {
  constexpr int V = 16 / sizeof(E);
  const bool vec = how == VECTORS;
  if (how == SHIFTED) {
    count_launch();
    return launch_wide_backward<E, true>(A, wide_for(A.d + V - 1, V), grid, s);
  }
  if (vec && ring_rows(A.d, V)) {
    const Ring r = ring_for(A.d, sizeof(E));
    cudaError_t e;
    if (A.d <= 1024)
      e = launch_ring<E, 32 / V, 12>(A, r, grid, s);
    else
      e = launch_ring<E, 64 / V, 8>(A, r, grid, s);
    if (e != cudaSuccess) return e;
  } else if (vec && wide_rows(A.d, V)) {
    count_launch();
    return launch_wide_backward<E, false>(A, wide_for(A.d, V), grid, s);
  } else {
    const bool wide = A.tpr > 32;
    const int nt = wide ? A.tpr : NT;
    const size_t sm = wide ? 0 : (size_t)nt * VALS * sizeof(float);   // 16 KB
    if (vec)
      launch_dependent(layer_norm_backward_kernel<E, V, 0>, dim3(grid), nt, sm, s, A);
    else if (A.tpr > 256)
      launch_dependent(layer_norm_backward_kernel<E, 1, 1024>, dim3(grid), nt, sm, s, A);
    else if (wide)
      launch_dependent(layer_norm_backward_kernel<E, 1, 256>, dim3(grid), nt, sm, s, A);
    else
      launch_dependent(layer_norm_backward_kernel<E, 1, 0>, dim3(grid), nt, sm, s, A);
  }
  count_launch();
  return cudaGetLastError();
}

// Blocks of the gradient's row pass: as many as are resident at once.
int backward_blocks(int64_t rows, int d, int v, Access how) {
  int64_t need, per_sm;
  const bool vec = how == VECTORS;
  if (how == SHIFTED) {
    const Wide w = wide_for(d + v - 1, v);
    return shifted_grid(rows, d, v, (int64_t)w.per_sm(backward_resident(w.nv * v)) * g16::device_sms());
  }
  if (vec && ring_rows(d, v)) {
    need = ceil_div(rows, ring_for(d, 16 / v).warps);
    per_sm = 1;
  } else if (vec && wide_rows(d, v)) {
    const Wide w = wide_for(d, v);
    need = rows;
    per_sm = w.per_sm(backward_resident(w.nv * v));
  } else {
    const int tpr = norm_tpr(d), nt = tpr > 32 ? tpr : NT;
    need = ceil_div(rows, nt / tpr);
    per_sm = nt <= 256 ? 512 / nt : 1;
  }
  const int64_t cap = per_sm * g16::device_sms();
  return (int)(need < cap ? need : cap);
}

}  // namespace

// The most that any alignment of the call's tensors takes.
int norm_backward_blocks(int64_t rows, int d, int dtype) {
  const int v = dtype == MEMLAYER_F32 ? 4 : 8;
  int most = 0;
  for (Access how : {ENTRIES, VECTORS, SHIFTED}) most = std::max(most, backward_blocks(rows, d, v, how));
  return most;
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
  const bool base = al16(a.x) && al16(a.residual) && al16(a.y) && al16(a.sum);
  Access how = ENTRIES;
  if (base && al16(a.scale) && al16(a.bias) && c.d_model % v == 0 && a.x_stride % v == 0 &&
      (!a.residual || a.residual_stride % v == 0))
    how = VECTORS;
  else if (base && shifted_rows(c.d_model, v) && a.x_stride == c.d_model &&
           (!a.residual || a.residual_stride == c.d_model))
    how = SHIFTED;
  switch (c.dtype) {
    case MEMLAYER_F16: return norm_forward_t<__half>(A, how, s);
    case MEMLAYER_BF16: return norm_forward_t<__nv_bfloat16>(A, how, s);
    default: return norm_forward_t<float>(A, how, s);
  }
}

cudaError_t launch_layer_norm_backward(const memlayer_norm_config& c, const memlayer_norm_grads& g, float* part,
                                       int* err, cudaStream_t s) {
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
  A.err = err;
  const int v = c.dtype == MEMLAYER_F32 ? 4 : 8;
  const bool base = al16(g.x) && al16(g.dy) && al16(g.dresidual) && al16(g.dx);
  Access how = ENTRIES;
  if (base && al16(g.scale) && c.d_model % v == 0 && g.x_stride % v == 0 && g.dy_stride % v == 0 &&
      (!g.dresidual || g.dresidual_stride % v == 0))
    how = VECTORS;
  else if (base && shifted_rows(c.d_model, v) && g.x_stride == c.d_model && g.dy_stride == c.d_model &&
           (!g.dresidual || g.dresidual_stride == c.d_model))
    how = SHIFTED;
  const int grid = backward_blocks(c.rows, c.d_model, v, how);
  cudaError_t e = cudaSuccess;
  if (grid > 0) switch (c.dtype) {
      case MEMLAYER_F16: e = norm_backward_t<__half>(A, how, grid, s); break;
      case MEMLAYER_BF16: e = norm_backward_t<__nv_bfloat16>(A, how, grid, s); break;
      default: e = norm_backward_t<float>(A, how, grid, s); break;
    }
  if (e != cudaSuccess) return e;
  count_launch();
  return launch_dependent(layer_norm_params_kernel, dim3((2 * c.d_model + 31) / 32), 1024, 0, s, part, grid, c.d_model,
                          g.dscale, g.dbias, err);
}

}  // namespace ml
