// The orthogonalised update (orth.cu) of matrices with a side of at most 128
// and another of at most 2048, in one launch: all of a matrix's steps inside
// a cluster of up to eight CTAs.  With S the smaller and L the larger side, X
// as an S x L matrix:
//
//   P = X X^T,   Q = a I + b P + c P P,   X <- Q X       `steps` times
//
// A CTA keeps up to 256 columns of X in shared memory as two f16 pieces
// (22 bits, scaled by 2^12 like the products of orth.cu).  It multiplies its
// columns' part of P on the tensor cores, the cluster adds the parts through
// distributed shared memory (each CTA some rows, in rank order), and every
// CTA then forms Q for itself and multiplies its own columns: X crosses HBM
// once each way, and a product costs its MMAs, the drain of its accumulators
// and a block barrier instead of a launch and the load of its operands.  Five
// steps of float32, launches of orth.cu against this: 12 x 64 x 64 91 -> 29 us,
// 128 x 128 103 -> 39, 4 x 128 x 256 116 -> 52, 64 x 1000 103 -> 60,
// 128 x 2048 121 -> 78 (of which the cluster's sums are 25), 1000 x 64 x 64
// 324 -> 183.  Latency bounds it: a step's products wait for each other.
//
// Shared memory holds the rows of X and of P in blocks of 64 columns, 128
// bytes a row with the 128-byte swizzle.  X is read both ways from the same
// bytes: K-major (k along the row) for P, MN-major (k down the rows) for Q X.
// Each 64 of k go to accumulators of their own in TMEM and are added in
// registers, rounding to nearest (the tensor cores add by truncation).
// Rows and columns past the matrix are zeros and stay zeros.  512 threads:
// between the products a step waits for what threads do, conversions and
// shared memory, and 256 took 1.2 times as long.
//
// A CTA takes most of an SM's shared memory, so no two of them meet on an SM
// and wait for each other's TMEM.  Waits are bounded; after one gave up the
// CTA goes on (its cluster's barriers need it) and the status word tells.
#include "gemm16.cuh"
#include "orth.cuh"
#include "pieces16.cuh"

namespace ml {

namespace {

constexpr int NT = 512;                        // four warps a TMEM lane quarter, 32 columns each at a time
constexpr int SIDE = 128, CHUNK = 256, MOST = 8;
constexpr uint32_t BLOCK = SIDE * 128;         // 64 columns
constexpr uint32_t X_PIECE = CHUNK / 64 * BLOCK, P_PIECE = 2 * BLOCK;
constexpr uint32_t SMEM = 1024 + 1024 + 2 * X_PIECE + 2 * P_PIECE;

struct ChainCtl {
  uint64_t done[2];
  double warp_sum[NT / 32];
  uint32_t tmem_base;
  int abort;
};

struct ChainArgs {
  const void* u;
  void* out;
  int m, n, S, L, tall;                        // tall: X is the transpose of the m x n matrix
  int C, lc, steps;                            // CTAs a matrix, columns of each (a multiple of 64)
  float a, b, c;
  double eps;
  int vec_in, vec_out;                         // eight columns in one access
  int* err;
};

template <typename E> __device__ __forceinline__ float up(E x);
template <> __device__ __forceinline__ float up(float x) { return x; }
template <> __device__ __forceinline__ float up(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename E> __device__ __forceinline__ E down(float x);
template <> __device__ __forceinline__ float down(float x) { return x; }
template <> __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }

// Descriptor of MN-major columns: blocks of 64 (leading byte offset) of
// 1024-byte atoms of 8 k (stride byte offset).
__device__ __forceinline__ uint64_t desc_columns(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(BLOCK >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ float4 ld_cluster(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at)
               : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster(uint32_t at, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}
__device__ __forceinline__ float4 ld_shared(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at)
               : "memory");
  return v;
}
__device__ __forceinline__ float ld_shared_f32(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float ld_half(uint32_t at) {
  unsigned short h;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(at) : "memory");
  return __half2float(__ushort_as_half(h));
}
__device__ __forceinline__ double ld_cluster_f64(uint32_t at) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at) : "memory");
  return v;
}

// The pieces' 16-byte chunk `c` of a row in a 64-column block.
__device__ __forceinline__ uint32_t chunk8(uint32_t block, int row, int c) {
  return block + row * 128 + ((c ^ (row & 7)) << 4);
}

// Eight values of a row as pieces.
__device__ __forceinline__ void put8(uint32_t at, uint32_t piece, const float (&x)[8]) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    __half2 a, b;
    g16::split2(x[2 * j], x[2 * j + 1], a, b);
    h[j] = *reinterpret_cast<const uint32_t*>(&a);
    l[j] = *reinterpret_cast<const uint32_t*>(&b);
  }
  g16::st_shared(at, h[0], h[1], h[2], h[3]);
  g16::st_shared(at + piece, l[0], l[1], l[2], l[3]);
}

// They again.
__device__ __forceinline__ void get8(uint32_t at, uint32_t piece, float (&x)[8]) {
  const float4 h = ld_shared(at), l = ld_shared(at + piece);
  const float a[4] = {h.x, h.y, h.z, h.w}, b[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&a[j]));
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&b[j]));
    x[2 * j] = u.x + v.x;
    x[2 * j + 1] = u.y + v.y;
  }
}

// Eight float32 values in the place of X's pieces, and back.
__device__ __forceinline__ void wait8(uint32_t at, const float (&x)[8]) {
  g16::st_shared(at, __float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  g16::st_shared(at + X_PIECE, __float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]),
                 __float_as_uint(x[7]));
}
__device__ __forceinline__ void waited8(uint32_t at, float (&x)[8]) {
  const float4 v = ld_shared(at), w = ld_shared(at + X_PIECE);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
}

// Eight neighbouring values of global memory, in one access.
template <typename E>
struct alignas(8 * sizeof(E)) Eight { E e[8]; };
template <typename E>
__device__ __forceinline__ Eight<E> read8(const E* p) {
  return *reinterpret_cast<const Eight<E>*>(p);
}
template <>
__device__ __forceinline__ Eight<float> read8(const float* p) {
  Eight<float> v;
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v.e[0]), "=f"(v.e[1]), "=f"(v.e[2]), "=f"(v.e[3]), "=f"(v.e[4]), "=f"(v.e[5]), "=f"(v.e[6]),
                 "=f"(v.e[7])
               : "l"(p));
  return v;
}
template <typename E>
__device__ __forceinline__ void write8(E* p, const Eight<E>& v) {
  *reinterpret_cast<Eight<E>*>(p) = v;
}
template <>
__device__ __forceinline__ void write8(float* p, const Eight<float>& v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v.e[0]), "f"(v.e[1]),
               "f"(v.e[2]), "f"(v.e[3]), "f"(v.e[4]), "f"(v.e[5]), "f"(v.e[6]), "f"(v.e[7])
               : "memory");
}

// The two-piece product of 64 k, small terms first; a whole warp calls, lane
// `one` issues (the operands stay in uniform registers).
__device__ __forceinline__ void mma_block(bool one, uint32_t d, uint64_t a, uint32_t a_piece, uint32_t astep,
                                          uint64_t b, uint32_t b_piece, uint32_t bstep, uint32_t idesc) {
  const uint64_t al = a + (a_piece >> 4), bl = b + (b_piece >> 4);
  if (!one) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) g16::mma_f16<1>(d, al + k * astep, b + k * bstep, idesc, k > 0);
#pragma unroll
  for (int k = 0; k < 4; ++k) g16::mma_f16<1>(d, a + k * astep, bl + k * bstep, idesc, 1);
#pragma unroll
  for (int k = 0; k < 4; ++k) g16::mma_f16<1>(d, a + k * astep, b + k * bstep, idesc, 1);
}

// 32 columns of an accumulator, and those of the accumulators [from, n),
// `apart` columns from each other, added to them.
__device__ __forceinline__ void take32(uint32_t taddr, float (&s)[32]) {
  uint32_t v[32];
  __syncwarp();
  tc::tmem_ld32(taddr, v);
  tc::tmem_wait_ld();
#pragma unroll
  for (int j = 0; j < 32; ++j) s[j] = __uint_as_float(v[j]);
}
__device__ __forceinline__ void add32(uint32_t taddr, int from, int n, uint32_t apart, float (&s)[32]) {
  for (int i = from; i < n; ++i) {
    float v[32];
    take32(taddr + i * apart, v);
#pragma unroll
    for (int j = 0; j < 32; ++j) s[j] += v[j];
  }
}

template <typename E>
__global__ void __launch_bounds__(NT, 1) orth_chain_kernel(const __grid_constant__ ChainArgs A) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  ChainCtl* ctl = reinterpret_cast<ChainCtl*>(smem);
  const uint32_t X = tc::smem_u32(smem) + 1024, P = X + 2 * X_PIECE;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, part = warp >> 2;
  const int row = (warp & 3) * 32 + lane;
  const int rank = (int)g16::cluster_rank();
  const int S = A.S, L = A.L, lc = A.lc, c0 = rank * lc, nblk = lc >> 6;
  volatile int* abort = &ctl->abort;
  if (t == 0) {
    tc::mbar_init(&ctl->done[0], 1);
    tc::mbar_init(&ctl->done[1], 1);
    ctl->abort = 0;
    tc::fence_mbar_init();
  }
  if (warp == 1) g16::tmem_alloc<1>(&ctl->tmem_base, 512);
  allow_next();
  wait_previous();
  if (blockIdx.x == 0 && t == 0) *A.err = 0;

  // ---- X_0 = U / (|U|_F + eps): eight columns of a row at a time --------------------
  const int64_t base = (int64_t)(blockIdx.x / A.C) * A.m * A.n;
  const int c8 = lc >> 3, bits = c8 > 16 ? 5 : c8 > 8 ? 4 : 3, items = A.tall ? SIDE * c8 : SIDE << bits;
  const int64_t step = A.tall ? A.n : 1;       // from a column of X to the next
  auto item = [&](int e, int& r, int& c) {     // neighbouring threads: neighbouring addresses
    r = A.tall ? e & (SIDE - 1) : e >> bits;
    c = A.tall ? e / SIDE : e & ((1 << bits) - 1);
    return e < items && c < c8;
  };
  // Eight columns of a row in global memory: at(r, c) on, step apart.
  auto at8 = [&](int r, int c) {
    const int64_t col = c0 + c * 8;
    return base + (A.tall ? col * A.n + r : r * (int64_t)A.n + col);
  };
  // The values wait as float32 where their pieces will be, four chunks in
  // flight.  Squares of float32 values leave its range: their sum is float64.
  constexpr int AHEAD = 4;
  double s0 = 0., s1 = 0.;
  auto take = [&](int e0, const float (&x)[AHEAD][8]) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      int r, c;
      if (!item(e0 + i * NT, r, c)) continue;
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        s0 = fma((double)x[i][j], (double)x[i][j], s0);
        s1 = fma((double)x[i][j + 1], (double)x[i][j + 1], s1);
      }
      wait8(chunk8(X + (c >> 3) * BLOCK, r, c & 7), x[i]);
    }
  };
  const E* u = reinterpret_cast<const E*>(A.u);
  if (A.vec_in) {
    for (int e0 = t; e0 < items; e0 += AHEAD * NT) {
      Eight<E> v[AHEAD];
      bool in[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        int r, c;
        in[i] = item(e0 + i * NT, r, c) && r < S && c0 + c * 8 < L;
        v[i] = read8(in[i] ? u + at8(r, c) : u);
      }
      float x[AHEAD][8];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = in[i] ? up(v[i].e[j]) : 0.f;
      take(e0, x);
    }
  } else {
    for (int e0 = t; e0 < items; e0 += AHEAD * NT) {
      E v[AHEAD][8];
      int left[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        int r, c;
        left[i] = item(e0 + i * NT, r, c) && r < S ? L - (c0 + c * 8) : 0;
        const E* p = u + at8(r, c);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = *(j < left[i] ? p + j * step : u);
      }
      float x[AHEAD][8];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = j < left[i] ? up(v[i][j]) : 0.f;
      take(e0, x);
    }
  }
  s0 += s1;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s0 += __shfl_xor_sync(FULL, s0, o);
  if (lane == 0) ctl->warp_sum[warp] = s0;
  __syncwarp();
  g16::cluster_sync();
  s0 = 0.;
  for (int i = lane; i < A.C * (NT / 32); i += 32)
    s0 += ld_cluster_f64(g16::map_to_cta(tc::smem_u32(&ctl->warp_sum[i % (NT / 32)]), i / (NT / 32)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s0 += __shfl_xor_sync(FULL, s0, o);
  // the factor as a power of two, which is exact, and a float32
  const double inv = (double)kOrthScale / (sqrt(s0) + A.eps);
  int e2 = 0;
  if (inv > 0. && inv < INFINITY) e2 = min(126, max(-126, (__double2hiint(inv) >> 20) - 1023));
  const float f1 = g16::pow2(e2), f2 = (float)(inv * (double)g16::pow2(-e2));
  for (int e0 = t; e0 < items; e0 += AHEAD * NT) {
    float x[AHEAD][8];
    uint32_t at[AHEAD];
    bool in[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      int r, c;
      in[i] = item(e0 + i * NT, r, c);
      at[i] = chunk8(X + (c >> 3) * BLOCK, r, c & 7);
      if (in[i]) waited8(at[i], x[i]);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (!in[i]) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = x[i][j] * f1 * f2;
      put8(at[i], X_PIECE, x[i]);
    }
  }

  const int nb0 = (nblk + 1) >> 1;             // blocks of the first signal
  const uint32_t id_p = g16::idesc_16(SIDE, SIDE, 0, 0, 0);
  const int nk = S > 64 ? 2 : 1;               // 64-k blocks of P and Q
  const bool one = g16::elect_one();
  uint32_t ph[2] = {0, 0};
  // Hands the operands just written to the tensor cores and has warp 0 issue.
  auto signal = [&](int i) {
    if (one) g16::commit<1>(&ctl->done[i]);
  };
  auto wait = [&](int i) {
    tc::mbar_wait(&ctl->done[i], ph[i], abort, A.err, 14);
    __syncwarp();
    tc::fence_after_sync();
  };
  auto multiply = [&](auto issue) {
    tc::fence_proxy_async_smem();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 0) {
      tc::fence_after_sync();
      issue(ctl->tmem_base);
      __syncwarp();
    }
  };
  constexpr float un = 1.f / kOrthScale;
  uint32_t lanes = 0;                          // this warp's TMEM lanes
  for (int k = 0; k < A.steps; ++k) {
    // opaque: the addresses below, kept over the steps, would spill
    int rw = row;
    uint32_t xs = X, ps = P;
    asm volatile("" : "+r"(rw), "+r"(xs), "+r"(ps));
    multiply([&](uint32_t tm) {
      for (int i = 0; i < nblk; ++i) {
        if (i == nb0) signal(1);
        const uint64_t d = tc::sdesc_k_sw128(X + i * BLOCK);
        mma_block(one, tm + i * SIDE, d, X_PIECE, 32 >> 4, d, X_PIECE, 32 >> 4, id_p);
      }
      if (nb0 == nblk) signal(1);
      signal(0);
    });
    lanes = ctl->tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    float p[32];
    wait(1);
    ph[1] ^= 1;
    take32(lanes + part * 32, p);
    add32(lanes + part * 32, 1, nb0, SIDE, p);
    wait(0);
    ph[0] ^= 1;
    add32(lanes + part * 32, nb0, nblk, SIDE, p);
    if (A.C > 1) {
      // rows of 512 bytes whose 16-byte chunks change places by row; P is
      // symmetric: chunks up to the diagonal (a CTA's share of the network is 14 bytes a cycle)
      auto chunk = [&](int r, int c) { return ps + r * 512 + ((c ^ (r & 31)) << 4); };
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (part * 8 + j <= rw >> 2)
          g16::st_shared(chunk(rw, part * 8 + j), __float_as_uint(p[4 * j]), __float_as_uint(p[4 * j + 1]),
                         __float_as_uint(p[4 * j + 2]), __float_as_uint(p[4 * j + 3]));
      g16::cluster_sync();
      // this CTA's chunks, in rank order (four rows of i + 1 chunks after four
      // of i); no other thread reads them, so the sums take their places in
      // every CTA at once
      const int G = (S + 3) >> 2, total = 2 * G * (G + 1);
      for (int e = total * rank / A.C + t; e < total * (rank + 1) / A.C; e += NT) {
        int g = (int)((sqrtf(2.f * e + 1.f) - 1.f) * 0.5f);
        while (2 * (g + 1) * (g + 2) <= e) ++g;
        while (2 * g * (g + 1) > e) --g;
        const int rem = e - 2 * g * (g + 1), r = rem / (g + 1);
        const uint32_t at = chunk(4 * g + r, rem - r * (g + 1));
        float4 s = ld_cluster(g16::map_to_cta(at, 0));
        for (int q0 = 1; q0 < A.C; q0 += 4) {  // the others, four in flight
          float4 v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q0 + q < A.C) v[q] = ld_cluster(g16::map_to_cta(at, q0 + q));
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q0 + q < A.C) s = make_float4(s.x + v[q].x, s.y + v[q].y, s.z + v[q].z, s.w + v[q].w);
        }
        for (int q = 0; q < A.C; ++q) st_cluster(g16::map_to_cta(at, q), s);
      }
      g16::cluster_sync();
      if (part < (warp & 3)) {                 // the warp's columns are before its rows
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 v = ld_shared(chunk(rw, part * 8 + j));
          p[4 * j] = v.x;
          p[4 * j + 1] = v.y;
          p[4 * j + 2] = v.z;
          p[4 * j + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const int r = max(rw, part * 32 + j), c = min(rw, part * 32 + j);
          p[j] = ld_shared_f32(chunk(r, c >> 2) + (c & 3) * 4);
        }
      }
      __syncthreads();                         // the pieces take its place
    }
    const uint32_t mine = ps + (part >> 1) * BLOCK;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = p[8 * c + j] * un;
      put8(chunk8(mine, rw, (part & 1) * 4 + c), P_PIECE, y);
    }
    multiply([&](uint32_t tm) {
      for (int g = 0; g < nk; ++g) {
        const uint64_t d = tc::sdesc_k_sw128(P + g * BLOCK);
        mma_block(one, tm + g * SIDE, d, P_PIECE, 32 >> 4, d, P_PIECE, 32 >> 4, id_p);
      }
      signal(0);
    });
    float q[32];
    wait(0);
    ph[0] ^= 1;
    take32(lanes + part * 32, q);
    add32(lanes + part * 32, 1, nk, SIDE, q);
    // P back from its pieces (32 registers a thread more, held over the
    // product, would spill), Q in their place
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t at = chunk8(mine, rw, (part & 1) * 4 + c);
      float y[8];
      get8(at, P_PIECE, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = fmaf(A.c * un, q[8 * c + j], A.b * y[j]);
      put8(at, P_PIECE, y);
    }
    if (part == (warp & 3)) {                   // the diagonal, where it went
      const uint32_t at = chunk8(mine, rw, (rw & 63) >> 3) + (rw & 7) * 2;
      const float x = ld_half(at) + ld_half(at + P_PIECE) + A.a * kOrthScale;
      const __half hi = __float2half_rn(x), lo = __float2half_rn(x - __half2float(hi));
      g16::st_shared16(at, __half_as_ushort(hi));
      g16::st_shared16(at + P_PIECE, __half_as_ushort(lo));
    }
    multiply([&](uint32_t tm) {
      for (int i = 0; i < 2; ++i) {            // the first half's columns, the others
        const int b0 = i ? nb0 : 0, nb = i ? nblk - nb0 : nb0;
        const uint32_t id_x = g16::idesc_16(SIDE, nb * 64, 0, 0, 1);
        for (int g = 0; g < nk && nb > 0; ++g)
          mma_block(one, tm + g * CHUNK + b0 * 64, tc::sdesc_k_sw128(P + g * BLOCK), P_PIECE, 32 >> 4,
                    desc_columns(X + b0 * BLOCK + g * 64 * 128), X_PIECE, 2048 >> 4, id_x);
        signal(i);
      }
    });
    // a warp's columns take the place of what no product reads any more
    const bool last = k + 1 == A.steps;
    for (int g = part; g < lc >> 5; g += 4) {
      if (g < 2 * nb0)
        wait(0);
      else
        wait(1);
      float v[32];
      const int cc = g * 32;
      take32(lanes + cc, v);
      add32(lanes + cc, 1, nk, CHUNK, v);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = v[8 * c + j] * un;
        const uint32_t at = chunk8(xs + (cc >> 6) * BLOCK, rw, ((cc & 63) >> 3) + c);
        if (last)
          wait8(at, x);
        else
          put8(at, X_PIECE, x);
      }
    }
    wait(1);                                   // by every warp: nobody falls a phase behind
    ph[0] ^= 1;
    ph[1] ^= 1;
  }
  // the result, neighbouring threads to neighbouring addresses
  __syncthreads();
#pragma unroll 2
  for (int e = t; e < items; e += NT) {
    int r, c;
    if (!item(e, r, c)) continue;
    const int left = r < S ? L - (c0 + c * 8) : 0;
    float x[8];
    waited8(chunk8(X + (c >> 3) * BLOCK, r, c & 7), x);
    E* p = reinterpret_cast<E*>(A.out) + at8(r, c);
    if (A.vec_out && left >= 8) {
      Eight<E> v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v.e[j] = down<E>(x[j] * un);
      write8(p, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) p[j * step] = down<E>(x[j] * un);
    }
  }
  if (*abort) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000) {}        // time for the MMAs in flight
  }
  __syncwarp();
  tc::fence_before_sync();
  g16::cluster_sync();                         // its shared memory is read no more
  if (warp == 1) {
    tc::fence_after_sync();
    g16::tmem_dealloc<1>(ctl->tmem_base, 512);
  }
}

template <typename E>
cudaError_t launch(const ChainArgs& a, int64_t batch, cudaStream_t s) {
  auto kern = orth_chain_kernel<E>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = g16::allow_smem(reinterpret_cast<const void*>(kern), &done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(batch * a.C));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  count_launch();
  return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace

bool orth_in_cluster(const memlayer_orth_config& c) {
  const int S = c.rows < c.cols ? c.rows : c.cols, L = c.rows < c.cols ? c.cols : c.rows;
  return S <= SIDE && L <= MOST * CHUNK;
}

cudaError_t launch_orth_chain(const memlayer_orth_config& c, const void* update, void* out, int* err, cudaStream_t s) {
  ChainArgs a{};
  a.u = update;
  a.out = out;
  a.m = c.rows;
  a.n = c.cols;
  a.tall = c.rows > c.cols;
  a.S = a.tall ? c.cols : c.rows;
  a.L = a.tall ? c.rows : c.cols;
  a.C = 1;
  while (a.C * CHUNK < a.L) a.C *= 2;
  a.lc = ((a.L + a.C - 1) / a.C + 63) / 64 * 64;
  a.steps = c.steps;
  a.a = c.a;
  a.b = c.b;
  a.c = c.c;
  a.eps = (double)c.epsilon;
  const bool rows8 = !a.tall && c.cols % 8 == 0;
  const uintptr_t mask = c.dtype == MEMLAYER_F32 ? 31 : 15;
  a.vec_in = rows8 && (reinterpret_cast<uintptr_t>(update) & mask) == 0;
  a.vec_out = rows8 && (reinterpret_cast<uintptr_t>(out) & mask) == 0;
  a.err = err;
  switch (c.dtype) {
    case MEMLAYER_F16: return launch<__half>(a, c.batch, s);
    case MEMLAYER_BF16: return launch<__nv_bfloat16>(a, c.batch, s);
    default: return launch<float>(a, c.batch, s);
  }
}

}  // namespace ml
