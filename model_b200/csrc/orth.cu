// Orthogonalised update of a batch of Dense kernels: the Newton-Schulz
// iteration towards the polar factor of the update U [m, n],
//
//   X_0 = U / (|U|_F + eps)
//   P = X X^T,  X <- (a I + b P + c P^2) X        (m <= n)
//   P = X^T X,  X <- X (a I + b P + c P^2)        (m > n: the smaller side)
//
// Three products a step on the 16-bit tensor cores (gemm16.cuh), operands as
// two f16 pieces (22 bits, like the float32 paths of loss.cu), accumulated
// in float32 with segments of k.  The polynomial is written so that no
// epilogue reads a matrix: the first product's epilogue writes P and
// R = b I + c P, the second's a I + R P, the third's the next X (the output's
// type in the last step).  Majors instead of transposes: the m > n products
// read X along its other index.  The first two are symmetric: only the tiles
// on and below the diagonal are computed, the epilogue writes the others as
// their transposes.  A long k with few tiles is cut into slices, whose float32
// partials a small kernel adds.  Matrices that a cluster's shared memory holds
// take orth_chain.cu instead.
//
// Entries of X, P, R and Q are bounded by their singular values, which the
// host bounds for the given coefficients before it launches (the usual
// (3.4445, -4.7750, 2.0315) keeps X below 1.21 and R, Q below 4.8), so the
// pieces use one fixed scale, 2^12.
#include "orth.cuh"

#include <math.h>

#include "gemm16.cuh"
#include "pieces16.cuh"

namespace ml {

namespace {

using g16::Maps;
using g16::Prod;
using g16::Sched;
using g16::Tile;

// Stages per segment of a product's k.  One (64 k, four steps) keeps the
// error at a float32 GEMM's; its drains take 1.35 times a long product's
// tensor time, so products of k > 512, whose float32 error is larger anyway,
// take two.
inline int seg_for(int64_t K) { return K > 512 ? 2 : 1; }
constexpr float SCALE = kOrthScale, BOUND = 15.f;   // 15 x 2^12 < 65504

// ---- |U|_F and the pieces of X_0 -----------------------------------------------
constexpr int NORM_CHUNKS = 1024;

template <typename E> __device__ __forceinline__ float up_f(E x);
template <> __device__ __forceinline__ float up_f(float x) { return x; }
template <> __device__ __forceinline__ float up_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float up_f(__nv_bfloat16 x) { return __bfloat162float(x); }

// Partial sums of squares in float64 (squares of float32 values overflow and
// underflow float32): chunk blockIdx.x of matrix blockIdx.y.
template <typename E>
__global__ void __launch_bounds__(256) orth_norm_kernel(const E* __restrict__ u, int64_t n, int chunks,
                                                        double* __restrict__ part) {
  __shared__ double red[8];
  allow_next();
  wait_previous();
  // whole 16-byte vectors per chunk; a matrix that starts or ends inside one
  // goes by single elements
  constexpr int V = 16 / sizeof(E);
  const int64_t per = ((n + chunks - 1) / chunks + V - 1) / V * V;
  const int64_t b = blockIdx.x * per, e = b + per < n ? b + per : n;
  const E* x = u + blockIdx.y * n;
  double s[4] = {0., 0., 0., 0.};
  auto take = [&](int j, float f) {
    const double v = f;
    s[j & 3] = fma(v, v, s[j & 3]);
  };
  if (((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(n * sizeof(E))) & 15) == 0) {
    struct alignas(16) Vec { E v[V]; };
    for (int64_t i = b + threadIdx.x * V; i < e; i += 2 * 256 * V) {
      Vec p = *reinterpret_cast<const Vec*>(x + i), q{};
      const bool two = i + 256 * V < e;
      if (two) q = *reinterpret_cast<const Vec*>(x + i + 256 * V);
#pragma unroll
      for (int j = 0; j < V; ++j) take(j, up_f(p.v[j]));
      if (two) {
#pragma unroll
        for (int j = 0; j < V; ++j) take(j, up_f(q.v[j]));
      }
    }
  } else {
    for (int64_t i = b + threadIdx.x; i < e; i += 1024) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j * 256 < e) take(j, up_f(x[i + j * 256]));
    }
  }
  double t = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(FULL, t, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) t += red[w];
    part[blockIdx.y * chunks + blockIdx.x] = t;
  }
}

// X_0's pieces, 8 columns a thread (zeros in the padding columns).
template <typename E>
__global__ void __launch_bounds__(256) orth_init_kernel(const E* __restrict__ u, int m, int n, int ld, double eps,
                                                        const double* __restrict__ part, int chunks,
                                                        __half* __restrict__ hi, __half* __restrict__ lo) {
  __shared__ double inv_s;
  allow_next();
  wait_previous();
  if (threadIdx.x < 32) {
    double t = 0.;
    for (int i = threadIdx.x; i < chunks; i += 32) t += part[blockIdx.y * chunks + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(FULL, t, o);
    if (threadIdx.x == 0) inv_s = (double)SCALE / (sqrt(t) + eps);
  }
  __syncthreads();
  const double inv = inv_s;
  const int c8 = ld >> 3;
  const int64_t items = (int64_t)m * c8, z = (int64_t)blockIdx.y;
  const E* x = u + z * m * n;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < items; e += (int64_t)gridDim.x * 256) {
    const int64_t r = e / c8;
    const int c = (int)(e - r * c8) * 8;
    const E* p = x + r * n + c;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < n ? (float)((double)up_f(p[j]) * inv) : 0.f;
    __half2 h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) g16::split2(v[2 * j], v[2 * j + 1], h[j], l[j]);
    const int64_t at = z * m * ld + r * ld + c;
    *reinterpret_cast<uint4*>(hi + at) = *reinterpret_cast<uint4*>(h);
    *reinterpret_cast<uint4*>(lo + at) = *reinterpret_cast<uint4*>(l);
  }
}

// ---- epilogue ----------------------------------------------------------------------
struct PolyArgs {
  CUtensorMap out[2][2];               // [first, second output][hi, lo]; out[0][0]: the plain output when type >= 0
  int64_t M;
  int N;
  int two;                             // a second output follows
  float s[2], diag[2];                 // output q = s[q] acc + diag[q] I (in scaled units)
  int type;                            // -1: pieces; -2: float32 partials of k slices (out[0][0]); else
                                       // memlayer_dtype of the plain output
  int tma;                             // the plain output's rows are 16 bytes apart
  void* plain;                         // [batch][M][N]
};

struct EpiPoly {
  static constexpr bool kSum = true, kStore = true;
  using Args = PolyArgs;
  float sum[128];
  uint32_t buf;
  StagingTurn turn;
  __device__ __forceinline__ void begin(const Args&, const Sched&, int, uint8_t* staging) {
    buf = tc::smem_u32(staging);
    turn = StagingTurn{};
  }
  static __device__ __forceinline__ void pieces(const CUtensorMap* map, uint32_t buf, const uint32_t (&v)[32],
                                                float s, float diag, int at, int col, int row0, int z, bool mirror) {
    uint32_t h[16], l[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float x = __uint_as_float(v[2 * j]) * s, y = __uint_as_float(v[2 * j + 1]) * s;
      if (at == 2 * j) x += diag;
      if (at == 2 * j + 1) y += diag;
      __half2 a, b;
      g16::split2(x, y, a, b);
      h[j] = *reinterpret_cast<const uint32_t*>(&a);
      l[j] = *reinterpret_cast<const uint32_t*>(&b);
    }
    g16::store_pieces(map, buf, h, l, col, row0, z);
    if (mirror) g16::store_pieces(map, buf, h, l, row0, col, z, true);
  }
  __device__ __forceinline__ void partial(const Args& A, uint32_t (&v)[32], int row0, int col, int z) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) g16::bulk_wait<0, true>();
    __syncwarp();
    g16::stage32(buf, lane, v);
    tc::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) g16::bulk_store(&A.out[0][0], buf, col, row0, z, false);
  }
  __device__ __forceinline__ void plain(const Args& A, uint32_t (&v)[32], int64_t row0, int col, int z) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * A.s[0]);
    const uint32_t b = g16::staging_place(turn, buf, A.type == MEMLAYER_F32, A.tma);
    g16::stage_as(A.type, b, lane, v);
    if (A.tma) {
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) g16::bulk_store(&A.out[0][0], b, col, (int)row0, z, false);
    } else {
      __syncwarp();
      g16::copy_rows(A.type, b, A.plain, (z * A.M + row0) * A.N + col, A.N, (int)(A.M - row0 < 32 ? A.M - row0 : 32),
                     A.N - col, false);
      __syncwarp();
    }
  }
  __device__ __forceinline__ void store(const Args& A, const Sched& S, const Tile& t, int64_t row, int half) {
    const int64_t row0 = row - (threadIdx.x & 31);
    const int hw = S.BN >> 1;
    const int col0 = t.nt * S.BN + half * hw;
    if (row0 >= A.M) return;
#pragma unroll
    for (int cc = 0; cc < 128; cc += 32) {
      if (cc >= hw || col0 + cc >= A.N) break;
      const int col = col0 + cc;
      uint32_t v[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(sum[cc + j]);
      if (A.type >= 0) {
        plain(A, v, row0, col, t.z);
      } else if (A.type == -2) {
        partial(A, v, (int)row0, col, t.ks * S.prod[0].batch + t.z);
      } else {
        const int64_t d = row - col;                         // the diagonal's column in this block
        const int at = d >= 0 && d < 32 ? (int)d : -1;
        const bool mirror = S.prod[0].tri && t.mt > t.nt;
        for (int q = 0; q < 1 + A.two; ++q)
          pieces(A.out[q], buf, v, A.s[q], A.diag[q], at, col, (int)row0, t.z, mirror);
      }
    }
  }
  __device__ __forceinline__ void end(const Args&, const Sched&, int) {}
};

// The slices' partials of a symmetric product [slices][batch][s][lds], added in
// slice order, to its outputs' pieces: a 32 x 32 block on or below the
// diagonal per thread block (the tiles above it were not computed), written
// as it is and transposed.
struct JoinArgs {
  const float* part;
  int slices, s, lds;
  int64_t se;                          // entries from hi to lo
  __half* out[2];
  int two;
  float sc[2], diag[2];
};

__global__ void __launch_bounds__(256) orth_join_kernel(JoinArgs A) {
  __shared__ float t[32][33];
  allow_next();
  wait_previous();
  int rb = (int)((sqrtf(8.f * blockIdx.x + 1.f) - 1.f) * 0.5f);
  while ((rb + 1) * (rb + 2) / 2 <= (int)blockIdx.x) ++rb;
  while (rb * (rb + 1) / 2 > (int)blockIdx.x) --rb;
  const int cb = blockIdx.x - rb * (rb + 1) / 2;
  const int64_t one = (int64_t)A.s * A.lds, all = one * gridDim.y, z = blockIdx.y;
  const int i = threadIdx.x >> 3, j0 = (threadIdx.x & 7) * 4;
  // lds is a multiple of 8: four columns are inside the pitch together
  const int r = rb * 32 + i, c = cb * 32 + j0;
  const bool in = r < A.s && c < A.lds;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (in) {
    const float* p = A.part + z * one + (int64_t)r * A.lds + c;
    for (int k = 0; k < A.slices; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(p + k * all);
      x[0] += v.x;
      x[1] += v.y;
      x[2] += v.z;
      x[3] += v.w;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) t[i][j0 + j] = x[j];
  __syncthreads();
  auto put = [&](int row, int col, const float (&v)[4]) {
    for (int q = 0; q < 1 + A.two; ++q) {
      alignas(8) __half2 h[2], l[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        g16::split2(v[2 * j] * A.sc[q] + (col + 2 * j == row ? A.diag[q] : 0.f),
                    v[2 * j + 1] * A.sc[q] + (col + 2 * j + 1 == row ? A.diag[q] : 0.f), h[j], l[j]);
      __half* o = A.out[q] + z * one + (int64_t)row * A.lds + col;
      *reinterpret_cast<uint2*>(o) = *reinterpret_cast<uint2*>(h);
      *reinterpret_cast<uint2*>(o + A.se) = *reinterpret_cast<uint2*>(l);
    }
  };
  if (in) put(r, c, x);
  if (rb != cb) {
    const int tr = cb * 32 + i, tc = rb * 32 + j0;
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = t[j0 + j][i];
    if (tr < A.s && tc < A.lds) put(tr, tc, y);
  }
}

// ---- plan -----------------------------------------------------------------------
int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

constexpr size_t O_ERR = 256, HEAD = 512;

struct Plan {
  int64_t B, m, n, s;                  // s: the smaller side
  bool tall;
  int64_t ldx, lds;
  size_t o_part, o_x[2], o_p, o_r, o_q, o_k, bytes;   // hi then lo in each
  int64_t xe, se;                      // entries of one piece of X, of an s x s matrix
};

struct Tiling {
  int cg, BN, tri, slices;
};

// Tile and slices of k with the least estimated time: rounds of tiles over
// the clusters, each its stages and an epilogue, in SM cycles as measured at
// 4096^3 (large tiles) and 256^3 (small ones); joining slices costs a small
// kernel.  Symmetric products take square tiles on and below the diagonal, or
// small ones everywhere (12 tiles of 128 x 128 took 176 us for 4 x 256 x 256,
// 32 of 128 x 64 148).
Tiling tiling(int64_t M, int64_t N, int64_t K, int64_t batch, bool symmetric) {
  struct Shape { int cg, BN, tri; double stage, epilogue; };
  const Shape all[4] = {{2, 256, 1, 1900, 6000}, {2, 128, 0, 1100, 4000}, {1, 128, 1, 1000, 4000}, {1, 64, 0, 750, 3000}};
  const int64_t kq = up(K, g16::BK) / g16::BK;
  Tiling best{1, 64, 0, 1};
  double least = 1e300;
  for (const Shape& t : all) {
    if (symmetric && t.cg == 2 && !t.tri) continue;
    const bool tri = symmetric && t.tri;
    const int64_t mt = up(M, 128 * t.cg) / (128 * t.cg), nt = up(N, t.BN) / t.BN;
    const int64_t tiles = (tri ? mt * (mt + 1) / 2 : mt * nt) * batch, clusters = g16::device_sms() / t.cg;
    for (int64_t n = 1; n <= (symmetric ? kq / 4 : 1) || n == 1; n *= 2) {
      if (n > 1 && tiles * n > clusters) break;
      const int64_t rounds = (tiles * n + clusters - 1) / clusters, per = (kq + n - 1) / n;
      const double cost = rounds * (per * t.stage + t.epilogue) + (n > 1 ? 8000 : 0);
      if (cost < least) {
        least = cost;
        best = {t.cg, t.BN, tri, (int)n};
      }
    }
  }
  return best;
}

bool make_plan(const memlayer_orth_config& c, Plan* out) {
  Plan p{};
  p.B = c.batch;
  p.m = c.rows;
  p.n = c.cols;
  p.tall = c.rows > c.cols;
  p.s = p.tall ? p.n : p.m;
  p.ldx = up(p.n, 8);
  p.lds = up(p.s, 8);
  p.xe = p.B * p.m * p.ldx;
  p.se = p.B * p.s * p.lds;
  if (orth_in_cluster(c)) {            // needs the status word only
    p.bytes = HEAD;
    *out = p;
    return true;
  }
  size_t off = HEAD;
  auto take = [&](int64_t bytes) {
    const size_t o = off;
    off += (size_t)up(bytes, 256);
    return o;
  };
  p.xe = up(p.xe, 128);                // the second piece starts 256-byte aligned
  p.se = up(p.se, 128);
  p.o_part = take(p.B * NORM_CHUNKS * 8);
  p.o_x[0] = take(2 * p.xe * 2);
  p.o_x[1] = take(2 * p.xe * 2);
  p.o_p = take(2 * p.se * 2);
  p.o_r = take(2 * p.se * 2);
  p.o_q = take(2 * p.se * 2);
  // partials of the first two products' slices
  const int s1 = tiling(p.s, p.s, p.tall ? p.m : p.n, p.B, true).slices, s2 = tiling(p.s, p.s, p.s, p.B, true).slices;
  const int sl = s1 > s2 ? s1 : s2;
  if (sl > 1) p.o_k = take((int64_t)sl * p.B * p.s * p.lds * 4);
  p.bytes = off;
  *out = p;
  return true;
}

#define OR_TRY(x)                             \
  do {                                        \
    const cudaError_t e_ = (x);               \
    if (e_ != cudaSuccess) return e_;         \
  } while (0)

struct Mat {
  const __half* p;                     // hi; lo is `lo` entries on
  int64_t lo, ld, batch;               // batch: entries between matrices
};

// One of the three products: its tiles and the maps of its operands (built
// once a call for each of the two buffers that X alternates between).
struct Product {
  Maps maps[2];
  Sched S;
  Tiling t;
  int64_t M, N;
};

// A(i, k): M rows; B(j, k): N rows; k of length K.  tri: the result is symmetric.
cudaError_t make_product(const Plan& p, const Mat (&a)[2], bool amn, const Mat (&b)[2], bool bmn, int64_t M, int64_t N,
                         int64_t K, bool tri, int buffers, Product* out) {
  Product& P = *out;
  P.t = tiling(M, N, K, p.B, tri);
  P.M = M;
  P.N = N;
  for (int k = 0; k < buffers; ++k)
    for (int q = 0; q < 2; ++q) {
      OR_TRY(g16::make_operand(&P.maps[k].a[0][q], a[k].p + q * a[k].lo, M, K, a[k].ld, amn, 128, 0, (int)p.B,
                               a[k].batch));
      OR_TRY(g16::make_operand(&P.maps[k].b[0][q], b[k].p + q * b[k].lo, N, K, b[k].ld, bmn, P.t.BN / P.t.cg, 0,
                               (int)p.B, b[k].batch));
    }
  Prod& r = P.S.prod[0];
  r.m_tiles = (int)(up(M, 128 * P.t.cg) / (128 * P.t.cg));
  r.n_tiles = (int)(up(N, P.t.BN) / P.t.BN);
  r.batch = (int)p.B;
  r.kq_total = (int)(up(K, g16::BK) / g16::BK);
  r.kq = (r.kq_total + P.t.slices - 1) / P.t.slices;
  r.splits = (r.kq_total + r.kq - 1) / r.kq;
  r.amn = amn;
  r.bmn = bmn;
  r.tri = P.t.tri;
  P.S.BN = P.t.BN;
  P.S.seg = seg_for(K);
  g16::distribute(&P.S, g16::device_sms() / P.t.cg, 0);
  return cudaSuccess;
}

cudaError_t launch(const Product& P, int buffer, const PolyArgs& ea, int* err, cudaStream_t s) {
  return P.t.cg == 2 ? g16::launch_one<EpiPoly, 2, 2, 2>(P.maps[buffer], P.S, ea, err, s)
                     : g16::launch_one<EpiPoly, 1, 2, 2>(P.maps[buffer], P.S, ea, err, s);
}

// A symmetric product to its outputs' pieces; `raw`: the partials of its slices as an output.
cudaError_t symmetric(const Plan& p, const Product& P, int buffer, const PolyArgs& ea, const PolyArgs& raw,
                      __half* o0, __half* o1, char* ws, cudaStream_t s) {
  int* err = reinterpret_cast<int*>(ws + O_ERR);
  if (P.S.prod[0].splits == 1) return launch(P, buffer, ea, err, s);
  OR_TRY(launch(P, buffer, raw, err, s));
  const JoinArgs j{reinterpret_cast<float*>(ws + p.o_k), P.S.prod[0].splits, (int)p.s, (int)p.lds, p.se, {o0, o1},
                   ea.two, {ea.s[0], ea.s[1]}, {ea.diag[0], ea.diag[1]}};
  const int64_t nb = (p.s + 31) / 32;
  count_launch();
  return launch_dependent(orth_join_kernel, dim3((unsigned)(nb * (nb + 1) / 2), (unsigned)p.B), 256, 0, s, j);
}

template <typename E>
cudaError_t start(const memlayer_orth_config& c, const Plan& p, const E* u, char* ws, cudaStream_t s) {
  const int64_t n = p.m * p.n;
  int64_t chunks = (n + 4095) / 4096;
  if (chunks > NORM_CHUNKS) chunks = NORM_CHUNKS;
  double* part = reinterpret_cast<double*>(ws + p.o_part);
  count_launch();
  OR_TRY(launch_dependent(orth_norm_kernel<E>, dim3((unsigned)chunks, (unsigned)p.B), 256, 0, s, u, n, (int)chunks,
                          part));
  const int64_t items = p.m * (p.ldx / 8);
  int64_t blocks = (items + 511) / 512;
  const int64_t cap = up(8 * g16::device_sms(), p.B) / p.B;
  if (blocks > cap) blocks = cap;
  __half* x = reinterpret_cast<__half*>(ws + p.o_x[0]);
  count_launch();
  return launch_dependent(orth_init_kernel<E>, dim3((unsigned)blocks, (unsigned)p.B), 256, 0, s, u, (int)p.m, (int)p.n,
                          (int)p.ldx, (double)c.epsilon, (const double*)part, (int)chunks, x, x + p.xe);
}

}  // namespace

bool orth_workspace(const memlayer_orth_config& c, size_t* bytes) {
  Plan p;
  if (!make_plan(c, &p)) return false;
  *bytes = p.bytes;
  return true;
}

bool orth_coefficients_ok(const memlayer_orth_config& cfg) {
  // Singular values start in [0, 1] and go through f(x) = x (a + b x^2 + c x^4);
  // every matrix of a step is bounded by its largest singular value.  f is
  // continuous and f(0) = 0, so a step takes [0, hi] to [0, max |f|] exactly,
  // and the maxima are at the ends or where a derivative is zero: no value in
  // between is missed (samples of [0, 1] missed some that grow without bound).
  const double a = cfg.a, b = cfg.b, c = cfg.c;
  double hi = 1.0;
  for (int k = 0; k < cfg.steps; ++k) {
    const double u = hi * hi;                              // u = x^2 in [0, u]
    const double r = fmax(fabs(b), fabs(b + c * u));
    auto q_at = [&](double v) { return a + (b + c * v) * v; };
    double q = fmax(fabs(a), fabs(q_at(u))), top = fabs(hi * q_at(u));
    if (c != 0.0 && -b / (2 * c) > 0.0 && -b / (2 * c) < u) q = fmax(q, fabs(q_at(-b / (2 * c))));
    double root[2] = {-1.0, -1.0};                         // of a + 3 b v + 5 c v^2
    if (c != 0.0) {
      const double d = 9 * b * b - 20 * a * c;
      if (d >= 0.0) {
        root[0] = (-3 * b + sqrt(d)) / (10 * c);
        root[1] = (-3 * b - sqrt(d)) / (10 * c);
      }
    } else if (b != 0.0) {
      root[0] = -a / (3 * b);
    }
    for (double v : root)
      if (v > 0.0 && v < u) top = fmax(top, sqrt(v) * fabs(q_at(v)));
    // (a NaN among the coefficients fails the comparisons: fmax drops it, the sum keeps it)
    if (!(u <= BOUND * 0.5) || !(r <= BOUND * 0.8) || !(q <= BOUND * 0.8) || !(a + b + c == a + b + c)) return false;
    hi = top;
  }
  return hi <= BOUND * 0.2;
}

cudaError_t launch_orthogonalize(const memlayer_orth_config& c, const void* update, void* out, char* ws,
                                 cudaStream_t s) {
  Plan p;
  if (!make_plan(c, &p)) return cudaErrorInvalidValue;
  int* err = reinterpret_cast<int*>(ws + O_ERR);
  if (p.B > 0 && orth_in_cluster(c)) return launch_orth_chain(c, update, out, err, s);
  OR_TRY(cudaMemsetAsync(err, 0, sizeof(int), s));
  if (p.B == 0) return cudaSuccess;
  switch (c.dtype) {
    case MEMLAYER_F16: OR_TRY(start(c, p, (const __half*)update, ws, s)); break;
    case MEMLAYER_BF16: OR_TRY(start(c, p, (const __nv_bfloat16*)update, ws, s)); break;
    default: OR_TRY(start(c, p, (const float*)update, ws, s)); break;
  }
  __half *x[2] = {reinterpret_cast<__half*>(ws + p.o_x[0]), reinterpret_cast<__half*>(ws + p.o_x[1])};
  __half *P = reinterpret_cast<__half*>(ws + p.o_p), *R = reinterpret_cast<__half*>(ws + p.o_r),
         *Q = reinterpret_cast<__half*>(ws + p.o_q);
  const Mat X[2] = {{x[0], p.xe, p.ldx, p.m * p.ldx}, {x[1], p.xe, p.ldx, p.m * p.ldx}};
  auto square = [&](const __half* q) { return Mat{q, p.se, p.lds, p.s * p.lds}; };
  const Mat MP[2] = {square(P), square(P)}, MR[2] = {square(R), square(R)}, MQ[2] = {square(Q), square(Q)};
  const int buffers = c.steps > 1 ? 2 : 1;
  Product gram{}, poly{}, apply{};
  OR_TRY(make_product(p, X, p.tall, X, p.tall, p.s, p.s, p.tall ? p.m : p.n, true, buffers, &gram));
  OR_TRY(make_product(p, MR, false, MP, false, p.s, p.s, p.s, true, 1, &poly));
  if (p.tall)
    OR_TRY(make_product(p, X, false, MQ, false, p.m, p.n, p.n, false, buffers, &apply));
  else
    OR_TRY(make_product(p, MQ, false, X, true, p.m, p.n, p.m, false, buffers, &apply));
  auto pieces = [&](CUtensorMap* map, __half* q, int64_t lo, int64_t rows, int64_t cols, int64_t ld) {
    for (int i = 0; i < 2; ++i) {
      const cudaError_t e = g16::make_store(map + i, q + i * lo, rows, cols, ld, MEMLAYER_F16, p.B, rows * ld);
      if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
  };
  auto sizes = [&](PolyArgs& a, const Product& q) {
    a.M = q.M;
    a.N = (int)q.N;
    a.type = -1;
  };
  PolyArgs a1{}, a2{}, a3[2]{}, last{}, r1{}, r2{};
  OR_TRY(pieces(a1.out[0], P, p.se, p.s, p.s, p.lds));
  OR_TRY(pieces(a1.out[1], R, p.se, p.s, p.s, p.lds));
  OR_TRY(pieces(a2.out[0], Q, p.se, p.s, p.s, p.lds));
  // accumulators carry SCALE^2, pieces SCALE
  sizes(a1, gram);
  a1.two = 1;
  a1.s[0] = 1.f / SCALE;
  a1.s[1] = c.c / SCALE;
  a1.diag[1] = c.b * SCALE;
  sizes(a2, poly);
  a2.s[0] = 1.f / SCALE;
  a2.diag[0] = c.a * SCALE;
  for (PolyArgs* r : {&r1, &r2}) {
    const Product& q = r == &r1 ? gram : poly;
    sizes(*r, q);
    r->type = -2;
    if (q.S.prod[0].splits > 1)
      OR_TRY(g16::make_store(&r->out[0][0], ws + p.o_k, p.s, p.s, p.lds, MEMLAYER_F32, q.S.prod[0].splits * p.B,
                             p.s * p.lds));
  }
  for (int k = 0; k < buffers; ++k) {
    sizes(a3[k], apply);
    a3[k].s[0] = 1.f / SCALE;
    OR_TRY(pieces(a3[k].out[0], x[k], p.xe, p.m, p.n, p.ldx));
  }
  const int64_t es = c.dtype == MEMLAYER_F32 ? 4 : 2;
  sizes(last, apply);
  last.type = c.dtype;
  last.s[0] = 1.f / (SCALE * SCALE);
  last.plain = out;
  last.tma = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && p.n * es % 16 == 0;
  if (last.tma) OR_TRY(g16::make_store(&last.out[0][0], out, p.m, p.n, p.n, c.dtype, p.B, p.m * p.n));
  for (int k = 0; k < c.steps; ++k) {
    OR_TRY(symmetric(p, gram, k & 1, a1, r1, P, R, ws, s));
    OR_TRY(symmetric(p, poly, 0, a2, r2, Q, nullptr, ws, s));
    OR_TRY(launch(apply, k & 1, k + 1 < c.steps ? a3[(k + 1) & 1] : last, err, s));
  }
  return cudaSuccess;
}

}  // namespace ml
