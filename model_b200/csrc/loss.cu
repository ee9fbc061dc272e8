// Softmax cross entropy over the vocabulary, fused with the output projection
// (the tied logits of memory_pool_model/model.py:125 under the trainer's
// integer-label cross entropy), and its gradient:
//
//   z = h W^T                       [T, V], never stored
//   lse_t = log sum_v exp z_tv,  loss_t = lse_t - z_t,target (0 when ignored)
//   dz_tv = p_tv (dloss_t + dlse_t) - [v == target] dloss_t,  p = exp(z - lse)
//   dh = dz W,  dW = dz^T h
//
// Forward: one pass of 16-bit tensor-core tiles (gemm16.cuh) over the
// vocabulary; the epilogue thread of a row keeps the running maximum and sum
// of its columns in registers along its cluster's run of tiles, so a row
// block leaves one (maximum, sum) pair per run and column half; a second
// kernel joins them.  Backward: the vocabulary in pieces; for each piece the
// logits are computed again, the epilogue turns them into dz (16 bits, the
// piece's [T, piece] matrix in the workspace), and one launch multiplies it
// both ways, dW of the piece and its part of dh.
//
// float32 operands run as two f16 pieces each (22 bits, see gemm16.cuh; h with
// a scale a token), dz too; 16-bit operands as they are.  dz of a 16-bit call
// has two pieces up to 128 tokens and is rounded once to the type beyond, half
// a step of each term.  It shows where one term is most of a sum, as a
// target's is: 8192 x 1024 over 32,768 bf16 is 2.4e-3 from the gradients in 64
// bits, 1999 x 512 over 30,011 f16 4.3e-4; two pieces leave the rounding of
// the results, 1.7e-3 and 3.9e-4, and take 2935 us for 1876 and 401 for 276.
// Statistics, exponentials and sums are float32.
#include "loss.cuh"

#include <float.h>

#include <type_traits>

#include "gemm16.cuh"
#include "pieces16.cuh"

namespace ml {

namespace {

int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

using g16::Maps;
using g16::Prod;
using g16::Sched;
using g16::Tile;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int STATUS_TARGET = 27;
// Stages per segment of k in the float32 gradient products: 192 k, 12 steps.
// dW of 1,000 tokens is 0.8e-6 off with 4, 0.58e-6 with 3, 0.45e-6 with 2
// (a float32 GEMM 0.56e-6); at 8192 x 256 x 16384 they take 296, 304, 367 us.
constexpr int SEG = 3;
// Stages per segment of the float32 logits, beyond a k of as many: there the
// loss is up to 0.6e-6 off, without segments 1.3e-6 at a k of 1024.
constexpr int LOGIT_SEG = 8;

template <typename E> __device__ __forceinline__ float to_f32(E x);
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename E> __device__ __forceinline__ E from_f32(float x);
template <> __device__ __forceinline__ float from_f32(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ int exp_of(const unsigned* amax) { return amax ? g16::scale_exp(*amax) : 0; }

// Factor that turns an accumulator of a token's logits back, from the scales'
// exponents: a normal float (beyond that range logits are zero or infinite for
// every purpose).
__device__ __forceinline__ float logit_unscale(int exp_h, int exp_w) {
  return g16::pow2(max(-100, min(126, -exp_h - exp_w)));
}

// ---- a scale for each token ----------------------------------------------------------
// f16 operands carry powers of two, and each token has its own.  With one for
// all of them a single huge token -- padding, too, where anything may stand --
// takes the others' bits (a row of 1e10 among ones of 1 put their lse 0.02
// off), and a token whose loss weighs 1e-9 of another's loses its dz.  h gets
// its scale from the token's largest entry (float32 only), dz from the larger
// of the token's two factors.  A logit and an entry of dh belong to one token,
// so the epilogues take the scales out by row.  dW sums over tokens, and what
// each of them adds has to carry the same power of two: there h is converted
// once more, a token's rows times the inverse of its dz scale, all of them
// such that the largest h / scale comes to 2^14 (a token's share of dW is that
// size times p).  That copy of h leaves out the tokens without a gradient, bf16
// too: their rows may hold anything, and zeros times a NaN would be in all of
// dW.  The first blocks look for the weight's largest magnitude meanwhile.
struct TokenArgs {
  AmaxMat w;
  const void* h;
  int64_t T, ldh, ld;
  int d, tpr;                          // tpr: threads a token, 32 or all
  __half *hi, *lo;                     // [T][ld] (float32)
  int* exp_h;                          // [T] exponent of h's scale (float32 forward)
  // the gradient's part (token null: none): a token's record, its target (-1:
  // none; PIECE_SKIP: no gradient at all) and exponent of dz's scale,
  // |p q - [target] g| <= 2 max(|q|, |g|) < 2^15; the largest exponent of
  // h / scale over the tokens that have a gradient
  const int* targets;
  const float *dloss, *dlse;
  int V, ignore;
  float4* token;
  int *tgt, *exp_g;
  unsigned* peak;
  int* err;
};

// What the epilogue of dz needs of a token, in one load: the factors of p and
// of the one-hot target, scaled; the target; the exponent of h's scale.
__device__ __forceinline__ float4 token_record(float q, float g, int target, int exp_h) {
  return make_float4(q, g, __int_as_float(target), __int_as_float(exp_h));
}

template <typename E>
__global__ void __launch_bounds__(PIECE_THREADS) loss_tokens_kernel(TokenArgs A) {
  constexpr int V = 16 / sizeof(E);
  constexpr bool F32 = sizeof(E) == 4, SCALED = !std::is_same<E, __nv_bfloat16>::value;
  struct alignas(16) Vec { E e[V]; };
  __shared__ unsigned red[PIECE_THREADS / 32], top_peak;
  allow_next();
  wait_previous();
  if ((int)blockIdx.x < A.w.blocks) {
    amax_block(A.w, blockIdx.x);
    return;
  }
  if (threadIdx.x == 0) top_peak = 0;
  __syncthreads();
  const int t = threadIdx.x & (A.tpr - 1), groups = PIECE_THREADS / A.tpr, d = A.d;
  const bool vec = A.ldh % V == 0 && d % V == 0 && (reinterpret_cast<uintptr_t>(A.h) & 15) == 0;
  const int64_t step = (int64_t)(gridDim.x - A.w.blocks) * groups;
  for (int64_t base = (int64_t)(blockIdx.x - A.w.blocks) * groups; base < A.T; base += step) {
    const int64_t row = base + threadIdx.x / A.tpr;
    const bool on = row < A.T;
    const E* x = reinterpret_cast<const E*>(A.h) + (on ? row : 0) * A.ldh;
    unsigned mx = 0;
    if (!SCALED) {
    } else if (vec) {
#pragma unroll 2
      for (int c = t * V; c < d; c += A.tpr * V) {
        const Vec v = *reinterpret_cast<const Vec*>(x + c);
#pragma unroll
        for (int j = 0; j < V; ++j) mx = max(mx, finite_bits(to_f32(v.e[j])));
      }
    } else {
      for (int c = t; c < d; c += A.tpr) mx = max(mx, finite_bits(to_f32(x[c])));
    }
    mx = __reduce_max_sync(FULL, mx);
    if (A.tpr > 32) {
      __syncthreads();                 // the slots of the token before are read
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mx;
      __syncthreads();
      for (int w = 0; w < PIECE_THREADS / 32; ++w) mx = max(mx, red[w]);
    }
    if (!on) continue;
    const int eh = F32 ? g16::scale_exp(mx) : 0;
    if (t == 0 && A.token) {
      const int v = A.targets[row];
      const bool in = v >= 0 && v < A.V && v != A.ignore;
      if (!in && v != A.ignore) atomicCAS(A.err, 0, STATUS_TARGET);
      const float g = in ? A.dloss[row] : 0.f, q = g + (A.dlse ? A.dlse[row] : 0.f);
      const bool none = g == 0.f && q == 0.f;
      const int target = none ? PIECE_SKIP : in ? v : -1;
      const int f = SCALED ? g16::scale_exp(max(finite_bits(g), finite_bits(q))) - 1 : 0;
      const float sg = g16::pow2(f);
      A.token[row] = token_record(q * sg, g * sg, target, eh);
      A.tgt[row] = target;
      if constexpr (SCALED) {
        A.exp_g[row] = f;
        if (!none && mx) atomicMax(&top_peak, piece_peak((int)(mx >> 23) - 127 - f));
      }
    }
    if constexpr (!F32) continue;
    if (t == 0 && A.exp_h) A.exp_h[row] = eh;
    const float sc = g16::pow2(eh);
    for (int c = t * 8; c < (int)A.ld; c += A.tpr * 8) {
      float v[8];
      if (vec && c + 8 <= d) {
        const float4 a = *reinterpret_cast<const float4*>(x + c), b = *reinterpret_cast<const float4*>(x + c + V);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < d ? to_f32(x[c + j]) : 0.f;
      }
      __half2 h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) g16::split2(v[2 * j] * sc, v[2 * j + 1] * sc, h[j], l[j]);
      *reinterpret_cast<uint4*>(A.hi + row * A.ld + c) = *reinterpret_cast<uint4*>(h);
      *reinterpret_cast<uint4*>(A.lo + row * A.ld + c) = *reinterpret_cast<uint4*>(l);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && top_peak) atomicMax(A.peak, top_peak);   // a maximum: the order does not matter
}

template <typename E>
cudaError_t launch_tokens(TokenArgs A, cudaStream_t s) {
  A.w.blocks = A.w.rows ? piece_blocks(A.w.rows * A.w.cols, 16) : 0;
  A.tpr = A.d <= 2048 ? 32 : PIECE_THREADS;
  const int64_t need = (A.T * A.tpr + PIECE_THREADS - 1) / PIECE_THREADS, cap = 8 * g16::device_sms();
  count_launch();
  return launch_dependent(loss_tokens_kernel<E>, dim3((unsigned)(A.w.blocks + (need < cap ? need : cap))), PIECE_THREADS,
                          0, s, A);
}

// log p of a logit whose forward may have been added in another order (the
// kernels of few tokens and the tiles differ, and lse may come from elsewhere):
// rounding of large logits does not make p more than 1.  A NaN stays.
__device__ __forceinline__ float at_most_0(float x) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(0.f));
  return r;
}

__device__ __forceinline__ unsigned long long pair(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}

// The 32 columns from cc on of an epilogue thread's row: from its accumulator,
// or from the sums of its segments.
struct FromTmem {
  uint32_t taddr;
  __device__ __forceinline__ void operator()(int cc, uint32_t (&v)[32]) const {
    tc::tmem_ld32(taddr + cc, v);
    tc::tmem_wait_ld();
  }
};
struct FromSums {
  const float (&sum)[128];
  __device__ __forceinline__ void operator()(int cc, uint32_t (&v)[32]) const {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(sum[cc + j]);
  }
};

// ---- forward epilogue ------------------------------------------------------------
struct StatsArgs {
  int64_t T;
  int V;
  const int* exp_h;                  // float32 operands: scales of the tokens and the weight (else null)
  const unsigned* amax_w;
  const int* targets;
  float2* part;                      // [slot][half][T] (maximum, sum of exp(z - maximum))
  float* zt;                         // [T] target logit
};

template <bool SUM>
struct EpiStats {
  static constexpr bool kSum = SUM, kStore = false;
  float sum[128];
  using Args = StatsArgs;
  float m, s, c, un;
  int mt, slot, target;
  int64_t row;
  bool any;

  __device__ __forceinline__ void begin(const Args& A, const Sched&, int cluster, uint8_t*) {
    mt = -1;
    slot = cluster;
    any = false;
  }
  __device__ __forceinline__ void flush(const Args& A, const Sched& S, int half) {
    if (!any || row >= A.T) return;
    // clusters before this one that hold tiles of the row block
    const int first = S.owner(mt * S.prod[0].n_tiles);
    A.part[((int64_t)(slot - first) * 2 + half) * A.T + row] = make_float2(m * un, s);
  }
  template <class Get>
  __device__ __forceinline__ void blocks(const Args& A, const Sched& S, const Tile& t, int64_t r, int half, Get get) {
    if (t.mt != mt) {
      flush(A, S, half);
      mt = t.mt;
      row = r;
      m = -INFINITY;
      s = 0.f;
      any = true;
      target = row < A.T ? A.targets[row] : -1;
      un = logit_unscale(A.exp_h && row < A.T ? A.exp_h[row] : 0, exp_of(A.amax_w));
      c = un * LOG2E;
    }
    const int hw = S.BN >> 1;
    const int col0 = t.nt * S.BN + half * hw;
#pragma unroll
    for (int cc = 0; cc < 128; cc += 32) {
      if (cc >= hw || col0 + cc >= A.V) break;   // the same for the whole warp
      uint32_t v[32];
      __syncwarp();
      get(cc, v);
      const int left = A.V - (col0 + cc);
      if (left < 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j >= left) v[j] = 0xFF800000u;   // -inf
      }
      float mx = __uint_as_float(v[0]);
#pragma unroll
      for (int j = 1; j < 32; ++j) mx = fmaxf(mx, __uint_as_float(v[j]));
      // the difference first, then the factor: at the maximum it is 0 whatever
      // the logits' size (v c - round(m c) is not: 4,000 for logits of 1e10),
      // and elsewhere its error goes by the difference, not by the logits.
      // Two columns an instruction: as many as one fused multiply-add each.
      const float mn = fmaxf(m, mx);
      const float ref = mn == -INFINITY ? 0.f : mn;
      const unsigned long long nr = pair(-ref, -ref), cc2 = pair(c, c);
      float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        unsigned long long x = pair(__uint_as_float(v[j]), __uint_as_float(v[j + 1]));
        asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(nr));
        asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(cc2));
        float e0, e1;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(e0), "=f"(e1) : "l"(x));
        a[j & 3] += g16::exp2_fast(e0);
        a[(j & 3) + 1] += g16::exp2_fast(e1);
      }
      s = fmaf(s, g16::exp2_fast((m - ref) * c), (a[0] + a[1]) + (a[2] + a[3]));
      m = mn;
      const unsigned at = (unsigned)(target - (col0 + cc));
      if (at < 32u && (int)at < left) {
        float z = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) z = at == j ? __uint_as_float(v[j]) : z;
        A.zt[row] = z * un;
      }
    }
  }
  __device__ __forceinline__ void tile(const Args& A, const Sched& S, const Tile& t, int64_t row, int half,
                                       uint32_t taddr) {
    blocks(A, S, t, row, half, FromTmem{taddr + half * (S.BN >> 1)});
  }
  __device__ __forceinline__ void store(const Args& A, const Sched& S, const Tile& t, int64_t row, int half) {
    blocks(A, S, t, row, half, FromSums{sum});
  }
  __device__ __forceinline__ void end(const Args& A, const Sched& S, int half) { flush(A, S, half); }
};

// Joins the partial (maximum, sum) pairs of a row, in slot order per lane and
// a fixed tree over the lanes.  One warp per row.
__global__ void __launch_bounds__(256) loss_join_kernel(const float2* __restrict__ part, const float* __restrict__ zt,
                                                        const int* __restrict__ targets, int64_t T, int V,
                                                        const __grid_constant__ Sched S, int rows_per_tile, int blocks,
                                                        int ignore,
                                                        float* __restrict__ loss, float* __restrict__ lse,
                                                        int* __restrict__ err) {
  allow_next();
  wait_previous();
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= T) return;
  int n = blocks;                      // one pair a block of the few-token kernel, else two a cluster
  if (n == 0) {
    const int mt = (int)(row / rows_per_tile), nt = S.prod[0].n_tiles;
    n = (S.owner(mt * nt + nt - 1) - S.owner(mt * nt) + 1) * 2;
  }
  float m = -INFINITY, s = 0.f;
  for (int i = lane; i < n; i += 32) {
    const float2 p = part[(int64_t)i * T + row];
    const float mn = fmaxf(m, p.x);
    const float ref = mn == -INFINITY ? 0.f : mn;
    s = s * exp2f((m - ref) * LOG2E) + p.y * exp2f((p.x - ref) * LOG2E);
    m = mn;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(FULL, m, o), s2 = __shfl_xor_sync(FULL, s, o);
    const float mn = fmaxf(m, m2);
    const float ref = mn == -INFINITY ? 0.f : mn;
    s = s * exp2f((m - ref) * LOG2E) + s2 * exp2f((m2 - ref) * LOG2E);
    m = mn;
  }
  if (lane == 0) {
    const float l = fmaf(log2f(s), LN2, m);
    lse[row] = l;
    const int t = targets[row];
    const bool in = t >= 0 && t < V;
    float x = 0.f;
    if (t != ignore) {
      x = in ? l - zt[row] : __int_as_float(0x7FC00000);
      if (!in) atomicCAS(err, 0, STATUS_TARGET);
    }
    loss[row] = x;
  }
}

// ---- few float32 tokens --------------------------------------------------------------
// Up to 24 float32 tokens: the weight is read once and everything else waits
// for it, while the two-piece form of the tensor cores would read it twice
// more.  A block takes 128 vocabulary entries, a thread one of them against
// four tokens (float32 FMAs, two columns an instruction); 64 columns of the
// block's rows at a time come through a ring of asynchronous copies, deep
// enough for all of a 256-wide row.  Over 16,384 entries of 256, on the device:
// 17 tokens 16.5 us instead of the 20.6 of pieces and tiles, 24 18.5 instead of
// 22.6, 32 22.6 instead of 20.8.
constexpr int FEW = 24, FEW_V = 128, FEW_K = 64, FEW_PITCH = FEW_K + 4, FEW_STAGES = 4, FEW_M = 4;

struct FewArgs {
  const float *h, *w;
  int64_t ldh, ldw;
  int T, V, d;
  const int* targets;
  float2* part;                        // [block][T]
  float* zt;
  int* err;
};

__device__ __forceinline__ void copy16(float* dst, const float* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::smem_u32(dst)), "l"(src), "r"(in ? 16 : 0)
               : "memory");
}

__global__ void __launch_bounds__(FEW_V * (FEW / FEW_M)) loss_few_kernel(FewArgs A) {
  extern __shared__ float4 few_raw[];
  float* ws = reinterpret_cast<float*>(few_raw);                       // [stages][128][68]
  float* hs = ws + FEW_STAGES * FEW_V * FEW_PITCH;                     // [tokens rounded up to 4][columns to 64]
  allow_next();
  wait_previous();
  const int t = threadIdx.x, nt = blockDim.x, v0 = blockIdx.x * FEW_V, chunks = (A.d + FEW_K - 1) / FEW_K;
  const int cols = chunks * FEW_K, tokens = nt / FEW_V * FEW_M;
  if (blockIdx.x == 0 && t == 0) *A.err = 0;
  auto fetch = [&](int c) {            // 16 lanes a row; zeros past the end
    if (c < chunks) {
      float* st = ws + (c % FEW_STAGES) * FEW_V * FEW_PITCH;
      const int col = c * FEW_K + (t & 15) * 4;
      for (int r = t >> 4; r < FEW_V; r += nt >> 4) {
        const bool in = v0 + r < A.V && col < A.d;
        copy16(st + r * FEW_PITCH + (t & 15) * 4, in ? A.w + (int64_t)(v0 + r) * A.ldw + col : A.w, in);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int e = t; e < tokens * (cols / 4); e += nt) {
    const int m = e / (cols / 4), k = (e - m * (cols / 4)) * 4;
    const bool in = m < A.T && k < A.d;
    copy16(hs + m * cols + k, in ? A.h + m * A.ldh + k : A.w, in);
  }
#pragma unroll
  for (int c = 0; c < FEW_STAGES - 1; ++c) fetch(c);                   // the tokens are in the first group
  const int r = t & (FEW_V - 1), m0 = t / FEW_V * FEW_M;               // a warp's tokens are the same
  unsigned long long acc[FEW_M] = {};                                  // (even columns, odd columns)
  for (int c = 0; c < chunks; ++c) {
    asm volatile("cp.async.wait_group %0;" ::"n"(FEW_STAGES - 2) : "memory");
    __syncthreads();                   // the chunk is in for every thread, the one before is read
    fetch(c + FEW_STAGES - 1);
    const ulonglong2* row =
        reinterpret_cast<const ulonglong2*>(ws + (c % FEW_STAGES) * FEW_V * FEW_PITCH + r * FEW_PITCH);
    const float* hk = hs + m0 * cols + c * FEW_K;
#pragma unroll
    for (int k4 = 0; k4 < FEW_K / 4; ++k4) {
      const ulonglong2 w = row[k4];
#pragma unroll
      for (int m = 0; m < FEW_M; ++m) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(hk + m * cols + k4 * 4);
        asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[m]) : "l"(w.x), "l"(x.x));
        asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[m]) : "l"(w.y), "l"(x.y));
      }
    }
  }
  // a token's 128 logits: one warp finds their maximum and sum
  __syncthreads();
  float* zs = ws;                      // [tokens][128]
#pragma unroll
  for (int m = 0; m < FEW_M; ++m) {
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(acc[m]));
    zs[(m0 + m) * FEW_V + r] = v0 + r < A.V ? a + b : -INFINITY;
  }
  __syncthreads();
  for (int m = t >> 5; m < A.T; m += nt >> 5) {
    const int lane = t & 31;
    float z[FEW_V / 32];
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < FEW_V / 32; ++i) {
      z[i] = zs[m * FEW_V + i * 32 + lane];
      mx = fmaxf(mx, z[i]);
    }
    mx = warp_max(mx);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < FEW_V / 32; ++i) s += g16::exp2_fast((z[i] - ref) * LOG2E);
    s = warp_sum(s);
    if (lane == 0) {
      A.part[(int64_t)blockIdx.x * A.T + m] = make_float2(mx, s);
      const unsigned at = (unsigned)(A.targets[m] - v0);
      if (at < FEW_V && v0 + (int)at < A.V) A.zt[m] = zs[m * FEW_V + at];
    }
  }
}

int few_threads(int64_t T) { return FEW_V * (int)((T + FEW_M - 1) / FEW_M); }

size_t few_smem(int64_t T, int d) {
  return (size_t)(FEW_STAGES * FEW_V * FEW_PITCH + up(T, FEW_M) * up(d, FEW_K)) * sizeof(float);
}

// Rows of 16-byte vectors, and the tokens fit beside the ring.
bool few_tokens(const memlayer_loss_config& c, const memlayer_loss_args& a) {
  auto rows16 = [](const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 4 == 0; };
  return c.dtype == MEMLAYER_F32 && c.tokens <= FEW && c.d_model % 4 == 0 && rows16(a.h, a.h_stride) &&
         rows16(a.weight, a.weight_stride) && few_smem(c.tokens, c.d_model) <= g16::SMEM_LIMIT;
}

// ---- backward ---------------------------------------------------------------------
struct GradArgs {
  int64_t T;
  int v0, vc;                          // the piece: columns [v0, v0 + vc)
  const unsigned* amax_w;
  const float* lse;
  const float4* token;                 // token_record
  CUtensorMap out[2];                  // dz: hi, lo
};

// dz as PIECES 16-bit matrices (hi, lo).
template <bool BF16, int PIECES, bool SUM>
struct EpiGrad {
  static constexpr bool kSum = SUM, kStore = true;
  float sum[128];
  using Args = GradArgs;
  uint32_t buf;
  int exp_w;
  StagingTurn turn;
  __device__ __forceinline__ void begin(const Args& A, const Sched&, int, uint8_t* staging) {
    buf = tc::smem_u32(staging);
    turn = StagingTurn{};
    exp_w = exp_of(A.amax_w);
  }
  template <class Get>
  __device__ __forceinline__ void blocks(const Args& A, const Sched& S, const Tile& t, int64_t row, int half,
                                         Get get) {
    // a warp whose 32 rows are past the last token has nothing to store, and
    // stages nothing: what it staged last may still be on its way
    if (row - (threadIdx.x & 31) >= A.T) return;
    float l = 0.f;
    float4 k = token_record(0.f, 0.f, -1, 0);
    if (row < A.T) {
      k = A.token[row];
      l = A.lse[row];
    }
    const float q = k.x, g = k.y, un = logit_unscale(__float_as_int(k.w), exp_w);
    const int tg = __float_as_int(k.z) - A.v0;
    const int hw = S.BN >> 1;
    const int col0 = t.nt * S.BN + half * hw;
#pragma unroll
    for (int cc = 0; cc < 128; cc += 32) {
      if (cc >= hw || col0 + cc >= A.vc) break;
      uint32_t v[32];
      __syncwarp();
      get(cc, v);
      float x[32];                     // p q, two columns an instruction where there is one
      const unsigned long long un2 = pair(un, un), nl2 = pair(-l, -l), log2e2 = pair(LOG2E, LOG2E), q2 = pair(q, q);
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        unsigned long long y = pair(__uint_as_float(v[j]), __uint_as_float(v[j + 1]));
        float a, b;
        asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(y) : "l"(un2), "l"(nl2));
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(y));
        y = pair(at_most_0(a), at_most_0(b));
        asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(y) : "l"(log2e2));
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(y));
        y = pair(g16::exp2_fast(a), g16::exp2_fast(b));
        asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(y) : "l"(q2));
        asm("mov.b64 {%0, %1}, %2;" : "=f"(x[j]), "=f"(x[j + 1]) : "l"(y));
      }
      const unsigned at = (unsigned)(tg - (col0 + cc));
      if (at < 32u) {
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = at == j ? x[j] - g : x[j];
      }
      if (q == 0.f && g == 0.f) {      // an ignored token: nothing, whatever its logits are
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = 0.f;
      }
      uint32_t h[16], o[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float a = x[2 * j], b = x[2 * j + 1];
        if constexpr (BF16) {
          const __nv_bfloat162 u = __floats2bfloat162_rn(a, b);
          h[j] = *reinterpret_cast<const uint32_t*>(&u);
          if constexpr (PIECES == 2) {
            const float2 f = __bfloat1622float2(u);
            const __nv_bfloat162 w = __floats2bfloat162_rn(a - f.x, b - f.y);
            o[j] = *reinterpret_cast<const uint32_t*>(&w);
          }
        } else if constexpr (PIECES == 2) {
          __half2 u, w;
          g16::split2(a, b, u, w);
          h[j] = *reinterpret_cast<const uint32_t*>(&u);
          o[j] = *reinterpret_cast<const uint32_t*>(&w);
        } else {
          const __half2 u = __floats2half2_rn(a, b);
          h[j] = *reinterpret_cast<const uint32_t*>(&u);
        }
      }
      const int lane = threadIdx.x & 31;
      if constexpr (PIECES == 2) {
        g16::store_pieces(A.out, buf, h, o, col0 + cc, (int)row, 0);   // lane 0 has the block's first row
      } else {                         // the halves of the staging buffer in turn
        const uint32_t b0 = g16::staging_place(turn, buf, false, true);
        g16::stage16(b0, lane, h);
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) g16::bulk_store(&A.out[0], b0, col0 + cc, (int)row, 0, false);
      }
    }
  }
  __device__ __forceinline__ void tile(const Args& A, const Sched& S, const Tile& t, int64_t row, int half,
                                       uint32_t taddr) {
    blocks(A, S, t, row, half, FromTmem{taddr + half * (S.BN >> 1)});
  }
  __device__ __forceinline__ void store(const Args& A, const Sched& S, const Tile& t, int64_t row, int half) {
    blocks(A, S, t, row, half, FromSums{sum});
  }
  __device__ __forceinline__ void end(const Args&, const Sched&, int) {}
};

// ---- gradient of few tokens ----------------------------------------------------------
// Up to 16 tokens of up to 1024 columns: the weight is read and its gradient
// written once, and the products are small enough for float32 FMAs.  A block
// takes 64 vocabulary entries at a time: a warp finds the logits of two of
// them (lanes along the columns), the block turns them into dz in shared
// memory, and a thread multiplies dz by its columns of h and of the weight
// (from L2 now): dW goes out, dh stays in registers over all of its entries.
// A second kernel adds the blocks' parts of dh in block order.  TM: tokens
// rounded up.
constexpr int FEWB = 16, FEWB_V = 64, FEWB_D = 1024, FEWB_T = 512;

// Groups of threads that share a block's entries where the columns leave threads over.
__host__ __device__ inline int few_groups(int d) {
  const int dp = (d + 31) / 32 * 32;
  return dp <= FEWB_T / 2 ? FEWB_T / dp : 1;
}

struct FewGradArgs {
  const void *h, *w;
  int64_t ldh, ldw;
  int T, V, d, ignore;
  const int* targets;
  const float *lse, *dloss, *dlse;
  void* dw;
  float* part;                         // [block][group][T][d]
  int* err;
};

template <typename E, int TM>
__global__ void __launch_bounds__(FEWB_T, TM <= 4 ? 2 : 1) loss_few_backward_kernel(const FewGradArgs A) {
  constexpr int COLS = FEWB_D / FEWB_T;
  extern __shared__ float4 few_raw[];
  float* dz = reinterpret_cast<float*>(few_raw);                       // [64][TM]
  float *q = dz + FEWB_V * TM, *g = q + TM, *l = g + TM;               // a token's factors and log sum
  int* tg = reinterpret_cast<int*>(l + TM);                            // and target (-1: none)
  float* hs = l + 2 * TM;                                              // [TM][d]
  allow_next();
  wait_previous();
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, d = A.d;
  const E *h = reinterpret_cast<const E*>(A.h), *w = reinterpret_cast<const E*>(A.w);
  E* dw = reinterpret_cast<E*>(A.dw);
  if (blockIdx.x == 0 && t == 0) *A.err = 0;
  __syncthreads();
  if (t < TM) {
    const int v = t < A.T ? A.targets[t] : A.ignore;
    const bool in = t < A.T && v >= 0 && v < A.V && v != A.ignore;
    if (t < A.T && !in && v != A.ignore && blockIdx.x == 0) atomicCAS(A.err, 0, STATUS_TARGET);
    g[t] = in ? A.dloss[t] : 0.f;
    q[t] = g[t] + (A.dlse && t < A.T ? A.dlse[t] : 0.f);
    l[t] = t < A.T ? A.lse[t] : 0.f;
    tg[t] = in ? v : -1;
  }
  __syncthreads();
  for (int e = t; e < TM * d; e += FEWB_T) {
    const int m = e / d;               // a token without a gradient: nothing, whatever its row holds
    hs[e] = m < A.T && !(q[m] == 0.f && g[m] == 0.f) ? to_f32(h[m * A.ldh + (e - m * d)]) : 0.f;
  }
  __syncthreads();
  const int groups = few_groups(d), width = groups > 1 ? (d + 31) / 32 * 32 : FEWB_T;
  const int group = groups > 1 ? t / width : 0, first = group < groups ? t - group * width : d;
  float hr[COLS][TM], acc[COLS][TM];
#pragma unroll
  for (int i = 0; i < COLS; ++i)
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      const int c = first + i * FEWB_T;
      hr[i][m] = c < d ? hs[m * d + c] : 0.f;
      acc[i][m] = 0.f;
    }
  const int tiles = (A.V - 1) / FEWB_V + 1;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int v0 = tile * FEWB_V, rows = min(FEWB_V, A.V - v0);
    for (int r = warp * 2; r < rows; r += FEWB_T / 32 * 2) {
      const E *w0 = w + (v0 + r) * A.ldw, *w1 = r + 1 < rows ? w0 + A.ldw : w0;
      float z[2][TM];
#pragma unroll
      for (int m = 0; m < TM; ++m) z[0][m] = z[1][m] = 0.f;
#pragma unroll 4
      for (int c = lane; c < d; c += 32) {
        const float a = to_f32(w0[c]), b = to_f32(w1[c]);
#pragma unroll
        for (int m = 0; m < TM; ++m) {
          const float x = hs[m * d + c];
          z[0][m] = fmaf(a, x, z[0][m]);
          z[1][m] = fmaf(b, x, z[1][m]);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int m = 0; m < TM; ++m) {
          const float x = warp_sum(z[i][m]);
          if (lane == 0) dz[(r + i) * TM + m] = x;      // r is even: inside the 64 rows
        }
    }
    __syncthreads();
    for (int e = t; e < rows * TM; e += FEWB_T) {
      const int m = e % TM, v = v0 + e / TM;
      float x = g16::exp2_fast(at_most_0(dz[e] - l[m]) * LOG2E) * q[m];
      if (tg[m] == v) x -= g[m];
      dz[e] = q[m] == 0.f && g[m] == 0.f ? 0.f : x;     // an ignored token: nothing, whatever its logits are
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < COLS; ++i) {
      const int c = first + i * FEWB_T;
      if (c >= d) break;
      const E* wc = w + v0 * A.ldw + c;
      E* dc = dw + (int64_t)v0 * d + c;
      auto entry = [&](int r) {
        const float x = to_f32(wc[r * A.ldw]);
        float o = 0.f;
#pragma unroll
        for (int m = 0; m < TM; ++m) {
          const float y = dz[r * TM + m];
          o = fmaf(y, hr[i][m], o);
          acc[i][m] = fmaf(y, x, acc[i][m]);
        }
        dc[(int64_t)r * d] = from_f32<E>(o);
      };
      if (groups == 1) {               // unrolled for its loads; with a stride between them it took 1.4 times as long
#pragma unroll 8
        for (int r = 0; r < rows; ++r) entry(r);
      } else {
#pragma unroll 4
        for (int r = group; r < rows; r += groups) entry(r);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < COLS; ++i) {
    const int c = first + i * FEWB_T;
    if (c >= d) break;
#pragma unroll
    for (int m = 0; m < TM; ++m)
      if (m < A.T) A.part[(((int64_t)blockIdx.x * groups + group) * A.T + m) * d + c] = acc[i][m];
  }
}

// out = the blocks' parts [blocks][n] added in block order: 32 groups of
// blocks an entry, then the groups in a fixed tree.
template <typename E>
__global__ void __launch_bounds__(1024) loss_few_dh_kernel(const float* __restrict__ part, int blocks, int n,
                                                           E* __restrict__ out) {
  __shared__ float red[32][33];
  allow_next();
  wait_previous();
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5, j = blockIdx.x * 32 + c;
  float x = 0.f;
  if (j < n) {
#pragma unroll 4
    for (int b = g; b < blocks; b += 32) x += part[(int64_t)b * n + j];
  }
  red[g][c] = x;
  __syncthreads();
  const float s = warp_sum(red[c][g]);
  if (c == 0 && blockIdx.x * 32 + g < n) out[blockIdx.x * 32 + g] = from_f32<E>(s);
}

// 16-bit tensor cores are ahead of more than four tokens where a block would
// take several times 64 entries (8 x 512 over 30,000 bf16 43 us for 50, 16 x
// 1024 over 32,768 72 for 169), and behind elsewhere: 5 x 112 over 7,933 bf16
// 25 for 14, 3 x 290 over 49,237 111 for 43, 4 x 856 over 10,146 float32 71
// for 33, 16 x 256 over 16,384 49 for 35.
bool few_backward(const memlayer_loss_config& c) {
  return c.tokens <= FEWB && c.d_model <= FEWB_D &&
         (c.tokens <= 4 || c.dtype == MEMLAYER_F32 || c.vocab_size <= FEWB_V * g16::device_sms());
}

int few_backward_blocks(const memlayer_loss_config& c) {
  const int most = g16::device_sms() * (c.tokens <= 4 ? 2 : 1), tiles = (c.vocab_size - 1) / FEWB_V + 1;
  return tiles < most ? tiles : most;
}

template <typename E, int TM>
cudaError_t launch_few_backward(const FewGradArgs& a, int blocks, void* dh, cudaStream_t s) {
  auto kern = loss_few_backward_kernel<E, TM>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = g16::allow_smem(reinterpret_cast<const void*>(kern), &done);
  if (e != cudaSuccess) return e;
  count_launch(2);
  e = launch_dependent(kern, dim3((unsigned)blocks), FEWB_T, (size_t)TM * (FEWB_V + 4 + a.d) * sizeof(float), s, a);
  if (e != cudaSuccess) return e;
  const int n = a.T * a.d;
  return launch_dependent(loss_few_dh_kernel<E>, dim3((unsigned)((n + 31) / 32)), 1024, 0, s, (const float*)a.part,
                          blocks * few_groups(a.d), n, reinterpret_cast<E*>(dh));
}

template <typename E>
cudaError_t few_backward_of(const FewGradArgs& a, int blocks, void* dh, cudaStream_t s) {
  if (a.T <= 4) return launch_few_backward<E, 4>(a, blocks, dh, s);
  if (a.T <= 8) return launch_few_backward<E, 8>(a, blocks, dh, s);
  return launch_few_backward<E, FEWB>(a, blocks, dh, s);
}

struct OutOne {
  CUtensorMap map;                     // out as staged stores write it (tma)
  int64_t M;
  int N;
  int64_t ld, slice;                   // slice: elements between the slices' partials
  void* out;
  int type;                            // memlayer_dtype of out
  int add;                             // float32 only: added to what is there
  int tma;                             // rows are 16 bytes apart
  // scales of the operands (null: none): dz's by row (dh), dW's common one, the weight's
  const int* exp_g;
  const unsigned *peak, *amax_w;
};
struct OutArgs { OutOne o[2]; };

// Plain outputs: out[row, col] = acc unscaled (+ what is there), float32 or
// the 16-bit type; slices write float32 partials.
template <bool SUM>
struct EpiOut {
  static constexpr bool kSum = SUM, kStore = true;
  using Args = OutArgs;
  float sum[128];                      // the thread's columns over the segments of k
  uint32_t buf;
  StagingTurn turn;                    // a cluster may have float32 partials of dh and 16-bit blocks of dW
  __device__ __forceinline__ void begin(const Args&, const Sched&, int, uint8_t* staging) {
    buf = tc::smem_u32(staging);
    turn = StagingTurn{};
  }
  // The warp's 32 rows x 32 columns.
  __device__ __forceinline__ void block(const OutOne& O, uint32_t (&v)[32], const g16::Unscale& un, int64_t row0,
                                        int col, int ks) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(un(__uint_as_float(v[j])));
    const uint32_t b = g16::staging_place(turn, buf, O.type == MEMLAYER_F32, O.tma);
    g16::stage_as(O.type, b, lane, v);
    if (O.tma) {
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) g16::bulk_store(&O.map, b, col, (int)row0, ks, O.add);
    } else {
      __syncwarp();
      g16::copy_rows(O.type, b, O.out, ks * O.slice + row0 * O.ld + col, O.ld,
                     (int)(O.M - row0 < 32 ? O.M - row0 : 32), O.N - col, O.add);
      __syncwarp();
    }
  }
  template <class Get>
  __device__ __forceinline__ void blocks(const Args& A, const Sched& S, const Tile& t, int64_t row, int half,
                                         Get get) {
    const OutOne& O = A.o[t.q];
    const g16::Unscale un(-(O.exp_g && row < O.M ? O.exp_g[row] : 0) - (O.peak ? piece_exp(*O.peak) : 0) - exp_of(O.amax_w));
    const int64_t row0 = row - (threadIdx.x & 31);
    const int hw = S.BN >> 1;
    const int col0 = t.nt * S.BN + half * hw;
#pragma unroll
    for (int cc = 0; cc < 128; cc += 32) {
      if (cc >= hw || col0 + cc >= O.N) break;
      uint32_t v[32];
      __syncwarp();
      get(cc, v);
      if (row0 < O.M) block(O, v, un, row0, col0 + cc, t.ks);
    }
  }
  __device__ __forceinline__ void tile(const Args& A, const Sched& S, const Tile& t, int64_t row, int half,
                                       uint32_t taddr) {
    blocks(A, S, t, row, half, FromTmem{taddr + half * (S.BN >> 1)});
  }
  __device__ __forceinline__ void store(const Args& A, const Sched& S, const Tile& t, int64_t row, int half) {
    blocks(A, S, t, row, half, FromSums{sum});
  }
  __device__ __forceinline__ void end(const Args&, const Sched&, int) {}
};

// out = the slices' partials added in slice order, in the storage type; four
// entries a thread (both buffers come 256-byte aligned or are written one by one).
__global__ void __launch_bounds__(256) loss_slices_kernel(const float* __restrict__ P, int S, int64_t n, void* out,
                                                          int type, int vec) {
  allow_next();
  wait_previous();
  auto put = [&](int64_t e, float x) {
    if (type == MEMLAYER_F32)
      reinterpret_cast<float*>(out)[e] = x;
    else if (type == MEMLAYER_F16)
      reinterpret_cast<__half*>(out)[e] = __float2half_rn(x);
    else
      reinterpret_cast<__nv_bfloat16*>(out)[e] = __float2bfloat16_rn(x);
  };
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
  if (vec) {
    for (int64_t e = at * 4; e < n; e += step * 4) {
      float4 x = *reinterpret_cast<const float4*>(P + e);
      for (int s = 1; s < S; ++s) {
        const float4 y = *reinterpret_cast<const float4*>(P + s * n + e);
        x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
      }
      if (type == MEMLAYER_F32) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + e) = x;
      } else {
        uint2 o;
        if (type == MEMLAYER_F16) {
          const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
          o = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        } else {
          const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
          o = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        }
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + e) = o;
      }
    }
  } else {
    for (int64_t e = at; e < n; e += step) {
      float x = P[e];
      for (int s = 1; s < S; ++s) x += P[s * n + e];
      put(e, x);
    }
  }
}

cudaError_t launch_slices(const float* P, int S, int64_t n, void* out, int type, cudaStream_t s) {
  const int vec = n % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  const int64_t items = vec ? n / 4 : n;
  int64_t blocks = (items + 255) / 256;
  const int64_t cap = 8 * g16::device_sms();
  if (blocks > cap) blocks = cap;
  count_launch();
  return launch_dependent(loss_slices_kernel, dim3((unsigned)blocks), 256, 0, s, P, S, n, out, type, vec);
}

// ---- plan -----------------------------------------------------------------------
struct Plan {
  int P, PZ;                           // pieces of h and W, of dz
  int cg, BN;                          // CTAs per tile; columns per tile of the logits
  int m_tiles, n_tiles;
  int slots;                           // partial pairs per row and column half
  int64_t ld;                          // row pitch of the 16-bit forms
  int vc;                              // columns of a vocabulary piece = row pitch of its dz
  int oBN, oNB;                        // columns per tile of the gradient products, tiles at once
  int s_h, s_w;                        // k slices of dh and of dW
  size_t o_hh, o_hl, o_eh, o_h2, o_wh, o_wl, o_part, o_zt, o_token, o_tgt, o_exp, o_g, o_g2, o_dh, o_dw, bytes;
};

constexpr size_t O_ERR = 256, O_AMAX = 512, HEAD = 1024;
enum { AMAX_W, PEAK };                 // words from O_AMAX on

// 16-bit matrices TMA can address: rows 16 bytes apart, 16-byte base.
bool tma_rows(const void* p, int64_t stride) { return stride % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int64_t kPieceBytes = 256ll << 20;   // dz of one vocabulary piece

Prod product(int64_t m_tiles, int64_t n_tiles, int splits, int64_t k, bool amn, bool bmn) {
  Prod p{};
  p.m_tiles = (int)m_tiles;
  p.n_tiles = (int)n_tiles;
  p.batch = 1;
  p.kq_total = (int)(up(k, g16::BK) / g16::BK);
  p.kq = (p.kq_total + splits - 1) / splits;
  p.splits = (p.kq_total + p.kq - 1) / p.kq;   // no empty slice
  p.amn = amn;
  p.bmn = bmn;
  return p;
}

// The two products of a piece of vc columns, the one with the longer tiles
// first; returns which place dh has.
int out_products(const Plan& p, int64_t T, int64_t vc, int64_t d, Sched* S) {
  const int rt = 128 * p.cg;
  const int64_t nd = up(d, p.oBN * p.oNB) / (p.oBN * p.oNB);
  const Prod w = product(up(vc, rt) / rt, nd, p.s_w, T, true, true);
  const Prod h = product(up(T, rt) / rt, nd, p.s_h, vc, false, true);
  const int at = h.kq > w.kq ? 0 : 1;
  S->prod[at] = h;
  S->prod[1 - at] = w;
  S->BN = p.oBN;
  S->seg = SEG;
  return at;
}

// Columns per piece and slices of k.
void piece_plan(int64_t T, int64_t V, int64_t d, int sms, Plan* p) {
  int64_t most = kPieceBytes / (2 * p->PZ) / (T ? T : 1);
  if (most < 256) most = 256;
  const int64_t n = (V + most - 1) / most;
  p->vc = (int)up((V + n - 1) / n, 256);
  const int rt = 128 * p->cg;
  const int64_t nd = up(d, p->oBN * p->oNB) / (p->oBN * p->oNB), kh = up(p->vc, 64) / 64, kw = up(T, 64) / 64;
  const double ideal = (double)(up(T, rt) / rt * nd * kh + up(p->vc, rt) / rt * nd * kw) / (sms / p->cg);
  const double cap = ideal * 1.25 < 16 ? 16 : ideal * 1.25;
  p->s_h = kh > cap ? (int)(kh / cap + 0.999) : 1;
  p->s_w = kw > cap ? (int)(kw / cap + 0.999) : 1;
}

bool plan(const memlayer_loss_config& c, bool backward, Plan* out) {
  Plan p{};
  const int64_t T = c.tokens, V = c.vocab_size, d = c.d_model;
  const bool f32 = c.dtype == MEMLAYER_F32;
  const int sms = g16::device_sms();
  p.P = f32 ? 2 : 1;
  // 16-bit dz rounds once more than the results; up to 128 tokens, where the
  // products wait for memory, a second piece makes it exact enough for free
  p.PZ = f32 || T <= 128 ? 2 : 1;
  p.cg = T > 128 ? 2 : 1;
  p.BN = p.cg == 2 ? 256 : 128;
  const int64_t mt = up(T, 128 * p.cg) / (128 * p.cg), nt = up(V, p.BN) / p.BN;
  if (mt * nt >= (1ll << 31)) return false;
  p.m_tiles = (int)mt;
  p.n_tiles = (int)nt;
  const int64_t total = mt * nt, cl = total < sms / p.cg ? total : sms / p.cg;
  const int64_t per = cl ? total / cl : 1;
  p.slots = (int)((nt + per - 1) / (per ? per : 1) + 1);
  p.ld = up(d, 8);
  size_t off = HEAD;
  auto take = [&](int64_t bytes) {
    const size_t o = off;
    off += (size_t)up(bytes, 256);
    return o;
  };
  if (backward && few_backward(c)) {
    p.o_dh = take((int64_t)few_backward_blocks(c) * few_groups(c.d_model) * T * d * 4);
    p.bytes = off;
    *out = p;
    return true;
  }
  // room for the 16-bit forms whether or not this call's strides need them
  p.o_hh = take(T * p.ld * 2);
  p.o_wh = take(V * p.ld * 2);
  if (f32) {
    p.o_hl = take(T * p.ld * 2);
    p.o_wl = take(V * p.ld * 2);
    if (!backward) p.o_eh = take(T * 4);
  }
  if (!backward) {
    const int64_t few = f32 && T <= FEW ? up(V, FEW_V) / FEW_V * T * 8 : 0, part = (int64_t)p.slots * 2 * T * 8;
    p.o_part = take(few > part ? few : part);
    p.o_zt = take(T * 4);
  } else {
    p.o_token = take(T * 16);
    p.o_tgt = take(T * 4);
    p.o_exp = take(T * 4);
    p.o_h2 = take(p.P * T * p.ld * 2);   // hi, lo
    p.oBN = d > 128 ? 256 : 128;
    // 16-bit products with an even number of column tiles take two at once:
    // 8192 x 1024 x 32768 bf16 791 us instead of 956, 1999 x 512 x 30011 f16
    // 100 instead of 124 (an odd one would multiply by columns that are not there)
    p.oNB = p.cg == 2 && p.PZ == 1 && up(d, 256) / 256 % 2 == 0 ? 2 : 1;
    piece_plan(T, V, d, sms, &p);
    p.o_g = take(T * p.vc * 2);
    if (p.PZ == 2) p.o_g2 = take(T * p.vc * 2);
    p.o_dh = take((int64_t)p.s_h * T * d * 4);
    p.o_dw = p.s_w > 1 ? take((int64_t)p.s_w * p.vc * d * 4) : 0;
  }
  p.bytes = off;
  *out = p;
  return true;
}

struct Operands {
  const void *h[2], *w[2], *h2[2];     // h2: dW's, a row every p.ld
  int64_t ldh, ldw;
};

#define LS_TRY(x)                             \
  do {                                        \
    const cudaError_t e_ = (x);               \
    if (e_ != cudaSuccess) return e_;         \
  } while (0)

// Operands in 16-bit form: the caller's where TMA can address them, else the
// workspace's.  g: the gradient's arguments, whose tokens it looks through (null: none).
cudaError_t prepare(const memlayer_loss_config& c, const memlayer_loss_args& a, const memlayer_loss_grads* g,
                    const Plan& p, char* ws, Operands* o, cudaStream_t s) {
  unsigned* amax = reinterpret_cast<unsigned*>(ws + O_AMAX);
  const bool f32 = c.dtype == MEMLAYER_F32;
  o->h[0] = a.h;
  o->w[0] = a.weight;
  o->ldh = a.h_stride;
  o->ldw = a.weight_stride;
  PiecesArgs B{};
  if (f32 || !tma_rows(a.weight, a.weight_stride)) {
    o->w[0] = ws + p.o_wh;
    o->w[1] = ws + p.o_wl;
    o->ldw = p.ld;
    B.m[0] = {a.weight, c.vocab_size, c.d_model, a.weight_stride, ws + p.o_wh, ws + p.o_wl, p.ld, amax + AMAX_W};
  }
  if (f32 || !tma_rows(a.h, a.h_stride)) {
    o->h[0] = ws + p.o_hh;
    o->h[1] = ws + p.o_hl;
    o->ldh = p.ld;
    if (!f32) B.m[1] = {a.h, c.tokens, c.d_model, a.h_stride, ws + p.o_hh, nullptr, p.ld};
  }
  const bool scaled = c.dtype != MEMLAYER_BF16;        // dz carries scales
  TokenArgs ta{{}, a.h, c.tokens, a.h_stride, p.ld, c.d_model, 0, (__half*)(ws + p.o_hh), (__half*)(ws + p.o_hl)};
  int *tgt = reinterpret_cast<int*>(ws + p.o_tgt), *exp_g = reinterpret_cast<int*>(ws + p.o_exp);
  if (f32) ta.w = {(const float*)a.weight, c.vocab_size, c.d_model, a.weight_stride, amax + AMAX_W, 0};
  if (g) {
    ta.targets = a.targets;
    ta.dloss = g->dloss;
    ta.dlse = g->dlse;
    ta.V = c.vocab_size;
    ta.ignore = c.ignore_index;
    ta.token = reinterpret_cast<float4*>(ws + p.o_token);
    ta.tgt = tgt;
    ta.exp_g = exp_g;
    ta.peak = amax + PEAK;
    ta.err = reinterpret_cast<int*>(ws + O_ERR);
  } else {
    ta.exp_h = reinterpret_cast<int*>(ws + p.o_eh);
  }
  if (f32)
    LS_TRY(launch_tokens<float>(ta, s));
  else if (g)
    LS_TRY(scaled ? launch_tokens<__half>(ta, s) : launch_tokens<__nv_bfloat16>(ta, s));
  if (g) {
    char *hi = ws + p.o_h2, *lo = hi + c.tokens * p.ld * 2;
    o->h2[0] = hi;
    o->h2[1] = lo;
    B.m[2] = {a.h, c.tokens, c.d_model, a.h_stride, hi, lo, p.ld, nullptr, tgt, scaled ? exp_g : nullptr,
              scaled ? amax + PEAK : nullptr};
  }
  return launch_pieces(B, c.dtype, s);
}

template <class EPI, int PA, int PB>
cudaError_t launch(int cg, const Maps& m, const Sched& S, const typename EPI::Args& ea, int* err, cudaStream_t s) {
  return cg == 2 ? g16::launch_one<EPI, 2, PA, PB>(m, S, ea, err, s)
                 : g16::launch_one<EPI, 1, PA, PB>(m, S, ea, err, s);
}

}  // namespace

bool loss_workspace(const memlayer_loss_config& c, bool backward, size_t* bytes) {
  Plan p;
  if (!plan(c, backward, &p)) return false;
  *bytes = p.bytes;
  return true;
}

cudaError_t launch_loss_forward(const memlayer_loss_config& c, const memlayer_loss_args& a, char* ws, cudaStream_t s) {
  Plan p;
  if (!plan(c, false, &p)) return cudaErrorInvalidValue;
  int* err = reinterpret_cast<int*>(ws + O_ERR);
  if (c.tokens > 0 && few_tokens(c, a)) {
    FewArgs f{(const float*)a.h, (const float*)a.weight, a.h_stride, a.weight_stride, (int)c.tokens, c.vocab_size,
              c.d_model, a.targets, reinterpret_cast<float2*>(ws + p.o_part), reinterpret_cast<float*>(ws + p.o_zt),
              err};
    static std::atomic<uint64_t> done{0};
    LS_TRY(g16::allow_smem(reinterpret_cast<const void*>(loss_few_kernel), &done));
    const int blocks = (c.vocab_size + FEW_V - 1) / FEW_V;
    count_launch(2);
    LS_TRY(launch_dependent(loss_few_kernel, dim3((unsigned)blocks), few_threads(c.tokens),
                            few_smem(c.tokens, c.d_model), s, f));
    return launch_dependent(loss_join_kernel, dim3((unsigned)((c.tokens + 7) / 8)), 256, 0, s, (const float2*)f.part,
                            (const float*)f.zt, a.targets, c.tokens, c.vocab_size, Sched{}, 1, blocks, c.ignore_index,
                            a.loss, a.lse, err);
  }
  LS_TRY(cudaMemsetAsync(ws + O_ERR, 0, HEAD - O_ERR, s));
  if (c.tokens == 0) return cudaSuccess;
  Operands o{};
  LS_TRY(prepare(c, a, nullptr, p, ws, &o, s));
  const int bf16 = c.dtype == MEMLAYER_BF16;
  Maps m{};
  for (int i = 0; i < p.P; ++i) {
    LS_TRY(g16::make_operand(&m.a[0][i], o.h[i], c.tokens, c.d_model, o.ldh, false, 128, bf16));
    LS_TRY(g16::make_operand(&m.b[0][i], o.w[i], c.vocab_size, c.d_model, o.ldw, false, p.BN / p.cg, bf16));
  }
  Sched S{};
  const int sms = g16::device_sms() / p.cg;
  S.prod[0] = product(p.m_tiles, p.n_tiles, 1, c.d_model, false, false);
  S.contiguous = 1;
  S.clusters = sms < S.prod[0].total() ? sms : S.prod[0].total();
  S.BN = p.BN;
  S.bf16 = bf16;
  const bool f32 = c.dtype == MEMLAYER_F32;
  StatsArgs ea{};
  ea.T = c.tokens;
  ea.V = c.vocab_size;
  ea.exp_h = f32 ? reinterpret_cast<int*>(ws + p.o_eh) : nullptr;
  ea.amax_w = f32 ? reinterpret_cast<unsigned*>(ws + O_AMAX) + AMAX_W : nullptr;
  ea.targets = a.targets;
  ea.part = reinterpret_cast<float2*>(ws + p.o_part);
  ea.zt = reinterpret_cast<float*>(ws + p.o_zt);
  S.seg = LOGIT_SEG;
  const bool sum = S.prod[0].kq > LOGIT_SEG;
  if (p.P == 1)
    LS_TRY((launch<EpiStats<false>, 1, 1>(p.cg, m, S, ea, err, s)));
  else if (sum)
    LS_TRY((launch<EpiStats<true>, 2, 2>(p.cg, m, S, ea, err, s)));
  else
    LS_TRY((launch<EpiStats<false>, 2, 2>(p.cg, m, S, ea, err, s)));
  count_launch();
  return launch_dependent(loss_join_kernel, dim3((unsigned)((c.tokens + 7) / 8)), 256, 0, s, (const float2*)ea.part,
                          (const float*)ea.zt, a.targets, c.tokens, c.vocab_size, S, 128 * p.cg, 0, c.ignore_index,
                          a.loss, a.lse, err);
}

cudaError_t launch_loss_backward(const memlayer_loss_config& c, const memlayer_loss_args& a,
                                 const memlayer_loss_grads& g, char* ws, cudaStream_t s) {
  Plan p;
  if (!plan(c, true, &p)) return cudaErrorInvalidValue;
  int* err = reinterpret_cast<int*>(ws + O_ERR);
  const int64_t T = c.tokens, V = c.vocab_size, d = c.d_model;
  if (T > 0 && few_backward(c)) {
    const FewGradArgs f{a.h, a.weight, a.h_stride, a.weight_stride, (int)T, c.vocab_size, c.d_model, c.ignore_index,
                        a.targets, g.lse, g.dloss, g.dlse, g.dweight, reinterpret_cast<float*>(ws + p.o_dh), err};
    const int blocks = few_backward_blocks(c);
    return c.dtype == MEMLAYER_F32   ? few_backward_of<float>(f, blocks, g.dh, s)
           : c.dtype == MEMLAYER_F16 ? few_backward_of<__half>(f, blocks, g.dh, s)
                                     : few_backward_of<__nv_bfloat16>(f, blocks, g.dh, s);
  }
  LS_TRY(cudaMemsetAsync(ws + O_ERR, 0, HEAD - O_ERR, s));
  const size_t esize = c.dtype == MEMLAYER_F32 ? 4 : 2;
  if (T == 0) return cudaMemsetAsync(g.dweight, 0, (size_t)V * d * esize, s);
  Operands o{};
  LS_TRY(prepare(c, a, &g, p, ws, &o, s));
  unsigned* words = reinterpret_cast<unsigned*>(ws + O_AMAX);
  const bool f32 = c.dtype == MEMLAYER_F32;
  const int bf16 = c.dtype == MEMLAYER_BF16;
  const unsigned *aw = f32 ? words + AMAX_W : nullptr, *peak = bf16 ? nullptr : words + PEAK;
  const int* exp_g = bf16 ? nullptr : reinterpret_cast<int*>(ws + p.o_exp);
  const float4* token = reinterpret_cast<float4*>(ws + p.o_token);
  uint16_t *gh = reinterpret_cast<uint16_t*>(ws + p.o_g), *gl = reinterpret_cast<uint16_t*>(ws + p.o_g2);
  float* acc_h = reinterpret_cast<float*>(ws + p.o_dh);
  const int sms = g16::device_sms() / p.cg;
  const int pieces = (int)((V + p.vc - 1) / p.vc);
  // dh in place when it needs no joining: one slice, and float32 or one piece
  const bool direct_h = p.s_h == 1 && (f32 || pieces == 1);
  auto al16 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  for (int i = 0; i < pieces; ++i) {
    const int v0 = i * p.vc;
    const int vc = (int)(V - v0 < p.vc ? V - v0 : p.vc);
    const int64_t woff = (int64_t)v0 * o.ldw * 2;
    // dz of the piece
    Maps m{};
    for (int q = 0; q < p.P; ++q) {
      LS_TRY(g16::make_operand(&m.a[0][q], o.h[q], T, d, o.ldh, false, 128, bf16));
      LS_TRY(g16::make_operand(&m.b[0][q], (const char*)o.w[q] + woff, vc, d, o.ldw, false, p.BN / p.cg, bf16));
    }
    Sched S{};
    S.prod[0] = product(p.m_tiles, (vc + p.BN - 1) / p.BN, 1, d, false, false);
    S.BN = p.BN;
    S.bf16 = bf16;
    g16::distribute(&S, sms, 0);
    GradArgs ga{T, v0, vc, aw, g.lse, token, {}};
    LS_TRY(g16::make_store(&ga.out[0], gh, T, p.vc, p.vc, f32 ? MEMLAYER_F16 : c.dtype));
    if (p.PZ == 2) LS_TRY(g16::make_store(&ga.out[1], gl, T, p.vc, p.vc, f32 ? MEMLAYER_F16 : c.dtype));
    S.seg = LOGIT_SEG;
    if (f32 && S.prod[0].kq > LOGIT_SEG)
      LS_TRY((launch<EpiGrad<false, 2, true>, 2, 2>(p.cg, m, S, ga, err, s)));
    else if (f32)
      LS_TRY((launch<EpiGrad<false, 2, false>, 2, 2>(p.cg, m, S, ga, err, s)));
    else if (bf16)
      LS_TRY(p.PZ == 2 ? (g16::launch_one<EpiGrad<true, 2, false>, 1, 1, 1>(m, S, ga, err, s))
                       : (g16::launch_one<EpiGrad<true, 1, false>, 2, 1, 1>(m, S, ga, err, s)));
    else
      LS_TRY(p.PZ == 2 ? (g16::launch_one<EpiGrad<false, 2, false>, 1, 1, 1>(m, S, ga, err, s))
                       : (g16::launch_one<EpiGrad<false, 1, false>, 2, 1, 1>(m, S, ga, err, s)));
    // dW of the piece = dz^T h; dh (+)= dz W of the piece
    Sched S2{};
    const int qh = out_products(p, T, vc, d, &S2), qw = 1 - qh;
    S2.bf16 = bf16;
    g16::distribute(&S2, sms, 2);
    Maps m2{};
    const uint16_t* gz[2] = {gh, gl};
    for (int q = 0; q < p.PZ; ++q) {
      LS_TRY(g16::make_operand(&m2.a[qw][q], gz[q], vc, T, p.vc, true, 0, bf16));
      LS_TRY(g16::make_operand(&m2.a[qh][q], gz[q], T, vc, p.vc, false, 128, bf16));
    }
    for (int q = 0; q < p.P; ++q) {
      LS_TRY(g16::make_operand(&m2.b[qw][q], o.h2[q], d, T, p.ld, true, 0, bf16));
      LS_TRY(g16::make_operand(&m2.b[qh][q], (const char*)o.w[q] + woff, d, vc, o.ldw, true, 0, bf16));
    }
    const int sw = S2.prod[qw].splits, sh = S2.prod[qh].splits;
    char* dwp = (char*)g.dweight + (size_t)v0 * d * esize;
    OutArgs ea{};
    auto out = [&](OutOne& O, int64_t M, void* q, int type, bool add, int slices, bool is_dh) {
      O.M = M;
      O.N = (int)d;
      O.ld = d;
      O.slice = M * d;
      O.out = q;
      O.type = type;
      O.add = add;
      O.tma = al16(q) && (d * (type == MEMLAYER_F32 ? 4 : 2)) % 16 == 0;
      O.exp_g = is_dh ? exp_g : nullptr;
      O.peak = is_dh ? nullptr : peak;
      O.amax_w = is_dh ? aw : nullptr;
      return O.tma ? g16::make_store(&O.map, q, M, d, d, type, slices, M * d) : cudaSuccess;
    };
    if (sw > 1)
      LS_TRY(out(ea.o[qw], vc, ws + p.o_dw, MEMLAYER_F32, false, sw, false));
    else
      LS_TRY(out(ea.o[qw], vc, dwp, c.dtype, false, 1, false));
    if (direct_h)
      LS_TRY(out(ea.o[qh], T, g.dh, c.dtype, i > 0, 1, true));
    else   // a shorter last piece may have fewer slices: the others keep what they hold
      LS_TRY(out(ea.o[qh], T, acc_h, MEMLAYER_F32, i > 0, sh, true));
    if (f32)
      LS_TRY((launch<EpiOut<true>, 2, 2>(p.cg, m2, S2, ea, err, s)));
    else
      LS_TRY(p.PZ == 2    ? (g16::launch_one<EpiOut<false>, 1, 2, 1>(m2, S2, ea, err, s))
             : p.oNB == 2 ? (g16::launch_one<EpiOut<false>, 2, 1, 1, 2>(m2, S2, ea, err, s))
                          : (g16::launch_one<EpiOut<false>, 2, 1, 1>(m2, S2, ea, err, s)));
    if (sw > 1)
      LS_TRY(launch_slices(reinterpret_cast<float*>(ws + p.o_dw), sw, (int64_t)vc * d, dwp, c.dtype, s));
    if (i == 0) p.s_h = sh;            // slices of the first (largest) piece
  }
  if (!direct_h) LS_TRY(launch_slices(acc_h, p.s_h, T * d, g.dh, c.dtype, s));
  return cudaSuccess;
}

}  // namespace ml
