// Persistent 16-bit tensor-core GEMM with exchangeable epilogues: the products
// of the vocabulary cross entropy (loss.cu) and of the orthogonalised update
// (orth.cu).
//
//   acc[i, j] = sum_k A(i, k) B(j, k)   in float32 TMEM accumulators
//
// An operand is one 16-bit matrix, or two (PA, PB = 2): the float32 matrix
// x s (s a power of two) as hi = f16(x s), lo = f16(x s - hi), 22 bits of it;
// then the product is hi.hi + hi.lo + lo.hi -- the dropped lo.lo is below
// 2^-22 -- at three 16-bit products, half the tensor time of the 3xTF32
// split (kind::tf32 runs at half the 16-bit rate).  The f16 range does for
// float32 data because s puts the largest entry at 2^14..2^15: entries down
// to 2^-18 of it keep all 22 bits, smaller ones an absolute error of 2^-40
// of it.
//
// The tensor cores add into TMEM by truncation: an entry loses up to one unit
// of its last place per 16-k step, always towards zero.  Over a k of
// thousands that is 1e-5 (measured: dh of a 9,000-entry vocabulary 2.4e-5
// off), too much for a float32 result.  So of a stage's two-piece products
// the small ones go first, while the accumulator is small, and epilogues that
// ask for it (kSum) get k in segments of S.seg stages, which they add in
// registers, rounding to nearest.
//
// Each operand is read as stored, by TMA with the 128-byte swizzle: K-major
// (k contiguous) or MN-major (the row index contiguous).  Rows past the end
// and the tail of k read as zeros.  z: independent products (batch).
//
// CTA = 12 warps: warps 0-7 epilogue (TMEM lane = output row; the two warps
// of a lane quarter take half of the columns each), warp 8 TMA producer, warp
// 9 MMA issuer, two idle ones that complete its warpgroup.  CG = 2 pairs two SMs on a 256-row tile: each CTA stages
// its own 128 rows of A and half of the rows of B, the leader issues for
// both, and each CTA drains its own 128 rows.  Accumulators are
// double-buffered in TMEM, so an epilogue runs beside the next tile's MMAs.
// NB = 2 takes two column tiles at once instead, an accumulator each: A is
// staged once for both.  TMA brings an SM 32 to 39 bytes a cycle whatever is
// asked of it (the bound of 16-bit products: 47 instead of 62 bytes a cycle at
// the tensor cores' full rate), and over a long k the drain that nothing
// overlaps is a few percent.
// Every mbarrier wait is bounded.
#pragma once

#include <atomic>

#include "dependent.cuh"
#include "staging_turn.cuh"
#include "tc_common.cuh"

namespace ml {
namespace g16 {

constexpr int THREADS = 384;
constexpr int EPI_WARPS = 8;
constexpr int BK = 64;                    // k elements per stage: 128-byte rows
constexpr int MAX_STAGES = 8;
constexpr uint32_t STAGING = 2 * STAGING_HALF;   // an epilogue warp's 32 rows x 128 bytes
constexpr uint32_t CTL_BYTES = 1024;
constexpr uint32_t SMEM_LIMIT = 227 * 1024;

struct Ctl {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], tfull[2], tempty[2];
  uint32_t tmem_base;
  int abort;
};

struct Maps {
  CUtensorMap a[2][2], b[2][2];           // [product of the launch][hi / lo]
};

struct Tile {
  int q, z, mt, nt, ks;                   // q: product of the launch
};

// One product: its tiles, cut into `splits` slices of kq BK-element stages.
struct Prod {
  int m_tiles, n_tiles, splits, batch;
  int kq, kq_total;
  uint32_t amn, bmn;                      // operand is MN-major
  int tri;                                // a symmetric result: only the tiles mt >= nt (square tiles)
  __host__ __device__ int tiles() const { return tri ? m_tiles * (m_tiles + 1) / 2 : m_tiles * n_tiles; }
  __host__ __device__ int total() const { return tiles() * splits * batch; }
};

// The tiles of one launch, over `clusters` clusters (CTAs or pairs).
// contiguous (one product, one slice): cluster c takes an equal run of the
// tiles, column tile fastest -- for an epilogue that keeps state along a row
// block.  Otherwise the first product's tiles go round the clusters, row
// tile fastest (neighbouring clusters share B), and the second product's,
// which are no longer than the first's, fill the clusters up to a common
// level in runs: the first `r` clusters, which have one long tile more, take
// x[0] each, the others x[1], and the first e[g] of a group one more.
struct Sched {
  Prod prod[2];
  int clusters, contiguous;
  int q, r, x[2], e[2];
  int BN;                                 // columns per tile (MMA N)
  int seg;                                // stages per segment (kSum)
  int stages;
  uint32_t bf16;                          // operand type
  // Where the contiguous run of cluster c begins.
  __host__ __device__ int first(int c) const { return (int)((int64_t)prod[0].total() * c / clusters); }
  // The cluster whose contiguous run holds tile `lin`.
  __host__ __device__ int owner(int lin) const {
    const int64_t n = prod[0].total();
    return (int)((((int64_t)lin + 1) * clusters + n - 1) / n) - 1;
  }
  __device__ __forceinline__ int count(int c) const {
    if (contiguous) return first(c + 1) - first(c);
    if (c >= clusters) return 0;
    const int g = c < r ? 0 : 1, i = g ? c - r : c;
    return q + (c < r) + x[g] + (i < e[g]);
  }
  __device__ __forceinline__ Tile tile(int c, int i) const {
    Tile t;
    if (contiguous) {
      const int lin = first(c) + i;
      t.mt = lin / prod[0].n_tiles;
      t.nt = lin - t.mt * prod[0].n_tiles;
      t.q = t.ks = t.z = 0;
      return t;
    }
    const int own = q + (c < r);
    int lin = c + i * clusters;
    t.q = 0;
    if (i >= own) {
      const int g = c < r ? 0 : 1, j = g ? c - r : c;
      lin = (g ? r * x[0] + e[0] : 0) + j * x[g] + min(j, e[g]) + (i - own);
      t.q = 1;
    }
    const Prod& p = prod[t.q];
    const int at = lin % p.tiles();
    lin /= p.tiles();
    if (p.tri) {
      int r = (int)((sqrtf(8.f * at + 1.f) - 1.f) * 0.5f);
      while ((r + 1) * (r + 2) / 2 <= at) ++r;
      while (r * (r + 1) / 2 > at) --r;
      t.mt = r;
      t.nt = at - r * (r + 1) / 2;
    } else {
      t.mt = at % p.m_tiles;
      t.nt = at / p.m_tiles;
    }
    t.ks = lin % p.splits;
    t.z = lin / p.splits;
    return t;
  }
  __device__ __forceinline__ int stages_of(const Tile& t) const {
    const int rem = prod[t.q].kq_total - t.ks * prod[t.q].kq;
    return rem < prod[t.q].kq ? rem : prod[t.q].kq;
  }
};

// Fills in the distribution over at most `most` clusters; the cost of a tile
// is its stages plus `over`.  Returns the largest cluster's cost.
double distribute(Sched* S, int most, double over);

// ---- PTX pieces ----------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ uint32_t map_to_cta(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// bar: a shared::cluster address (CG = 2: the leader's barrier).
template <int CG>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
        "%4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
        "[%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Arrives on the barrier (of both CTAs of a pair) once the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            tc::smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    tc::mma_commit(bar);
}

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t cols) {
  if constexpr (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(dst)),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tc::tmem_alloc(dst, cols);
  }
}

template <int CG>
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
  else
    tc::tmem_dealloc(addr, cols);
}

// Descriptor of an MN-major tile: 64 rows (128 bytes) x 64 k per block, each
// block 8 KB of 128-byte k rows in 1024-byte swizzle atoms of 8 k.  Leading
// byte offset: block to block along the row index; stride byte offset: atom
// to atom along k.
__device__ __forceinline__ uint64_t sdesc_mn_sw128(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// Instruction descriptor of kind::f16: D float32, A and B both f16 or both
// bf16, each K-major or MN-major.
__device__ __forceinline__ uint32_t idesc_16(int M, int N, uint32_t bf16, uint32_t amn, uint32_t bmn) {
  return (1u << 4) | (bf16 << 7) | (bf16 << 10) | (amn << 15) | (bmn << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// 2^x (ex2.approx: 2 ulp).
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// ---- staged stores ---------------------------------------------------------------
// An epilogue thread holds a row; a warp's stores straight from registers
// would touch 32 rows each.  Instead a warp writes 32 rows x 32 columns into
// its staging buffer (swizzled as the tensor map says) and one thread hands
// the block to a bulk tensor store, which clips it at the matrix's edges.
template <int N, bool READ>
__device__ __forceinline__ void bulk_wait() {
  if constexpr (READ)
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
  else
    asm volatile("cp.async.bulk.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void bulk_store(const CUtensorMap* map, uint32_t src, int x, int y, int z, bool add) {
  if (add)
    asm volatile(
        "cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
            reinterpret_cast<uint64_t>(map)),
        "r"(src), "r"(x), "r"(y), "r"(z)
        : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(src), "r"(x), "r"(y), "r"(z)
                 : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// The place of the warp's next staged block, free to be written (staging_turn.cuh).
__device__ __forceinline__ uint32_t staging_place(StagingTurn& turn, uint32_t buf, bool wide, bool bulk) {
  const StagingTurn::Place p = turn.next(wide, bulk);
  if ((threadIdx.x & 31) == 0) {
    if (p.stand)
      bulk_wait<1, true>();
    else
      bulk_wait<0, true>();
  }
  __syncwarp();
  return buf + p.offset;
}

__device__ __forceinline__ void st_shared16(uint32_t at, uint32_t a) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"((uint16_t)a) : "memory");
}

__device__ __forceinline__ void st_shared(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// The calling lane's row of 32 16-bit values (64 bytes, 64-byte swizzle) /
// of 32 floats (128 bytes, 128-byte swizzle).
__device__ __forceinline__ void stage16(uint32_t buf, int lane, const uint32_t (&h)[16]) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    st_shared(buf + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4), h[4 * c], h[4 * c + 1], h[4 * c + 2], h[4 * c + 3]);
}
__device__ __forceinline__ void stage32(uint32_t buf, int lane, const uint32_t (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    st_shared(buf + lane * 128 + ((c ^ (lane & 7)) << 4), v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
}
// Entry (row, column) of a staged block.
__device__ __forceinline__ uint32_t at16(uint32_t buf, int r, int c) {
  return buf + r * 64 + (((c >> 3) ^ ((r >> 1) & 3)) << 4) + (c & 7) * 2;
}
__device__ __forceinline__ uint32_t at32(uint32_t buf, int r, int c) {
  return buf + r * 128 + (((c >> 2) ^ (r & 7)) << 4) + (c & 3) * 4;
}

// The calling lane's row of 32 16-bit values as a column of the block (its transpose).
__device__ __forceinline__ void stage16_transposed(uint32_t buf, int lane, const uint32_t (&h)[16]) {
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    st_shared16(at16(buf, 2 * c, lane), h[c]);
    st_shared16(at16(buf, 2 * c + 1, lane), h[c] >> 16);
  }
}

// The calling lane's row of 32 float32 values staged in the output's type.
__device__ __forceinline__ void stage_as(int dtype, uint32_t buf, int lane, const uint32_t (&v)[32]) {
  if (dtype == MEMLAYER_F32) {
    stage32(buf, lane, v);
    return;
  }
  uint32_t h[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float x = __uint_as_float(v[2 * j]), y = __uint_as_float(v[2 * j + 1]);
    if (dtype == MEMLAYER_BF16) {
      const __nv_bfloat162 u = __floats2bfloat162_rn(x, y);
      h[j] = *reinterpret_cast<const uint32_t*>(&u);
    } else {
      const __half2 u = __floats2half2_rn(x, y);
      h[j] = *reinterpret_cast<const uint32_t*>(&u);
    }
  }
  stage16(buf, lane, h);
}

// A staged block to rows that TMA cannot address: a row per pass, a column
// per lane; `at`: the block's first entry, `rows` x `cols` of it inside.
__device__ __forceinline__ void copy_rows(int dtype, uint32_t buf, void* out, int64_t at, int64_t ld, int rows,
                                          int cols, bool add) {
  const int lane = threadIdx.x & 31;
  if (lane >= cols) return;
  for (int r0 = 0; r0 < rows; r0 += 8) {   // eight loads in flight
    if (dtype == MEMLAYER_F32) {
      float* p = reinterpret_cast<float*>(out) + at + r0 * ld + lane;
      float old[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) old[r] = add && r0 + r < rows ? p[r * ld] : 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        float x;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at32(buf, r0 + r, lane)) : "memory");
        if (r0 + r < rows) p[r * ld] = old[r] + x;
      }
    } else {
      uint16_t* p = reinterpret_cast<uint16_t*>(out) + at + r0 * ld + lane;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        uint16_t x;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(at16(buf, r0 + r, lane)) : "memory");
        if (r0 + r < rows) p[r * ld] = x;
      }
    }
  }
}

// The warp's block of two matrices of 16-bit pieces (hi, lo), a half of the
// staging buffer each, or its transpose.  One proxy fence for both: fences
// are most of what a small product's stores take.
__device__ __forceinline__ void store_pieces(const CUtensorMap* map, uint32_t buf, const uint32_t (&h)[16],
                                             const uint32_t (&l)[16], int x, int y, int z,
                                             bool transposed = false) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) bulk_wait<0, true>();
  __syncwarp();
  if (transposed) {
    stage16_transposed(buf, lane, h);
    stage16_transposed(buf + 2048, lane, l);
  } else {
    stage16(buf, lane, h);
    stage16(buf + 2048, lane, l);
  }
  tc::fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    bulk_store(map, buf, x, y, z, false);
    bulk_store(map + 1, buf + 2048, x, y, z, false);
  }
}

// A segment's columns (32, 64 or 128) added to a thread's sums.  They have to
// stay in registers (hence the redistribution of the CTA's): spilled, a
// segment's drain took 4,000 to 6,000 cycles instead of 700.
__device__ __forceinline__ void add_segment(uint32_t taddr, float (&sum)[128], int cols, int sg) {
#pragma unroll
  for (int c = 0; c < 128; c += 64) {
    if (c >= cols) break;
    uint32_t v[32], w[32];
    tc::tmem_ld32(taddr + c, v);
    tc::tmem_ld32(taddr + (cols > 32 ? c + 32 : c), w);
    tc::tmem_wait_ld();
    if (sg == 0) {
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        sum[c + j] = __uint_as_float(v[j]);
        sum[c + 32 + j] = __uint_as_float(w[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        sum[c + j] += __uint_as_float(v[j]);
        sum[c + 32 + j] += __uint_as_float(w[j]);
      }
    }
  }
}

// ---- power-of-two scales ---------------------------------------------------------
// amax: the float bits of the largest finite magnitude (0: no entry or all
// zero).  scale_of puts it in [2^14, 2^15); the exponent is clamped so that
// both the scale and its inverse are normal floats.
__device__ __forceinline__ int scale_exp(unsigned amax) {
  if (amax == 0) return 0;
  const int e = (int)(amax >> 23) - 127;   // a subnormal maximum counts as 2^-127
  const int s = 14 - e;
  return s > 126 ? 126 : s;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ float scale_of(const unsigned* amax) { return amax ? pow2(scale_exp(*amax)) : 1.0f; }

// x 2^e of a product's accumulator, e beyond one float's exponent range too.
struct Unscale {
  float a, b;
  __device__ __forceinline__ explicit Unscale(int e) {
    const int e1 = max(-126, min(127, e));
    a = pow2(e1);
    b = pow2(max(-126, min(127, e - e1)));
  }
  __device__ __forceinline__ float operator()(float x) const { return x * a * b; }
};

// ---- the kernel --------------------------------------------------------------------
__host__ __device__ inline uint32_t a_bytes() { return 128 * 128; }                  // one piece, one stage, one CTA
__host__ __device__ inline uint32_t b_bytes(int BN, int cg) { return (uint32_t)(BN / cg) * 128; }

// What a CTA's roles share.
struct Cta {
  Ctl* ctl;
  uint8_t* ring;
  volatile int* abort;
  int* err;
  uint32_t rank, stage_bytes, tmem_base;
  int cluster, stages;
};

// Positions in the stage ring and between the two accumulators, kept by each role.
struct RingPos {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++s == stages) {
      s = 0;
      ph ^= 1;
    }
  }
};
struct AccPos {
  int acc = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    acc ^= 1;
    if (acc == 0) ph ^= 1;
  }
};

// Barriers and TMEM; all threads call.
template <int CG, int PA, int PB, int NB>
__device__ __forceinline__ Cta begin_cta(uint8_t* smem_raw, int BN, int stages, int* err) {
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Cta c;
  c.ctl = reinterpret_cast<Ctl*>(smem);
  c.ring = smem + CTL_BYTES;
  c.abort = &c.ctl->abort;
  c.err = err;
  c.rank = CG == 2 ? cluster_rank() : 0;
  c.stage_bytes = PA * a_bytes() + NB * PB * b_bytes(BN, CG);
  c.cluster = blockIdx.x / CG;
  c.stages = stages;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      tc::mbar_init(&c.ctl->full[s], 1);
      tc::mbar_init(&c.ctl->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(&c.ctl->tfull[b], 1);
      tc::mbar_init(&c.ctl->tempty[b], CG * EPI_WARPS);
    }
    c.ctl->abort = 0;
    tc::fence_mbar_init();
  }
  if (threadIdx.x >> 5 == 9) tmem_alloc<CG>(&c.ctl->tmem_base, 512);
  tc::fence_before_sync();
  if constexpr (CG == 2)
    cluster_sync();
  else
    __syncthreads();
  tc::fence_after_sync();
  c.tmem_base = c.ctl->tmem_base;
  return c;
}

template <int CG>
__device__ __forceinline__ void end_cta(const Cta& c) {
  __syncwarp();
  tc::fence_before_sync();
  if constexpr (CG == 2)
    cluster_sync();
  else
    __syncthreads();
  if (threadIdx.x >> 5 == 9) {
    tc::fence_after_sync();
    tmem_dealloc<CG>(c.tmem_base, 512);
  }
}

// Epilogue warps: the cluster's tiles of one product.
template <class EPI, int CG, int NB>
__device__ __forceinline__ bool drain(const Cta& c, EPI& epi, const typename EPI::Args& ea, const Sched& S, AccPos& at) {
  constexpr bool SUM = EPI::kSum;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp & 3, half = warp >> 2;
  const int cnt = S.count(c.cluster);
  uint32_t tempty[2];
  for (int b = 0; b < 2; ++b) {
    tempty[b] = tc::smem_u32(&c.ctl->tempty[b]);
    if constexpr (CG == 2) tempty[b] = map_to_cta(tempty[b], 0);
  }
  for (int i = 0; i < cnt; ++i) {
    Tile t = S.tile(c.cluster, i);
    const int64_t row = (int64_t)t.mt * (128 * CG) + c.rank * 128 + quarter * 32 + lane;
    const int nseg = SUM ? (S.stages_of(t) + S.seg - 1) / S.seg : NB;
    t.nt *= NB;
    for (int sg = 0; sg < nseg; ++sg) {    // segments of k, or the column tiles
      if (!__all_sync(FULL, tc::mbar_wait(&c.ctl->tfull[at.acc], at.ph, c.abort, c.err, 15))) return false;
      tc::fence_after_sync();
      const uint32_t taddr = c.tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(at.acc * 256);
      if constexpr (SUM)
        add_segment(taddr + half * (S.BN >> 1), epi.sum, S.BN >> 1, sg);
      else
        epi.tile(ea, S, t, row, half, taddr);
      if constexpr (!SUM) ++t.nt;
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2)
          arrive_cluster(tempty[at.acc]);
        else
          tc::mbar_arrive(&c.ctl->tempty[at.acc]);
      }
      if constexpr (SUM) {                 // the accumulator is free before the stores
        if (sg == nseg - 1) epi.store(ea, S, t, row, half);
      }
      at.next();
    }
  }
  return true;
}

// Producer (one thread): the stages of the cluster's tiles.
template <int CG, int PA, int PB, int NB>
__device__ __forceinline__ bool produce(const Cta& c, const Maps& maps, const Sched& S, RingPos& at) {
  const uint32_t ab = a_bytes(), bb = b_bytes(S.BN, CG);
  const int cnt = S.count(c.cluster);
  for (int i = 0; i < cnt; ++i) {
    const Tile t = S.tile(c.cluster, i);
    const int nk = S.stages_of(t);
    const uint32_t amn = S.prod[t.q].amn, bmn = S.prod[t.q].bmn;
    const int ar = t.mt * (128 * CG) + (int)c.rank * 128;
    const int br = t.nt * NB * S.BN + (int)c.rank * (S.BN / CG);
    for (int kc = 0; kc < nk; ++kc) {
      if (!tc::mbar_wait(&c.ctl->empty[at.s], at.ph ^ 1, c.abort, c.err, 11)) return false;
      const int k = (t.ks * S.prod[t.q].kq + kc) * BK;
      const uint32_t st = tc::smem_u32(c.ring + (size_t)at.s * c.stage_bytes);
      if (c.rank == 0) tc::mbar_expect_tx(&c.ctl->full[at.s], CG * c.stage_bytes);
      uint32_t bar = tc::smem_u32(&c.ctl->full[at.s]);
      if constexpr (CG == 2) bar = map_to_cta(bar, 0);
#pragma unroll
      for (int p = 0; p < PA; ++p) {
        const uint32_t da = st + p * ab;
        const CUtensorMap* ma = &maps.a[t.q][p];
        if (amn) {
          tma_load_3d<CG>(da, ma, bar, ar, k, t.z);
          tma_load_3d<CG>(da + 8192, ma, bar, ar + 64, k, t.z);
        } else {
          tma_load_3d<CG>(da, ma, bar, k, ar, t.z);
        }
      }
#pragma unroll
      for (int p = 0; p < NB * PB; ++p) {  // the column tiles' pieces
        const uint32_t db = st + PA * ab + p * bb;
        const CUtensorMap* mb = &maps.b[t.q][p % PB];
        const int r = br + p / PB * S.BN;
        if (bmn) {
          for (int n = 0; n < S.BN / CG; n += 64) tma_load_3d<CG>(db + (n >> 6) * 8192, mb, bar, r + n, k, t.z);
        } else {
          tma_load_3d<CG>(db, mb, bar, k, r, t.z);
        }
      }
      at.next(c.stages);
    }
  }
  return true;
}

// Producer, at the end: every stage read (in a pair: the leader's arrivals on
// this CTA's barriers are in); after a wait that gave up, time for the copies
// in flight to land.
__device__ __forceinline__ void finish_producing(const Cta& c, bool ok, RingPos& at) {
  for (int j = 0; j < c.stages && ok; ++j) {
    ok = tc::mbar_wait(&c.ctl->empty[at.s], at.ph ^ 1, c.abort, c.err, 11);
    at.next(c.stages);
  }
  if (!ok) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000) {}    // about a millisecond
  }
}

__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// MMA issuer (a whole warp, of the leader in a pair): every lane walks the
// tiles, one issues.  The operands are then the same in every lane for the
// compiler, too, and stay in uniform registers, where the instruction wants
// them; issued by one lane of a divergent branch, twelve MMAs took 1,100 to
// 1,750 cycles whatever their size.
template <int CG, int PA, int PB, int NB, bool SUM>
__device__ __forceinline__ bool issue(const Cta& c, const Sched& S, RingPos& at, AccPos& ac) {
  const uint32_t ab = a_bytes() >> 4, bb = b_bytes(S.BN, CG) >> 4;
  const uint32_t ring = tc::smem_u32(c.ring);
  const int cnt = S.count(c.cluster);
  const bool one = elect_one();
  for (int i = 0; i < cnt; ++i) {
    const Tile t = S.tile(c.cluster, i);
    const int nk = S.stages_of(t);
    const uint32_t amn = S.prod[t.q].amn, bmn = S.prod[t.q].bmn;
    const uint32_t idesc = idesc_16(128 * CG, S.BN, S.bf16, amn, bmn);
    // 16 k: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major block
    const uint32_t astep = amn ? 2048 >> 4 : 32 >> 4, bstep = bmn ? 2048 >> 4 : 32 >> 4;
    const uint64_t adesc = amn ? sdesc_mn_sw128(0) : tc::sdesc_k_sw128(0);
    const uint64_t bdesc = bmn ? sdesc_mn_sw128(0) : tc::sdesc_k_sw128(0);
    const int nseg = SUM ? (nk + S.seg - 1) / S.seg : 1;
    for (int sg = 0; sg < nseg; ++sg) {
      if (NB == 1) {
        if (!__all_sync(FULL, tc::mbar_wait(&c.ctl->tempty[ac.acc], ac.ph ^ 1, c.abort, c.err, 12))) return false;
        tc::fence_after_sync();
      }
      const int kc0 = nk * sg / nseg, kc1 = nk * (sg + 1) / nseg;
      for (int kc = kc0; kc < kc1; ++kc) {
        if (!__all_sync(FULL, tc::mbar_wait(&c.ctl->full[at.s], at.ph, c.abort, c.err, 13))) return false;
        tc::fence_after_sync();
        // descriptors hold addresses in 16 bytes, 14 bits of them; the steps stay inside
        const uint32_t sa = ((ring + at.s * c.stage_bytes) >> 4) & 0x3FFF, sb = sa + PA * ab;
        const uint64_t a0 = adesc + sa;
        const uint32_t more = kc > kc0;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          if (NB == 2 && kc == kc0) {      // each column tile waits for its own accumulator
            if (!__all_sync(FULL, tc::mbar_wait(&c.ctl->tempty[nb], ac.ph ^ 1, c.abort, c.err, 12))) return false;
            tc::fence_after_sync();
          }
          const uint32_t d = c.tmem_base + (uint32_t)((NB == 2 ? nb : ac.acc) * 256);
          const uint64_t b0 = bdesc + sb + nb * PB * bb;
          if (one) {
            if constexpr (PA == 2) {
#pragma unroll
              for (int k16 = 0; k16 < BK / 16; ++k16)
                mma_f16<CG>(d, a0 + ab + k16 * astep, b0 + k16 * bstep, idesc, k16 ? 1 : more);
            }
            if constexpr (PB == 2) {
#pragma unroll
              for (int k16 = 0; k16 < BK / 16; ++k16)
                mma_f16<CG>(d, a0 + k16 * astep, b0 + bb + k16 * bstep, idesc, k16 || PA == 2 ? 1 : more);
            }
#pragma unroll
            for (int k16 = 0; k16 < BK / 16; ++k16)
              mma_f16<CG>(d, a0 + k16 * astep, b0 + k16 * bstep, idesc, k16 || PA + PB > 2 ? 1 : more);
            if (nb == NB - 1) commit<CG>(&c.ctl->empty[at.s]);
            if (kc == kc1 - 1) commit<CG>(&c.ctl->tfull[NB == 2 ? nb : ac.acc]);
          }
        }
        __syncwarp();
        at.next(c.stages);
      }
      ac.next();
      if (NB == 2) ac.next();
    }
  }
  return true;
}

template <int PA, int PB>
__device__ __forceinline__ void prefetch(const Maps& maps, const Sched& S) {
  for (int q = 0; q < 2 && S.prod[q].m_tiles > 0; ++q)
    for (int p = 0; p < 2; ++p) {
      if (p < PA) tc::prefetch_tmap(&maps.a[q][p]);
      if (p < PB) tc::prefetch_tmap(&maps.b[q][p]);
    }
}

// kSum keeps 128 sums a thread: 384 x 168 registers dealt out again, 256 x 224
// + 128 x 56.
template <bool SUM>
__device__ __forceinline__ void more_registers() {
  if constexpr (SUM) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
}
template <bool SUM>
__device__ __forceinline__ void fewer_registers() {
  if constexpr (SUM) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
}

template <class EPI, int CG, int PA, int PB, int NB>
__global__ void __launch_bounds__(THREADS, 1)
    gemm16_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Sched S,
                  const __grid_constant__ typename EPI::Args ea, int* err) {
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cta c = begin_cta<CG, PA, PB, NB>(smem_raw, S.BN, S.stages, err);
  allow_next();
  wait_previous();
  if (warp < EPI_WARPS) {
    more_registers<EPI::kSum>();
    EPI epi;
    AccPos at;
    epi.begin(ea, S, c.cluster, c.ring + (size_t)c.stages * c.stage_bytes + warp * STAGING);
    drain<EPI, CG, NB>(c, epi, ea, S, at);
    epi.end(ea, S, warp >> 2);
    if constexpr (EPI::kStore) {
      if (lane == 0) bulk_wait<0, false>();   // the stores are done with the staging buffers
    }
  } else {
    fewer_registers<EPI::kSum>();
    if (warp == 8 && lane == 0) {
      prefetch<PA, PB>(maps, S);
      RingPos at;
      const bool ok = produce<CG, PA, PB, NB>(c, maps, S, at);
      finish_producing(c, ok, at);
    } else if (warp == 9 && c.rank == 0) {
      RingPos at;
      AccPos ac;
      issue<CG, PA, PB, NB, EPI::kSum>(c, S, at, ac);
    }
  }
  end_cta<CG>(c);
}

// ---- host side -------------------------------------------------------------------
// One 16-bit operand: rows x k (per batch), K-major (row pitch `pitch`) or
// MN-major (k rows of `pitch` elements).  pitch and bstride in elements,
// multiples of 8; base 16-byte aligned.  box_rows: rows staged per CTA.
cudaError_t make_operand(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int64_t pitch, bool mn,
                         int box_rows, int bf16, int batch = 1, int64_t bstride = 0);

// A matrix written by staged stores: rows x cols of 16-bit or float32
// entries, row pitch in elements (rows 16 bytes apart), z of them.
cudaError_t make_store(CUtensorMap* map, void* base, int64_t rows, int64_t cols, int64_t pitch, int dtype,
                       int64_t z = 1, int64_t zstride = 0);

inline uint32_t stage_size(int BN, int cg, int pa, int pb, int nb) {
  return pa * a_bytes() + nb * pb * b_bytes(BN, cg);
}

inline int smem_stages(int BN, int cg, int pa, int pb, int nb, bool store) {
  const int n = (int)((SMEM_LIMIT - 1024 - CTL_BYTES - (store ? EPI_WARPS * STAGING : 0)) / stage_size(BN, cg, pa, pb, nb));
  return n > MAX_STAGES ? MAX_STAGES : n;
}

int device_sms();
// Lets `kernel` use all of an SM's shared memory, once per device (`done`: its devices so far).
cudaError_t allow_smem(const void* kernel, std::atomic<uint64_t>* done);

template <class EPI, int CG, int PA, int PB, int NB = 1>
cudaError_t launch_one(const Maps& maps, Sched S, const typename EPI::Args& ea, int* err, cudaStream_t s) {
  static_assert(NB == 1 || !EPI::kSum, "segments use both accumulators");
  S.stages = smem_stages(S.BN, CG, PA, PB, NB, EPI::kStore);
  const size_t smem = 1024 + CTL_BYTES + (size_t)S.stages * stage_size(S.BN, CG, PA, PB, NB) +
                      (EPI::kStore ? EPI_WARPS * STAGING : 0);
  auto kern = gemm16_kernel<EPI, CG, PA, PB, NB>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), &done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(S.clusters * CG);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, kern, maps, S, ea, err);
  count_launch();
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace g16
}  // namespace ml
