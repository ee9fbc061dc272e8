// Host side of the 16-bit tensor-core GEMM (gemm16.cuh) and the kernel that
// puts its operands into 16-bit form: float32 matrices split into f16 pieces,
// 16-bit matrices whose rows TMA cannot address copied.
#include <cudaTypedefs.h>

#include <atomic>
#include <mutex>

#include "gemm16.cuh"

#include "pieces16.cuh"

namespace ml {

namespace {

constexpr int NTH = PIECE_THREADS;

// 8 columns a thread: hi / lo pieces of x s (float32 source) or a copy
// (16-bit source; scaled: f16), zeros in the padding columns.
template <typename E>
__global__ void __launch_bounds__(NTH) pieces_kernel(PiecesArgs A) {
  allow_next();
  wait_previous();
  int i = 0, b = blockIdx.x;
  while (b >= A.m[i].blocks) b -= A.m[i++].blocks;
  const PiecesMat M = A.m[i];
  const int c8 = (int)(M.ld >> 3);
  const int64_t n = M.rows * c8;
  const E* src = reinterpret_cast<const E*>(M.x);
  const int e0 = M.peak ? piece_exp(*M.peak) : sizeof(E) == 4 && M.amax ? g16::scale_exp(*M.amax) : 0;
  constexpr int V = 16 / sizeof(E);
  struct alignas(16) Vec { E e[V]; };
  const bool vec = M.pitch % V == 0 && (reinterpret_cast<uintptr_t>(M.x) & 15) == 0;
  for (int64_t e = (int64_t)b * NTH + threadIdx.x; e < n; e += (int64_t)M.blocks * NTH) {
    const int64_t r = e / c8;
    const int c = (int)(e - r * c8) * 8;
    const E* p = src + r * M.pitch + c;
    alignas(16) E v[8];
    if (M.row_tgt && M.row_tgt[r] == PIECE_SKIP) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = E(0);
    } else if (vec && c + 8 <= M.cols) {
#pragma unroll
      for (int j = 0; j < 8; j += V) *reinterpret_cast<Vec*>(v + j) = *reinterpret_cast<const Vec*>(p + j);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < M.cols ? p[j] : E(0);
    }
    const g16::Unscale sc(M.row_exp ? e0 - M.row_exp[r] : e0);
    if constexpr (sizeof(E) == 4) {
      __half2 h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) g16::split2(sc(v[2 * j]), sc(v[2 * j + 1]), h[j], l[j]);
      *reinterpret_cast<uint4*>(reinterpret_cast<__half*>(M.hi) + r * M.ld + c) = *reinterpret_cast<uint4*>(h);
      *reinterpret_cast<uint4*>(reinterpret_cast<__half*>(M.lo) + r * M.ld + c) = *reinterpret_cast<uint4*>(l);
    } else {
      if (M.row_exp) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __half_as_ushort(__float2half_rn(sc(__half2float(__ushort_as_half(v[j])))));
      }
      *reinterpret_cast<uint4*>(reinterpret_cast<E*>(M.hi) + r * M.ld + c) = *reinterpret_cast<uint4*>(v);
    }
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode16_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

}  // namespace

namespace g16 {

int device_sms() {
  static std::atomic<int> known[64];       // by device; 0: not asked yet
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;   // sizes can be asked for without a GPU
  if (dev < 64 && (sms = known[dev].load(std::memory_order_relaxed))) return sms;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  if (dev < 64) known[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

cudaError_t allow_smem(const void* kernel, std::atomic<uint64_t>* done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit && (done->load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_LIMIT);
  if (e == cudaSuccess) done->fetch_or(bit, std::memory_order_relaxed);
  return e;
}

cudaError_t make_operand(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int64_t pitch, bool mn,
                         int box_rows, int bf16, int batch, int64_t bstride) {
  auto enc = encode16_fn();
  if (!enc) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)(mn ? rows : k), (cuuint64_t)(mn ? k : rows), (cuuint64_t)batch};
  const cuuint64_t strides[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)(batch > 1 ? bstride : pitch * dims[1]) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)(mn ? 64 : box_rows), 1}, one[3] = {1, 1, 1};
  const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                         const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t make_store(CUtensorMap* map, void* base, int64_t rows, int64_t cols, int64_t pitch, int dtype, int64_t z,
                       int64_t zstride) {
  auto enc = encode16_fn();
  if (!enc) return cudaErrorNotSupported;
  const bool f32 = dtype == MEMLAYER_F32;
  const cuuint64_t es = f32 ? 4 : 2;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)z};
  const cuuint64_t strides[2] = {pitch * es, (cuuint64_t)(z > 1 ? zstride : pitch * rows) * es};
  const cuuint32_t box[3] = {32, 32, 1}, one[3] = {1, 1, 1};
  const CUresult r =
      enc(map,
          f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
              : dtype == MEMLAYER_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
          3, base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
          f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

double distribute(Sched* S, int most, double over) {
  const int n0 = S->prod[0].total(), n1 = S->prod[1].total();
  int C = n0 + n1 < most ? n0 + n1 : most;
  if (C < 1) C = 1;
  S->clusters = C;
  S->q = n0 / C;
  S->r = n0 % C;
  S->x[0] = S->x[1] = S->e[0] = S->e[1] = 0;
  const double c0 = S->prod[0].kq + over, c1 = S->prod[1].kq + over;
  double load[2] = {(S->q + 1) * c0, S->q * c0};
  const int size[2] = {S->r, C - S->r};
  int left = n1;
  while (left > 0) {                       // a round of the less loaded group at a time
    const int g = size[0] > 0 && load[0] < load[1] ? 0 : 1;
    load[g] += c1;
    if (left >= size[g]) {
      S->x[g]++;
      left -= size[g];
    } else {
      S->e[g] = left;
      left = 0;
    }
  }
  return size[0] > 0 && load[0] > load[1] ? load[0] : load[1];
}

}  // namespace g16

cudaError_t launch_pieces(PiecesArgs A, int dtype, cudaStream_t s) {
  int total = 0;
  for (PiecesMat& M : A.m) {
    const int64_t n = M.rows * (M.ld >> 3);
    M.blocks = n ? piece_blocks(n, 2) : 0;
    total += M.blocks;
  }
  if (!total) return cudaSuccess;
  count_launch();
  // 16-bit sources: their bits as they are
  return dtype == MEMLAYER_F32 ? launch_dependent(pieces_kernel<float>, dim3(total), NTH, 0, s, A)
                               : launch_dependent(pieces_kernel<unsigned short>, dim3(total), NTH, 0, s, A);
}

}  // namespace ml
