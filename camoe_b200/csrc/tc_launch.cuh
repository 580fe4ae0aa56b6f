// Host side of tc_gemm.cuh: tensor maps, grid and launch.
#pragma once

#include <atomic>

#include "tc_gemm.cuh"

namespace camoe {
namespace tm {
int status(cudaError_t e);  // timemix.cu
}  // namespace tm

namespace tc {

// `depth` row-major bf16 matrices [rows][inner], one behind the other
struct Matrix {
  const void* base = nullptr;
  int64_t inner = 0, rows = 0, depth = 0;
};

inline int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return n;
}

// opt in to the dynamic shared memory once per kernel and device
template <typename K>
cudaError_t allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// A, B and (K2 > 0) the second pair.  The box of an operand whose k is contiguous
// has all its rows of a stage; one whose m or n is contiguous, 64 rows of k.
template <int kCG, int kBN, bool kAMN, bool kBMN, bool kWGrad, int kEpi>
int launch(const Matrix& A, const Matrix& B, const Matrix& A2, const Matrix& B2, const Args& a, cudaStream_t s) {
  using Sh = Shape<kCG, kBN, kEpi>;
  if (!tma::bind_context()) return camoe::tm::status(cudaErrorNoDevice);
  CUtensorMap m[4];
  const int ra = kAMN ? 64 : 128, rb = kBMN ? 64 : kBN / kCG;
  bool ok = tma::encode_3d_sw128(&m[0], A.base, A.inner, A.rows, A.depth, ra) &&
            tma::encode_3d_sw128(&m[1], B.base, B.inner, B.rows, B.depth, rb);
  if (kEpi == kDRelu2)  // A2: h, B2: low, in the epilogue's boxes of 32 rows
    ok = ok && tma::encode_2d_rows(&m[2], A2.base, 2 * A2.inner, A2.rows, 64, 32) &&
         (a.low == nullptr || tma::encode_2d_rows(&m[3], a.low, low_stride(a.N), a.R, 32, 32));
  else if (a.K2 > 0)
    ok = ok && tma::encode_3d_sw128(&m[2], A2.base, A2.inner, A2.rows, A2.depth, ra) &&
         tma::encode_3d_sw128(&m[3], B2.base, B2.inner, B2.rows, B2.depth, rb);
  else
    m[2] = m[0], m[3] = m[1];
  if (kEpi == kDRelu2 && a.low == nullptr) m[3] = m[2];
  if (!ok) return camoe::tm::status(cudaErrorInvalidValue);
  const int64_t nt = (a.N + kBN - 1) / kBN;
  const int64_t rt = kWGrad ? static_cast<int64_t>(a.groups) * ((a.M + Sh::kBM - 1) / Sh::kBM)
                            : a.R / Sh::kBM + (a.R < a.groups ? a.R : a.groups);
  if (nt * rt > 0x7fffffffLL) return 3;  // CAMOE_ERR_SHAPE
  int64_t pairs = sm_count() / kCG;
  if (pairs < 1) return camoe::tm::status(cudaErrorNoDevice);
  if (nt * rt < pairs) pairs = nt * rt > 0 ? nt * rt : 1;
  const auto kernel = gemm_kernel<kCG, kBN, kAMN, kBMN, kWGrad, kEpi>;
  static std::atomic<uint64_t> opted{0};
  constexpr int smem = smem_bytes<kCG, kBN, kEpi>();
  if (const int st = camoe::tm::status(allow_smem(kernel, smem, opted))) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(pairs * kCG));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCG;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kCG > 1 ? 1 : 0;
  return camoe::tm::status(cudaLaunchKernelEx(&cfg, kernel, m[0], m[1], m[2], m[3], a));
}

}  // namespace tc
}  // namespace camoe
