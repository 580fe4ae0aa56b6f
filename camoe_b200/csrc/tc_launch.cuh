// Host side of tc_gemm.cuh: tensor maps, grid and launch.
#pragma once

#include <atomic>

#include "tc_gemm.cuh"
#include "tc_thin.cuh"

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

// kBlocks: pairs of a group and a row tile at most
inline int64_t most_blocks(int64_t R, int64_t groups, int64_t tile) {
  return (R + tile - 1) / tile + (R < groups ? R : groups);
}

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

// A, B and (kJoined) the second pair.  The box of an operand whose k is contiguous
// has all its rows of a stage; one whose m or n is contiguous, 64 rows of k.
template <int kBN, bool kAMN, bool kBMN, int kMode, int kEpi>
int launch(const Matrix& A, const Matrix& B, const Matrix& A2, const Matrix& B2, const Args& a, cudaStream_t s) {
  using Sh = Shape<kBN, kEpi>;
  if (!tma::bind_context()) return camoe::tm::status(cudaErrorNoDevice);
  CUtensorMap m[6];
  const int ra = kAMN ? 64 : 128, rb = Sh::box(kBMN);
  bool ok = tma::encode_3d_sw128(&m[0], A.base, A.inner, A.rows, A.depth, ra) &&
            tma::encode_3d_sw128(&m[1], B.base, B.inner, B.rows, B.depth, rb);
  m[2] = m[4] = m[5] = m[0], m[3] = m[1];  // where a kernel has no use for them
  if (kEpi == kDRelu2)  // A2: h
    ok = ok && tma::encode_2d_rows(&m[2], A2.base, 2 * A2.inner, A2.rows, 64, 32);
  else if (kMode == kJoined || (kMode == kWeights && a.M2 > 0))
    ok = ok && tma::encode_3d_sw128(&m[2], A2.base, A2.inner, A2.rows, A2.depth, ra) &&
         tma::encode_3d_sw128(&m[3], B2.base, B2.inner, B2.rows, B2.depth, rb);
  // the epilogue's boxes of 32 x 32
  if (a.scatter == nullptr)
    ok = ok && tma::encode_2d_rows(&m[4], a.out, 2 * static_cast<int64_t>(a.N),
                                   kMode == kWeights  ? static_cast<int64_t>(a.groups) * a.M
                                   : kMode == kBlocks ? most_blocks(a.R, a.groups, Sh::kBM) * Sh::kBM
                                                      : a.R, 64, 32);
  if (kMode == kWeights && a.M2 > 0)
    ok = ok && tma::encode_2d_rows(&m[5], a.out2, 2 * static_cast<int64_t>(a.N2), static_cast<int64_t>(a.groups) * a.M2, 64, 32);
  if (a.low != nullptr) ok = ok && tma::encode_2d_rows(&m[5], a.low, low_stride(a.N), a.R, 32, 32);
  if (!ok) return camoe::tm::status(cudaErrorInvalidValue);
  const int64_t nt = (a.N + kBN - 1) / kBN;
  const int64_t rt = kMode == kWeights  ? static_cast<int64_t>(a.groups) * ((a.M + Sh::kBM - 1) / Sh::kBM)
                     : kMode == kJoined ? (a.R + Sh::kBM - 1) / Sh::kBM
                     : kMode == kBlocks ? most_blocks(a.R, a.groups, Sh::kBM)
                                        : a.R / Sh::kBM + (a.R < a.groups ? a.R : a.groups);
  const int64_t more = kMode == kWeights ? static_cast<int64_t>(a.groups) * ((a.M2 + Sh::kBM - 1) / Sh::kBM) *
                                               ((a.N2 + kBN - 1) / kBN)
                                         : 0;
  const int64_t tiles = nt * rt + more;
  if (tiles > 0x3fffffffLL) return 3;  // CAMOE_ERR_SHAPE
  int64_t pairs = sm_count() / kCG;
  if (pairs < 1) return camoe::tm::status(cudaErrorNoDevice);
  if (2 * tiles < pairs) pairs = tiles > 0 ? 2 * tiles : 1;  // a tile may be done as two halves
  const auto kernel = gemm_kernel<kBN, kAMN, kBMN, kMode, kEpi>;
  static std::atomic<uint64_t> opted{0};
  constexpr int smem = smem_bytes<kBN, kEpi>();
  static_assert(smem <= 227 * 1024, "a CTA's shared memory");
  if (const int st = camoe::tm::status(allow_smem(kernel, smem, opted))) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(pairs * kCG));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kCG;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return camoe::tm::status(cudaLaunchKernelEx(&cfg, kernel, m[0], m[1], m[2], m[3], m[4], m[5], a));
}

}  // namespace tc

namespace thin {

// CTAs per tile of 128 outputs: as many as keep all of them on the SMs at once, two per
// SM, with two pieces of k at least for each
inline int split_of(int64_t tiles, int64_t K, int least) {
  const int64_t nk = (K + tc::kBK - 1) / tc::kBK, room = 2 * tc::sm_count();
  int s = least;
  while (s < 8 && tiles * s * 2 <= room && nk >= 4 * s) s *= 2;
  return s;
}

// `groups` that can have rows, `row_tiles` started apart (1: one after the other);
// The kernel may start before the one before it in the stream has ended: it waits
// for that one before it reads what that one may have written, and in every case
// before it ends.
template <int kN, int kEpi>
int launch(const void* x, const void* w, Args a, int64_t groups, int64_t row_tiles, cudaStream_t s) {
  if (!tma::bind_context()) return camoe::tm::status(cudaErrorNoDevice);
  CUtensorMap mw, mx;
  if (!tma::encode_3d_sw128(&mw, w, a.K, a.O, a.groups, kM) || !tma::encode_3d_sw128(&mx, x, a.K, a.R, 1, kN))
    return camoe::tm::status(cudaErrorInvalidValue);
  const int64_t tiles = (a.O + kM - 1) / kM;
  a.split = split_of(tiles * groups * row_tiles, a.K, kEpi == kAdapter ? kN / kAdd : 1);
  const auto kernel = thin_kernel<kN, kEpi>;
  static std::atomic<uint64_t> opted{0};
  if (const int st = camoe::tm::status(tc::allow_smem(kernel, smem_bytes<kN>(kEpi == kAdapter ? 256 : 0), opted)))
    return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * a.split), static_cast<unsigned>(groups),
                     static_cast<unsigned>(row_tiles));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem_bytes<kN>(kEpi == kAdapter ? a.D : 0);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(a.split);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return camoe::tm::status(cudaLaunchKernelEx(&cfg, kernel, mw, mx, a));
}

}  // namespace thin
}  // namespace camoe
