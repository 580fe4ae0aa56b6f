// The experts' squared-ReLU products over sorted rows (declared in
// include/camoe_experts.h): forward in two grouped products, backward in four
// (three launches).
//
//   h    = relu(xs w_up^T)^2          rows, K = C, k contiguous in both
//   ys   = h w_down^T                 rows, K = F
//   dpre = (dys w_down) 2 sqrt(h)     rows, K = C, w_down read with n contiguous
//   dxs  = dpre w_up                  rows, K = F, w_up read with n contiguous
//   dw_up   = dpre^T xs               sums over an expert's rows
//   dw_down = dys^T h
//
// h and dpre are held in bf16, the type of the products' operands.  relu(pre) is
// not kept: it is sqrt(h).  For the backward h is kept with 8 bits more than
// bf16 (one byte each): without them the root of the rounded h would add half of
// its rounding error to dpre's own (2.49e-3 against 2.35e-3 of dxs and dw_up in the
// 2-norm, 16384 rows x 1024 x 4096, where one rounding is 1.7e-3).
#include "camoe_experts.h"
#include "tc_gemm.cuh"
#include "tc_launch.cuh"

namespace camoe {
namespace tm {
int status(cudaError_t e);  // timemix.cu
}  // namespace tm

unsigned int ffn_timeouts() {
  unsigned int n = 0;
  if (cudaMemcpyFromSymbol(&n, g_wkv7_timeouts, sizeof(n)) != cudaSuccess) return ~0u;
  return n;
}

namespace ffn {

// Few rows per expert: the weights' bytes decide, and tiles of a few rows read them
// at HBM rate; with more the products count, and 256-row tiles are faster.
bool few_rows(int64_t R, int64_t E) { return R <= 32 * E; }

// Both products of 8 experts of 1024 x 4096 (134 MB), us for 16, 32 and 64 rows each and
// for as many rows unevenly spread: 32 (35), 35 (38) and 42 (66) here, 43, 44 and
// 45 for all in 256-row tiles.
template <int kEpi>
int thin_product(const bf16* x, const bf16* w, const int* offsets, bf16* out, int8_t* low, int64_t R, int64_t E,
                 int64_t O, int64_t K, bool second, cudaStream_t st) {
  thin::Args a{};
  a.offsets = offsets;
  a.groups = static_cast<int>(E);
  a.R = R;
  a.O = static_cast<int>(O);
  a.K = static_cast<int>(K);
  a.second = a.zero_tail = second ? 1 : 0;
  a.out = out;
  a.low = low;
  const int64_t groups = E < R ? E : R;
  // Up to four rows per expert on average: 16 at a time (24.5 us against 26.8 for 1 to
  // 18 rows each); otherwise 64 (30.5 against 38.4 with 32, for 2 to 44 rows).  Two
  // row tiles start side by side, for the experts with more rows than that.
  if (R <= 16) return thin::launch<16, kEpi>(x, w, a, groups, 1, st);
  if (R <= 4 * E) return thin::launch<16, kEpi>(x, w, a, groups, 2, st);
  return thin::launch<64, kEpi>(x, w, a, groups, R <= 64 ? 1 : 2, st);
}

tc::Args args(const int* offsets, int64_t E, int64_t R, int64_t N, int64_t K, void* out) {
  tc::Args a{};
  a.offsets = offsets;
  a.groups = static_cast<int>(E);
  a.R = R;
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.out = static_cast<bf16*>(out);
  return a;
}

// rows x grouped weights; w is [E][N][K], or [E][K][N] where kBMN; h for kDRelu2
template <bool kBMN, int kEpi>
int rows_product(const void* x, const void* w, const tc::Args& a, int64_t E, cudaStream_t st,
                 const void* h = nullptr) {
  return tc::launch<256, false, kBMN, tc::kRows, kEpi>(
      {x, a.K, a.R, 1}, kBMN ? tc::Matrix{w, a.N, a.K, E} : tc::Matrix{w, a.K, a.N, E}, {h, a.N, a.R, 1},
      {}, a, st);
}

int check(const int* offsets, int64_t R, int64_t E, int64_t C, int64_t F) {
  if (R < 0 || E < 1 || C < 1 || F < 1) return 1;
  if (E > 1024 || C % 8 != 0 || F % 8 != 0) return 2;
  if (R > 0x7fffffffLL || C > (1 << 24) || F > (1 << 24)) return 3;
  return offsets == nullptr ? 1 : 0;
}

template <typename... Ptr>
bool aligned(Ptr... p) {
  uintptr_t all = 0;
  ((all |= reinterpret_cast<uintptr_t>(p)), ...);
  return (all & 15u) == 0;
}

}  // namespace ffn
}  // namespace camoe

extern "C" {

int camoe_ex_ffn_fwd(const void* xs, const void* w_up, const void* w_down, const int32_t* offsets, void* h,
                     void* h_low, void* ys, int64_t R, int64_t E, int64_t C, int64_t F, void* stream) {
  using namespace camoe;
  using namespace camoe::ffn;
  if (const int st = check(offsets, R, E, C, F)) return st;
  if (R == 0) return 0;
  if (xs == nullptr || w_up == nullptr || w_down == nullptr || h == nullptr || ys == nullptr) return 1;
  if (!aligned(xs, w_up, w_down, h, h_low, ys) || reinterpret_cast<uintptr_t>(offsets) % 4 != 0) return 4;
  int8_t* low = static_cast<int8_t*>(h_low);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (few_rows(R, E)) {
    const int st = thin_product<tc::kRelu2>(static_cast<const bf16*>(xs), static_cast<const bf16*>(w_up), offsets,
                                      static_cast<bf16*>(h), low, R, E, F, C, false, s);
    if (st != 0) return st;
    return thin_product<tc::kPlain>(static_cast<const bf16*>(h), static_cast<const bf16*>(w_down), offsets,
                               static_cast<bf16*>(ys), nullptr, R, E, C, F, true, s);
  }
  tc::Args up = args(offsets, E, R, F, C, h);
  up.low = low;
  if (const int st = rows_product<false, tc::kRelu2>(xs, w_up, up, E, s)) return st;
  tc::Args down = args(offsets, E, R, C, F, ys);
  down.zero_tail = 1;
  return rows_product<false, tc::kPlain>(h, w_down, down, E, s);
}

int camoe_ex_ffn_bwd(const void* dys, const void* xs, const void* w_up, const void* w_down,
                     const int32_t* offsets, const void* h, const void* h_low, void* dpre, void* dxs, void* dw_up,
                     void* dw_down, int64_t R, int64_t E, int64_t C, int64_t F, void* stream) {
  using namespace camoe;
  using namespace camoe::ffn;
  if (const int st = check(offsets, R, E, C, F)) return st;
  if (!aligned(dys, xs, w_up, w_down, h, h_low, dpre, dxs, dw_up, dw_down) ||
      reinterpret_cast<uintptr_t>(offsets) % 4 != 0)
    return 4;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (R == 0) {
    const size_t bytes = static_cast<size_t>(E * C * F) * sizeof(bf16);
    if (dw_up != nullptr)
      if (const int st = camoe::tm::status(cudaMemsetAsync(dw_up, 0, bytes, s))) return st;
    return dw_down != nullptr ? camoe::tm::status(cudaMemsetAsync(dw_down, 0, bytes, s)) : 0;
  }
  if (dys == nullptr || h == nullptr) return 1;
  if (dxs != nullptr || dw_up != nullptr) {
    if (w_down == nullptr || dpre == nullptr) return 1;
    tc::Args a = args(offsets, E, R, F, C, dpre);
    a.low = static_cast<int8_t*>(const_cast<void*>(h_low));  // read only
    if (const int st = rows_product<true, tc::kDRelu2>(dys, w_down, a, E, s, h)) return st;
  }
  if (dxs != nullptr) {
    if (w_up == nullptr) return 1;
    tc::Args a = args(offsets, E, R, C, F, dxs);
    a.zero_tail = 1;
    if (const int st = rows_product<true, tc::kPlain>(dpre, w_up, a, E, s)) return st;
  }
  if (dw_up == nullptr && dw_down == nullptr) return 0;
  if (dw_up != nullptr && xs == nullptr) return 1;
  // both weight gradients in one launch: one start and end, one last round of tiles
  const tc::Matrix up[2] = {{dpre, F, R, 1}, {xs, C, R, 1}}, down[2] = {{dys, C, R, 1}, {h, F, R, 1}};
  tc::Args a = args(offsets, E, R, dw_up != nullptr ? C : F, 0, dw_up != nullptr ? dw_up : dw_down);
  a.M = static_cast<int>(dw_up != nullptr ? F : C);
  if (dw_up == nullptr)
    return tc::launch<256, true, true, tc::kWeights, tc::kPlain>(down[0], down[1], {}, {}, a, s);
  if (dw_down != nullptr) {
    a.M2 = static_cast<int>(C);
    a.N2 = static_cast<int>(F);
    a.out2 = static_cast<bf16*>(dw_down);
  }
  return tc::launch<256, true, true, tc::kWeights, tc::kPlain>(up[0], up[1], down[0], down[1], a, s);
}

}  // extern "C"
