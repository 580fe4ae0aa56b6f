// Products of few rows with grouped weights: what a generated token needs.
//
//   out[p][o] = f(sum over k of x[p][k] W_g[o][k]) for the rows p of group g
//
// With a few rows per group the weights' bytes are the whole cost, so a block
// owns 16 weight rows and streams them once from HBM to registers; nothing is
// staged in shared memory.  The products run on warp-level mma (m16n8k16, the
// weights as the 16-row operand, 8 rows of x as its columns), which is far from
// its limit here.  Both operands index k alike, so k may be permuted: lane
// (g, t) of a warp holds k = 8 t .. 8 t + 7 of a 32-deep piece, one 16-byte load
// per operand row, which are two mma steps.  The eight warps take alternate
// pieces (512 contiguous bytes of each weight row per turn of the block), and
// their sums are added in a fixed order through shared memory.
#pragma once

#include "wkv7_common.cuh"

namespace camoe {
namespace thin {

constexpr int kThreads = 256;
constexpr int kWarps = 8;
constexpr int kO = 16;  // weight rows per block

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// weights are read once: keep them out of the way of what is read again
__device__ __forceinline__ uint4 ld_once(const bf16* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// sums[o][r] = sum over k of w[o][k] x[r][k] for 16 weight rows from `w` (of
// which n_o exist) and 8 kN rows from `x` (n_r exist): called by the whole
// block, leaves the sums in `red` (kWarps x 16 x 8 kN floats).
template <int kN>
__device__ __forceinline__ void block_sums(const bf16* __restrict__ w, int n_o, const bf16* __restrict__ x,
                                           int n_r, int K, float* red) {
  constexpr int kU = kN >= 4 ? 2 : 4;  // pieces in flight per warp
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  float acc[kN][4];
#pragma unroll
  for (int i = 0; i < kN; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  const bool o0 = g < n_o, o1 = g + 8 < n_o;
  const bf16* w0 = w + static_cast<int64_t>(o0 ? g : 0) * K;
  const bf16* w1 = w + static_cast<int64_t>(o1 ? g + 8 : 0) * K;
  for (int k0 = warp * 32; k0 < K; k0 += kWarps * 32 * kU) {
    uint4 a[kU][2], b[kU][kN];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int k = k0 + u * kWarps * 32 + 8 * t;
      const bool in = k < K;  // K is a multiple of 8
      a[u][0] = in && o0 ? ld_once(w0 + k) : zero;
      a[u][1] = in && o1 ? ld_once(w1 + k) : zero;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int r = 8 * i + g;
        b[u][i] = in && r < n_r ? *reinterpret_cast<const uint4*>(x + static_cast<int64_t>(r) * K + k) : zero;
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        mma16816(acc[i], a[u][0].x, a[u][1].x, a[u][0].y, a[u][1].y, b[u][i].x, b[u][i].y);
        mma16816(acc[i], a[u][0].z, a[u][1].z, a[u][0].w, a[u][1].w, b[u][i].z, b[u][i].w);
      }
  }
  float* mine = red + warp * (kO * 8 * kN);
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    float* p = mine + 8 * i + 2 * t;
    *reinterpret_cast<float2*>(p + g * (8 * kN)) = make_float2(acc[i][0], acc[i][1]);
    *reinterpret_cast<float2*>(p + (g + 8) * (8 * kN)) = make_float2(acc[i][2], acc[i][3]);
  }
  __syncthreads();
}

// the sum of weight row o and row r
template <int kN>
__device__ __forceinline__ float total(const float* red, int o, int r) {
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) s += red[w * (kO * 8 * kN) + o * (8 * kN) + r];
  return s;
}

}  // namespace thin
}  // namespace camoe
