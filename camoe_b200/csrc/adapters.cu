// A projection with the low-rank adapter of each row beside it (declared in
// include/camoe_experts.h):
//   y[n] = weight x[n] + scale[a] up[a] (down[a] x[n]),  a = adapter[n]
//
// Few rows (a token of each of many requests): two launches, or one for the fewest.
// low[n] = scale[a] down[a] x[n] in fp32, a warp per output; then the projection
// with the weights streamed once (tc_thin.cuh; it starts while the first kernel
// runs), to whose sums each output adds its row of up times low, in fp32, before
// the one rounding.
//
// Many rows (prompts): the rows are sorted by adapter, low = scale (xs down^T) is one
// grouped product (rounded to bf16, the type of the next product's operand), and
// the projection's sum runs over [x | low] against [weight | up[a]]: an adapter is
// D more columns of k for the row tiles that hold rows of it, which add to its own
// rows only (kBlocks and kJoined in tc_gemm.cuh), so row tiles are full whatever
// the adapters' shares.  The result goes to the row that it came from.
#include "camoe_experts.h"
#include "tc_launch.cuh"

namespace camoe {
namespace rows {
size_t sort_bytes(int64_t N, int64_t k, int64_t E);  // experts_rows.cu
int sort_rows(const void* x, const int* group, void* xs, int* offsets, int* position, int* source, void* work,
              int64_t N, int L, int64_t V, cudaStream_t st);
}  // namespace rows

unsigned int adapter_timeouts() {
  unsigned int n = 0;
  if (cudaMemcpyFromSymbol(&n, g_wkv7_timeouts, sizeof(n)) != cudaSuccess) return ~0u;
  return n;
}

namespace adapt {

constexpr int kThreads = 256;

// low[n][d] = scale[a] (x[n] . down[a][d]): a warp per (n, d)
__global__ void __launch_bounds__(kThreads) low_kernel(const bf16* __restrict__ x,
                                                       const bf16* __restrict__ down,
                                                       const int* __restrict__ adapter,
                                                       const float* __restrict__ scale,
                                                       float* __restrict__ low, int C, int D, int L) {
  thin::allow_next();
  const int n = blockIdx.y, lane = threadIdx.x & 31;
  const int d = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int a = adapter[n];
  if (a < 0 || a >= L || d >= D) return;
  const uint4* xp = reinterpret_cast<const uint4*>(x + static_cast<int64_t>(n) * C);
  const uint4* dp = reinterpret_cast<const uint4*>(down + (static_cast<int64_t>(a) * D + d) * C);
  constexpr int kDeep = 4;  // loads in flight
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  float s = 0.0f;
  for (int v0 = lane; v0 < C / 8; v0 += 32 * kDeep) {
    uint4 p[kDeep], q[kDeep];
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const bool in = v0 + 32 * u < C / 8;
      p[u] = in ? xp[v0 + 32 * u] : zero;
      q[u] = in ? dp[v0 + 32 * u] : zero;
    }
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      if (v0 + 32 * u >= C / 8) continue;
      const __nv_bfloat162* ph = reinterpret_cast<const __nv_bfloat162*>(&p[u]);
      const __nv_bfloat162* qh = reinterpret_cast<const __nv_bfloat162*>(&q[u]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = __bfloat1622float2(ph[e]), g = __bfloat1622float2(qh[e]);
        s = fmaf(f.x, g.x, s);
        s = fmaf(f.y, g.y, s);
      }
    }
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
  if (lane == 0) low[static_cast<int64_t>(n) * D + d] = scale != nullptr ? scale[a] * s : s;
}

// Rows that are streamed rather than sorted: few, and with little of the adapters' own
// work, which each row does for itself there.  B200, us streamed / in tiles, rows
// that mix L adapters, N x C x M x D, L:  128 x 2048 x 2048 x 32, 64: 19 / 64;
// 256 x 2048 x 2048 x 32, 64: 31 / 69;  384: 51 / 58;  512 x 1024 x 1024 x 16, 12:
// 24 / 27;  512 x 1024 x 1024 x 64, 3: 51 / 23;  256 x 2048 x 4096 x 128, 64: 133 / 88.
// Up to 128 rows all are streamed: 128 x 2048 x 2048 x 128, 64 45 / 82;  64 x 2048 x
// 4096 x 256, 64 80 / 93;  16: 30 / 56.  The rule is not the best at the highest
// ranks: 128 x 2048 x 4096 x 256, 64 147 / 112;  128 x 1024 x 1024 x 256, 3 43 / 27.
bool few_rows(int64_t N, int64_t M, int64_t D) { return N <= 128 || (N <= 512 && N * M * D <= (24 << 20)); }

// A few rows whose low-rank parts are little work for each CTA of a cluster of four
// (64 KB of down read at most): every tile of the projection works them out for
// itself, in one launch.  B200, us here / with a launch of their own, N x C x D:
// 1 x 1024 x 16 6.9 / 8.3, 8 x 1024 x 16 7.3 / 8.3, 1 x 2048 x 64 15.7 / 10.3.
bool own_low(int64_t N, int64_t C, int64_t D) { return N <= 8 && (N + 3) / 4 * C * D <= 32 * 1024; }

size_t up16(size_t n) { return (n + 15) / 16 * 16; }

constexpr int64_t kTile = 256;  // rows of a tile
int64_t blocks(int64_t N, int64_t L) { return tc::most_blocks(N, L, kTile); }

struct Layout {  // of the workspace
  size_t low, xs, offsets, position, source, sort, total;
};
Layout layout(int64_t N, int64_t C, int64_t M, int64_t D, int64_t L) {
  Layout w{};
  const size_t n = static_cast<size_t>(N);
  if (few_rows(N, M, D)) {
    w.total = up16(n * static_cast<size_t>(D) * sizeof(float));
    return w;
  }
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += up16(bytes);
    return here;
  };
  w.low = take(static_cast<size_t>(blocks(N, L)) * kTile * static_cast<size_t>(D) * sizeof(bf16));
  w.xs = take(n * static_cast<size_t>(C) * sizeof(bf16));
  w.offsets = take(static_cast<size_t>(L + 2) * sizeof(int));
  w.position = take(n * sizeof(int));
  w.source = take(n * sizeof(int));
  w.sort = take(rows::sort_bytes(N, 1, L));
  w.total = at;
  return w;
}

int check(int64_t N, int64_t C, int64_t M, int64_t D, int64_t L) {
  if (N < 0 || C < 1 || M < 1 || D < 1 || L < 1) return 1;
  if (C % 8 != 0 || M % 8 != 0 || D % 8 != 0 || D > 256 || L > 1024) return 2;
  if (N > (1 << 27) || C > (1 << 24) || M > (1 << 24)) return 3;
  return 0;
}

template <int kBN>
int low_product(const bf16* xs, const void* down, const tc::Args& a, int64_t L, cudaStream_t st) {
  return tc::launch<kBN, false, false, tc::kBlocks, tc::kScale>({xs, a.K, a.R, 1}, {down, a.K, a.N, L}, {}, {}, a, st);
}

}  // namespace adapt
}  // namespace camoe

extern "C" {

size_t camoe_ad_work_bytes(int64_t N, int64_t C, int64_t M, int64_t D, int64_t L) {
  return camoe::adapt::check(N, C, M, D, L) == 0 ? camoe::adapt::layout(N, C, M, D, L).total : 0;
}

int camoe_ad_linear(const void* x, const void* weight, const void* down, const void* up, const int32_t* adapter,
                    const float* scale, void* y, void* work, size_t work_bytes, int64_t N, int64_t C, int64_t M,
                    int64_t D, int64_t L, void* stream) {
  using namespace camoe;
  using namespace camoe::adapt;
  if (const int st = check(N, C, M, D, L)) return st;
  if (N == 0) return 0;
  for (const void* p : {x, weight, down, up, static_cast<const void*>(adapter), static_cast<const void*>(y),
                        static_cast<const void*>(work)})
    if (p == nullptr) return 1;
  for (const void* p : {x, weight, down, up, static_cast<const void*>(y), static_cast<const void*>(work)})
    if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) return 4;
  if ((reinterpret_cast<uintptr_t>(adapter) | reinterpret_cast<uintptr_t>(scale)) % 4 != 0) return 4;
  const Layout w = layout(N, C, M, D, L);
  if (work_bytes < w.total) return 5;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  unsigned char* base = static_cast<unsigned char*>(work);
  const int c = static_cast<int>(C), m = static_cast<int>(M), d = static_cast<int>(D), l = static_cast<int>(L);
  const bf16* xb = static_cast<const bf16*>(x);
  if (few_rows(N, M, D)) {
    float* low = static_cast<float*>(work);
    const bool own = own_low(N, C, D);
    if (!own) {
      low_kernel<<<dim3((d + 7) / 8, static_cast<unsigned>(N)), kThreads, 0, s>>>(
          xb, static_cast<const bf16*>(down), adapter, scale, low, c, d, l);
      if (const int st = camoe::tm::status(cudaGetLastError())) return st;
    }
    thin::Args t{};
    t.groups = 1;
    t.R = N;
    t.O = m;
    t.K = c;
    t.out = static_cast<bf16*>(y);
    t.up = static_cast<const bf16*>(up);
    t.adapter = adapter;
    t.low_rank = own ? nullptr : low;
    t.x = xb;
    t.down = static_cast<const bf16*>(down);
    t.scale = scale;
    t.D = d;
    t.L = l;
    t.second = own ? 0 : 1;  // the first kernel has waited for what is before it
    // row tiles of 32 started apart: their adapters' work runs side by side, and
    // the weights of all but one come from L2
    return N <= 16 ? thin::launch<16, thin::kAdapter>(x, weight, t, 1, 1, s)
                   : thin::launch<32, thin::kAdapter>(x, weight, t, 1, (N + 31) / 32, s);
  }
  bf16* low = reinterpret_cast<bf16*>(base + w.low);
  bf16* xs = reinterpret_cast<bf16*>(base + w.xs);
  int* offsets = reinterpret_cast<int*>(base + w.offsets);
  int* source = reinterpret_cast<int*>(base + w.source);
  if (const int st = rows::sort_rows(x, adapter, xs, offsets, reinterpret_cast<int*>(base + w.position), source,
                                     base + w.sort, N, l, C / 8, s))
    return st;
  tc::Args a{};
  a.offsets = offsets;
  a.groups = l;
  a.R = N;
  a.N = d;
  a.K = c;
  a.out = low;
  a.scale = scale;
  const int st = D <= 64 ? low_product<64>(xs, down, a, L, s)
                         : (D <= 128 ? low_product<128>(xs, down, a, L, s) : low_product<256>(xs, down, a, L, s));
  if (st != 0) return st;
  a.N = m;
  a.K2 = d;
  a.out = static_cast<bf16*>(y);
  a.scale = nullptr;
  a.scatter = source;
  return tc::launch<256, false, false, tc::kJoined, tc::kPlain>(
      {xs, C, N, 1}, {weight, C, M, 1}, {low, D, blocks(N, L) * kTile, 1}, {up, D, M, L}, a, s);
}

}  // extern "C"
