// Products of few rows with grouped weights on the tensor cores: what generated
// tokens need.
//
//   out[p][o] = f(sum over k of W_g[o][k] x[p][k]) for the rows p of group g
//
// The weights' bytes are the cost: 128 weight rows are the M of a product and up
// to kN rows of x its N, so a 16 KB box of weights is read once from HBM, by TMA,
// and used for all rows of its group (kN at a time).  What counts is that all
// SMs have loads in flight from the first to the last moment:
//   * a tile of 128 outputs is split over a cluster of 1 to 8 CTAs along k, so
//     that even one token's two experts fill the SMs; two CTAs fit an SM;
//   * a CTA's loads are a ring of 64-deep pieces, the first of which (weights
//     only) are asked for before the kernel that makes x has ended, where the
//     launch allows it (a programmatic dependent launch);
//   * the CTAs of a cluster add their accumulators through distributed shared
//     memory, each for its share of the rows, in the order of their ranks
//     (deterministic), and apply f.
// Measured (B200): see the launch rules in experts_ffn.cu and adapters.cu.
#pragma once

#include "tc_gemm.cuh"

namespace camoe {
namespace thin {

constexpr int kThreads = 192;  // producer, product issue, four epilogue warps
constexpr int kM = 128;        // weight rows per tile
constexpr int kMaxStages = 5;
constexpr uint32_t kWBytes = kM * 128;

struct Args {
  const int* offsets;  // [groups + 1], or null: one group of all rows
  int groups;
  int64_t R;
  int O, K;
  int split;           // CTAs per tile (the cluster's size)
  int second;          // offsets and weights are older than the kernel before this one, x is not
  int zero_tail;       // write zeros to the rows behind the last group
  bf16* out;
  int8_t* low;         // tc::kRelu2: as in tc_gemm.cuh, or null
  // kAdapter: out += up[a] low[p], a = adapter[p]; low is low_rank [R, D], or (null)
  // scale[a] down[a] x[p], which the kernel works out
  const bf16* up;
  const int* adapter;
  const float* low_rank;
  const bf16 *x, *down;
  const float* scale;
  int D, L;
};

constexpr int kAdapter = 16;  // an epilogue next to those of tc_gemm.cuh

template <int kN>
struct Shape {
  static constexpr uint32_t kStage = kWBytes + kN * 128;
  static constexpr int kFit = 96 * 1024 / static_cast<int>(kStage);  // two CTAs on an SM
  static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
  static constexpr uint32_t kCols = kN < 32 ? 32 : kN;  // tensor-memory columns
};
struct Control {
  uint64_t full[kMaxStages], empty[kMaxStages], acc;
  uint32_t tmem;
};
// plus kAdapter's rows of low_rank
template <int kN>
__host__ __device__ constexpr int smem_bytes(int rank) {
  return Shape<kN>::kStages * static_cast<int>(Shape<kN>::kStage) + static_cast<int>(sizeof(Control)) + 1024 +
         16 * rank * static_cast<int>(sizeof(float));
}

__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float load_peer(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile(
      "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.f32 %0, [a];\n}\n"
      : "=f"(v)
      : "r"(addr), "r"(rank));
  return v;
}

// The y-th group that has rows; false where there are fewer.
__device__ __forceinline__ bool nth_group(const Args& a, int y, int* g, int64_t* r0, int64_t* r1) {
  if (a.offsets == nullptr) {
    *g = 0;
    *r0 = 0;
    *r1 = a.R;
    return y == 0;
  }
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int e0 = 0; e0 < a.groups; e0 += 32) {
    const int e = e0 + lane;
    int64_t p = 0, q = 0;
    if (e < a.groups) {
      p = a.offsets[e];
      q = a.offsets[e + 1];
      p = p < 0 ? 0 : (p < a.R ? p : a.R);
      q = q < 0 ? 0 : (q < a.R ? q : a.R);
    }
    unsigned has = __ballot_sync(0xffffffffu, q > p);
    const int n = __popc(has);
    if (y < before + n) {
      for (int i = before; i < y; ++i) has &= has - 1;
      const int src = __ffs(has) - 1;
      *g = e0 + src;
      *r0 = __shfl_sync(0xffffffffu, p, src);
      *r1 = __shfl_sync(0xffffffffu, q, src);
      return true;
    }
    before += n;
  }
  return false;
}

// f, and the store of output o of row p
template <int kEpi>
__device__ __forceinline__ void put(const Args& a, int64_t p, int o, float v) {
  if (kEpi != kAdapter) v = tc::finish<kEpi>(v, 0.0f, 1.0f);
  const bf16 hi = __float2bfloat16_rn(v);
  a.out[p * a.O + o] = hi;
  if (kEpi == tc::kRelu2 && a.low != nullptr)
    a.low[p * tc::low_stride(a.O) + o] = static_cast<int8_t>(tc::low_bits(v, hi));
}

// kAdapter: what the adapters add to output o of up to kAdd rows p, p + step, ...
// below end.  kAddRows rows at a time and 16 columns of up each, so that their
// loads overlap; those of the first step are made by fetch(), before `low`, the
// rows' low_rank in shared memory ([kAdd][D]), is there.
constexpr int kAdd = 16, kAddRows = 8;
struct AdapterAdd {
  const uint4* u[kAddRows];
  uint4 w[kAddRows][2];
  __device__ __forceinline__ void rows(const Args& a, int64_t p, int step, int64_t end, int o) {
#pragma unroll
    for (int j = 0; j < kAddRows; ++j) {
      const int64_t q = p + static_cast<int64_t>(step) * j;
      const int ad = q < end && o < a.O ? a.adapter[q] : -1;
      u[j] = ad >= 0 && ad < a.L ? reinterpret_cast<const uint4*>(a.up + (static_cast<int64_t>(ad) * a.O + o) * a.D)
                                 : nullptr;
    }
  }
  __device__ __forceinline__ void fetch(int d, int n) {
#pragma unroll
    for (int j = 0; j < kAddRows; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (u[j] != nullptr && d + h < n) w[j][h] = u[j][d + h];
  }
  __device__ __forceinline__ void sum(int d, int D, const float* low, float* add) {
#pragma unroll
    for (int j = 0; j < kAddRows; ++j) {
      if (u[j] == nullptr) continue;
      float s = add[j];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (d + h >= D / 8) continue;
        const float4* l = reinterpret_cast<const float4*>(low + j * D + 8 * (d + h));
        const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&w[j][h]);
        const float4 l0 = l[0], l1 = l[1];
        const float2 f0 = __bfloat1622float2(b[0]), f1 = __bfloat1622float2(b[1]), f2 = __bfloat1622float2(b[2]),
                     f3 = __bfloat1622float2(b[3]);
        s = fmaf(f0.x, l0.x, s);
        s = fmaf(f0.y, l0.y, s);
        s = fmaf(f1.x, l0.z, s);
        s = fmaf(f1.y, l0.w, s);
        s = fmaf(f2.x, l1.x, s);
        s = fmaf(f2.y, l1.y, s);
        s = fmaf(f3.x, l1.z, s);
        s = fmaf(f3.y, l1.w, s);
      }
      add[j] = s;
    }
  }
};

// low[q][d] = scale (down[d] x) for this CTA's rows, by its four epilogue warps: where
// the rows are so few that a launch of its own costs more
__device__ __forceinline__ void own_low(const Args& a, int64_t p, int step, int64_t end, float* low) {
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - 2;
  constexpr int kDeep = 4;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int q = 0; q < kAdd && p + static_cast<int64_t>(step) * q < end; ++q) {
    const int64_t row = p + static_cast<int64_t>(step) * q;
    const int ad = a.adapter[row];
    if (ad < 0 || ad >= a.L) continue;
    const float scale = a.scale != nullptr ? a.scale[ad] : 1.0f;
    const uint4* x = reinterpret_cast<const uint4*>(a.x + row * a.K);
    for (int d = warp * kDeep; d < a.D; d += 4 * kDeep) {  // D is a multiple of 8
      const uint4* w = reinterpret_cast<const uint4*>(a.down + (static_cast<int64_t>(ad) * a.D + d) * a.K);
      const int n = a.K / 8;
      float s[kDeep] = {};
      for (int v0 = lane; v0 < n; v0 += 64) {
        uint4 xv[2], wv[2][kDeep];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool in = v0 + 32 * h < n;
          xv[h] = in ? x[v0 + 32 * h] : zero;
#pragma unroll
          for (int e = 0; e < kDeep; ++e) wv[h][e] = in ? w[static_cast<int64_t>(e) * n + v0 + 32 * h] : zero;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (v0 + 32 * h >= n) continue;
          const __nv_bfloat162* xb = reinterpret_cast<const __nv_bfloat162*>(&xv[h]);
#pragma unroll
          for (int e = 0; e < kDeep; ++e) {
            const __nv_bfloat162* wb = reinterpret_cast<const __nv_bfloat162*>(&wv[h][e]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = __bfloat1622float2(xb[i]), g = __bfloat1622float2(wb[i]);
              s[e] = fmaf(f.x, g.x, s[e]);
              s[e] = fmaf(f.y, g.y, s[e]);
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < kDeep; ++e) {
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) s[e] += __shfl_xor_sync(0xffffffffu, s[e], m);
        if (lane == e) low[q * a.D + d + e] = scale * s[e];
      }
    }
  }
}

// The sums over the cluster of rows r, r + split, ... (those below `rows`), rank by
// rank; all loads of kPeerRows rows are in flight at once.
constexpr int kPeerRows = 4;
__device__ __forceinline__ void peer_sums(uint32_t part, int r, int split, int rows, float (&v)[kPeerRows]) {
  float x[kPeerRows][8];
#pragma unroll
  for (int e = 0; e < kPeerRows; ++e)
#pragma unroll
    for (int q = 0; q < 8; ++q)
      x[e][q] = q < split && r + e * split < rows ? load_peer(part + 4u * kM * (r + e * split), static_cast<uint32_t>(q))
                                                  : 0.0f;
#pragma unroll
  for (int e = 0; e < kPeerRows; ++e) {
    v[e] = x[e][0];
#pragma unroll
    for (int q = 1; q < 8; ++q) v[e] += x[e][q];
  }
}

__device__ __forceinline__ void ld_cols(float (&v)[16], uint32_t taddr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;\n"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
        "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}

// grid: x = tiles of 128 outputs x split (a cluster along x), y = groups that
// have rows, z = row tiles that start apart.
template <int kN, int kEpi>
__global__ void __launch_bounds__(kThreads, 2) thin_kernel(const __grid_constant__ CUtensorMap mw,
                                                        const __grid_constant__ CUtensorMap mx, const Args a) {
  using Sh = Shape<kN>;
  constexpr int S = Sh::kStages;
  static_assert(S * Sh::kStage >= kN * kM * 4, "the ring also holds the accumulators for the sum over the cluster");
  extern __shared__ __align__(128) unsigned char raw[];
  unsigned char* ring = raw + ((1024u - (sm_addr(raw) & 1023u)) & 1023u);
  Control& c = *reinterpret_cast<Control*>(ring + S * Sh::kStage);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = a.split, rank = static_cast<int>(blockIdx.x) % split, tile = static_cast<int>(blockIdx.x) / split;
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&mw)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&mx)) : "memory");
    for (int s = 0; s < S; ++s) {
      mbar_init(&c.full[s], 1);
      mbar_init(&c.empty[s], 1);
    }
    mbar_init(&c.acc, 1);
    mbar_fence_init();
  }
  if (!a.second) wait_previous();
  // Not before this wait: a second kernel reads offsets and weights before its own,
  // so what comes before the first one has to be done by the time it may start.
  allow_next();
  if (a.zero_tail && blockIdx.y == 0) {
    const int64_t pieces = a.O / 8, used = a.offsets != nullptr ? a.offsets[a.groups] : a.R;
    uint4* out = reinterpret_cast<uint4*>(a.out);
    for (int64_t i = (used > 0 ? used : 0) * pieces + static_cast<int64_t>(blockIdx.x) * kThreads + tid;
         i < a.R * pieces; i += static_cast<int64_t>(gridDim.x) * kThreads)
      out[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  int g;
  int64_t r0, r1;
  if (!nth_group(a, static_cast<int>(blockIdx.y), &g, &r0, &r1)) {  // the whole cluster
    if (a.second) wait_previous();
    return;
  }
  const int nk = (a.K + tc::kBK - 1) / tc::kBK, per = (nk + split - 1) / split;
  const int k0 = rank * per < nk ? rank * per : nk, k1 = k0 + per < nk ? k0 + per : nk;
  if (warp == 1) tc::tmem_alloc<1>(&c.tmem, Sh::kCols);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = c.tmem, ring0 = sm_addr(ring);
  const int64_t start = r0 + static_cast<int64_t>(blockIdx.z) * kN, step = static_cast<int64_t>(gridDim.z) * kN;
  const int o = tile * kM + 32 * (warp & 3) + lane;
  int i = 0, it = 0;  // pieces and row tiles so far
  float add[kAdd];    // kAdapter: kN / split rows at most, which the launch sees to
  bool ok = true;
  for (int64_t p = start; p < r1; p += step, ++it) {
    if (warp == 0) {
      if (lane == 0) {
        const int row = static_cast<int>(p);
        const auto load_w = [&](int s, int k) {
          mbar_arrive_expect_tx(&c.full[s], Sh::kStage);
          tc::load_box<1>(ring0 + s * Sh::kStage, &mw, k * tc::kBK, tile * kM, g, sm_addr(&c.full[s]));
        };
        const auto load_x = [&](int s, int k) {
          tc::load_box<1>(ring0 + s * Sh::kStage + kWBytes, &mx, k * tc::kBK, row, 0, sm_addr(&c.full[s]));
        };
        int k = k0;
        if (it == 0) {  // the first pieces' weights do not wait for x
          const int first = k1 - k0 < S ? k1 - k0 : S;
          for (int j = 0; j < first; ++j) load_w(j, k0 + j);
          if (a.second) wait_previous();
          for (int j = 0; j < first; ++j) load_x(j, k0 + j);
          k += first;
          i = first;
        }
        for (; ok && k < k1; ++k, ++i) {
          const int s = i % S;
          if (i >= S && !(ok = mbar_wait(&c.empty[s], static_cast<uint32_t>((i / S - 1) & 1)))) break;
          load_w(s, k);
          load_x(s, k);
        }
        if (!ok)  // after a wait that ran out: the copies in flight end first
          for (int q = i > S ? i - S : 0; q < i; ++q) mbar_wait(&c.full[q % S], static_cast<uint32_t>((q / S) & 1));
      }
    } else if (warp == 1) {
      if (lane == 0) {
        constexpr uint32_t idesc = tc::instr<false, false>(kM, kN);
        tc::fence_after();
        for (int k = k0; ok && k < k1; ++k, ++i) {
          const int s = i % S;
          if (!(ok = mbar_wait(&c.full[s], static_cast<uint32_t>((i / S) & 1)))) break;
          tc::fence_after();
          const uint32_t sw = ring0 + s * Sh::kStage;
#pragma unroll
          for (int q = 0; q < tc::kBK / 16; ++q)
            tc::mma<1>(tmem, tc::desc<false>(sw + tc::kStep<false> * q),
                       tc::desc<false>(sw + kWBytes + tc::kStep<false> * q), idesc, k > k0 || q > 0);
          tc::commit<1>(&c.empty[s]);
        }
        if (k1 > k0) tc::commit<1>(&c.acc);
      }
    }
    const int rows = r1 - p < kN ? static_cast<int>(r1 - p) : kN;
    if (warp >= 2) {
      if (kEpi == kAdapter) {  // while the weights arrive
        float* low = reinterpret_cast<float*>(ring + S * Sh::kStage + sizeof(Control));
        const int64_t end = r1 < p + kN ? r1 : p + kN;
        AdapterAdd f;
        f.rows(a, p + rank, split, end, o);
        f.fetch(0, a.D / 8);
        wait_previous();
        named_sync(1, 128);  // the last row tile's are no longer read
        if (a.low_rank == nullptr)
          own_low(a, p + rank, split, end, low);
        else
          for (int q = 0; q < kAdd && p + rank + q * split < end; ++q)
            for (int d = tid - 64; d < a.D; d += 128) low[q * a.D + d] = a.low_rank[(p + rank + q * split) * a.D + d];
        named_sync(1, 128);
#pragma unroll
        for (int j = 0; j < kAdd; ++j) add[j] = 0.0f;
#pragma unroll
        for (int j = 0; j < kAdd; j += kAddRows) {
          if (p + rank + j * split >= end) break;
          if (j > 0) {
            f.rows(a, p + rank + j * split, split, end, o);
            f.fetch(0, a.D / 8);
          }
          for (int d = 0; d < a.D / 8; d += 2) {
            f.sum(d, a.D, low + j * a.D, add + j);
            f.fetch(d + 2, a.D / 8);
          }
        }
      }
      if (k1 > k0) ok = tc::warp_wait(&c.acc, static_cast<uint32_t>(it & 1)) && ok;
      tc::fence_after();
      float* part = reinterpret_cast<float*>(ring) + (32 * (warp & 3) + lane);
#pragma unroll 1
      for (int c0 = 0; c0 < kN; c0 += 16) {
        if (c0 >= rows) break;
        float v[16];
        if (k1 > k0) {
          ld_cols(v, tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + static_cast<uint32_t>(c0));
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = 0.0f;
        }
        if (split == 1) {
          if (o < a.O) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (c0 + e < rows) put<kEpi>(a, p + c0 + e, o, kEpi == kAdapter && kN == kAdd ? v[e] + add[e] : v[e]);
          }
        } else {  // every product has read the ring: it holds the sums now
#pragma unroll
          for (int e = 0; e < 16; ++e) part[(c0 + e) * kM] = v[e];
        }
        __syncwarp();
      }
      tc::fence_before();
    }
    __syncwarp();
    if (split > 1) {
      cluster_sync();
      if (warp >= 2 && o < a.O) {
        const uint32_t part = ring0 + 4u * static_cast<uint32_t>(32 * (warp & 3) + lane);
        if (kEpi == kAdapter) {
#pragma unroll
          for (int j = 0; j < kAdd; j += kPeerRows) {
            if (rank + j * split >= rows) break;
            float v[kPeerRows];
            peer_sums(part, rank + j * split, split, rows, v);
#pragma unroll
            for (int e = 0; e < kPeerRows; ++e)
              if (rank + (j + e) * split < rows) put<kEpi>(a, p + rank + (j + e) * split, o, v[e] + add[j + e]);
          }
        } else {
          for (int r = rank; r < rows; r += kPeerRows * split) {
            float v[kPeerRows];
            peer_sums(part, r, split, rows, v);
#pragma unroll
            for (int e = 0; e < kPeerRows; ++e)
              if (r + e * split < rows) put<kEpi>(a, p + r + e * split, o, v[e]);
          }
        }
      }
      fence_proxy_async();  // the ring's next writer is TMA
      cluster_sync();
    } else {
      __syncthreads();
    }
  }
  __syncthreads();
  if (warp == 1) tc::tmem_free<1>(tmem, Sh::kCols);
}

}  // namespace thin
}  // namespace camoe
