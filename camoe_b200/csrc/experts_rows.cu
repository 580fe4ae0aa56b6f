// Tokens sorted by expert and back (declared in include/camoe_experts.h).
//
// The sort is a counting sort that keeps the slots' order: the row of slot s is
//   #{s' : e(s') < e(s)} + #{s' < s : e(s') = e(s)}
// with an unused slot counted as expert E, so every slot has exactly one row and
// the rows behind offsets[E] are those of the unused slots (which get zeros).
// Counts are integers and nothing depends on the order in which blocks run.
//
// Up to kSmallSlots slots one launch does it all: each token's block counts its
// own slots' rows by reading the whole index once (a warp per slot) and copies
// its row.  Above that every chunk of slots has a block that places them: it adds
// up the slots of the chunks before it (up to 8192 slots of few experts by reading
// the whole index itself, otherwise from counts per chunk that a first launch makes)
// and a warp's of the warps before it.  The copy follows; the launches overlap (programmatic
// dependent launches), so that x is loaded by the time the rows are known.
//
// The copies are bound by HBM: a thread holds 16 bytes (or one element where the
// width or an address is no multiple of 16 bytes) of a row of each of kTokens
// tokens, so that enough loads are in flight; a token's row is read once and
// written k times.
#include "camoe_experts.h"
#include "wkv7_common.cuh"

namespace camoe {
namespace tm {
int status(cudaError_t e);  // timemix.cu
}  // namespace tm

namespace rows {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSmallSlots = 2048;
constexpr int kMaxExperts = 1024;
constexpr int kMaxSlots = 64;  // per token
constexpr unsigned kFull = 0xffffffffu;

// the expert of slot s, E for an unused one
template <typename I>
__device__ __forceinline__ int bin_of(const I* index, int64_t s, int E) {
  const I e = index[s];
  return e >= 0 && e < static_cast<I>(E) ? static_cast<int>(e) : E;
}

// exclusive scan of v over the block (kThreads threads); total in *sum
__device__ __forceinline__ int block_scan(int v, int* sum) {
  __shared__ int part[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(kFull, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // part may still be read from an earlier call
  if (lane == 31) part[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    before += w < warp ? part[w] : 0;
    all += part[w];
  }
  *sum = all;
  return before + x - v;
}

// ---- a row in pieces of type P (uint4: 16 bytes; otherwise one element)

template <typename T, typename P>
struct Piece {
  static constexpr int n = sizeof(P) / sizeof(T);
};
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(bf16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, typename P>
__device__ __forceinline__ void widen(const P& p, float (&f)[Piece<T, P>::n]) {
  const T* t = reinterpret_cast<const T*>(&p);
#pragma unroll
  for (int i = 0; i < Piece<T, P>::n; ++i) f[i] = to_f(t[i]);
}
template <typename T, typename P>
__device__ __forceinline__ P narrow(const float (&f)[Piece<T, P>::n]) {
  P p;
  T* t = reinterpret_cast<T*>(&p);
#pragma unroll
  for (int i = 0; i < Piece<T, P>::n; ++i) t[i] = from_f<T>(f[i]);
  return p;
}
template <typename P>
__device__ __forceinline__ P zero_piece() {
  P p;
  memset(&p, 0, sizeof(P));
  return p;
}

// ---- sort

// One block per token, and one more for the offsets.
// kKeep: the slots outside [0, E) are kept, as one more group behind the others
template <typename I, typename P, bool kKeep>
__global__ void __launch_bounds__(kThreads) small_kernel(const P* __restrict__ x,
                                                         const I* __restrict__ index,
                                                         P* __restrict__ xs, int* __restrict__ offsets,
                                                         int* __restrict__ position,
                                                         int* __restrict__ source, int N, int k, int E,
                                                         int64_t V) {
  const int S = N * k, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x == static_cast<unsigned>(N)) {
    __shared__ int count[kMaxExperts + 1];
    for (int e = threadIdx.x; e <= E; e += kThreads) count[e] = 0;
    __syncthreads();
    for (int s = threadIdx.x; s < S; s += kThreads) atomicAdd(&count[bin_of(index, s, E)], 1);
    __syncthreads();
    const int per = (E + kThreads) / kThreads;  // ceil((E + 1) / kThreads)
    const int first = threadIdx.x * per;
    int mine = 0, all;
    for (int e = first; e < first + per && e <= E; ++e) mine += count[e];
    int at = block_scan(mine, &all);
    for (int e = first; e < first + per && e <= E; ++e) {
      offsets[e] = at;
      at += count[e];
    }
    if (kKeep && threadIdx.x == 0) offsets[E + 1] = S;
    return;
  }
  __shared__ int row[kMaxSlots];
  const int n = blockIdx.x;
  for (int j = warp; j < k; j += kWarps) {
    const int s = n * k + j, b = bin_of(index, s, E);
    int before = 0;
    for (int i = lane; i < S; i += 32) {
      const int o = bin_of(index, i, E);
      before += o < b || (o == b && i < s);
    }
    before = __reduce_add_sync(kFull, before);
    if (lane == 0) {
      const bool used = kKeep || b < E;
      row[j] = used ? before : -1 - before;
      position[s] = used ? before : -1;
      source[before] = used ? s : -1;
    }
  }
  if (xs == nullptr) return;
  __syncthreads();
  for (int64_t v = threadIdx.x; v < V; v += kThreads) {
    const P p = x[n * V + v];
    for (int j = 0; j < k; ++j) {
      const int r = row[j];
      if (r >= 0)
        xs[r * V + v] = p;
      else
        xs[(-1 - r) * V + v] = zero_piece<P>();
    }
  }
}

constexpr int kSortThreads = 512, kSortWarps = kSortThreads / 32, kSortDeep = 4;

// slots per block, a multiple of kSortThreads: at most 256 blocks
inline int64_t chunk_of(int64_t S) {
  const int64_t c = ((S + 255) / 256 + kSortThreads - 1) / kSortThreads * kSortThreads;
  return c > 2 * kSortThreads ? c : 2 * kSortThreads;
}
// Whether each block counts all slots itself, one launch less: dearer on the device
// (every block reads all slots and sums a counter per warp and expert) and cheaper for
// the host, which bounds such calls.  us a call in a loop, with the copy of rows of
// 1024 bf16, so / in two launches, and on the device behind queued work: 2600 slots of 8
// experts 11.1 / 14.4 (10.3 / 8.3), 8192 of 8 12.4 / 14.5 (12.4 / 10.3), 8192 of 16
// 14.4 / 14.6 (14.4 / 10.3), 8192 of 24 16.4 / 14.6 (16.4 / 10.3), 8192 of 200 20.5 /
// 14.4 (20.6 / 12.4).
constexpr int kAloneExperts = 16;
inline bool alone(int64_t S, int64_t E) { return S <= 8192 && E <= kAloneExperts; }
// Shared memory of place_kernel, and the most that any call asks for (alone with few
// experts asks for little): the limit is set to that one, so that host threads with
// sorts of different sizes do not lower each other's before a launch.
constexpr int place_smem(bool solo, int E) {
  return ((solo ? 2 : 1) * kSortWarps + 2) * (E + 1) * static_cast<int>(sizeof(int));
}
constexpr int kPlaceSmem = place_smem(false, kMaxExperts);
static_assert(place_smem(true, kAloneExperts) <= kPlaceSmem, "the most of any call");
inline int64_t chunks_of(int64_t S) { return (S + chunk_of(S) - 1) / chunk_of(S); }

// slots of each expert in each chunk: counts[chunk][expert]
template <typename I>
__global__ void __launch_bounds__(kSortThreads) count_kernel(const I* __restrict__ index,
                                                             int* __restrict__ counts, int64_t S,
                                                             int64_t chunk, int E) {
  __shared__ int count[kMaxExperts + 1];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int e = threadIdx.x; e <= E; e += kSortThreads) count[e] = 0;
  __syncthreads();
  const int64_t s0 = blockIdx.x * chunk, s1 = s0 + chunk < S ? s0 + chunk : S;
  for (int64_t s = s0 + threadIdx.x; s < s1; s += kSortThreads) atomicAdd(&count[bin_of(index, s, E)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += kSortThreads)
    counts[static_cast<int64_t>(blockIdx.x) * (E + 1) + e] = count[e];
}

// The rows of a chunk's slots.  Warp w owns the w-th contiguous share of the
// chunk; `seen` counts a warp's slots of each expert, then holds the rows of the
// chunk before them.
template <typename I, bool kKeep>
__global__ void __launch_bounds__(kSortThreads)
    place_kernel(const I* __restrict__ index, const int* counts, int* __restrict__ offsets,
                 int* __restrict__ position, int* __restrict__ source, int64_t S, int64_t chunk, int E) {
  extern __shared__ int seen[];  // [kSortWarps][E + 1], then [E + 1] all slots, [E + 1] those of earlier chunks
  __shared__ int part[kSortWarps];
  int *all = seen + kSortWarps * (E + 1), *first = all + E + 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int i = threadIdx.x; i < (kSortWarps + 2) * (E + 1); i += kSortThreads) seen[i] = 0;
  __syncthreads();
  int* mine = seen + warp * (E + 1);
  const int64_t share = chunk / kSortWarps, s0 = blockIdx.x * chunk + warp * share;
  const int64_t s1 = s0 + share < S ? s0 + share : S;
  for (int64_t t = s0; t < s1; t += 32 * kSortDeep) {  // kSortDeep steps' loads at once
    int bin[kSortDeep];
#pragma unroll
    for (int u = 0; u < kSortDeep; ++u) {
      const int64_t s = t + 32 * u + lane;
      bin[u] = s < s1 ? bin_of(index, s, E) : E + 1;
    }
#pragma unroll
    for (int u = 0; u < kSortDeep; ++u)
      if (bin[u] <= E) atomicAdd(&mine[bin[u]], 1);
  }
  if (counts == nullptr) {  // the block counts all slots for itself, a warp's in its own counters
    int* temp = first + E + 1;  // [kSortWarps][E + 1]
    int* own = temp + warp * (E + 1);
    for (int i = threadIdx.x; i < kSortWarps * (E + 1); i += kSortThreads) temp[i] = 0;
    const int64_t cut = blockIdx.x * chunk;
    for (int half = 0; half < 2; ++half) {  // the slots before the chunk, then the others
      __syncthreads();  // temp is cleared; its sum over the first half is taken before the second adds to it
      const int64_t end = half == 0 ? cut : S;
      for (int64_t t = (half == 0 ? 0 : cut) + warp * 32; t < end; t += 32 * kSortWarps * kSortDeep) {
        int bin[kSortDeep];
#pragma unroll
        for (int u = 0; u < kSortDeep; ++u) {
          const int64_t s = t + u * 32 * kSortWarps + lane;
          bin[u] = s < end ? bin_of(index, s, E) : E + 1;
        }
#pragma unroll
        for (int u = 0; u < kSortDeep; ++u) {
          const unsigned same = __match_any_sync(kFull, bin[u]);
          if (bin[u] <= E && (same & ((1u << lane) - 1u)) == 0) own[bin[u]] += __popc(same);
          __syncwarp();
        }
      }
      __syncthreads();
      for (int e = threadIdx.x; e <= E; e += kSortThreads) {
        int n = 0;
        for (int w = 0; w < kSortWarps; ++w) n += temp[w * (E + 1) + e];
        (half == 0 ? first : all)[e] = n;
      }
    }
  } else {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the counts
    const int chunks = gridDim.x;
    for (int i = threadIdx.x; i < chunks * (E + 1); i += kSortThreads) {
      const int n = counts[i], c = i / (E + 1), e = i - c * (E + 1);
      if (n == 0) continue;
      atomicAdd(&all[e], n);
      if (c < static_cast<int>(blockIdx.x)) atomicAdd(&first[e], n);
    }
  }
  __syncthreads();
  // rows before expert e: a scan over the experts, `per` of them per thread
  const int per = (E + kSortThreads) / kSortThreads, e0 = threadIdx.x * per;
  int n = 0;
  for (int e = e0; e < e0 + per && e <= E; ++e) n += all[e];
  int x = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(kFull, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) part[warp] = x;
  __syncthreads();
  int at = x - n;
  for (int w = 0; w < warp; ++w) at += part[w];
  for (int e = e0; e < e0 + per && e <= E; ++e) {
    if (blockIdx.x == 0) offsets[e] = at;
    first[e] += at;
    at += all[e];
  }
  if (kKeep && blockIdx.x == 0 && threadIdx.x == 0) offsets[E + 1] = static_cast<int>(S);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += kSortThreads) {
    int r = first[e];
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = seen[w * (E + 1) + e];
      seen[w * (E + 1) + e] = r;
      r += c;
    }
  }
  __syncthreads();
  for (int64_t t = s0; t < s1; t += 32 * kSortDeep) {
    int bin[kSortDeep];
#pragma unroll
    for (int u = 0; u < kSortDeep; ++u) {
      const int64_t s = t + 32 * u + lane;
      bin[u] = s < s1 ? bin_of(index, s, E) : E + 1;
    }
#pragma unroll
    for (int u = 0; u < kSortDeep; ++u) {
      const unsigned same = __match_any_sync(kFull, bin[u]);
      const int ahead = __popc(same & ((1u << lane) - 1u));
      const int r = bin[u] <= E ? mine[bin[u]] + ahead : 0;
      __syncwarp();
      if (bin[u] <= E && ahead == 0) mine[bin[u]] += __popc(same);
      __syncwarp();
      if (bin[u] > E) continue;
      const bool used = kKeep || bin[u] < E;
      const int64_t s = t + 32 * u + lane;
      position[s] = used ? r : -1;
      source[r] = used ? static_cast<int>(s) : -1;
    }
  }
}

// ---- copies: blockDim.x threads along a row, blockDim.y groups of kTokens tokens
// kTokens apart; the first kTailBlocks blocks write zeros behind offsets[E].

constexpr int kTokens = 2, kTailBlocks = 148;

template <typename P>
__device__ __forceinline__ void zero_rows(const int* offsets, int E, P* rows, int64_t R, int64_t V) {
  const int64_t threads = static_cast<int64_t>(blockDim.x) * blockDim.y;
  const int64_t used = offsets[E] > 0 ? offsets[E] : 0;
  for (int64_t i = used * V + blockIdx.x * threads + threadIdx.y * blockDim.x + threadIdx.x; i < R * V;
       i += kTailBlocks * threads)
    rows[i] = zero_piece<P>();
}

template <typename P>
__global__ void __launch_bounds__(kThreads) copy_kernel(const P* __restrict__ x, const int* position,
                                                        const int* offsets, P* __restrict__ xs, int64_t N, int k,
                                                        int E, int64_t V, bool tail) {
  if (tail && blockIdx.x < kTailBlocks) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    zero_rows(offsets, E, xs, N * k, V);
    return;
  }
  const int64_t n0 = (static_cast<int64_t>(blockIdx.x) - (tail ? kTailBlocks : 0)) * (blockDim.y * kTokens) + threadIdx.y;
  for (int64_t v = threadIdx.x; v < V; v += blockDim.x) {
    P p[kTokens];
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      const int64_t n = n0 + u * blockDim.y;
      p[u] = n < N ? x[n * V + v] : zero_piece<P>();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the sort, which the loads of x do not need
    for (int j0 = 0; j0 < k; j0 += 4) {  // the rows of four slots, then their stores
      int r[kTokens][4];
#pragma unroll
      for (int u = 0; u < kTokens; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t n = n0 + u * blockDim.y;
          r[u][j] = n < N && j0 + j < k ? position[n * k + j0 + j] : -1;
        }
#pragma unroll
      for (int u = 0; u < kTokens; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r[u][j] >= 0) xs[r[u][j] * V + v] = p[u];  // below N k: the sort's own
    }
  }
}

// kPer tokens per thread
template <typename T, typename P, bool kWeighted, int kPer>
__global__ void __launch_bounds__(kThreads) combine_kernel(const P* __restrict__ rows,
                                                           const float* __restrict__ weight,
                                                           const int* __restrict__ position,
                                                           P* __restrict__ out, int64_t N, int k,
                                                           int64_t V) {
  constexpr int n_el = Piece<T, P>::n;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (blockDim.y * kPer) + threadIdx.y;
  for (int64_t v = threadIdx.x; v < V; v += blockDim.x) {
    float acc[kPer][n_el];
#pragma unroll
    for (int u = 0; u < kPer; ++u)
#pragma unroll
      for (int i = 0; i < n_el; ++i) acc[u][i] = 0.0f;
    for (int j0 = 0; j0 < k; j0 += 2) {  // the loads of two slots of all tokens, then their sums
      int64_t r[kPer][2];
      P p[kPer][2];
#pragma unroll
      for (int u = 0; u < kPer; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int64_t n = n0 + u * blockDim.y;
          r[u][j] = n < N && j0 + j < k ? position[n * k + j0 + j] : -1;
          if (r[u][j] >= N * k) r[u][j] = -1;
        }
#pragma unroll
      for (int u = 0; u < kPer; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (r[u][j] >= 0) p[u][j] = rows[r[u][j] * V + v];
#pragma unroll
      for (int u = 0; u < kPer; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (r[u][j] < 0) continue;
          float f[n_el];
          widen<T, P>(p[u][j], f);
          const float w = kWeighted ? weight[(n0 + u * blockDim.y) * k + j0 + j] : 1.0f;
#pragma unroll
          for (int i = 0; i < n_el; ++i) acc[u][i] = kWeighted ? fmaf(w, f[i], acc[u][i]) : acc[u][i] + f[i];
        }
    }
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int64_t n = n0 + u * blockDim.y;
      if (n < N) out[n * V + v] = narrow<T, P>(acc[u]);
    }
  }
}

// a warp per token: its row of dout is held while its slots' rows are read and written
template <typename T, typename P>
__global__ void __launch_bounds__(kThreads) combine_bwd_kernel(
    const P* __restrict__ dout, const P* __restrict__ ys, const float* __restrict__ weight,
    const int* __restrict__ position, const int* __restrict__ offsets, P* __restrict__ dys,
    float* __restrict__ dweight, int64_t N, int k, int E, int64_t V) {
  constexpr int n_el = Piece<T, P>::n, kGroup = 2, kDeep = 4;
  if (dys != nullptr && blockIdx.x < kTailBlocks) {
    zero_rows(offsets, E, dys, N * k, V);
    return;
  }
  const int lane = threadIdx.x & 31;
  const int64_t n = (static_cast<int64_t>(blockIdx.x) - (dys != nullptr ? kTailBlocks : 0)) * kWarps + (threadIdx.x >> 5);
  if (n >= N) return;
  for (int j0 = 0; j0 < k; j0 += kGroup) {
    int64_t r[kGroup];
    float w[kGroup], dot[kGroup];
#pragma unroll
    for (int j = 0; j < kGroup; ++j) {
      r[j] = j0 + j < k ? position[n * k + j0 + j] : -1;
      if (r[j] >= N * k) r[j] = -1;
      w[j] = r[j] >= 0 ? weight[n * k + j0 + j] : 0.0f;
      dot[j] = 0.0f;
    }
    for (int64_t v0 = lane; v0 < V; v0 += 32 * kDeep) {
      P d[kDeep], y[kDeep][kGroup];
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        const int64_t v = v0 + 32 * u;
        if (v >= V) continue;
        d[u] = dout[n * V + v];
#pragma unroll
        for (int j = 0; j < kGroup; ++j)
          if (r[j] >= 0 && dweight != nullptr) y[u][j] = ys[r[j] * V + v];
      }
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        const int64_t v = v0 + 32 * u;
        if (v >= V) continue;
        float df[n_el];
        widen<T, P>(d[u], df);
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
          if (r[j] < 0) continue;
          float g[n_el];
          if (dweight != nullptr) {
            widen<T, P>(y[u][j], g);
#pragma unroll
            for (int i = 0; i < n_el; ++i) dot[j] = fmaf(df[i], g[i], dot[j]);
          }
          if (dys != nullptr) {
#pragma unroll
            for (int i = 0; i < n_el; ++i) g[i] = w[j] * df[i];
            dys[r[j] * V + v] = narrow<T, P>(g);
          }
        }
      }
    }
    if (dweight != nullptr) {
#pragma unroll
      for (int j = 0; j < kGroup; ++j) {
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) dot[j] += __shfl_xor_sync(kFull, dot[j], m);
        if (lane == 0 && j0 + j < k) dweight[n * k + j0 + j] = r[j] >= 0 ? dot[j] : 0.0f;
      }
    }
  }
}

// threads along a row of V pieces: a power of two from 32 to kThreads
inline dim3 row_block(int64_t V) {
  int tx = 32;
  while (tx < kThreads && tx < V) tx *= 2;
  return dim3(tx, kThreads / tx);
}
inline int64_t blocks(int64_t N, const dim3& b, int per) { return (N + b.y * per - 1) / (b.y * per); }

// C elements of 2 or 4 bytes as 16-byte pieces: 0 where that cannot be
template <typename... Ptr>
int64_t pieces(int64_t C, int size, Ptr... p) {
  uintptr_t all = 0;
  ((all |= reinterpret_cast<uintptr_t>(p)), ...);
  return (C * size) % 16 == 0 && (all & 15u) == 0 ? C * size / 16 : 0;
}

// whether all pointers are at multiples of `size` bytes
template <typename... Ptr>
bool at_multiples(int size, Ptr... p) {
  uintptr_t all = 0;
  ((all |= reinterpret_cast<uintptr_t>(p)), ...);
  return all % static_cast<uintptr_t>(size) == 0;
}

int check(int64_t N, int64_t k, int64_t E, int64_t C, int dtype) {
  if (dtype != 0 && dtype != 1) return 2;
  if (N < 0 || k < 1 || E < 1 || C < 0) return 1;
  if (k > kMaxSlots || E > kMaxExperts) return 2;
  if (N > 0x7fffffffLL / k || C > 0x7fffffffLL) return 3;
  return 0;
}

template <typename I, typename P, bool kKeep>
int sort(const P* x, const I* index, P* xs, int* offsets, int* position, int* source, int* work, int64_t N, int k, int E, int64_t V, cudaStream_t st) {
  const int64_t S = N * k;
  if (S <= kSmallSlots) {
    small_kernel<I, P, kKeep><<<static_cast<unsigned>(N + 1), kThreads, 0, st>>>(
        x, index, xs, offsets, position, source, static_cast<int>(N), k, E, V);
    return camoe::tm::status(cudaGetLastError());
  }
  const int64_t chunk = chunk_of(S);
  const unsigned g = static_cast<unsigned>(chunks_of(S));
  const bool solo = alone(S, E);
  if (!solo) {
    count_kernel<I><<<g, kSortThreads, 0, st>>>(index, work, S, chunk, E);
    if (const int e = camoe::tm::status(cudaGetLastError())) return e;
  }
  const int smem = place_smem(solo, E);
  const auto place = place_kernel<I, kKeep>;
  if (smem > 48 * 1024)
    if (const int e = camoe::tm::status(cudaFuncSetAttribute(place, cudaFuncAttributeMaxDynamicSharedMemorySize, kPlaceSmem)))
      return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(g);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = solo ? 0 : 1;  // by itself it reads the index at once
  if (const int e = camoe::tm::status(cudaLaunchKernelEx(&cfg, place, index,
                                                         static_cast<const int*>(solo ? nullptr : work), offsets,
                                                         position, source, S, chunk, E)))
    return e;
  if (xs == nullptr || V == 0) return 0;
  const dim3 b = row_block(V);
  cfg.gridDim = dim3(static_cast<unsigned>(blocks(N, b, kTokens) + (kKeep ? 0 : kTailBlocks)));
  cfg.blockDim = b;
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return camoe::tm::status(cudaLaunchKernelEx(&cfg, copy_kernel<P>, x, static_cast<const int*>(position),
                                              static_cast<const int*>(offsets), xs, N, k, E, V, !kKeep));
}

template <typename P>
int sort_index(const void* x, const void* index, int index_bytes, void* xs, int* offsets, int* position,
               int* source, int* work, int64_t N, int k, int E, int64_t V, cudaStream_t st) {
  const P* xp = static_cast<const P*>(x);
  P* xsp = static_cast<P*>(xs);
  return index_bytes == 4
             ? sort<int32_t, P, false>(xp, static_cast<const int32_t*>(index), xsp, offsets, position,
                                       source, work, N, k, E, V, st)
             : sort<int64_t, P, false>(xp, static_cast<const int64_t*>(index), xsp, offsets, position,
                                       source, work, N, k, E, V, st);
}

size_t sort_bytes(int64_t N, int64_t k, int64_t E) {
  if (N * k <= kSmallSlots || alone(N * k, E)) return 0;
  return static_cast<size_t>(chunks_of(N * k)) * static_cast<size_t>(E + 1) * sizeof(int);
}

// For the adapters (adapters.cu): rows of 16-byte pieces by their group, the rows of no group behind
// the others; offsets has L + 2 entries, row r of xs is row source[r] of x.
int sort_rows(const void* x, const int* group, void* xs, int* offsets, int* position, int* source,
              void* work, int64_t N, int L, int64_t V, cudaStream_t st) {
  return sort<int32_t, uint4, true>(static_cast<const uint4*>(x), group, static_cast<uint4*>(xs), offsets,
                                    position, source, static_cast<int*>(work), N, 1, L, V, st);
}

template <typename T, typename P>
int combine(const void* in, const float* weight, const int* position, void* out, int64_t N, int k,
            int64_t V, cudaStream_t st) {
  const dim3 b = row_block(V);
  const P* p = static_cast<const P*>(in);
  P* o = static_cast<P*>(out);
  // few tokens: one per thread, so that all SMs have some
  const bool many = N >= 4096;
  const unsigned g = static_cast<unsigned>(blocks(N, b, many ? 2 : 1));
  if (weight != nullptr) {
    if (many)
      combine_kernel<T, P, true, 2><<<g, b, 0, st>>>(p, weight, position, o, N, k, V);
    else
      combine_kernel<T, P, true, 1><<<g, b, 0, st>>>(p, weight, position, o, N, k, V);
  } else if (many) {
    combine_kernel<T, P, false, 2><<<g, b, 0, st>>>(p, weight, position, o, N, k, V);
  } else {
    combine_kernel<T, P, false, 1><<<g, b, 0, st>>>(p, weight, position, o, N, k, V);
  }
  return camoe::tm::status(cudaGetLastError());
}

template <typename T, typename P>
int combine_bwd(const void* dout, const void* ys, const float* weight, const int* offsets,
                const int* position, void* dys, float* dweight, int64_t N, int k, int E, int64_t V,
                cudaStream_t st) {
  const int64_t g = (N + kWarps - 1) / kWarps + (dys != nullptr ? kTailBlocks : 0);
  combine_bwd_kernel<T, P><<<static_cast<unsigned>(g), kThreads, 0, st>>>(
      static_cast<const P*>(dout), static_cast<const P*>(ys), weight, position, offsets, static_cast<P*>(dys),
      dweight, N, k, E, V);
  return camoe::tm::status(cudaGetLastError());
}

}  // namespace rows
}  // namespace camoe

extern "C" {

size_t camoe_ex_dispatch_work_bytes(int64_t N, int64_t k, int64_t E) {
  using namespace camoe::rows;
  return check(N, k, E, 1, 0) == 0 ? sort_bytes(N, k, E) : 0;
}

int camoe_ex_dispatch(const void* x, int dtype, const void* index, int index_bytes, void* xs,
                      int32_t* offsets, int32_t* position, int32_t* source, void* work,
                      size_t work_bytes, int64_t N, int64_t k, int64_t E, int64_t C, void* stream) {
  using namespace camoe::rows;
  if (const int st = check(N, k, E, C, dtype)) return st;
  if (index_bytes != 4 && index_bytes != 8) return 2;
  if (offsets == nullptr) return 1;
  if (!at_multiples(4, offsets)) return 4;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (N == 0)
    return camoe::tm::status(cudaMemsetAsync(offsets, 0, static_cast<size_t>(E + 1) * sizeof(int), s));
  if (index == nullptr || position == nullptr || source == nullptr || (xs != nullptr && x == nullptr)) return 1;
  if (!at_multiples(dtype == 0 ? 2 : 4, x, xs) || !at_multiples(index_bytes, index) ||
      !at_multiples(4, offsets, position, source, work))
    return 4;
  const size_t need = sort_bytes(N, k, E);
  if (need > 0 && work == nullptr) return 1;
  if (work_bytes < need) return 5;
  int* w = static_cast<int*>(work);
  const int kk = static_cast<int>(k), e = static_cast<int>(E);
  const int64_t V = pieces(C, dtype == 0 ? 2 : 4, x, xs);
  if (V > 0) return sort_index<uint4>(x, index, index_bytes, xs, offsets, position, source, w, N, kk, e, V, s);
  if (dtype == 0)
    return sort_index<uint16_t>(x, index, index_bytes, xs, offsets, position, source, w, N, kk, e, C, s);
  return sort_index<uint32_t>(x, index, index_bytes, xs, offsets, position, source, w, N, kk, e, C, s);
}

int camoe_ex_combine(const void* in, int dtype, const float* weight, const int32_t* position, void* out,
                     int64_t N, int64_t k, int64_t C, void* stream) {
  using namespace camoe;
  using namespace camoe::rows;
  if (const int st = check(N, k, 1, C, dtype)) return st;
  if (N == 0 || C == 0) return 0;
  if (in == nullptr || position == nullptr || out == nullptr) return 1;
  if (!at_multiples(dtype == 0 ? 2 : 4, in, out) || !at_multiples(4, weight, position)) return 4;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int kk = static_cast<int>(k);
  const int64_t V = pieces(C, dtype == 0 ? 2 : 4, in, out);
  if (dtype == 0)
    return V > 0 ? combine<bf16, uint4>(in, weight, position, out, N, kk, V, s)
                 : combine<bf16, bf16>(in, weight, position, out, N, kk, C, s);
  return V > 0 ? combine<float, uint4>(in, weight, position, out, N, kk, V, s)
               : combine<float, float>(in, weight, position, out, N, kk, C, s);
}

int camoe_ex_combine_bwd(const void* dout, int dtype, const void* ys, const float* weight,
                         const int32_t* offsets, const int32_t* position, void* dys, float* dweight,
                         int64_t N, int64_t k, int64_t E, int64_t C, void* stream) {
  using namespace camoe;
  using namespace camoe::rows;
  if (const int st = check(N, k, E, C, dtype)) return st;
  if (N == 0 || (dys == nullptr && dweight == nullptr)) return 0;
  if (position == nullptr || weight == nullptr || (dys != nullptr && offsets == nullptr)) return 1;
  if (C > 0 && (dout == nullptr || (dweight != nullptr && ys == nullptr))) return 1;
  if (!at_multiples(dtype == 0 ? 2 : 4, dout, ys, dys) || !at_multiples(4, weight, offsets, position, dweight)) return 4;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int kk = static_cast<int>(k), e = static_cast<int>(E);
  const int64_t V = pieces(C, dtype == 0 ? 2 : 4, dout, ys, dys);
  if (dtype == 0)
    return V > 0 ? combine_bwd<bf16, uint4>(dout, ys, weight, offsets, position, dys, dweight, N, kk, e, V, s)
                 : combine_bwd<bf16, bf16>(dout, ys, weight, offsets, position, dys, dweight, N, kk, e, C, s);
  return V > 0 ? combine_bwd<float, uint4>(dout, ys, weight, offsets, position, dys, dweight, N, kk, e, V, s)
               : combine_bwd<float, float>(dout, ys, weight, offsets, position, dys, dweight, N, kk, e, C, s);
}

}  // extern "C"
