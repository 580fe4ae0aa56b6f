// Products of grouped rows on the 5th-generation tensor cores (tcgen05): one
// kernel for the experts' six products and the adapters' two.
//
// kRows: for the rows p of group g (p in [offsets[g], offsets[g + 1]))
//     out[p][n] = sum over k of A[p][k] B_g[n][k]
//   A's rows have k contiguous; B_g is stored [N][K] (k contiguous) or [K][N]
//   (n contiguous), which is a bit of the instruction descriptor.
// kWeights (weight gradients): out_g[m][n] = sum over the rows p of g of
//   A[p][m] B[p][n], both stored with m or n contiguous.
// kBlocks and kJoined (adapters), over row tiles of the whole array, which the
//   groups' rows cut as they may:
//   kBlocks: for each group and row tile that share rows a block of the tile's
//     rows with the group's product in its own rows and zeros in the others;
//   kJoined: out[p][n] = sum over k of A[p][k] B[n][k] + sum over the groups g of
//     p's tile of sum over d of block[p][d] B2_g[n][d].  A group's product leaves
//     the accumulator's other rows as they are (zeros there would not do: 0 x inf
//     is NaN, and one group's B2 would reach the rows of the others).
//
// One pair of CTAs on two SMs (kCG = 2) per tile of 128 kCG rows x kBN
// columns, persistent over the tiles:
//   * warp 0 streams 64-deep pieces of A and B through a ring of stages by TMA
//     (128-byte swizzle); a piece that passes the end of a matrix reads zeros;
//   * warp 1 issues the products, K = 16 at a time, into one of two accumulators
//     in tensor memory, so that
//   * warps 2-9 read the other one (an output row per thread) and write the
//     previous tile meanwhile, turned through shared memory so that a warp's
//     stores are 64-byte row segments.
// A row tile starts at its group's first row and may reach into the next
// group's rows: those outputs are not written.  Where the sum runs over the
// rows (weight gradients) the last piece of a group is cleared behind the
// group's last row in both operands (0 x inf would not be 0).
//
// A pair splits a tile by rows for A and the output and by columns for B, so each
// SM loads half of B: 32 KB instead of 48 KB per 64-deep piece of 128 x 256
// outputs per SM.
//
// Every wait on an mbarrier is bounded (wkv7_sync.cuh); a wait that runs out is
// counted in camoe_wkv7_device_errors() and ends the roles' loops.
#pragma once

#include "wkv7_common.cuh"
#include "wkv7_sync.cuh"
#include "wkv7_tma.cuh"

namespace camoe {
namespace tc {

constexpr int kCG = 2;            // CTAs of a tile: a pair, on two SMs
constexpr int kBK = 64;           // depth of a stage: one 128-byte swizzled row of bf16
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;  // producer, product issue, epilogue
constexpr int kMaxGroups = 1025;  // 1024 and the rows of no group
constexpr int kRingBytes = 192 * 1024;
constexpr uint32_t kBox = 64 * 128;  // a box of 64 columns x 64 rows

enum Mode : int { kRows = 0, kWeights = 1, kBlocks = 2, kJoined = 3 };
enum Epilogue : int {
  kPlain = 0,   // out = acc
  kRelu2 = 1,   // out = relu(acc)^2
  kDRelu2 = 2,  // out = acc 2 sqrt(h): the derivative of relu^2 from its value (maps ma2: h, mlow: low)
  kScale = 3,   // out = acc scale[group]
};

// rows of low start at multiples of 16 bytes
__host__ __device__ constexpr int64_t low_stride(int64_t n) { return (n + 15) / 16 * 16; }

struct Args {
  const int* offsets;    // [groups + 1]
  int groups;
  int64_t R;             // rows of A (the sorted arrays)
  int M, N, K;           // M: weight gradients only
  int K2;                // kJoined: depth of the blocks (maps ma2: blocks, mb2: B2)
  int M2, N2;            // kWeights: a second product in the same launch, or 0 (maps ma2, mb2, mlow: out2)
  bf16* out2;
  int zero_tail;         // write zeros to the rows behind the last group
  bf16* out;
  int8_t* low;           // [R, low_stride(N)] (kRelu2, kDRelu2) or null: the 8 bits of the value below bf16's
  const float* scale;    // [groups] or null (kScale)
  const int* scatter;    // output row of row p, or null
};

// Per epilogue warp: 32 rows x 32 columns of bf16, and of bytes
constexpr uint32_t kOutBytes = 32 * 64, kLowBytes = 32 * 32;

template <int kBN, int kEpi>
struct Shape {
  static constexpr int kBM = 128 * kCG;
  static constexpr uint32_t kABytes = 128 * 128;          // per CTA and stage
  static constexpr uint32_t kBBytes = kBN / kCG * 128;
  // kDRelu2 reads h a step ahead: two staging buffers per warp, in place of a stage
  static constexpr int kBufs = kEpi == kDRelu2 ? 2 : 1;
  static constexpr int kFit = (kRingBytes - (kBufs - 1) * kEpiWarps * static_cast<int>(kOutBytes + kLowBytes)) / (kABytes + kBBytes);
  static constexpr int kStages = kFit < 10 ? kFit : 10;
  static constexpr uint32_t kStaging = kEpiWarps * kBufs * (kOutBytes + kLowBytes);
  // columns of B in a TMA box: half of a CTA's share, or 64 where they are contiguous
  __host__ __device__ static constexpr int box(bool mn) { return mn ? 64 : (kBN == 256 ? kBN / kCG / 2 : kBN / kCG); }
  static constexpr uint32_t kCols = 2 * kBN;              // two accumulators
};

struct Control {
  uint64_t full[10], empty[10], tail[10], peer_tail[10], acc_full[2], acc_empty[2], drained, aux[kEpiWarps][2];
  uint32_t tmem;
  int tiles[kMaxGroups + 1];  // row tiles of the groups before each
  int first[kMaxGroups + 1];  // the groups' first rows, clamped to R
};

template <int kBN, int kEpi>
__host__ __device__ constexpr int smem_bytes() {
  using Sh = Shape<kBN, kEpi>;
  return Sh::kStages * static_cast<int>(Sh::kABytes + Sh::kBBytes) + static_cast<int>(Sh::kStaging) +
         static_cast<int>(sizeof(Control)) + 1024;
}

// ---- PTX

// mbarrier address in the CTA `rank` of the pair
__device__ __forceinline__ uint32_t bar_at(uint64_t* bar, uint32_t rank) {
  uint32_t a = sm_addr(bar);
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(rank));
  return a;
}
// The scopes matter for speed: a release or an acquire at cluster scope waits
// for the thread's memory traffic (0.8 us per stage of the ring when every
// stage's barrier had them), and the ring needs none: TMA and the products order
// themselves, and the epilogue's tcgen05 fences order tensor memory.  Only the
// pieces that a CTA clears by ordinary stores are released to the pair's leader.
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_release(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// bounded wait that sees what the pair's other CTA released
__device__ __forceinline__ bool wait_acquire(uint64_t* bar, uint32_t parity) {
  long long t0 = 0, limit = 0;
  while (true) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(sm_addr(bar)), "r"(parity)
        : "memory");
    if (done) return true;
    if (limit == 0) {
      t0 = clock64();
      limit = *static_cast<volatile long long*>(&g_wkv7_wait_limit);
    } else if (clock64() - t0 > limit) {
      atomicAdd(&g_wkv7_timeouts, 1u);
      return false;
    }
  }
}
// the whole warp waits, and leaves together when one of its lanes gave up
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}
// box at (x, y, z) into this CTA's shared memory, completing on the barrier at `bar`
template <int kCtas>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                         uint32_t bar) {
  if (kCtas > 1)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
template <int kCtas>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  if (kCtas > 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm_addr(slot)),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm_addr(slot)),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <int kCtas>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
  if (kCtas > 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}
template <int kCtas>
__device__ __forceinline__ void mma(uint32_t tmem, uint64_t da, uint64_t db, uint32_t idesc, bool add) {
  if (kCtas > 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem),
        "l"(da), "l"(db), "r"(idesc), "r"(add ? 1u : 0u)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem),
        "l"(da), "l"(db), "r"(idesc), "r"(add ? 1u : 0u)
        : "memory");
}
// Which of a pair's 256 accumulator rows a product leaves as they are: bit r % 32 of
// word r / 32 for row r, all but rows [first, end).
struct Rows {
  uint32_t off[8];
  __device__ __forceinline__ void all_but(int first, int end) {
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const int lo = first - 32 * w, hi = end - 32 * w;
      const uint32_t below = lo <= 0 ? 0u : (lo < 32 ? (1u << lo) - 1u : ~0u);
      const uint32_t from = hi >= 32 ? 0u : (hi > 0 ? ~0u << hi : ~0u);
      off[w] = below | from;
    }
  }
};
// a pair's product that adds to the other rows only
__device__ __forceinline__ void mma_rows(uint32_t tmem, uint64_t da, uint64_t db, uint32_t idesc, const Rows& r) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, 1, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%4, %5, %6, %7, %8, %9, %10, %11}, p;\n\t}\n" ::"r"(tmem),
      "l"(da), "l"(db), "r"(idesc), "r"(r.off[0]), "r"(r.off[1]), "r"(r.off[2]), "r"(r.off[3]), "r"(r.off[4]),
      "r"(r.off[5]), "r"(r.off[6]), "r"(r.off[7])
      : "memory");
}
// arrive on the barrier (in both CTAs of a pair) once the products issued so far are done
template <int kCtas>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if (kCtas > 1)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            sm_addr(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(sm_addr(bar))
                 : "memory");
}
// true in one lane of the (converged) warp, the same one each time
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}" : "=r"(p));
  return p != 0;
}
// box at (x, y) of a map from this CTA's shared memory (bulk-group completion)
__device__ __forceinline__ void store_box(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(x), "r"(y), "r"(0), "r"(src)
      : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 32 consecutive accumulator columns of this thread's TMEM lane (the wait is in the
// same statement, so that no use of v can be moved before it)
__device__ __forceinline__ void ld32(uint32_t (&v)[32], uint32_t taddr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
        "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
        "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle (layout type 2), descriptor
// version 1, 1024 bytes between groups of 8 rows.  K contiguous: the rows are M
// (or N) and the leading offset is not used.  M (or N) contiguous: the rows are
// K and the leading offset is the bytes between boxes of 64 columns.
template <bool kMN>
__device__ __forceinline__ uint64_t desc(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) |
         (static_cast<uint64_t>(kMN ? (kBox >> 4) : 1u) << 16) | (static_cast<uint64_t>(1024u >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// bytes between K = 16 steps within a stage
template <bool kMN>
constexpr uint32_t kStep = kMN ? 16 * 128 : 32;

// Instruction descriptor of kind::f16: fp32 accumulator, bf16 A and B, the
// operands' majors (bits 15, 16: set for M or N contiguous), N / 8, M / 16.
template <bool kAMN, bool kBMN>
__host__ __device__ constexpr uint32_t instr(int M, int N) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (kAMN ? 1u << 15 : 0u) | (kBMN ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// ---- tiles

struct Tile {
  int group, n0, width;  // width: columns, kBN or half of it
  int64_t row0, row1;  // the group's rows from the tile's first (weight gradients: all of the group's)
  int m0;              // weight gradients: first output row
  int nk1, nk;         // pieces of the first pair, of both
  int tile;            // kBlocks: block; kJoined: row tile
  int64_t lead;        // kBlocks: rows of the tile before the group's
  bool second;         // kWeights: of the second product
};

template <int kBN, int kMode>
struct Tiles {
  const Args& a;
  const Control& c;
  int nt, mt, nt2, mt2;
  int whole, jobs;  // tiles done whole, and these with the halves of the others
  __device__ Tiles(const Args& args, const Control& ctl) : a(args), c(ctl) {
    nt = (a.N + kBN - 1) / kBN;
    mt = kMode == kWeights ? (a.M + (128 * kCG) - 1) / (128 * kCG) : 0;
    nt2 = kMode == kWeights ? (a.N2 + kBN - 1) / kBN : 0;
    mt2 = kMode == kWeights ? (a.M2 + (128 * kCG) - 1) / (128 * kCG) : 0;
    const int total = kMode == kWeights ? a.groups * (mt * nt + mt2 * nt2)
                      : kMode == kJoined ? static_cast<int>((a.R + 128 * kCG - 1) / (128 * kCG)) * nt
                                         : c.tiles[a.groups] * nt;
    // Tiles left for a last round that would leave half of the workers or more
    // without one are done as halves of kBN / 2 columns, which take half the time.
    const int workers = gridDim.x / kCG, left = total % workers;
    const bool halves = kBN == 256 && 2 * left <= workers;
    whole = halves ? total - left : total;
    jobs = halves ? whole + 2 * left : total;
  }
  __device__ int64_t first(int g) const { return c.first[g]; }
  // kJoined: the first group at or behind g with rows of the row tile, `groups` if none
  __device__ int next_group(int g, int tile) const {
    const int64_t end = static_cast<int64_t>(tile + 1) * (128 * kCG);
    while (g < a.groups && c.first[g + 1] <= c.first[g]) ++g;
    return g < a.groups && c.first[g] < end ? g : a.groups;
  }
  __device__ int group_at(int64_t row) const {  // the last group that starts at or before the row
    int lo = 0, hi = a.groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (c.first[mid] <= row) lo = mid; else hi = mid;
    }
    return lo;
  }
  __device__ Tile get(int job) const {
    Tile x;
    int t = job < whole ? job : whole + (job - whole) / 2;
    x.second = kMode == kWeights && t >= a.groups * mt * nt;
    if (x.second) t -= a.groups * mt * nt;
    const int nts = x.second ? nt2 : nt, mts = x.second ? mt2 : mt;
    const int rt = t / nts;
    x.width = job < whole ? kBN : kBN / 2;
    x.n0 = (t - rt * nts) * kBN + (job < whole ? 0 : (job - whole) % 2 * (kBN / 2));
    if (kMode == kWeights) {
      x.group = rt / mts;
      x.m0 = (rt - x.group * mts) * (128 * kCG);
      x.row0 = first(x.group);
      x.row1 = first(x.group + 1);
      x.nk1 = x.nk = x.row1 > x.row0 ? static_cast<int>((x.row1 - x.row0 + kBK - 1) / kBK) : 0;
    } else if (kMode == kJoined) {
      x.group = group_at(static_cast<int64_t>(rt) * (128 * kCG));
      if (c.first[x.group + 1] <= static_cast<int64_t>(rt) * (128 * kCG)) ++x.group;  // ends before the tile
      x.m0 = 0;
      x.tile = rt;
      x.row0 = static_cast<int64_t>(rt) * (128 * kCG);
      x.row1 = a.R;
      x.nk1 = x.nk = (a.K + kBK - 1) / kBK;
      const int each = (a.K2 + kBK - 1) / kBK;
      for (int g = next_group(x.group, rt); g < a.groups; g = next_group(g + 1, rt)) x.nk += each;
    } else {
      int lo = 0, hi = a.groups;  // the last group whose first row tile is at most rt
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (c.tiles[mid] <= rt) lo = mid; else hi = mid;
      }
      x.group = lo;
      x.m0 = 0;
      x.tile = rt;
      x.row0 = first(lo) + static_cast<int64_t>(rt - c.tiles[lo]) * (128 * kCG);
      x.row1 = first(lo + 1);
      if (kMode == kBlocks) {
        x.row0 = (first(lo) / (128 * kCG) + rt - c.tiles[lo]) * (128 * kCG);
        x.lead = first(lo) - x.row0;
      }
      x.nk1 = x.nk = (a.K + kBK - 1) / kBK;
    }
    return x;
  }
};

// A value as its bf16 rounding and 8 more bits: what an operand of the products
// cannot hold but a derivative can use.  d: the value's bits behind the rounded
// one's, rounded to a multiple of 256; its second byte is kept.
__device__ __forceinline__ int low_word(float v, uint32_t hi) {
  const int d = static_cast<int>(__float_as_uint(v) - hi + 128u);
  return d < 32767 ? d : 32767;
}
__device__ __forceinline__ int low_bits(float v, bf16 hi) {
  return low_word(v, static_cast<uint32_t>(__bfloat16_as_ushort(hi)) << 16) >> 8;
}
// byte i of `low`, signed, in place
template <int i>
__device__ __forceinline__ float with_low(uint32_t hi, uint32_t low) {
  uint32_t d;  // bytes 3 and 2: the byte's sign (bit 3 of a selector), 1: the byte, 0: zero
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(low), "r"(0u), "n"((8 + i) << 12 | (8 + i) << 8 | i << 4 | 4));
  return __uint_as_float(hi + d);
}
// one instruction, 1 ulp: its result is multiplied and rounded to bf16
__device__ __forceinline__ float fast_sqrt(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float relu(float x) {  // NaN stays NaN
  float y;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
  return y;
}
template <int kEpi>
__device__ __forceinline__ float finish(float x, float aux, float scale) {
  if (kEpi == kRelu2) {
    const float y = relu(x);
    return y * y;
  }
  if (kEpi == kDRelu2) return x * (2.0f * fast_sqrt(aux));
  if (kEpi == kScale) return x * scale;
  return x;
}

// 16-byte piece q of row r in a warp's staging buffers: swizzled (as TMA swizzles rows
// of 64 and of 32 bytes), so that both a thread per row and four (two) threads
// per row touch all banks
__device__ __forceinline__ uint32_t out_at(int r, int q) { return r * 64 + ((q ^ ((r >> 1) & 3)) << 4); }
__device__ __forceinline__ uint32_t low_at(int r, int q) { return r * 32 + ((q ^ ((r >> 2) & 1)) << 4); }

template <int kBN, bool kAMN, bool kBMN, int kMode, int kEpi>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb,
                const __grid_constant__ CUtensorMap ma2, const __grid_constant__ CUtensorMap mb2,
                const __grid_constant__ CUtensorMap mo, const __grid_constant__ CUtensorMap mlow, const Args a) {
  using Sh = Shape<kBN, kEpi>;
  constexpr int S = Sh::kStages, kBBox = Sh::box(kBMN);
  constexpr uint32_t kStage = Sh::kABytes + Sh::kBBytes;
  extern __shared__ __align__(128) unsigned char raw[];
  unsigned char* ring = raw + ((1024u - (sm_addr(raw) & 1023u)) & 1023u);
  unsigned char* staging = ring + S * kStage;
  Control& c = *reinterpret_cast<Control*>(staging + Sh::kStaging);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int worker = blockIdx.x / kCG, workers = gridDim.x / kCG;

  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&ma)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&mb)) : "memory");
    for (int s = 0; s < S; ++s) {
      mbar_init(&c.full[s], 1);
      mbar_init(&c.empty[s], 1);
      mbar_init(&c.tail[s], 1);
      mbar_init(&c.peer_tail[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&c.acc_full[b], 1);
      mbar_init(&c.acc_empty[b], kEpiWarps * kCG);
    }
    mbar_init(&c.drained, 1);
    for (int w = 0; w < kEpiWarps; ++w)
      for (int b = 0; b < Sh::kBufs; ++b) mbar_init(&c.aux[w][b], 1);
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc<kCG>(&c.tmem, Sh::kCols);
  // Up to here the kernel may run beside the one before it in the stream
  // (programmatic dependent launch); what follows reads what that one wrote.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 2) {  // the groups' first rows and row tiles
    // rows are clamped to R: whatever the offsets hold, nothing outside the arrays is touched
    const auto clamped = [&](int g) {
      const int64_t o = a.offsets[g];
      return o < 0 ? 0 : (o < a.R ? o : a.R);
    };
    int carry = 0;
    for (int g0 = 0; g0 < a.groups; g0 += 32) {
      const int g = g0 + lane;
      int n = 0;
      if (g < a.groups) {
        const int64_t r0 = clamped(g), r1 = clamped(g + 1);
        if (r1 > r0)
          n = kMode == kRows ? static_cast<int>((r1 - r0 + Sh::kBM - 1) / Sh::kBM)
                             : static_cast<int>((r1 - 1) / Sh::kBM - r0 / Sh::kBM + 1);
        c.first[g] = static_cast<int>(r0);
      }
      int x = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      if (g < a.groups) c.tiles[g] = carry + x - n;
      carry += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) {
      c.tiles[a.groups] = carry;
      c.first[a.groups] = static_cast<int>(clamped(a.groups));
    }
  }
  fence_before();
  __syncthreads();
  pair_sync();
  fence_after();
  const uint32_t tmem = c.tmem, ring0 = sm_addr(ring);
  const Tiles<kBN, kMode> tiles(a, c);

  // Producer and product issue run as whole warps of which an elected lane acts: with
  // the operands uniform over the warp the issue is short (a branch on the lane
  // number made a 64-deep piece of 256 x 128 outputs take 0.31 us, whatever its
  // size; elected, 0.20 us).
  if (warp == 0) {
    int loaded = 0, s = 0;  // pieces loaded so far; their stage
    uint32_t round = 0;     // of the ring
    bool ok = true;
    for (int t = worker; ok && t < tiles.jobs; t += workers) {
      const Tile x = tiles.get(t);
      const int row = static_cast<int>(x.row0) + static_cast<int>(rank) * 128;
      const int m = x.m0 + static_cast<int>(rank) * 128, n = x.n0 + static_cast<int>(rank) * (x.width / kCG);
      const bool two = x.width / kCG > kBBox;  // boxes of B beyond the first
      const int boxes = x.width / kCG / kBBox;
      const uint32_t bytes = Sh::kABytes + static_cast<uint32_t>(x.width / kCG) * 128u;
      const bool cut = kMode == kWeights && ((x.row1 - x.row0) % kBK) != 0;
      const int each = (a.K2 + kBK - 1) / kBK;
      int part = 0, group = 0, block = 0;  // kJoined
      for (int j = 0; j < x.nk; ++j) {
        if (round > 0 && !(ok = warp_wait(&c.empty[s], (round - 1) & 1u))) break;
        if (kMode == kJoined && j >= x.nk1) {  // the next 64 columns of the group's block, or the next group's
          if (++part == each || j == x.nk1) {
            part = 0;
            group = tiles.next_group(j == x.nk1 ? x.group : group + 1, x.tile);
            block = (c.tiles[group] + x.tile - c.first[group] / Sh::kBM) * Sh::kBM;
          }
        }
        if (elect_one()) {
          const bool last = cut && j == x.nk - 1;
          // a piece to be cleared lands on this CTA's own barrier
          const uint32_t bar = last ? sm_addr(&c.tail[s]) : bar_at(&c.full[s], 0);
          if (last)
            mbar_arrive_expect_tx(&c.tail[s], bytes);
          else if (rank == 0)  // for both CTAs: the pair's loads complete on the leader's barrier
            mbar_arrive_expect_tx(&c.full[s], kCG * bytes);
          const uint32_t sa = ring0 + s * kStage, sb = sa + Sh::kABytes;
          if (kMode == kWeights) {
            const int r = static_cast<int>(x.row0) + j * kBK;
            const CUtensorMap* pa = x.second ? &ma2 : &ma;
            const CUtensorMap* pb = x.second ? &mb2 : &mb;
            load_box<kCG>(sa, pa, m, r, 0, bar);
            load_box<kCG>(sa + kBox, pa, m + 64, r, 0, bar);
            load_box<kCG>(sb, pb, n, r, 0, bar);
            for (int q = 1; q < boxes; ++q) load_box<kCG>(sb + q * kBox, pb, n + 64 * q, r, 0, bar);
          } else {
            const bool one = kMode != kJoined || j < x.nk1;
            const int k = one ? j * kBK : part * kBK;
            const CUtensorMap* pa = one ? &ma : &ma2;
            const CUtensorMap* pb = one ? &mb : &mb2;
            const int z = kMode == kJoined ? (one ? 0 : group) : x.group;
            load_box<kCG>(sa, pa, k, one ? row : block + static_cast<int>(rank) * 128, 0, bar);
            if (kBMN) {
              load_box<kCG>(sb, pb, n, k, z, bar);
              for (int q = 1; q < boxes; ++q) load_box<kCG>(sb + q * kBox, pb, n + 64 * q, k, z, bar);
            } else {
              load_box<kCG>(sb, pb, k, n, z, bar);
              if (two) load_box<kCG>(sb + kBBox * 128, pb, k, n + kBBox, z, bar);
            }
          }
        }
        __syncwarp();
        ++loaded;
        if (++s == S) s = 0, ++round;
      }
    }
    // after a wait that ran out: this CTA's shared memory outlives the copies into it
    if (!ok && rank == 0)
      for (int q = loaded > S ? loaded - S : 0; q < loaded; ++q)
        mbar_wait(&c.full[q % S], static_cast<uint32_t>((q / S) & 1));
  } else if (warp == 1) {
    int done = 0, s = 0;
    uint32_t round = 0;
    uint32_t tail_phase = 0;  // a bit per stage
    bool ok = true;
    for (int t = worker; ok && t < tiles.jobs; t += workers) {
      const Tile x = tiles.get(t);
      const int tail = kMode == kWeights ? static_cast<int>((x.row1 - x.row0) % kBK) : 0;
      if (x.nk == 0) continue;
      const uint32_t idesc = x.width == kBN ? instr<kAMN, kBMN>(Sh::kBM, kBN) : instr<kAMN, kBMN>(Sh::kBM, kBN / 2);
      const int boxes = static_cast<int>((Sh::kABytes + static_cast<uint32_t>(x.width / kCG) * 128u) / kBox);
      const int b = done & 1;
      if (rank == 0) {
        if (done >= 2 && !(ok = warp_wait(&c.acc_empty[b], static_cast<uint32_t>((done / 2 - 1) & 1)))) break;
        fence_after();
      }
      // the products of the stage that is next, and what they free
      const auto stage = [&](bool last, const auto& products) {
        if (rank == 0) {
          if (!(ok = warp_wait(&c.full[s], round & 1u))) return;
          fence_after();
          if (elect_one()) {
            products(tmem + static_cast<uint32_t>(b * kBN), ring0 + s * kStage);
            commit<kCG>(&c.empty[s]);
            if (last) commit<kCG>(&c.acc_full[b]);
          }
          __syncwarp();
        }
        if (++s == S) s = 0, ++round;
      };
      const auto plain = [&](uint32_t acc, uint32_t sa, bool add) {
#pragma unroll
        for (int k = 0; k < kBK / 16; ++k)
          mma<kCG>(acc, desc<kAMN>(sa + kStep<kAMN> * k), desc<kBMN>(sa + Sh::kABytes + kStep<kBMN> * k), idesc,
                   add || k > 0);
      };
      for (int j = 0; ok && j < x.nk1; ++j) {
        if (kMode == kWeights && tail != 0 && j == x.nk - 1) {
          if (!(ok = warp_wait(&c.tail[s], (tail_phase >> s) & 1u))) break;
          tail_phase ^= 1u << s;
#pragma unroll 1
          for (int q = 0; q < boxes; ++q)
            for (uint32_t o = tail * 128 + lane * 16; o < kBox; o += 512)
              *reinterpret_cast<uint4*>(ring + s * kStage + q * kBox + o) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async();
          __syncwarp();
          if (rank != 0) {
            if (lane == 0) arrive_release(bar_at(&c.peer_tail[s], 0));
          } else {
            if (!(ok = __all_sync(0xffffffffu, wait_acquire(&c.peer_tail[s], ((tail_phase >> s) & 1u) ^ 1u))))
              break;
            if (lane == 0) mbar_arrive(&c.full[s]);  // the stage's phase, which no load completes
            __syncwarp();
          }
        }
        stage(j == x.nk - 1, [&](uint32_t acc, uint32_t sa) { plain(acc, sa, j > 0); });
      }
      if (kMode == kJoined) {
        const int each = (a.K2 + kBK - 1) / kBK, row0 = static_cast<int>(x.row0);
        const int row1 = x.row1 - x.row0 < Sh::kBM ? static_cast<int>(x.row1) : row0 + Sh::kBM;
        int group = x.group;
        for (int j = x.nk1; ok && j < x.nk; ++group) {  // as the producer goes through the groups
          group = tiles.next_group(group, x.tile);
          const int first = c.first[group], end = c.first[group + 1];
          Rows others;
          others.all_but(first - row0, end - row0);
          for (int part = 0; ok && part < each; ++part, ++j) {
            if (first <= row0 && end >= row1)
              stage(j == x.nk - 1, [&](uint32_t acc, uint32_t sa) { plain(acc, sa, true); });
            else
              stage(j == x.nk - 1, [&](uint32_t acc, uint32_t sa) {
#pragma unroll
                for (int k = 0; k < kBK / 16; ++k)
                  mma_rows(acc, desc<kAMN>(sa + kStep<kAMN> * k), desc<kBMN>(sa + Sh::kABytes + kStep<kBMN> * k),
                           idesc, others);
              });
          }
        }
      }
      ++done;
    }
    if (!ok && rank == 0) {  // the products in flight end before tensor memory is freed
      if (elect_one()) commit<kCG>(&c.drained);
      mbar_wait(&c.drained, 0);
    }
    __syncwarp();
  } else {
    // two warps per 32 rows (a warp reads the tensor-memory lanes of its number mod 4), half of the columns each
    const int quarter = warp & 3, ew = warp - 2, half = ew >> 2;
    unsigned char* outs = staging + ew * (Sh::kBufs * kOutBytes);
    unsigned char* all_lows = staging + kEpiWarps * Sh::kBufs * kOutBytes + ew * (Sh::kBufs * kLowBytes);
    int steps = 0, asked = 0;  // kDRelu2: boxes of h this warp has read, and asked for
    const auto fetch = [&](int step, int n, int64_t row) {  // 32 columns of h and low
      asked = step + 1;
      if (lane != 0) return;
      uint64_t* bar = &c.aux[ew][step & 1];
      mbar_arrive_expect_tx(bar, kOutBytes + (a.low != nullptr ? kLowBytes : 0));
      load_box<1>(sm_addr(outs + (step & 1) * kOutBytes), &ma2, n, static_cast<int>(row), 0, sm_addr(bar));
      if (a.low != nullptr)
        load_box<1>(sm_addr(all_lows + (step & 1) * kLowBytes), &mlow, n, static_cast<int>(row), 0, sm_addr(bar));
    };
    int done = 0;
    bool ok = true;
    for (int t = worker; ok && t < tiles.jobs; t += workers) {
      const Tile x = tiles.get(t);
      const int b = done & 1;
      const bool have = x.nk > 0;
      const int M = x.second ? a.M2 : a.M, N = x.second ? a.N2 : a.N;
      bf16* const dest = x.second ? a.out2 : a.out;
      // the warp's 32 rows: the first, and how many of them exist
      const int in_tile = static_cast<int>(rank) * 128 + 32 * quarter;
      const int64_t row0 = (kMode == kWeights  ? static_cast<int64_t>(x.group) * M + x.m0
                            : kMode == kBlocks ? static_cast<int64_t>(x.tile) * Sh::kBM
                                               : x.row0) + in_tile;
      const int64_t left = (kMode == kWeights ? M - x.m0 : kMode == kBlocks ? Sh::kBM : x.row1 - x.row0) - in_tile;
      // kBlocks: this lane's row is the group's
      const bool live = kMode != kBlocks || (in_tile + lane >= x.lead && x.row0 + in_tile + lane < x.row1);
      const int rows = left < 32 ? (left > 0 ? static_cast<int>(left) : 0) : 32;
      const float scale = kEpi == kScale && a.scale != nullptr && live ? a.scale[x.group] : 1.0f;
      int to = 0;  // where this lane's row goes
      if (kMode != kWeights && a.scatter != nullptr && lane < rows) to = a.scatter[row0 + lane];
      const int begin = half * (x.width / 2), end = begin + x.width / 2;
      const int cols = N - x.n0 < end ? N - x.n0 : end;
      if (kEpi == kDRelu2 && rows > 0 && begin < cols) {
        if (lane == 0) bulk_wait_read();
        fetch(steps, x.n0 + begin, row0);
      }
      if (have && !(ok = warp_wait(&c.acc_full[b], static_cast<uint32_t>((done / 2) & 1)))) break;
      fence_after();
      if (have && begin >= cols && lane == 0) arrive_at(bar_at(&c.acc_empty[b], 0));
#pragma unroll 1
      for (int c0 = begin; c0 < cols; c0 += 32) {
        uint32_t v[32];
        if (have) {
          ld32(v, tmem + (static_cast<uint32_t>(32 * quarter) << 16) + static_cast<uint32_t>(b * kBN + c0));
          if (c0 + 32 >= cols) {  // read to the end: the accumulator is free
            fence_before();
            __syncwarp();
            if (lane == 0) arrive_at(bar_at(&c.acc_empty[b], 0));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0u;
        }
        if (rows == 0) continue;  // the whole warp
        if (!live) {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0u;
        }
        unsigned char* out = outs;
        unsigned char* lows = all_lows;
        if (kEpi == kDRelu2) {  // h lies where the result will be staged
          if (c0 + 32 < cols) {
            if (lane == 0) bulk_wait_read();  // the box before this one was stored from there
            fetch(steps + 1, x.n0 + c0 + 32, row0);
          }
          out += (steps & 1) * kOutBytes;
          lows += (steps & 1) * kLowBytes;
          if (!(ok = warp_wait(&c.aux[ew][steps & 1], static_cast<uint32_t>((steps >> 1) & 1)))) break;
          ++steps;
        } else {  // the last store has read the staging buffers
          if (lane == 0) bulk_wait_read();
          __syncwarp();
        }
        uint4 low4 = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4 av = make_uint4(0u, 0u, 0u, 0u);
          uint2 lv = make_uint2(0u, 0u);
          if (kEpi == kDRelu2) {
            av = *reinterpret_cast<const uint4*>(out + out_at(lane, q));
            if (a.low != nullptr) lv = *reinterpret_cast<const uint2*>(lows + low_at(lane, q / 2) + 8 * (q % 2));
          }
          const uint32_t ah[4] = {av.x, av.y, av.z, av.w}, al[2] = {lv.x, lv.y};
          uint32_t o4[4], l[2] = {0u, 0u};
#pragma unroll
          for (int e = 0; e < 2; ++e) {  // four columns
            float y[4], h[4] = {};
            if (kEpi == kDRelu2) {
              h[0] = with_low<0>(ah[2 * e] << 16, al[e]);
              h[1] = with_low<1>(ah[2 * e] & 0xffff0000u, al[e]);
              h[2] = with_low<2>(ah[2 * e + 1] << 16, al[e]);
              h[3] = with_low<3>(ah[2 * e + 1] & 0xffff0000u, al[e]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = finish<kEpi>(__uint_as_float(v[8 * q + 4 * e + i]), h[i], scale);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const __nv_bfloat162 two = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
              o4[2 * e + i] = *reinterpret_cast<const uint32_t*>(&two);
            }
            if (kEpi == kRelu2 && a.low != nullptr) {
              const uint32_t l01 = __byte_perm(low_word(y[0], o4[2 * e] << 16),
                                               low_word(y[1], o4[2 * e] & 0xffff0000u), 0x0051);
              const uint32_t l23 = __byte_perm(low_word(y[2], o4[2 * e + 1] << 16),
                                               low_word(y[3], o4[2 * e + 1] & 0xffff0000u), 0x0051);
              l[e] = __byte_perm(l01, l23, 0x5410);
            }
          }
          const uint4 o = make_uint4(o4[0], o4[1], o4[2], o4[3]);
          *reinterpret_cast<uint4*>(out + out_at(lane, q)) = o;
          if (kEpi == kRelu2 && a.low != nullptr) {
            if (q % 2 == 0) {
              low4.x = l[0], low4.y = l[1];
            } else {
              low4.z = l[0], low4.w = l[1];
              *reinterpret_cast<uint4*>(lows + low_at(lane, q / 2)) = low4;
            }
          }
        }
        const int n = x.n0 + c0;
        // Whole boxes of 32 rows go out by TMA; with loads and stores through registers
        // in its place kDRelu2 took 127 us against 122 for 16384 rows x 1024 x 4096 (the
        // others within 1 us).
        if (rows == 32 && (kMode == kWeights || a.scatter == nullptr)) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            store_box(x.second ? &mlow : &mo, sm_addr(out), n, static_cast<int>(row0));
            if (kEpi == kRelu2 && a.low != nullptr) store_box(&mlow, sm_addr(lows), n, static_cast<int>(row0));
            bulk_commit();
          }
          __syncwarp();
          continue;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * i + (lane >> 2), m = n + 8 * (lane & 3);
          const int64_t dst = kMode != kWeights && a.scatter != nullptr ? __shfl_sync(0xffffffffu, to, r) : row0 + r;
          if (r < rows && m < N)
            *reinterpret_cast<uint4*>(dest + dst * N + m) =
                *reinterpret_cast<const uint4*>(out + out_at(r, lane & 3));
        }
        if (kEpi == kRelu2 && a.low != nullptr) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = 16 * i + (lane >> 1), m = n + 16 * (lane & 1);
            if (r >= rows || m >= N) continue;
            *reinterpret_cast<uint4*>(a.low + (row0 + r) * low_stride(N) + m) =
                *reinterpret_cast<const uint4*>(lows + low_at(r, lane & 1));
          }
        }
        if (kEpi == kDRelu2) fence_proxy_async();  // the next box lands here
        __syncwarp();
      }
      if (have) ++done;
    }
    if (lane == 0) bulk_wait_all();
    for (; !ok && steps < asked; ++steps)  // as above: the copies in flight end first
      mbar_wait(&c.aux[ew][steps & 1], static_cast<uint32_t>((steps >> 1) & 1));
    if (kMode != kWeights && a.zero_tail) {
      const int64_t pieces = a.N / 8;
      const int64_t end = a.R * pieces;
      uint4* out = reinterpret_cast<uint4*>(a.out);
      const int64_t step = static_cast<int64_t>(gridDim.x) * (32 * kEpiWarps);
      for (int64_t i = tiles.first(a.groups) * pieces + static_cast<int64_t>(blockIdx.x) * (32 * kEpiWarps) + (tid - 64); i < end;
           i += step)
        out[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  fence_before();
  __syncthreads();
  pair_sync();
  if (warp == 1) tmem_free<kCG>(tmem, Sh::kCols);
}

}  // namespace tc
}  // namespace camoe
