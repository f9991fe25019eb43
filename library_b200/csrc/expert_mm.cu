// The experts' products: a block-diagonal matrix times a dense one, with bias, activation and residual
// in the epilogue, and the gradient with respect to the blocks.
//   Z[p,n] = sum_k X[p,k] op(W_e)[k,n] + bias[e,n],   Y[p,n] = act(Z[p,n]) + R[p,n]   for p in segment e
//   dW_e   = dZ_e^T X_e  (or its transpose)
//
// expert_mm_kernel runs both: persistent pairs of CTAs whose tcgen05.mma (M = 256, N up to 256) shares the N operand between the two
// SMs, operands staged by TMA in a ring of six 32 KB stages per CTA, two accumulators in tensor memory so that a tile's epilogue runs
// behind the next tile's MMAs.  expert_mm_few_kernel takes products of few rows, whose work is the weights' bytes.
// The MMA's M side (lanes of tensor memory) is always the output's
// contiguous dimension, its N side the output's rows: a warp of the epilogue then writes 32
// neighbouring elements of a row, and the N of an MMA, which the instruction takes in steps of 16,
// follows a ragged segment closely.
//
// What bounds the pair kernel: power.  In a run of seconds (1,000 W, about 1.35 GHz) 32,768 x 2,048 times 2,048 x 4,096 in bf16 takes
// 441-446 us (1,235 TFLOP/s) against 417 us for a library product of the same sizes; in short bursts 1,370 TFLOP/s, 1,450 at
// K = N = 4,096.  Spread over 32 experts it takes 487 us (520 MB more of weights from HBM), with uneven segments 518 us.  The tile
// order matters for that reason: pairs that work at a time take all column blocks of few row tiles (448 us); groups of eight
// column blocks 452, of four 479 us (more distinct rows of X cross the fabric).
#include <cuda.h>

#include <atomic>

#include "expert_act.h"
#include "expert_launch.h"
#include "expert_vec.h"

namespace asp {
namespace {

// ---- PTX helpers --------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// Address of the same shared-memory location in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_u32(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
// (for threads whose reads of a peer's memory have been used and that have nothing to make visible: no wait for their stores)
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
// Arrivals take a cluster address: the CTA's own barrier or a peer's.  The producer's carries no data of
// its own (the copies complete on the barrier by themselves), so it is relaxed: a release at cluster
// scope waits for the warp's earlier operations, once per stage.
__device__ __forceinline__ void mbar_arrive_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// An arrival that only says that reads of an accumulator have completed (after tcgen05.wait::ld).  A release at cluster scope would
// wait for the epilogue's global stores.
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Bounded wait on a barrier of this CTA: false if the phase did not complete within `limit` polls.  A poll parks the warp for up to two
// microseconds or until the phase completes: a warp that polls flat out costs power, and power is what limits the products.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint32_t limit) {
  for (uint32_t i = 0; i < limit; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(2000)
        : "memory");
    if (ok) return true;
  }
  return false;
}
// The same for what a peer's threads wrote before they arrived with a release at cluster scope.
__device__ __forceinline__ bool mbar_wait_peers(uint32_t bar, uint32_t parity, uint32_t limit) {
  for (uint32_t i = 0; i < limit; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(2000)
        : "memory");
    if (ok) return true;
  }
  return false;
}
// One lane of the converged warp, in a form that tells the compiler that exactly one thread runs the guarded code.
__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(pred));
  return pred != 0;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// TMA loads into this CTA's shared memory.  The .cta_group::2 form may complete on a barrier of either CTA of the pair.
// CG: CTAs of the MMA.
template <int CG>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map),
        "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map),
        "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
// Shared-memory descriptor of a 128-byte-swizzled operand.  K-major: rows of 64 elements (128 bytes), groups of
// eight rows 1,024 bytes apart.  MN-major: 64 x 64 boxes (a row of 128 bytes per k), groups of eight k 1,024
// bytes apart, the next 64 elements one box (8,192 bytes) further.
__device__ __forceinline__ uint64_t umma_desc(uint32_t saddr, uint32_t lbo_bytes) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo_bytes >> 4) & 0x3FFFu) << 16) | ((uint64_t)(1024u >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
template <int CG>
__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// The barrier (of both CTAs of a pair, at the same offset) is arrived on when the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void umma_commit(uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"((uint16_t)3)
                 : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
  if constexpr (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t cols) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// ---- the tile kernel ----------------------------------------------------------------------------
constexpr int kKC = 64;                        // contraction per stage: 128 bytes of a 16-bit type
constexpr int kTileM = 128;                    // M of a CTA: lanes of tensor memory
constexpr int kTileJ = 256;                    // N of an MMA, at most: rows of the output per tile
constexpr int kPairM = 2 * kTileM;             // columns of the output per tile
constexpr int kABytes = kTileM * kKC * 2;      // 16 KB
constexpr int kMmStages = 6;
constexpr int kMmStage = kABytes + kTileJ / 2 * kKC * 2;  // a CTA's 128 columns of M and its half of N: 32 KB
constexpr int kBoxBytes = 64 * 128;            // an MN-major box
constexpr int kEpiParts = 2;                   // epilogue warps per quarter of the lanes
constexpr int kEpiWarp0 = 4, kEpiWarps = 4 * kEpiParts;
constexpr int kMmThreads = (kEpiWarp0 + kEpiWarps) * 32;
constexpr int kTmemCols = 512;                 // two accumulators of 256 columns
// Polls of a bounded wait: seconds, and more than a tile of `chunks` stages can take.  Below 2^31, so that twice the limit and the
// peers' margin stay a number of 32 bits.
inline uint32_t wait_limit(alphasparseHandle_t h, int64_t chunks) {
  const HandleImpl* i = impl(h);
  if (i->expert_wait) return i->expert_wait;
  return (1u << 21) + (uint32_t)(chunks < (1 << 23) ? 128 * chunks : (1 << 30));
}

// Which contraction the kernel runs.
enum MmKind {
  kFwdT = 0,  // M = output features (W_e stored N x K, K-major),  N = rows of the segment (X, K-major), over K
  kFwdN = 1,  // M = output features (W_e stored K x N, MN-major), N = rows of the segment (X, K-major), over K
  kGradW = 2  // M = columns of dW_e, N = rows of dW_e (both MN-major), over the rows of the segment
};

struct MmArgs {
  const int32_t* off;
  int segments, rows;
  int m_total;        // columns of the output (contiguous)
  int j_total;        // kGradW: rows of a block of dW
  int k;              // kFwd*: contraction length
  int box_rows;       // kFwd*: rows of X per TMA box
  uint32_t types;     // operand type bits of the instruction descriptor
  void* y;
  int64_t ldy;
  const void* r;
  int64_t ldr;
  void* z;
  int64_t ldz;
  const void* bias;
  int64_t ldb;
  int bias_type;
  int act;
  uint32_t limit;     // polls of a wait; bit 31 (kWaitDropCopy): testing
  int* err;
};

__device__ __forceinline__ int clamp_row(const int32_t* off, int e, int rows) {
  const int v = off[e];
  return v < 0 ? 0 : v > rows ? rows : v;
}
template <typename T>
__device__ __forceinline__ float load_as(const void* p, int64_t i) { return Wide<T>::up(((const T*)p)[i]); }
__device__ __forceinline__ float load_bias(const void* p, int64_t i, int t) {
  return t == ALPHA_R_32F ? ((const float*)p)[i] : t == ALPHA_R_16F ? load_as<__half>(p, i) : load_as<__nv_bfloat16>(p, i);
}

struct Tile {
  int e;           // segment
  int m0;          // first column of the output (of the CTA pair)
  int row0, rows;  // rows of the output: first (of the whole matrix), how many
  int width;       // N of the MMA (rows rounded up to 16)
  int k0, klen;    // contraction range
};

// s_tile[e] = tiles of ROWS rows of the segments before e (s_tile[segments]: of all, returned).  All THREADS of the CTA; consecutive
// segments per thread.  s_warp: a word per warp.
template <int THREADS, int ROWS>
__device__ __forceinline__ int segment_tiles(const int* s_off, int segments, int* s_tile, int* s_warp) {
  constexpr int kPer = (ALPHASPARSE_MAX_EXPERTS + THREADS - 1) / THREADS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int cnt[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = tid * kPer + i;
    const int n = e < segments ? s_off[e + 1] - s_off[e] : 0;
    cnt[i] = n > 0 ? (n + ROWS - 1) / ROWS : 0;
    sum += cnt[i];
  }
  int v = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += s_warp[w];
    all += s_warp[w];
  }
  int run = before + v - sum;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = tid * kPer + i;
    if (e < segments) s_tile[e] = run;
    run += cnt[i];
  }
  if (tid == 0) s_tile[segments] = all;
  return all;
}
// Row tile j: its segment and rows (the segment's rows are spread evenly over its tiles).  Whole warp; every lane gets the same answer.
__device__ __forceinline__ void row_tile(int j, int segments, const int* s_off, const int* s_tile, Tile& x) {
  const int lane = threadIdx.x & 31;
  // the segment: the last one whose first tile is not past j (two ballots over up to 1,024 segments)
  const unsigned hi = __ballot_sync(0xffffffffu, lane * 32 < segments && s_tile[lane * 32 < segments ? lane * 32 : 0] <= j);
  const int blk = 31 - __clz(hi);
  const int i = blk * 32 + lane;
  const unsigned lo = __ballot_sync(0xffffffffu, i < segments && s_tile[i < segments ? i : 0] <= j);
  x.e = blk * 32 + 31 - __clz(lo);
  const int b = s_off[x.e], n = s_off[x.e + 1] - b, tiles = s_tile[x.e + 1] - s_tile[x.e];
  const int w = ((n + tiles - 1) / tiles + 15) & ~15;
  const int at = (j - s_tile[x.e]) * w;
  x.row0 = b + at;
  x.rows = n - at < w ? n - at : w;
}

// Tile t of the launch.  Whole warp; every lane gets the same answer.
template <int KIND>
__device__ __forceinline__ Tile tile_of(int t, const MmArgs& a, const int* s_off, const int* s_tile, int mblocks, int jblocks) {
  Tile x;
  if constexpr (KIND == kGradW) {
    const int per = mblocks * jblocks;
    x.e = t / per;
    const int i = t % per, j = i / mblocks;
    x.m0 = (i % mblocks) * kPairM;
    const int left = a.j_total - j * kTileJ;
    x.rows = left < kTileJ ? left : kTileJ;
    x.row0 = j * kTileJ;  // within the block of dW
    x.k0 = s_off[x.e];
    x.klen = s_off[x.e + 1] > x.k0 ? s_off[x.e + 1] - x.k0 : 0;
  } else {
    x.m0 = (t % mblocks) * kPairM;
    row_tile(t / mblocks, a.segments, s_off, s_tile, x);
    x.k0 = 0;
    x.klen = a.k;
  }
  x.width = (x.rows + 15) & ~15;
  return x;
}

constexpr int kCols = 16;  // (32 at a time spilled registers; 8 take a third longer)
// The epilogue of kCols rows (n of them exist, all if FULL) of output column m, from row `row` of the output on: v holds the
// sums.  Each optional operand is one guarded loop, not a test per element.
template <typename TO>
__device__ __forceinline__ void load_residual(const MmArgs& a, int64_t row, int m, int n, TO (&res)[kCols]) {
  const TO* r = (const TO*)a.r + row * a.ldr + m;
#pragma unroll
  for (int c = 0; c < kCols; ++c, r += a.ldr)
    if (c < n) res[c] = *r;
}
template <typename TO, int ACT, bool FULL>
__device__ __forceinline__ void finish_values(const MmArgs& a, int64_t row, int m, int n, float bias, const TO (&res)[kCols],
                                              float (&v)[kCols]) {
#pragma unroll
  for (int c = 0; c < kCols; ++c) v[c] += bias;
  if (a.z) {
    TO* z = (TO*)a.z + row * a.ldz + m;
#pragma unroll
    for (int c = 0; c < kCols; ++c, z += a.ldz)
      if (FULL || c < n) *z = Wide<TO>::down(v[c]);
  }
#pragma unroll
  for (int c = 0; c < kCols; c += 2) activate2<ACT>(v[c], v[c + 1]);
  if (a.r) {
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      if (FULL || c < n) v[c] += Wide<TO>::up(res[c]);
  }
  TO* y = (TO*)a.y + row * a.ldy + m;
#pragma unroll
  for (int c = 0; c < kCols; ++c, y += a.ldy)
    if (FULL || c < n) *y = Wide<TO>::down(v[c]);
}
// A warp's share of a tile: every PARTS-th block of kCols rows.
template <typename TO, int ACT, int PARTS = kEpiParts>
__device__ __forceinline__ void finish_tile(const MmArgs& a, const Tile& x, int m, int part, uint32_t tmem, bool in, float bias,
                                            int64_t out_row0) {
  for (int c0 = part * kCols; c0 < x.rows; c0 += PARTS * kCols) {
    TO res[kCols];
    if (a.r && in) load_residual<TO>(a, out_row0 + c0, m, x.rows - c0, res);
    __syncwarp();  // tensor memory is read by the converged warp; past the last column `in` differs between its lanes
    uint32_t acc[kCols];
    tmem_ld16(tmem + (uint32_t)c0, acc);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    if (in) {
      float v[kCols];
#pragma unroll
      for (int c = 0; c < kCols; ++c) v[c] = x.klen <= 0 ? 0.f : __uint_as_float(acc[c]);  // an empty sum: no MMA wrote them
      if (c0 + kCols <= x.rows) finish_values<TO, ACT, true>(a, out_row0 + c0, m, kCols, bias, res, v);
      else finish_values<TO, ACT, false>(a, out_row0 + c0, m, x.rows - c0, bias, res, v);
    }
    __syncwarp();
  }
}

// Warp roles: 0 TMA producer, 1 MMA issuer, 2 clearing of ragged tails (kGradW), 4 and up epilogue.
template <int KIND, typename TO>
__global__ void __launch_bounds__(kMmThreads, 1)
expert_mm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ MmArgs a) {
  extern __shared__ unsigned char smem_raw[];
  // swizzled tiles need a 1,024-byte aligned base; the offset is the same in both CTAs of a pair
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char* gen = smem_raw + (base - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(gen + kMmStages * kMmStage);
  const uint32_t bar0 = base + kMmStages * kMmStage;
  const uint32_t full = bar0, empty = bar0 + 8 * kMmStages, tail = bar0 + 16 * kMmStages, acc_full = bar0 + 24 * kMmStages,
                 acc_empty = acc_full + 16;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + 3 * kMmStages + 4);
  int* s_fail = reinterpret_cast<int*>(s_tmem + 1);
  int* s_off = s_fail + 1;                             // segments + 1
  int* s_tile = s_off + ALPHASPARSE_MAX_EXPERTS + 1;   // segments + 1
  __shared__ int s_warp[kMmThreads / 32];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t limit = a.limit & ~kWaitDropCopy;
  const uint32_t rank = cluster_rank();
  const int mblocks = (a.m_total + kPairM - 1) / kPairM;
  const int jblocks = KIND == kGradW ? (a.j_total + kTileJ - 1) / kTileJ : 0;

  if (tid == 0) {
    for (int i = 0; i < kMmStages; ++i) {
      mbar_init(full + 8 * i, 2);  // an arrival per CTA
      mbar_init(empty + 8 * i, 1);
      mbar_init(tail + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, 2 * kEpiWarps);
    }
    *s_fail = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc<2>(smem_u32(s_tmem), kTmemCols);
  if (tid == 32 * 3) {
    prefetch_map(&map_a);
    prefetch_map(&map_b);
  }
  __syncthreads();
  cluster_arrive();  // this CTA's barriers are ready (the wait is below, behind the kernel's other waits)
  dependents_go();   // tensor memory is allocated
  dependency_wait();
  for (int i = tid; i <= a.segments; i += kMmThreads) s_off[i] = a.off ? clamp_row(a.off, i, a.rows) : (i == 0 ? 0 : a.rows);
  __syncthreads();
  int total;
  if constexpr (KIND == kGradW) {
    total = a.segments * mblocks * jblocks;
  } else {
    const int all = segment_tiles<kMmThreads, kTileJ>(s_off, a.segments, s_tile, s_warp);
    total = all * mblocks;
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_wait();  // the peer's barriers are ready
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *s_tmem;
  const int first = (int)blockIdx.x / 2, stride = (int)gridDim.x / 2;
  bool ok = true;

  if (warp == 0) {
    // ---------------- producer: this CTA's half of every stage ----------------
    int st = 0;
    uint32_t ph = 0;
    for (int t = first; t < total && ok; t += stride) {
      const Tile x = tile_of<KIND>(t, a, s_off, s_tile, mblocks, jblocks);
      const int m = x.m0 + (int)rank * kTileM;
      const int half = x.width / 2;  // rows of the B operand in this CTA
      const int j = x.row0 + (int)rank * half;
      const int box = KIND == kGradW ? 64 : a.box_rows, boxes = (half + box - 1) / box;
      const uint32_t bytes = kABytes + (uint32_t)(boxes * box * 128);
      for (int c = 0; c < x.klen; c += kKC) {
        if (!__all_sync(0xffffffffu, mbar_wait(empty + 8 * st, ph ^ 1u, limit))) {
          ok = false;
          break;
        }
        if (elect_one()) {
          const uint32_t sa = base + st * kMmStage, sb = sa + kABytes;
          // a last chunk that has to be cleared completes on the CTA's own barrier; warp 2 passes it on
          const bool own = KIND == kGradW && x.klen - c < kKC && ((x.klen - c) & 15) != 0;
          const uint32_t bar = peer_u32(own ? tail + 8 * st : full + 8 * st, own ? rank : 0);
          mbar_arrive_tx(bar, bytes);
          if (a.limit & kWaitDropCopy) {
            // testing: announced but not issued, so that every role's wait runs out
          } else if constexpr (KIND == kFwdT) {
            tma_3d<2>(sa, &map_a, c, m, x.e, bar);
          } else if constexpr (KIND == kFwdN) {
            tma_3d<2>(sa, &map_a, m, c, x.e, bar);
            tma_3d<2>(sa + kBoxBytes, &map_a, m + 64, c, x.e, bar);
          } else {
            tma_2d<2>(sa, &map_a, m, x.k0 + c, bar);
            tma_2d<2>(sa + kBoxBytes, &map_a, m + 64, x.k0 + c, bar);
          }
          for (int b = 0; b < boxes; ++b) {
            if constexpr (KIND == kGradW) tma_2d<2>(sb + b * kBoxBytes, &map_b, j + b * 64, x.k0 + c, bar);
            else tma_2d<2>(sb + b * box * 128, &map_b, c, j + b * box, bar);
          }
        }
        __syncwarp();
        if (++st == kMmStages) {
          st = 0;
          ph ^= 1u;
        }
      }
    }
    // no stage is left with an arrival on its way to this CTA
    for (int i = 0; i < kMmStages && ok; ++i) {
      ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * st, ph ^ 1u, limit));
      if (++st == kMmStages) {
        st = 0;
        ph ^= 1u;
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (the pair's first CTA) ----------------
    if (rank == 0) {
      int st = 0, n = 0;
      uint32_t ph = 0;
      constexpr uint32_t kMajor = KIND == kFwdN ? (1u << 15) : KIND == kGradW ? (1u << 15) | (1u << 16) : 0u;
      const uint32_t idesc0 = (1u << 4) | a.types | kMajor | ((uint32_t)(kPairM >> 4) << 24);
      constexpr uint32_t kStepA = KIND == kFwdT ? 2u : 128u, kStepB = KIND == kGradW ? 128u : 2u;  // 16 elements of k, in 16 bytes
      for (int t = first; t < total && ok; t += stride, ++n) {
        const Tile x = tile_of<KIND>(t, a, s_off, s_tile, mblocks, jblocks);
        const int buf = n & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(acc_empty + 8 * buf, (uint32_t)(((n >> 1) & 1) ^ 1), limit))) {
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem + (uint32_t)buf * kTileJ, idesc = idesc0 | ((uint32_t)(x.width >> 3) << 17);
        for (int c = 0; c < x.klen; c += kKC) {
          if (!__all_sync(0xffffffffu, mbar_wait(full + 8 * st, ph, limit))) {
            ok = false;
            break;
          }
          // (zeros that a warp of the peer stored in its tail)
          if (KIND == kGradW && x.klen - c < kKC) asm volatile("fence.acq_rel.cluster;" ::: "memory");
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (elect_one()) {
            const uint64_t da = umma_desc(base + st * kMmStage, kBoxBytes), db = umma_desc(base + st * kMmStage + kABytes, kBoxBytes);
            const int left = x.klen - c, steps = left >= kKC ? kKC / 16 : (left + 15) / 16;
            for (int s = 0; s < steps; ++s) umma<2>(d, da + s * kStepA, db + s * kStepB, idesc, c > 0 || s > 0 ? 1u : 0u);
            umma_commit<2>(empty + 8 * st);
          }
          __syncwarp();
          if (++st == kMmStages) {
            st = 0;
            ph ^= 1u;
          }
        }
        if (ok && elect_one()) umma_commit<2>(acc_full + 8 * buf);
        __syncwarp();
      }
    }
  } else if (warp == 2) {
    if constexpr (KIND == kGradW) {
      // ---------------- ragged tails: the rows of the next segment (or none) behind the last one ----------------
      int chunk = 0;
      uint32_t phases = 0;  // of the tail barriers, a bit per stage
      for (int t = first; t < total && ok; t += stride) {
        const Tile x = tile_of<KIND>(t, a, s_off, s_tile, mblocks, jblocks);
        const int chunks = (x.klen + kKC - 1) / kKC, left = x.klen - (chunks - 1) * kKC;
        chunk += chunks;
        if (chunks == 0 || (left & 15) == 0) continue;
        const int st = (chunk - 1) % kMmStages;
        if (!__all_sync(0xffffffffu, mbar_wait(tail + 8 * st, (phases >> st) & 1u, limit))) {
          ok = false;
          break;
        }
        phases ^= 1u << st;
        const int to = (left + 15) & ~15, n16 = (to - left) * 8;   // 16-byte words per box
        const int boxes = 2 + (x.width / 2 + 63) / 64;
        unsigned char* s = gen + st * kMmStage;
        for (int i = lane; i < n16 * boxes; i += 32)  // whole rows of 128 bytes: the swizzle does not matter
          *reinterpret_cast<uint4*>(s + (i / n16) * kBoxBytes + left * 128 + (i % n16) * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(peer_u32(full + 8 * st, 0));
        __syncwarp();
      }
    }
  } else if (warp >= kEpiWarp0) {
    // ---------------- epilogue: lane = column of the output, accumulator column = row ----------------
    const int quarter = warp & 3, part = (warp - kEpiWarp0) >> 2;
    int n = 0;
    for (int t = first; t < total && ok; t += stride, ++n) {
      const Tile x = tile_of<KIND>(t, a, s_off, s_tile, mblocks, jblocks);
      const int buf = n & 1;
      const int m = x.m0 + (int)rank * kTileM + quarter * 32 + lane;
      const bool in = m < a.m_total;
      const float bias = a.bias && in ? load_bias(a.bias, (int64_t)x.e * a.ldb + m, a.bias_type) : 0.f;
      const int64_t out_row0 = KIND == kGradW ? (int64_t)x.e * a.j_total + x.row0 : (int64_t)x.row0;
      if (a.r) {
        // the tile's residual on its way to L2 while the accumulator is still being formed: a row per lane of the epilogue
        const int row = (warp - kEpiWarp0) * 32 + lane, m_cta = x.m0 + (int)rank * kTileM;
        const TO* r = (const TO*)a.r + (out_row0 + row) * a.ldr + m_cta;
        for (int c = 0; row < x.rows && c < kTileM && m_cta + c < a.m_total; c += 128 / (int)sizeof(TO))
          asm volatile("prefetch.global.L2 [%0];" ::"l"(r + c));
      }
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full + 8 * buf, (uint32_t)((n >> 1) & 1), limit))) {
        ok = false;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t d = tmem + (uint32_t)buf * kTileJ + ((uint32_t)(quarter * 32) << 16);
      switch (KIND == kGradW ? ALPHASPARSE_ACT_NONE : a.act) {
        case ALPHASPARSE_ACT_RELU: finish_tile<TO, ALPHASPARSE_ACT_RELU>(a, x, m, part, d, in, bias, out_row0); break;
        case ALPHASPARSE_ACT_GELU: finish_tile<TO, ALPHASPARSE_ACT_GELU>(a, x, m, part, d, in, bias, out_row0); break;
        case ALPHASPARSE_ACT_SILU: finish_tile<TO, ALPHASPARSE_ACT_SILU>(a, x, m, part, d, in, bias, out_row0); break;
        default: finish_tile<TO, ALPHASPARSE_ACT_NONE>(a, x, m, part, d, in, bias, out_row0); break;
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      if (lane == 0) mbar_arrive_relaxed(peer_u32(acc_empty + 8 * buf, 0));
    }
  }
  __syncwarp();
  if (!ok && lane == 0) *s_fail = 1;
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*s_fail) {
    // a wait ran out: say so, and give copies and MMAs still in flight time to land before the memory goes
    if (tid == 0) *a.err = 1;
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  cluster_sync();  // the peer's MMAs read this CTA's shared memory, its arrivals land here
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1) tmem_free<2>(tmem, kTmemCols);
}

// ---- few rows: the weights' bytes are the work ----------------------------------------------------
// (and, for gradients, few tiles: a long contraction would run on few SMs).
// One output tile of 128 columns x up to J rows per CLUSTER, whose CTAs share the contraction: each streams its
// part of K through a ring of its own (several CTAs per SM, so that many loads are in flight),
// leaves its fp32 sums in shared memory and tells its peers, and CTA r adds up the rows r, r + size, ... over all
// CTAs in rank order (through distributed shared memory) and finishes them.  No workspace, no atomics.
constexpr int kFewThreads = 192;
constexpr int kFewStages = 4;
constexpr int kFewBox = 16;                                  // rows of X per TMA box
template <int J> struct Few {
  static constexpr int kStage = kABytes + J * kKC * 2;
  static constexpr int kSmem = 1024 + kFewStages * kStage + 8 * (2 * kFewStages + 2) + 8;
  static_assert(kFewStages * kStage >= J * kTileM * 4, "the sums take the ring's place");
};
constexpr int kFewTmem = 64;
// The wait for the cluster's sums takes twice the limit of the other waits and this many polls more: a CTA that gives up after its own
// limit still arrives, so its peers do not give up before it.  (Memory does not depend on it: no CTA leaves before the
// cluster's last barrier, which every CTA reaches, since every wait before it ends.)
constexpr uint32_t kPeerPolls = 1u << 20;

// Row tile j (of at most J rows) over all segments: false if there are fewer tiles.  Whole warp, without shared memory: a lane counts
// the tiles of consecutive segments, the lanes' sums are scanned, and the lane that holds tile j finds its segment.
template <int J>
__device__ __forceinline__ bool few_tile(int j, const MmArgs& a, Tile& x) {
  const int lane = threadIdx.x & 31;
  if (!a.off) {
    x.e = 0;
    x.row0 = j * J;
    if (x.row0 >= a.rows) return false;
    x.rows = a.rows - x.row0 < J ? a.rows - x.row0 : J;
    x.width = (x.rows + 15) & ~15;
    return true;
  }
  auto at = [&](int e) { return clamp_row(a.off, e, a.rows); };
  const int per = (a.segments + 31) / 32, e0 = lane * per < a.segments ? lane * per : a.segments;
  const int e1 = e0 + per < a.segments ? e0 + per : a.segments;
  int sum = 0, prev = at(e0);
#pragma unroll 4
  for (int e = e0; e < e1; ++e) {
    const int next = at(e + 1);
    sum += next > prev ? (next - prev + J - 1) / J : 0;
    prev = next;
  }
  int incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  int found = -1, lo = 0, n = 0, k = 0;
  const bool mine = incl - sum <= j && j < incl;
  if (mine) {
    k = j - (incl - sum);
    prev = at(e0);
    for (int e = e0; e < e1 && found < 0; ++e) {
      const int next = at(e + 1), tiles = next > prev ? (next - prev + J - 1) / J : 0;
      if (k < tiles) {
        found = e;
        lo = prev;
        n = next - prev;
      } else {
        k -= tiles;
        prev = next;
      }
    }
  }
  const unsigned who = __ballot_sync(0xffffffffu, mine);
  if (who == 0) return false;
  const int src = __ffs(who) - 1;
  x.e = __shfl_sync(0xffffffffu, found, src);
  lo = __shfl_sync(0xffffffffu, lo, src);
  n = __shfl_sync(0xffffffffu, n, src);
  k = __shfl_sync(0xffffffffu, k, src);
  x.row0 = lo + k * J;
  x.rows = n - k * J < J ? n - k * J : J;
  x.width = (x.rows + 15) & ~15;
  return true;
}

__device__ __forceinline__ float ld_peer(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

constexpr int kFewSplit = 8;  // CTAs that may share a tile's contraction (the portable cluster size)

template <typename TO, int ACT>
__device__ __forceinline__ void finish_shared(const MmArgs& a, const Tile& x, int64_t row0, int m, int col, uint32_t sums, uint32_t rank,
                                              uint32_t size, bool in, float bias) {
  if (!in) return;
  // two rows at a time, the sums of all CTAs asked for before the first is added
  for (int j0 = (int)rank; j0 < x.rows; j0 += (int)size * 2) {
    const int j1 = j0 + (int)size;
    const bool second = j1 < x.rows;
    float p[2][kFewSplit];
#pragma unroll
    for (int c = 0; c < kFewSplit; ++c) {
      if ((uint32_t)c < size) {
        const uint32_t from = peer_u32(sums, c) + (uint32_t)col * 4u;
        p[0][c] = ld_peer(from + (uint32_t)(j0 * kTileM) * 4u);
        if (second) p[1][c] = ld_peer(from + (uint32_t)(j1 * kTileM) * 4u);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i == 1 && !second) break;
      const int64_t row = row0 + (i == 0 ? j0 : j1);
      TO res;
      if (a.r) res = ((const TO*)a.r)[row * a.ldr + m];
      float w = 0.f;
#pragma unroll
      for (int c = 0; c < kFewSplit; ++c)
        if ((uint32_t)c < size) w += p[i][c];
      w += bias;
      if (a.z) ((TO*)a.z)[row * a.ldz + m] = Wide<TO>::down(w);
      w = activate<ACT>(w);
      if (a.r) w += Wide<TO>::up(res);
      ((TO*)a.y)[row * a.ldy + m] = Wide<TO>::down(w);
    }
  }
}

template <int KIND, int J, typename TO>
__global__ void __launch_bounds__(kFewThreads)
expert_mm_few_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ MmArgs a,
                     int log_size) {
  constexpr int kStage = Few<J>::kStage;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char* gen = smem_raw + (base - raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(gen + kFewStages * kStage);
  const uint32_t full = base + kFewStages * kStage, empty = full + 8 * kFewStages, acc_full = empty + 8 * kFewStages, ready = acc_full + 8;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + 2 * kFewStages + 2);
  int* s_fail = reinterpret_cast<int*>(s_tmem + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t limit = a.limit & ~kWaitDropCopy;
  const int size = 1 << log_size;
  const uint32_t rank = blockIdx.x & (uint32_t)(size - 1);  // in the cluster
  const int mblocks = (a.m_total + kTileM - 1) / kTileM, t = (int)(blockIdx.x >> log_size);
  if (tid == 0) {
    for (int i = 0; i < kFewStages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(ready, size);
    *s_fail = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc<1>(smem_u32(s_tmem), kFewTmem);
  if (tid == 64) {
    prefetch_map(&map_a);
    prefetch_map(&map_b);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *s_tmem;
  cluster_arrive();  // this CTA's barriers are ready; waited for when the contraction is done, so at no cost
  dependents_go();  // tensor memory is allocated
  dependency_wait();
  Tile x;
  int64_t out_row0;
  if constexpr (KIND == kGradW) {
    const int per = mblocks * ((a.j_total + J - 1) / J);
    x.e = t / per;
    x.row0 = t % per / mblocks * J;
    x.rows = a.j_total - x.row0 < J ? a.j_total - x.row0 : J;
    x.width = (x.rows + 15) & ~15;
    x.k0 = a.off ? clamp_row(a.off, x.e, a.rows) : 0;
    x.klen = (a.off ? clamp_row(a.off, x.e + 1, a.rows) : a.rows) - x.k0;
    out_row0 = (int64_t)x.e * a.j_total + x.row0;
  } else {
    if (!few_tile<J>(t / mblocks, a, x)) {  // the whole cluster: the grid covers the most tiles these sizes can have
      if (warp == 1) tmem_free<1>(tmem, kFewTmem);
      cluster_wait();
      return;
    }
    x.k0 = 0;
    x.klen = a.k;
    out_row0 = x.row0;
  }
  x.m0 = (t % mblocks) * kTileM;
  const int chunks = x.klen > 0 ? (x.klen + kKC - 1) / kKC : 0;
  const int c0 = (int)(((uint32_t)chunks * rank) >> log_size), c1 = (int)(((uint32_t)chunks * (rank + 1)) >> log_size);
  bool ok = true;
  if (warp == 0) {
    const int boxes = KIND == kGradW ? 0 : x.width / kFewBox;
    const uint32_t bytes = kABytes + (uint32_t)(KIND == kGradW ? kBoxBytes : boxes * kFewBox * 128);
    int st = 0;
    uint32_t ph = 0;
    for (int c = c0; c < c1; ++c) {
      if (!__all_sync(0xffffffffu, mbar_wait(empty + 8 * st, ph ^ 1u, limit))) {
        ok = false;
        break;
      }
      if (elect_one()) {
        const uint32_t sa = base + st * kStage, sb = sa + kABytes, bar = full + 8 * st;
        mbar_arrive_tx(bar, bytes);
        if ((a.limit & kWaitDropCopy) && rank == 0) {
          // testing, as in the kernel above; one CTA of a cluster, so that its peers have to wait for one that gives up
        } else if constexpr (KIND == kFwdT) {
          tma_3d<1>(sa, &map_a, c * kKC, x.m0, x.e, bar);
        } else if constexpr (KIND == kGradW) {
          tma_2d<1>(sa, &map_a, x.m0, x.k0 + c * kKC, bar);
          tma_2d<1>(sa + kBoxBytes, &map_a, x.m0 + 64, x.k0 + c * kKC, bar);
        } else {
          tma_3d<1>(sa, &map_a, x.m0, c * kKC, x.e, bar);
          tma_3d<1>(sa + kBoxBytes, &map_a, x.m0 + 64, c * kKC, x.e, bar);
        }
        if constexpr (KIND == kGradW) tma_2d<1>(sb, &map_b, x.row0, x.k0 + c * kKC, bar);
        for (int b = 0; b < boxes; ++b) tma_2d<1>(sb + b * kFewBox * 128, &map_b, c * kKC, x.row0 + b * kFewBox, bar);
      }
      __syncwarp();
      if (++st == kFewStages) {
        st = 0;
        ph ^= 1u;
      }
    }
  } else if (warp == 1) {
    int st = 0;
    uint32_t ph = 0;
    constexpr uint32_t kMajor = KIND == kFwdN ? (1u << 15) : KIND == kGradW ? (1u << 15) | (1u << 16) : 0u;
    const uint32_t idesc = (1u << 4) | a.types | kMajor | ((uint32_t)(x.width >> 3) << 17) | ((uint32_t)(kTileM >> 4) << 24);
    constexpr uint32_t kStepA = KIND == kFwdT ? 2u : 128u, kStepB = KIND == kGradW ? 128u : 2u;
    for (int c = c0; c < c1; ++c) {
      if (!__all_sync(0xffffffffu, mbar_wait(full + 8 * st, ph, limit))) {
        ok = false;
        break;
      }
      const int left = x.klen - c * kKC;
      if (KIND == kGradW && left < kKC && (left & 15) != 0) {
        // rows of the next segment (or none) behind the last one: zeros up to the MMA's sixteen
        const int n16 = (((left + 15) & ~15) - left) * 8;
        unsigned char* tile = gen + st * kStage;
        for (int i = lane; i < 3 * n16; i += 32)  // whole rows of 128 bytes: the swizzle does not matter
          *reinterpret_cast<uint4*>(tile + (i / n16) * kBoxBytes + left * 128 + (i % n16) * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (elect_one()) {
        const uint64_t da = umma_desc(base + st * kStage, kBoxBytes), db = umma_desc(base + st * kStage + kABytes, kBoxBytes);
        const int steps = left >= kKC ? kKC / 16 : (left + 15) / 16;
        for (int s = 0; s < steps; ++s) umma<1>(tmem, da + s * kStepA, db + s * kStepB, idesc, c > c0 || s > 0 ? 1u : 0u);
        umma_commit<1>(empty + 8 * st);
      }
      __syncwarp();
      if (++st == kFewStages) {
        st = 0;
        ph ^= 1u;
      }
    }
    if (ok && elect_one()) umma_commit<1>(acc_full);
    __syncwarp();
  }
  const int quarter = warp & 3;
  const int col = quarter * 32 + lane, m = x.m0 + col;
  const bool epilogue = warp >= 2, in = epilogue && m < a.m_total;
  float bias = 0.f;
  if (epilogue) {
    if (a.bias && in) bias = load_bias(a.bias, (int64_t)x.e * a.ldb + m, a.bias_type);
    ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0u, limit));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (ok && size == 1) {
      const uint32_t d = tmem + ((uint32_t)(quarter * 32) << 16);
      switch (KIND == kGradW ? (int)ALPHASPARSE_ACT_NONE : a.act) {
        case ALPHASPARSE_ACT_RELU: finish_tile<TO, ALPHASPARSE_ACT_RELU, 1>(a, x, m, 0, d, in, bias, out_row0); break;
        case ALPHASPARSE_ACT_GELU: finish_tile<TO, ALPHASPARSE_ACT_GELU, 1>(a, x, m, 0, d, in, bias, out_row0); break;
        case ALPHASPARSE_ACT_SILU: finish_tile<TO, ALPHASPARSE_ACT_SILU, 1>(a, x, m, 0, d, in, bias, out_row0); break;
        default: finish_tile<TO, ALPHASPARSE_ACT_NONE, 1>(a, x, m, 0, d, in, bias, out_row0); break;
      }
    } else if (ok) {
      // every MMA of this CTA is done: the ring's memory takes the sums, [row][column]
      float* sums = reinterpret_cast<float*>(gen);
      for (int j0 = 0; j0 < x.rows; j0 += kCols) {
        uint32_t acc[kCols];
        tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)j0, acc);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          if (j0 + c < x.rows) sums[(j0 + c) * kTileM + col] = c0 < c1 ? __uint_as_float(acc[c]) : 0.f;
      }
    }
  }
  __syncwarp();
  if (!ok && lane == 0) *s_fail = 1;
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*s_fail) {
    if (tid == 0) *a.err = 1;
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
  }
  cluster_wait();
  if (size > 1) {
    // this CTA's sums are complete: every peer is told, and waits for all of them (a barrier instruction of the cluster takes a
    // microsecond, arrivals on each other's barriers half of that)
    if (tid < size) mbar_arrive(peer_u32(ready, tid));
    if (epilogue && !__all_sync(0xffffffffu, mbar_wait_peers(ready, 0u, 2 * limit + kPeerPolls))) {
      *s_fail = 1;
      if (tid == 64) *a.err = 1;
    }
  }
  if (epilogue && size > 1 && !*s_fail) {
    switch (KIND == kGradW ? (int)ALPHASPARSE_ACT_NONE : a.act) {
      case ALPHASPARSE_ACT_RELU: finish_shared<TO, ALPHASPARSE_ACT_RELU>(a, x, out_row0, m, col, base, rank, (uint32_t)size, in, bias); break;
      case ALPHASPARSE_ACT_GELU: finish_shared<TO, ALPHASPARSE_ACT_GELU>(a, x, out_row0, m, col, base, rank, (uint32_t)size, in, bias); break;
      case ALPHASPARSE_ACT_SILU: finish_shared<TO, ALPHASPARSE_ACT_SILU>(a, x, out_row0, m, col, base, rank, (uint32_t)size, in, bias); break;
      default: finish_shared<TO, ALPHASPARSE_ACT_NONE>(a, x, out_row0, m, col, base, rank, (uint32_t)size, in, bias); break;
    }
  }
  __syncwarp();
  if (size > 1) {
    // the epilogue's warps have read their peers' sums; warp 0's arrivals on the peers' barriers must have landed (a peer that gave up
    // `ready` has not waited for them)
    if (warp == 0) cluster_arrive();
    else cluster_arrive_relaxed();
  }
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1) tmem_free<1>(tmem, kFewTmem);
  if (size > 1) cluster_wait();  // no CTA leaves while a peer can reach its shared memory
}

// ---- operands the TMA cannot take: aligned copies -----------------------------------------------
struct Copy16 {
  const void* in;
  void* out;
  int64_t rows, ld, ldo;  // in units of the copy
  int cols;
  int64_t block;          // rows of an expert's block (0: all rows are wanted); those of experts without rows are left out
};
// Up to two matrices in one launch, in units of 4 bytes where every row starts on such a boundary, else of 2; a warp per row, sixteen
// loads in flight per lane (bound by HBM: 1 GB moved for 27 blocks of 3,224 x 2,965).
template <typename U>
__global__ void __launch_bounds__(256)
expert_repack_kernel(const __grid_constant__ Copy16 a, const __grid_constant__ Copy16 b, const int32_t* off, int rows) {
  dependency_wait();
  dependents_go();
  const int lane = threadIdx.x & 31;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5; i < a.rows + b.rows; i += (int64_t)gridDim.x * 8) {
    const Copy16& m = i < a.rows ? a : b;
    const int64_t r = i < a.rows ? i : i - a.rows;
    if (m.block && off) {
      const int e = (int)(r / m.block);
      if (clamp_row(off, e, rows) >= clamp_row(off, e + 1, rows)) continue;
    }
    const U* in = (const U*)m.in + r * m.ld;
    U* out = (U*)m.out + r * m.ldo;
    constexpr int kBatch = 16;
    for (int c = lane; c < m.cols; c += 32 * kBatch) {
      U v[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (c + 32 * k < m.cols) v[k] = in[c + 32 * k];
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (c + 32 * k < m.cols) out[c + 32 * k] = v[k];
    }
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
               ? reinterpret_cast<EncodeTiledFn>(p)
               : nullptr;
  }();
  return fn;
}

// A 16-bit operand ready for the TMA: base on 16 bytes, rows a multiple of 16 bytes apart.
struct Operand {
  void* p;
  int64_t rows, cols, ld;
  alphasparseDataType type;
};
bool tma_ready(alphasparseDnMatDescr_t m) {
  return m->rows == 0 || m->cols == 0 || ((reinterpret_cast<uintptr_t>(m->values) & 15) == 0 && (m->ld & 7) == 0);
}
int64_t padded8(int64_t cols) { return (cols + 7) & ~(int64_t)7; }
size_t repack_bytes(alphasparseDnMatDescr_t m) {
  return tma_ready(m) ? 0 : (((size_t)m->rows * (size_t)padded8(m->cols) * 2 + 255) & ~(size_t)255);
}
size_t repack_bytes(alphasparseDnMatDescr_t a, alphasparseDnMatDescr_t b) {
  const size_t n = repack_bytes(a) + repack_bytes(b);
  return n ? n + 256 : 0;
}
// (block: rows of an expert's block of mb, 0 if mb is not stacked)
alphasparseStatus_t ready_operands(alphasparseHandle_t h, alphasparseDnMatDescr_t ma, alphasparseDnMatDescr_t mb, int64_t block,
                                   const int32_t* off, void* buffer, Operand* a, Operand* b) {
  unsigned char* scratch = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(buffer) + 255) & ~(uintptr_t)255);
  Copy16 copies[2] = {};
  alphasparseDnMatDescr_t m[2] = {ma, mb};
  Operand* o[2] = {a, b};
  bool words = true;
  for (int i = 0; i < 2; ++i) {
    *o[i] = {m[i]->values, m[i]->rows, m[i]->cols, m[i]->ld, m[i]->data_type};
    if (tma_ready(m[i])) continue;
    o[i]->p = scratch;
    o[i]->ld = padded8(m[i]->cols);
    copies[i] = {m[i]->values, o[i]->p, m[i]->rows, m[i]->ld, o[i]->ld, (int)m[i]->cols, i == 1 ? block : 0};
    words &= (reinterpret_cast<uintptr_t>(m[i]->values) & 3) == 0 && (m[i]->ld & 1) == 0 && (m[i]->cols & 1) == 0;
    scratch += repack_bytes(m[i]);
  }
  const int64_t blocks = (copies[0].rows + copies[1].rows + 7) / 8, most = 8 * (int64_t)impl(h)->sm_count;
  if (blocks == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
  if (words)
    for (Copy16& c : copies) c.ld /= 2, c.ldo /= 2, c.cols /= 2;
  return launch_chained(h, words ? expert_repack_kernel<uint32_t> : expert_repack_kernel<uint16_t>,
                        dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, 1, copies[0], copies[1], off, (int)ma->rows);
}

// blocks > 0: a third dimension over stacked blocks of rows / blocks rows each (out-of-range rows of a block read as
// zero, not as the next block's).
alphasparseStatus_t tensor_map(CUtensorMap* map, const Operand& o, int64_t blocks, uint32_t box_cols, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
  const cuuint32_t rank = blocks > 0 ? 3 : 2;
  const int64_t per = blocks > 0 ? o.rows / blocks : o.rows;
  const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)per, (cuuint64_t)blocks};
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)o.ld * 2 * (cuuint64_t)per};
  const cuuint32_t box[3] = {box_cols, box_rows, 1}, ones[3] = {1, 1, 1};
  const CUresult r = fn(map, o.type == ALPHA_R_16F ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, o.p, dims,
                        strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ALPHA_SPARSE_STATUS_SUCCESS : ALPHA_SPARSE_STATUS_INVALID_VALUE;
}

uint32_t type_bits(alphasparseDataType t) { return t == ALPHA_R_16BF ? (1u << 7) | (1u << 10) : 0u; }

// The most shared memory a kernel may take, set once per device.
template <typename K>
alphasparseStatus_t allow_smem(K* kernel, int bytes, int device, std::atomic<uint64_t>* done) {
  const uint64_t bit = uint64_t(1) << (device & 63);
  if (device < 64 && (done->load(std::memory_order_relaxed) & bit)) return ALPHA_SPARSE_STATUS_SUCCESS;
  ASP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done->fetch_or(bit, std::memory_order_relaxed);
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

template <int KIND, typename TO>
alphasparseStatus_t launch_mm(alphasparseHandle_t h, const CUtensorMap& ma, const CUtensorMap& mb, const MmArgs& a, int64_t tiles) {
  constexpr size_t smem = 1024 + (size_t)kMmStages * kMmStage + 8 * (3 * kMmStages + 4) + 8 + 8 * (ALPHASPARSE_MAX_EXPERTS + 1);
  static std::atomic<uint64_t> done{0};
  const auto kernel = expert_mm_kernel<KIND, TO>;
  const alphasparseStatus_t s = allow_smem(kernel, (int)smem, h->device, &done);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  const int64_t most = impl(h)->sm_count / 2;
  return launch_chained(h, kernel, dim3((unsigned)((tiles < most ? tiles : most) * 2)), dim3(kMmThreads), smem, 2, ma, mb, a);
}
template <int KIND>
alphasparseStatus_t launch_mm(alphasparseHandle_t h, const CUtensorMap& ma, const CUtensorMap& mb, const MmArgs& a, int64_t tiles,
                              alphasparseDataType out) {
  switch (out) {
    case ALPHA_R_32F: return launch_mm<KIND, float>(h, ma, mb, a, tiles);
    case ALPHA_R_16F: return launch_mm<KIND, __half>(h, ma, mb, a, tiles);
    default: return launch_mm<KIND, __nv_bfloat16>(h, ma, mb, a, tiles);
  }
}

template <int KIND, int J, typename TO>
alphasparseStatus_t launch_few(alphasparseHandle_t h, const CUtensorMap& ma, const CUtensorMap& mb, const MmArgs& a, int64_t tiles,
                               int64_t chunks) {
  static std::atomic<uint64_t> done{0};
  const auto kernel = expert_mm_few_kernel<KIND, J, TO>;
  const alphasparseStatus_t s = allow_smem(kernel, Few<J>::kSmem, h->device, &done);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  // CTAs that share a tile's contraction: as many as fit the device at once, a ring's worth of stages each
  const int resident = (J == 16 ? 3 : 2) * impl(h)->sm_count;
  int log_size = 0;
  while ((1 << log_size) < kFewSplit && (tiles << log_size) * 2 <= resident && chunks >= ((2 * kFewStages) << log_size)) ++log_size;
  return launch_chained(h, kernel, dim3((unsigned)(tiles << log_size)), dim3(kFewThreads), Few<J>::kSmem, 1 << log_size, ma, mb, a, log_size);
}
template <int KIND, int J>
alphasparseStatus_t launch_few(alphasparseHandle_t h, const CUtensorMap& ma, const CUtensorMap& mb, const MmArgs& a, int64_t tiles,
                               int64_t chunks, alphasparseDataType out) {
  switch (out) {
    case ALPHA_R_32F: return launch_few<KIND, J, float>(h, ma, mb, a, tiles, chunks);
    case ALPHA_R_16F: return launch_few<KIND, J, __half>(h, ma, mb, a, tiles, chunks);
    default: return launch_few<KIND, J, __nv_bfloat16>(h, ma, mb, a, tiles, chunks);
  }
}

bool type16(alphasparseDataType t) { return t == ALPHA_R_16F || t == ALPHA_R_16BF; }

struct MmShape {
  int64_t rows, n, k;
};
// Which kernel: 0 the pair kernel, else the one for few rows per segment with tiles of 16 (1) or 64 rows (2).  Up to 16 rows per
// segment the weights' bytes are the work and many small CTAs draw them faster (64 experts x 2,048 x 1,408, 64 to 1,024 rows: 74-76 us
// against 85-87; at 2,048 rows 89 against 87).  Beyond, it is the number of tiles that decides: where pair tiles would leave half of
// the pairs idle and the small tiles still fit the device at once, the small ones run (one 4,096 x 4,096 layer, 32 / 128 / 256 rows:
// 15 / 18 / 24 us against 26 / 28 / 29; 512 rows 35 against 30; eight 2,048 x 2,048 layers, 256 rows: 23 against 22).
// How the rows are spread is not known on the host.  Where most go to one expert, its weights are read once per 16 rows, from L2: at
// 64 experts x 2,048 x 1,408 and the rule's limit of 1,024 rows 60 us against 69 when they are even, 66 against 70 with half of them at
// one expert, 77 against 69 with 961; at 512 rows 64 against 68 with 449 at one.  It loses more with more experts: 256 of them, 4,096 rows,
// 225 against 236 when even, 260 against 243 with half at one, 104 against 29 with all at one.
int few_rows(alphasparseHandle_t h, const MmShape& s, int64_t filled) {
  const int64_t pairs = (s.rows / kTileJ + filled) * ((s.n + kPairM - 1) / kPairM);
  if (s.rows <= 16 * filled) return 1;
  const int64_t small = (s.rows / 64 + filled) * ((s.n + kTileM - 1) / kTileM);
  return pairs * 4 <= impl(h)->sm_count && small <= 2 * (int64_t)impl(h)->sm_count ? 2 : 0;
}
alphasparseStatus_t check_mm(alphasparseHandle_t h, alphasparseOperation_t op, int64_t segments, const int32_t* off,
                             alphasparseDnMatDescr_t x, alphasparseDnMatDescr_t w, alphasparseDnMatDescr_t y, MmShape* shape) {
  if (!h) return ALPHA_SPARSE_STATUS_INVALID_HANDLE;
  if (!x || !w || !y) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  if (op != ALPHA_SPARSE_OPERATION_NON_TRANSPOSE && op != ALPHA_SPARSE_OPERATION_TRANSPOSE)
    return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
  alphasparseStatus_t s = expert_check_segments(segments, off);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (!type16(x->data_type) || w->data_type != x->data_type ||
      (y->data_type != x->data_type && y->data_type != ALPHA_R_32F))
    return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
  const int64_t n = y->cols, k = x->cols;
  if ((s = expert_check_mat(x, -1, -1)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if ((s = expert_check_mat(y, x->rows, -1)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  const bool nk = op == ALPHA_SPARSE_OPERATION_TRANSPOSE;
  if ((s = expert_check_mat(w, segments * (nk ? n : k), nk ? k : n)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  *shape = {x->rows, n, k};
  return ALPHA_SPARSE_STATUS_SUCCESS;
}
alphasparseStatus_t check_grad_w(alphasparseHandle_t h, alphasparseOperation_t op, int64_t segments, const int32_t* off,
                                 alphasparseDnMatDescr_t x, alphasparseDnMatDescr_t dz, alphasparseDnMatDescr_t dw) {
  if (!h) return ALPHA_SPARSE_STATUS_INVALID_HANDLE;
  if (!x || !dz || !dw) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  if (op != ALPHA_SPARSE_OPERATION_NON_TRANSPOSE && op != ALPHA_SPARSE_OPERATION_TRANSPOSE)
    return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
  alphasparseStatus_t s = expert_check_segments(segments, off);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (!type16(x->data_type) || dz->data_type != x->data_type ||
      (dw->data_type != x->data_type && dw->data_type != ALPHA_R_32F))
    return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
  if ((s = expert_check_mat(x, -1, -1)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if ((s = expert_check_mat(dz, x->rows, -1)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  const bool nk = op == ALPHA_SPARSE_OPERATION_TRANSPOSE;
  return expert_check_mat(dw, segments * (nk ? dz->cols : x->cols), nk ? x->cols : dz->cols);
}

}  // namespace
}  // namespace asp

using namespace asp;

extern "C" {

alphasparseStatus_t alphasparseExpertMM_bufferSize(alphasparseHandle_t h, alphasparseOperation_t op, int64_t segments,
                                                   const int32_t* off, alphasparseDnMatDescr_t x,
                                                   alphasparseDnMatDescr_t w, alphasparseDnMatDescr_t y, size_t* size) {
  if (!size) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  MmShape shape;
  const alphasparseStatus_t s = check_mm(h, op, segments, off, x, w, y, &shape);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  *size = repack_bytes(x, w);
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

alphasparseStatus_t alphasparseExpertMM(alphasparseHandle_t h, alphasparseOperation_t op, int64_t segments,
                                        const int32_t* off, alphasparseDnMatDescr_t x, alphasparseDnMatDescr_t w,
                                        alphasparseDnMatDescr_t bias, alphasparseActivation_t act,
                                        alphasparseDnMatDescr_t r, alphasparseDnMatDescr_t z, alphasparseDnMatDescr_t y,
                                        void* buffer) {
  MmShape shape;
  alphasparseStatus_t s = check_mm(h, op, segments, off, x, w, y, &shape);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if ((int)act < ALPHASPARSE_ACT_NONE || (int)act > ALPHASPARSE_ACT_SILU) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
  if ((r && r->data_type != y->data_type) || (z && z->data_type != y->data_type) ||
      (bias && bias->data_type != x->data_type && bias->data_type != ALPHA_R_32F))
    return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
  if (bias && (s = expert_check_mat(bias, segments, shape.n)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (r && (s = expert_check_mat(r, shape.rows, shape.n)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (z && (s = expert_check_mat(z, shape.rows, shape.n)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (shape.rows == 0 || shape.n == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
  if (!buffer && repack_bytes(x, w)) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  if (!impl(h)->dev_err) return ALPHA_SPARSE_STATUS_NOT_INITIALIZED;  // a handle that alphasparseGetHandle has not set up
  DeviceScope dev(h->device);
  ASP_CUDA(dev.status);
  const bool nk = op == ALPHA_SPARSE_OPERATION_TRANSPOSE;
  Operand ox, ow;
  if ((s = ready_operands(h, x, w, nk ? shape.n : shape.k, off, buffer, &ox, &ow)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  MmArgs a = {};
  a.off = off;
  a.segments = (int)segments;
  a.rows = (int)shape.rows;
  a.m_total = (int)shape.n;
  a.k = (int)shape.k;
  // at most: every segment with rows ends in a tile of its own
  const int64_t filled = segments < shape.rows ? segments : shape.rows;
  const int few = few_rows(h, shape, filled);
  // rows of X per box: whole halves of a tile where segments fill tiles, less where a box would mostly fetch rows of other segments
  a.box_rows = few ? kFewBox : shape.rows > 256 * filled ? 128 : shape.rows > 64 * filled ? 64 : 32;
  a.types = type_bits(x->data_type);
  a.y = y->values;
  a.ldy = y->ld;
  if (r) a.r = r->values, a.ldr = r->ld;
  if (z) a.z = z->values, a.ldz = z->ld;
  if (bias) a.bias = bias->values, a.ldb = bias->ld, a.bias_type = (int)bias->data_type;
  a.act = (int)act;
  a.limit = wait_limit(h, shape.k / kKC);
  a.err = impl(h)->dev_err;
  CUtensorMap mw = {}, mx = {};
  if (shape.k > 0) {
    if ((s = tensor_map(&mw, ow, segments, 64, nk ? kTileM : kKC)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
    if ((s = tensor_map(&mx, ox, 0, kKC, (uint32_t)a.box_rows)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  }
  if (few) {
    const int j = few == 1 ? 16 : 64;
    const int64_t chunks = (shape.k + kKC - 1) / kKC;
    const int64_t tiles = (shape.rows / j + filled) * ((shape.n + kTileM - 1) / kTileM);
    if (few == 1)
      return nk ? launch_few<kFwdT, 16>(h, mw, mx, a, tiles, chunks, y->data_type) : launch_few<kFwdN, 16>(h, mw, mx, a, tiles, chunks, y->data_type);
    return nk ? launch_few<kFwdT, 64>(h, mw, mx, a, tiles, chunks, y->data_type) : launch_few<kFwdN, 64>(h, mw, mx, a, tiles, chunks, y->data_type);
  }
  const int64_t tiles = (shape.rows / kTileJ + filled) * ((shape.n + kPairM - 1) / kPairM);
  return nk ? launch_mm<kFwdT>(h, mw, mx, a, tiles, y->data_type) : launch_mm<kFwdN>(h, mw, mx, a, tiles, y->data_type);
}

alphasparseStatus_t alphasparseExpertMM_gradW_bufferSize(alphasparseHandle_t h, alphasparseOperation_t op,
                                                         int64_t segments, const int32_t* off,
                                                         alphasparseDnMatDescr_t x, alphasparseDnMatDescr_t dz,
                                                         alphasparseDnMatDescr_t dw, size_t* size) {
  if (!size) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  const alphasparseStatus_t s = check_grad_w(h, op, segments, off, x, dz, dw);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  *size = repack_bytes(x, dz);
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

alphasparseStatus_t alphasparseExpertMM_gradW(alphasparseHandle_t h, alphasparseOperation_t op, int64_t segments,
                                              const int32_t* off, alphasparseDnMatDescr_t x, alphasparseDnMatDescr_t dz,
                                              alphasparseDnMatDescr_t dw, void* buffer) {
  alphasparseStatus_t s = check_grad_w(h, op, segments, off, x, dz, dw);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  const bool nk = op == ALPHA_SPARSE_OPERATION_TRANSPOSE;
  alphasparseDnMatDescr_t m = nk ? x : dz, j = nk ? dz : x;  // columns and rows of a block of dW
  if (m->cols == 0 || j->cols == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
  if (!buffer && repack_bytes(x, dz)) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  if (!impl(h)->dev_err) return ALPHA_SPARSE_STATUS_NOT_INITIALIZED;  // a handle that alphasparseGetHandle has not set up
  DeviceScope dev(h->device);
  ASP_CUDA(dev.status);
  Operand om, oj;
  if ((s = ready_operands(h, m, j, 0, nullptr, buffer, &om, &oj)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  MmArgs a = {};
  a.off = off;
  a.segments = (int)segments;
  a.rows = (int)x->rows;
  a.m_total = (int)m->cols;
  a.j_total = (int)j->cols;
  a.types = type_bits(x->data_type);
  a.y = dw->values;
  a.ldy = dw->ld;
  a.limit = wait_limit(h, x->rows / kKC);
  a.err = impl(h)->dev_err;
  CUtensorMap mm = {}, mj = {};
  if (x->rows > 0) {
    if ((s = tensor_map(&mm, om, 0, 64, kKC)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
    if ((s = tensor_map(&mj, oj, 0, 64, kKC)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  }
  const int64_t tiles = segments * ((m->cols + kPairM - 1) / kPairM) * ((j->cols + kTileJ - 1) / kTileJ);
  if (tiles >= (int64_t(1) << 31)) return ALPHA_SPARSE_STATUS_INVALID_SIZE;
  // as in few_rows: small tiles, and clusters that share the rows of a segment, where pair tiles would leave half of the pairs idle and
  // the contraction is long (two segments, 3,879 rows, 432 x 232: 24 us with dX against 32; below 512 rows a segment it loses 2 us)
  const int64_t small = segments * ((m->cols + kTileM - 1) / kTileM) * ((j->cols + 63) / 64);
  if (x->rows > 512 * segments && tiles * 4 <= impl(h)->sm_count && small <= 2 * (int64_t)impl(h)->sm_count)
    return launch_few<kGradW, 64>(h, mm, mj, a, small, x->rows / (segments * kKC), dw->data_type);
  return launch_mm<kGradW>(h, mm, mj, a, tiles, dw->data_type);
}

}  // extern "C"
