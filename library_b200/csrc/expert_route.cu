// The routing matrix of a mixture-of-experts layer: tokens sorted by expert, and back.
//
// The routing matrix is tokens x experts with topk entries per row, so its row offsets need no
// array; what has to be built is the column-wise form, the order an expert reads its tokens in.
//   sort      position[s] = offset[e_s] + |{s' < s : e_s' = e_s}|   (a stable counting sort by expert)
//   dispatch  Xs[position[t,j]] = X[t]
//   combine   Y[t] = sum_j w[t,j] Ys[position[t,j]] + R[t]
//   gradient  dYs[position[t,j]] = w[t,j] dY[t],   dw[t,j] = <dY[t], Ys[position[t,j]]>
// All row movement is organised by token: a row of X, dY or R is read once however many experts
// it goes to, and only `position` is needed, never its inverse.
#include <cooperative_groups.h>

#include <algorithm>

#include "expert_launch.h"
#include "expert_vec.h"

namespace cg = cooperative_groups;

namespace asp {
namespace {

constexpr int kSortWarps = 16;
constexpr int kSortThreads = kSortWarps * 32;
constexpr int kSortCluster = 8;                  // CTAs of the one-launch sort (portable cluster size)
constexpr int kSortBatch = 4;                    // ids a lane asks for at a time
// Slots above which the sort runs on the whole device in two launches instead of one cluster: at 16,384 the cluster's CTAs hold four
// steps a warp (5.3 us); at 65,536 it would take 10.4 us.
constexpr int64_t kSortClusterSlots = 1 << 14;

// Shared memory of a sorting CTA: counts[experts][kSortRow] (a column per warp; the odd stride keeps a row's and a column's
// accesses off the same banks), then totals, all and base[experts], then a word per warp.
constexpr int kSortRow = kSortWarps + 1;
constexpr int sort_words(int experts) { return experts * kSortRow + 3 * experts + kSortWarps; }

// The slots of a warp, a multiple of 32 from `begin` on.  Warps and CTAs take ascending ranges, so that counting by CTA, then warp and
// slot is the stable order.
struct SlotRange {
  int64_t begin, end;
};
__device__ __forceinline__ SlotRange warp_slots(int64_t slots) {
  const int64_t parts = (int64_t)gridDim.x * kSortWarps, part = (int64_t)blockIdx.x * kSortWarps + (threadIdx.x >> 5);
  const int64_t per = (slots + parts * 32 - 1) / (parts * 32) * 32, begin = per * part;
  return {begin, begin + per < slots ? begin + per : slots};
}
template <typename Id>
__device__ __forceinline__ void load_ids(const Id* ids, int64_t s, int64_t end, int experts, int (&id)[kSortBatch]) {
#pragma unroll
  for (int i = 0; i < kSortBatch; ++i) {
    id[i] = -1;
    if (s + 32 * i < end) {
      const Id v = ids[s + 32 * i];
      if (v >= 0 && v < (Id)experts) id[i] = (int)v;
    }
  }
}

// counts[e][w]: the slots of e that the CTA's warps before w hold.  totals[e]: the CTA's.
template <typename Id>
__device__ __forceinline__ void count_slots(const Id* ids, int experts, SlotRange r, int* counts, int* totals) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int id[kSortBatch];
  load_ids(ids, r.begin + lane, r.end, experts, id);  // on their way while the counts are cleared
  for (int i = tid; i < experts * kSortRow; i += kSortThreads) counts[i] = 0;
  __syncthreads();
  for (int64_t s = r.begin + lane;;) {
#pragma unroll
    for (int i = 0; i < kSortBatch; ++i)
      if (id[i] >= 0) atomicAdd(&counts[id[i] * kSortRow + warp], 1);  // whole numbers: the order does not matter
    s += 32 * kSortBatch;
    if (s - lane >= r.end) break;
    load_ids(ids, s, r.end, experts, id);
  }
  __syncthreads();
  const int sub = lane % kSortWarps;
  for (int e0 = warp * 2; e0 < experts; e0 += kSortWarps * 2) {  // half a warp per expert
    const int e = e0 + lane / kSortWarps;
    const int c = e < experts ? counts[e * kSortRow + sub] : 0;
    int v = c;
#pragma unroll
    for (int o = 1; o < kSortWarps; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (sub >= o) v += u;
    }
    if (e < experts) {
      counts[e * kSortRow + sub] = v - c;
      if (sub == kSortWarps - 1) totals[e] = v;
    }
  }
  __syncthreads();
}

// position[] of the warp's slots: base[e] is where the CTA's first slot of e goes.
template <typename Id, int BITS>
__device__ __forceinline__ void place_slots(const Id* ids, int experts, SlotRange r, int* counts, const int* base,
                                            int32_t* __restrict__ position) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int64_t s = r.begin + lane; s - lane < r.end; s += 32 * kSortBatch) {
    int id[kSortBatch];
    load_ids(ids, s, r.end, experts, id);
#pragma unroll
    for (int i = 0; i < kSortBatch; ++i) {
      if (s - lane + 32 * i >= r.end) break;
      const int e = id[i];
      // lanes with the same expert: a ballot per bit of the number
      unsigned same = __ballot_sync(0xffffffffu, e >= 0);
#pragma unroll
      for (int b = 0; b < BITS; ++b) {
        const bool bit = (e & (1 << b)) != 0;
        same &= __ballot_sync(0xffffffffu, bit) ^ (bit ? 0u : ~0u);
      }
      const int before = __popc(same & ((1u << lane) - 1u));
      int* count = &counts[(e >= 0 ? e : 0) * kSortRow + warp];
      const int at = *count;  // the warp's own column
      __syncwarp();
      if (e >= 0 && before == 0) *count = at + __popc(same);
      __syncwarp();
      if (s + 32 * i < r.end) position[s + 32 * i] = e >= 0 ? base[e] + at + before : -1;
    }
  }
}

// Exclusive prefix over the experts of all[e], in place, consecutive experts per thread; returns the sum.
__device__ int scan_experts(int* all, int experts, int* warp_sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kPer = (ALPHASPARSE_MAX_EXPERTS + kSortThreads - 1) / kSortThreads;
  int n[kPer], mine = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    n[i] = tid * kPer + i < experts ? all[tid * kPer + i] : 0;
    mine += n[i];
  }
  int v = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kSortWarps; ++w) {
    const int s = warp_sums[w];
    if (w < warp) before += s;
    sum += s;
  }
  int run = before + v - mine;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (tid * kPer + i < experts) all[tid * kPer + i] = run;
    run += n[i];
  }
  __syncthreads();
  return sum;
}
// The whole sort in one launch of one thread-block cluster: counts meet in distributed shared memory.
template <typename Id, int BITS>
__global__ void __launch_bounds__(kSortThreads)
route_sort_cluster_kernel(const Id* ids, int64_t slots, int experts, int32_t* __restrict__ offsets,
                          int32_t* __restrict__ position) {
  extern __shared__ int sort_smem[];
  int* counts = sort_smem;
  int* totals = counts + experts * kSortRow;
  int* all = totals + experts;
  int* base = all + experts;
  int* warp_sums = base + experts;
  dependency_wait();
  dependents_go();
  cg::cluster_group cl = cg::this_cluster();
  const int size = (int)gridDim.x, cta = (int)blockIdx.x;  // the grid is one cluster
  const SlotRange r = warp_slots(slots);
  count_slots(ids, experts, r, counts, totals);
  if (size > 1) cl.sync();
  for (int e = threadIdx.x; e < experts; e += kSortThreads) {
    int sum = totals[e], before = 0;
    if (size > 1) {
      int n[kSortCluster];  // (all peers' totals asked for at once)
#pragma unroll
      for (int c = 0; c < kSortCluster; ++c) n[c] = c < size ? *cl.map_shared_rank(totals + e, c) : 0;
      sum = 0;
#pragma unroll
      for (int c = 0; c < kSortCluster; ++c) {
        if (c < cta) before += n[c];
        sum += n[c];
      }
    }
    all[e] = sum;
    base[e] = before;
  }
  if (size > 1) cl.sync();  // every CTA has read its peers' totals: none may leave before
  else __syncthreads();
  const int kept = scan_experts(all, experts, warp_sums);
  for (int e = threadIdx.x; e < experts; e += kSortThreads) {
    if (cta == 0) offsets[e] = all[e];
    base[e] += all[e];
  }
  if (cta == 0 && threadIdx.x == 0) offsets[experts] = kept;
  __syncthreads();
  place_slots<Id, BITS>(ids, experts, r, counts, base, position);
}

// The same on the whole device in two launches, for long inputs: the CTAs' totals before[b][e]; then every CTA adds them up for itself,
// those of the CTAs before it and all of them, and places its slots.
template <typename Id>
__global__ void __launch_bounds__(kSortThreads)
route_sort_count_kernel(const Id* ids, int64_t slots, int experts, int* __restrict__ before) {
  extern __shared__ int sort_smem[];
  int* totals = sort_smem + experts * kSortRow;
  dependency_wait();
  dependents_go();
  count_slots(ids, experts, warp_slots(slots), sort_smem, totals);
  for (int e = threadIdx.x; e < experts; e += kSortThreads) before[(size_t)blockIdx.x * experts + e] = totals[e];
}
template <typename Id, int BITS>
__global__ void __launch_bounds__(kSortThreads)
route_sort_place_kernel(const Id* ids, int64_t slots, int experts, const int* before,
                        int32_t* __restrict__ offsets, int32_t* __restrict__ position) {
  extern __shared__ int sort_smem[];
  int* counts = sort_smem;
  int* totals = counts + experts * kSortRow;
  int* all = totals + experts;
  int* base = all + experts;
  int* warp_sums = base + experts;
  const SlotRange r = warp_slots(slots);
  for (int e = threadIdx.x; e < experts; e += kSortThreads) all[e] = base[e] = 0;
  dependency_wait();
  dependents_go();
  count_slots(ids, experts, r, counts, totals);
  const int parts = experts < kSortThreads ? kSortThreads / experts : 1, blocks = (int)gridDim.x;
  for (int i = threadIdx.x; i < parts * experts; i += kSortThreads) {
    const int e = i % experts;
    int sum = 0, mine = 0;
#pragma unroll 8
    for (int b = i / experts; b < blocks; b += parts) {
      const int c = before[(size_t)b * experts + e];
      sum += c;
      mine += b < (int)blockIdx.x ? c : 0;
    }
    atomicAdd(&all[e], sum);
    atomicAdd(&base[e], mine);
  }
  __syncthreads();
  const int kept = scan_experts(all, experts, warp_sums);
  for (int e = threadIdx.x; e < experts; e += kSortThreads) {
    if (blockIdx.x == 0) offsets[e] = all[e];
    base[e] += all[e];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) offsets[experts] = kept;
  __syncthreads();
  place_slots<Id, BITS>(ids, experts, r, counts, base, position);
}

// ---- row movement ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;

// A warp takes a token's stretch of 32 * U packs: loads it once, stores it to every sorted row.  Bound by HBM's writes: 1 KB per warp takes
// 56.6 us with the sort for 8,192 tokens x 8 rows of 2,048 bf16 (302 MB), 2 KB 58.9, 512 bytes 57.1 us.
template <typename T, int V, int U>
__global__ void __launch_bounds__(kRowThreads)
route_dispatch_kernel(const T* x, int64_t ldx, T* __restrict__ xs, int64_t ldxs,
                      const int32_t* position, int tokens, int topk, int packs, int stretches, int xs_rows) {
  const int lane = threadIdx.x & 31;
  const int64_t task = ((int64_t)blockIdx.x * kRowThreads + threadIdx.x) >> 5;
  dependency_wait();
  dependents_go();
  if (task >= (int64_t)tokens * stretches) return;
  const int t = (int)(task / stretches), c0 = (int)(task % stretches) * (32 * U) + lane;
  Pack<T, V> row[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (c0 + 32 * u < packs) row[u] = load_pack<T, V>(x + (int64_t)t * ldx + (int64_t)(c0 + 32 * u) * V);
  const int32_t* pos = position + (int64_t)t * topk;
  for (int j0 = 0; j0 < topk; j0 += 32) {
    const int mine = j0 + lane < topk ? pos[j0 + lane] : -1;
    const int n = topk - j0 < 32 ? topk - j0 : 32;
    for (int j = 0; j < n; ++j) {
      const int p = __shfl_sync(0xffffffffu, mine, j);
      if ((unsigned)p >= (unsigned)xs_rows) continue;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + 32 * u < packs) store_pack<T, V>(xs + (int64_t)p * ldxs + (int64_t)(c0 + 32 * u) * V, row[u]);
    }
  }
}

// A warp takes a token's stretch of 32 * U packs of Y and adds up the sorted rows, J of them in flight.  Bound by HBM: what counts is how
// many bytes an SM has on the way and how long the pieces of a row are.  1 KB of four rows per warp and three CTAs per SM: 53 us for
// 8,192 tokens x 8 rows of 2,048 bf16 with a residual (322 MB: 50 us at 6.4 TB/s); 512 bytes of four rows 59 us, of eight rows 64 us;
// warps that walk over several stretches 90 us (neighbouring stretches of a row then run at different times).
template <typename T, int V, int U, int J>
__global__ void __launch_bounds__(kRowThreads, 3)
route_combine_kernel(const T* ys, int64_t ldys, const float* weights, const T* r, int64_t ldr,
                     T* y, int64_t ldy, const int32_t* position, int tokens, int topk, int packs,
                     int stretches, int ys_rows) {
  const int lane = threadIdx.x & 31;
  const int64_t task = ((int64_t)blockIdx.x * kRowThreads + threadIdx.x) >> 5;
  dependency_wait();
  dependents_go();
  if (task >= (int64_t)tokens * stretches) return;
  const int t = (int)(task / stretches), c0 = (int)(task % stretches) * (32 * U) + lane;
  float acc[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int v = 0; v < V; ++v) acc[u][v] = 0.f;
  Pack<T, V> res[U];
  if (r) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + 32 * u < packs) res[u] = load_pack<T, V>(r + (int64_t)t * ldr + (int64_t)(c0 + 32 * u) * V);
  }
  for (int j0 = 0; j0 < topk; j0 += 32) {
    int mine = -1;
    float w_mine = 1.f;
    if (j0 + lane < topk) {
      mine = position[(int64_t)t * topk + j0 + lane];
      if (weights) w_mine = weights[(int64_t)t * topk + j0 + lane];
    }
    const int n = topk - j0 < 32 ? topk - j0 : 32;
    for (int j = 0; j < n; j += J) {
      Pack<T, V> in[J][U];
#pragma unroll
      for (int i = 0; i < J; ++i) {
        const int p = __shfl_sync(0xffffffffu, mine, (j + i) & 31);
        if (j + i < n && (unsigned)p < (unsigned)ys_rows) {
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c0 + 32 * u < packs) in[i][u] = load_pack<T, V>(ys + (int64_t)p * ldys + (int64_t)(c0 + 32 * u) * V);
        }
      }
#pragma unroll
      for (int i = 0; i < J; ++i) {
        const int p = __shfl_sync(0xffffffffu, mine, (j + i) & 31);
        const float w = __shfl_sync(0xffffffffu, w_mine, (j + i) & 31);
        if (j + i >= n || (unsigned)p >= (unsigned)ys_rows) continue;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (c0 + 32 * u < packs) {
#pragma unroll
            for (int v = 0; v < V; ++v) acc[u][v] = fmaf(w, in[i][u].at(v), acc[u][v]);
          }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (c0 + 32 * u < packs) {
      if (r) {
#pragma unroll
        for (int v = 0; v < V; ++v) acc[u][v] += res[u].at(v);
      }
      store_pack<T, V>(y + (int64_t)t * ldy + (int64_t)(c0 + 32 * u) * V, round_pack<T, V>(acc[u]));
    }
}

// Sums of J values over the lanes of a warp (J a power of two, at most 32): lane l ends with the sum of value l % J.
// While more than one value is left, each step sends half of them to the partner and adds the half that comes back:
// 5 shuffles for J = 2 instead of 10.
template <int J>
__device__ __forceinline__ float reduce_values(float (&v)[J], int lane) {
#pragma unroll
  for (int n = J / 2; n > 0; n /= 2) {
    const bool up = (lane & n) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, n);
    }
  }
#pragma unroll
  for (int o = J; o < 32; o *= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}

// Gradient of combine.  blockDim.y tokens per CTA, blockDim.x threads on a token's row (whole warps).  J slots at a time: their rows
// of Ys are all asked for before the first is used; their dot products are added up over lanes, then over the row's warps, in a
// fixed order.  Bound by HBM (435 MB at 8,192 tokens x 6 rows of 2,048 bf16: 68 us at 6.4 TB/s): 1 KB of two rows per warp in flight,
// two tokens per CTA and four CTAs per SM take 71.7 us; 512 bytes of four rows 82 us (one token per CTA 90), of eight rows 105 us.
constexpr int kGradThreads = 128;  // of a token
template <typename T, int V, int U, int J>
__global__ void __launch_bounds__(kRowThreads, 4)
route_combine_grad_kernel(const T* dy, int64_t lddy, const T* ys, int64_t ldys,
                          const float* weights, T* dys, int64_t lddys, float* __restrict__ dweights,
                          const int32_t* position, int tokens, int topk, int packs, int rows) {
  __shared__ float part[kRowThreads / 32][J];
  const int t = (int)blockIdx.x * (int)blockDim.y + (int)threadIdx.y;
  dependency_wait();
  dependents_go();
  const int lane = threadIdx.x & 31;
  const int warps = (int)blockDim.x >> 5, row_warp0 = (int)threadIdx.y * warps, my_warp = row_warp0 + ((int)threadIdx.x >> 5);
  int p_mine = -1;
  float w_mine = 1.f;
  for (int j0 = 0; j0 < topk; j0 += J) {
    if ((j0 & 31) == 0) {  // lane i of every warp holds slot i of the next 32
      p_mine = -1;
      if (t < tokens && j0 + lane < topk) {
        p_mine = position[(int64_t)t * topk + j0 + lane];
        if (weights) w_mine = weights[(int64_t)t * topk + j0 + lane];
      }
    }
    float dot[J];
#pragma unroll
    for (int i = 0; i < J; ++i) dot[i] = 0.f;
    if (t < tokens) {
      // (whole warps step together: the shuffles below need every lane)
      for (int c0 = (int)threadIdx.x - lane; c0 < packs; c0 += (int)blockDim.x * U) {
        Pack<T, V> g[U], in[J][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = c0 + lane + (int)blockDim.x * u;
          if (c < packs) g[u] = load_pack<T, V>(dy + (int64_t)t * lddy + (int64_t)c * V);
        }
        if (dweights) {
#pragma unroll
          for (int i = 0; i < J; ++i) {
            const int p = __shfl_sync(0xffffffffu, p_mine, (j0 + i) & 31);
            if ((unsigned)p >= (unsigned)rows) continue;
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int c = c0 + lane + (int)blockDim.x * u;
              if (c < packs) in[i][u] = load_pack<T, V>(ys + (int64_t)p * ldys + (int64_t)c * V);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < J; ++i) {
          const int p = __shfl_sync(0xffffffffu, p_mine, (j0 + i) & 31);
          const float w = __shfl_sync(0xffffffffu, w_mine, (j0 + i) & 31);
          if ((unsigned)p >= (unsigned)rows) continue;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int c = c0 + lane + (int)blockDim.x * u;
            if (c >= packs) continue;
            float out[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
              const float gv = g[u].at(v);
              if (dweights) dot[i] = fmaf(gv, in[i][u].at(v), dot[i]);
              out[v] = w * gv;
            }
            if (dys) store_pack<T, V>(dys + (int64_t)p * lddys + (int64_t)c * V, round_pack<T, V>(out));
          }
        }
        __syncwarp();
      }
    }
    if (!dweights) continue;
    const float sum_mine = reduce_values<J>(dot, lane);
    if (lane < J) part[my_warp][lane] = sum_mine;
    __syncthreads();
    if (t < tokens && (int)threadIdx.x < J && j0 + (int)threadIdx.x < topk) {
      float sum = 0.f;
      for (int k = 0; k < warps; ++k) sum += part[row_warp0 + k][threadIdx.x];
      dweights[(int64_t)t * topk + j0 + threadIdx.x] = sum;
    }
    if (j0 + J < topk) __syncthreads();  // part is written again
  }
}

alphasparseStatus_t check_routing(alphasparseHandle_t h, alphasparseRoutingDescr_t r) {
  if (!h) return ALPHA_SPARSE_STATUS_INVALID_HANDLE;
  if (!r || !r->init) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

template <typename F>
alphasparseStatus_t by_type(alphasparseDataType t, F f) {
  switch (t) {
    case ALPHA_R_32F: return f(float());
    case ALPHA_R_16F: return f(__half());
    case ALPHA_R_16BF: return f(__nv_bfloat16());
    default: return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
  }
}

// CTAs of the two-launch sort: four steps a warp or more, no more than one per SM.
int64_t sort_blocks(alphasparseHandle_t h, int64_t slots) { return std::min<int64_t>((slots + 2047) / 2048, impl(h)->sm_count); }

template <typename Id, int BITS>
alphasparseStatus_t run_sort(alphasparseHandle_t h, alphasparseRoutingDescr_t r, void* buffer) {
  const int64_t slots = r->tokens * r->topk;
  const int experts = (int)r->experts;
  const Id* ids = (const Id*)r->expert_ids;
  const size_t smem = sizeof(int) * (size_t)sort_words(experts);
  const int most = (int)sizeof(int) * sort_words(ALPHASPARSE_MAX_EXPERTS);
  if (slots <= kSortClusterSlots) {
    const auto kernel = route_sort_cluster_kernel<Id, BITS>;
    if (smem > 48 * 1024) ASP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    int ctas = 1;  // a CTA per 2,048 slots (four steps of its warps), as far as a cluster goes
    while (ctas < kSortCluster && ctas * 2048 < slots) ctas *= 2;
    return launch_chained(h, kernel, dim3(ctas), dim3(kSortThreads), smem, ctas, ids, slots, experts, r->expert_offsets, r->position);
  }
  const int blocks = (int)sort_blocks(h, slots);
  int* before = reinterpret_cast<int*>((reinterpret_cast<uintptr_t>(buffer) + 15) & ~(uintptr_t)15);
  const auto count = route_sort_count_kernel<Id>;
  const auto place = route_sort_place_kernel<Id, BITS>;
  if (smem > 48 * 1024) {
    ASP_CUDA(cudaFuncSetAttribute(count, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    ASP_CUDA(cudaFuncSetAttribute(place, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
  }
  const alphasparseStatus_t s = launch_chained(h, count, dim3(blocks), dim3(kSortThreads), smem, 1, ids, slots, experts, before);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  return launch_chained(h, place, dim3(blocks), dim3(kSortThreads), smem, 1, ids, slots, experts, before, r->expert_offsets, r->position);
}
template <typename Id>
alphasparseStatus_t run_sort(alphasparseHandle_t h, alphasparseRoutingDescr_t r, void* buffer) {
  return r->experts <= 64 ? run_sort<Id, 6>(h, r, buffer) : run_sort<Id, 10>(h, r, buffer);
}
static_assert(ALPHASPARSE_MAX_EXPERTS <= 1 << 10, "ten ballots tell the experts apart");

// Warps for tokens x stretches, as a grid; 0 when there is nothing to do.
int64_t row_blocks(int64_t tokens, int64_t stretches) { return (tokens * stretches * 32 + kRowThreads - 1) / kRowThreads; }

template <typename T, int V>
alphasparseStatus_t run_dispatch(alphasparseHandle_t h, alphasparseRoutingDescr_t r, alphasparseDnMatDescr_t x,
                                 alphasparseDnMatDescr_t xs) {
  constexpr int U = packs_per_lane<T, V>(32);
  const int64_t packs = x->cols / V, stretches = (packs + 32 * U - 1) / (32 * U);
  const int64_t blocks = row_blocks(r->tokens, stretches);
  if (blocks >= (int64_t(1) << 31)) return ALPHA_SPARSE_STATUS_INVALID_SIZE;
  return launch_chained(h, route_dispatch_kernel<T, V, U>, dim3((unsigned)blocks), dim3(kRowThreads), 0, 1,
      (const T*)x->values, x->ld, (T*)xs->values, xs->ld, r->position, (int)r->tokens, (int)r->topk, (int)packs,
      (int)stretches, (int)xs->rows);
}

template <typename T, int V>
alphasparseStatus_t run_combine(alphasparseHandle_t h, alphasparseRoutingDescr_t r, alphasparseDnMatDescr_t ys,
                                const float* weights, alphasparseDnMatDescr_t res, alphasparseDnMatDescr_t y) {
  constexpr int U = packs_per_lane<T, V>(32);
  const int64_t packs = y->cols / V, stretches = (packs + 32 * U - 1) / (32 * U);
  const int64_t blocks = row_blocks(r->tokens, stretches);
  if (blocks >= (int64_t(1) << 31)) return ALPHA_SPARSE_STATUS_INVALID_SIZE;
  return launch_chained(h, route_combine_kernel<T, V, U, 4>, dim3((unsigned)blocks), dim3(kRowThreads), 0, 1,
      (const T*)ys->values, ys->ld, weights, res ? (const T*)res->values : nullptr, res ? res->ld : 0, (T*)y->values,
      y->ld, r->position, (int)r->tokens, (int)r->topk, (int)packs, (int)stretches, (int)ys->rows);
}

template <typename T, int V>
alphasparseStatus_t run_combine_grad(alphasparseHandle_t h, alphasparseRoutingDescr_t r, alphasparseDnMatDescr_t dy,
                                     alphasparseDnMatDescr_t ys, const float* weights, alphasparseDnMatDescr_t dys,
                                     float* dweights, int64_t rows) {
  const int64_t packs = dy->cols / V;
  int x = 32;
  constexpr int U = packs_per_lane<T, V>(32);
  while (x < kGradThreads && (int64_t)x * U < packs) x *= 2;
  const int y = kRowThreads / x;
  const int64_t blocks = (r->tokens + y - 1) / y;
  return launch_chained(h, route_combine_grad_kernel<T, V, U, 2>, dim3((unsigned)blocks), dim3(x, y), 0, 1,
      (const T*)dy->values, dy->ld, ys ? (const T*)ys->values : nullptr, ys ? ys->ld : 0, weights,
      dys ? (T*)dys->values : nullptr, dys ? dys->ld : 0, dweights, r->position, (int)r->tokens, (int)r->topk, (int)packs,
      (int)rows);
}

}  // namespace
}  // namespace asp

using namespace asp;

extern "C" {

alphasparseStatus_t alphasparseRoutingSort_bufferSize(alphasparseHandle_t h, alphasparseRoutingDescr_t r, size_t* size) {
  if (!size) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  const alphasparseStatus_t s = check_routing(h, r);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  *size = r->tokens * r->topk <= kSortClusterSlots ? 0 : sizeof(int) * (size_t)(sort_blocks(h, r->tokens * r->topk) * r->experts) + 16;
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

alphasparseStatus_t alphasparseRoutingSort(alphasparseHandle_t h, alphasparseRoutingDescr_t r, void* buffer) {
  const alphasparseStatus_t s = check_routing(h, r);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (r->tokens > 0 && !r->expert_ids) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  if (r->tokens * r->topk > kSortClusterSlots && !buffer) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  DeviceScope dev(h->device);
  ASP_CUDA(dev.status);
  return r->id_type == ALPHA_SPARSE_INDEXTYPE_I64 ? run_sort<int64_t>(h, r, buffer) : run_sort<int32_t>(h, r, buffer);
}

alphasparseStatus_t alphasparseRoutingDispatch(alphasparseHandle_t h, alphasparseRoutingDescr_t r,
                                               alphasparseDnMatDescr_t x, alphasparseDnMatDescr_t xs) {
  alphasparseStatus_t s = check_routing(h, r);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (!x || !xs) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  if (!expert_type(x->data_type) || xs->data_type != x->data_type) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
  if ((s = expert_check_mat(x, r->tokens, -1)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if ((s = expert_check_mat(xs, -1, x->cols)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (r->tokens == 0 || x->cols == 0 || xs->rows == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
  DeviceScope dev(h->device);
  ASP_CUDA(dev.status);
  return by_type(x->data_type, [&](auto t) {
    using T = decltype(t);
    return by_pack<T>([&](auto v) { return run_dispatch<T, decltype(v)::value>(h, r, x, xs); }, x, xs);
  });
}

alphasparseStatus_t alphasparseRoutingCombine(alphasparseHandle_t h, alphasparseRoutingDescr_t r,
                                              alphasparseDnMatDescr_t ys, const float* weights,
                                              alphasparseDnMatDescr_t res, alphasparseDnMatDescr_t y) {
  alphasparseStatus_t s = check_routing(h, r);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (!ys || !y) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  if (!expert_type(y->data_type) || ys->data_type != y->data_type || (res && res->data_type != y->data_type))
    return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
  if ((s = expert_check_mat(y, r->tokens, -1)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if ((s = expert_check_mat(ys, -1, y->cols)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (res && (s = expert_check_mat(res, r->tokens, y->cols)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (r->tokens == 0 || y->cols == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
  DeviceScope dev(h->device);
  ASP_CUDA(dev.status);
  return by_type(y->data_type, [&](auto t) {
    using T = decltype(t);
    return by_pack<T>([&](auto v) { return run_combine<T, decltype(v)::value>(h, r, ys, weights, res, y); }, ys, res, y);
  });
}

alphasparseStatus_t alphasparseRoutingCombineGrad(alphasparseHandle_t h, alphasparseRoutingDescr_t r,
                                                  alphasparseDnMatDescr_t dy, alphasparseDnMatDescr_t ys,
                                                  const float* weights, alphasparseDnMatDescr_t dys, float* dweights) {
  alphasparseStatus_t s = check_routing(h, r);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (!dy || (dweights && !ys) || (!dys && !dweights)) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  if (!expert_type(dy->data_type) || (ys && ys->data_type != dy->data_type) || (dys && dys->data_type != dy->data_type))
    return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
  if ((s = expert_check_mat(dy, r->tokens, -1)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (ys && (s = expert_check_mat(ys, -1, dy->cols)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (dys && (s = expert_check_mat(dys, ys ? ys->rows : -1, dy->cols)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (r->tokens == 0 || (dy->cols == 0 && !dweights)) return ALPHA_SPARSE_STATUS_SUCCESS;
  DeviceScope dev(h->device);
  ASP_CUDA(dev.status);
  const int64_t rows = dys ? dys->rows : ys->rows;
  return by_type(dy->data_type, [&](auto t) {
    using T = decltype(t);
    return by_pack<T>([&](auto v) { return run_combine_grad<T, decltype(v)::value>(h, r, dy, ys, weights, dys, dweights, rows); }, dy,
                      ys, dys);
  });
}

}  // extern "C"
