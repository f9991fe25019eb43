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

#include "expert_vec.h"

namespace cg = cooperative_groups;

namespace asp {
namespace {

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortCluster = 8;             // CTAs of the one-launch sort (portable cluster size)
// Slots above which the sort runs on the whole device in three launches instead of one cluster.
constexpr int64_t kSortClusterSlots = 1 << 18;

struct SlotRange {
  int begin, end;
};
// Warps own contiguous, ascending slot ranges (multiples of 32 slots), so that counting in warp
// order and then in lane order is the stable order.
__device__ __forceinline__ SlotRange warp_slots(int slots, int part, int parts) {
  const int64_t per = ((int64_t)slots + (int64_t)parts * 32 - 1) / ((int64_t)parts * 32) * 32;
  const int64_t b = per * part, e = b + per;
  return {(int)(b < slots ? b : slots), (int)(e < slots ? e : slots)};
}
template <typename Id>
__device__ __forceinline__ int expert_of(const Id* __restrict__ ids, int slot, int experts) {
  const Id v = ids[slot];
  return v >= 0 && v < (Id)experts ? (int)v : -1;
}

// counts[w][e] of this CTA's warps, then its exclusive prefix over the warps; totals[e] of the CTA.
template <typename Id>
__device__ void count_slots(const Id* __restrict__ ids, int slots, int experts, int part0, int parts, int* counts,
                            int* totals) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < kSortWarps * experts; i += kSortThreads) counts[i] = 0;
  __syncthreads();
  const SlotRange r = warp_slots(slots, part0 + warp, parts);
  int* mine = counts + warp * experts;
  for (int s = r.begin + lane; s < r.end; s += 32) {
    const int e = expert_of(ids, s, experts);
    if (e >= 0) atomicAdd(&mine[e], 1);  // whole numbers: the order does not matter
  }
  __syncthreads();
  for (int e = tid; e < experts; e += kSortThreads) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = counts[w * experts + e];
      counts[w * experts + e] = sum;
      sum += c;
    }
    totals[e] = sum;
  }
  __syncthreads();
}

// position[] of this CTA's slots; counts[w][e] already holds where warp w's first slot of e goes.
template <typename Id>
__device__ void place_slots(const Id* __restrict__ ids, int slots, int experts, int part0, int parts, int* counts,
                            int32_t* __restrict__ position) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const SlotRange r = warp_slots(slots, part0 + warp, parts);
  int* mine = counts + warp * experts;
  for (int s0 = r.begin; s0 < r.end; s0 += 32) {
    const int s = s0 + lane;
    const int e = s < r.end ? expert_of(ids, s, experts) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    const int base = e >= 0 ? mine[e] : 0;
    __syncwarp();
    if (e >= 0 && before == 0) mine[e] = base + __popc(same);
    __syncwarp();
    if (s < r.end) position[s] = e >= 0 ? base + before : -1;
  }
}

// Exclusive prefix over the experts of all[e] (experts <= 2 * kSortThreads), in place; returns the sum.
__device__ int scan_experts(int* all, int experts, int* warp_sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int i0 = 2 * tid, i1 = 2 * tid + 1;
  const int a = i0 < experts ? all[i0] : 0, b = i1 < experts ? all[i1] : 0;
  int v = a + b;
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
  const int excl = before + v - (a + b);
  if (i0 < experts) all[i0] = excl;
  if (i1 < experts) all[i1] = excl + a;
  __syncthreads();
  return sum;
}
static_assert(ALPHASPARSE_MAX_EXPERTS <= 2 * kSortThreads, "scan_experts holds two experts per thread");

// The whole sort in one launch of one thread-block cluster: counts meet in distributed shared memory.
// Shared: counts[warps][experts], totals[experts], all[experts], warp_sums[warps].
template <typename Id>
__global__ void __launch_bounds__(kSortThreads)
route_sort_cluster_kernel(const Id* __restrict__ ids, int slots, int experts, int32_t* __restrict__ offsets,
                          int32_t* __restrict__ position) {
  extern __shared__ int sort_smem[];
  int* counts = sort_smem;
  int* totals = counts + kSortWarps * experts;
  int* all = totals + experts;
  int* warp_sums = all + experts;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), size = (int)cl.num_blocks();
  count_slots(ids, slots, experts, rank * kSortWarps, size * kSortWarps, counts, totals);
  cl.sync();
  int before[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = (int)threadIdx.x + i * kSortThreads;
    if (e < experts) {
      int sum = 0;
      for (int c = 0; c < size; ++c) {
        const int n = *cl.map_shared_rank(totals + e, c);
        if (c < rank) before[i] += n;
        sum += n;
      }
      all[e] = sum;
    }
  }
  cl.sync();  // every CTA has read its peers' totals: none may leave before, and all[] is complete
  const int kept = scan_experts(all, experts, warp_sums);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = (int)threadIdx.x + i * kSortThreads;
    if (e < experts) {
      if (rank == 0) offsets[e] = all[e];
      const int base = all[e] + before[i];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) counts[w * experts + e] += base;
    }
  }
  if (rank == 0 && threadIdx.x == 0) offsets[experts] = kept;
  __syncthreads();
  place_slots(ids, slots, experts, rank * kSortWarps, size * kSortWarps, counts, position);
}

// The same in three launches for long inputs: CTA totals, their prefix over the CTAs and the experts, places.
template <typename Id, bool PLACE>
__global__ void __launch_bounds__(kSortThreads)
route_sort_pass_kernel(const Id* __restrict__ ids, int slots, int experts, int* __restrict__ block_base,
                       int32_t* __restrict__ position) {
  extern __shared__ int sort_smem[];
  int* counts = sort_smem;
  int* totals = counts + kSortWarps * experts;
  const int part0 = (int)blockIdx.x * kSortWarps, parts = (int)gridDim.x * kSortWarps;
  count_slots(ids, slots, experts, part0, parts, counts, totals);
  int* base = block_base + (size_t)blockIdx.x * experts;
  if constexpr (!PLACE) {
    for (int e = threadIdx.x; e < experts; e += kSortThreads) base[e] = totals[e];
  } else {
    for (int i = threadIdx.x; i < kSortWarps * experts; i += kSortThreads) counts[i] += base[i % experts];
    __syncthreads();
    place_slots(ids, slots, experts, part0, parts, counts, position);
  }
}
__global__ void __launch_bounds__(kSortThreads)
route_sort_scan_kernel(int* __restrict__ block_base, int blocks, int experts, int32_t* __restrict__ offsets) {
  __shared__ int all[ALPHASPARSE_MAX_EXPERTS];
  __shared__ int warp_sums[kSortWarps];
  for (int e = threadIdx.x; e < experts; e += kSortThreads) {
    int sum = 0;
#pragma unroll 8
    for (int b = 0; b < blocks; ++b) sum += block_base[(size_t)b * experts + e];
    all[e] = sum;
  }
  __syncthreads();
  const int kept = scan_experts(all, experts, warp_sums);
  for (int e = threadIdx.x; e < experts; e += kSortThreads) {
    int run = all[e];
    offsets[e] = run;
#pragma unroll 8
    for (int b = 0; b < blocks; ++b) {
      const int c = block_base[(size_t)b * experts + e];
      block_base[(size_t)b * experts + e] = run;
      run += c;
    }
  }
  if (threadIdx.x == 0) offsets[experts] = kept;
}

// ---- row movement ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;

// A warp takes a token's stretch of 32 * U packs: loads it once, stores it to every sorted row.
template <typename T, int V, int U>
__global__ void __launch_bounds__(kRowThreads)
route_dispatch_kernel(const T* __restrict__ x, int64_t ldx, T* __restrict__ xs, int64_t ldxs,
                      const int32_t* __restrict__ position, int tokens, int topk, int packs, int stretches, int xs_rows) {
  const int lane = threadIdx.x & 31;
  const int64_t task = ((int64_t)blockIdx.x * kRowThreads + threadIdx.x) >> 5;
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

// A warp takes a token's stretch of 32 * U packs of Y and adds up the sorted rows, J of them in flight.
template <typename T, int V, int U, int J>
__global__ void __launch_bounds__(kRowThreads)
route_combine_kernel(const T* __restrict__ ys, int64_t ldys, const float* __restrict__ weights, const T* r, int64_t ldr,
                     T* y, int64_t ldy, const int32_t* __restrict__ position, int tokens, int topk, int packs,
                     int stretches, int ys_rows) {
  const int lane = threadIdx.x & 31;
  const int64_t task = ((int64_t)blockIdx.x * kRowThreads + threadIdx.x) >> 5;
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
      float w[J];
      bool kept[J];
#pragma unroll
      for (int i = 0; i < J; ++i) {
        const int p = __shfl_sync(0xffffffffu, mine, (j + i) & 31);
        w[i] = __shfl_sync(0xffffffffu, w_mine, (j + i) & 31);
        kept[i] = j + i < n && (unsigned)p < (unsigned)ys_rows;
        if (kept[i]) {
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c0 + 32 * u < packs) in[i][u] = load_pack<T, V>(ys + (int64_t)p * ldys + (int64_t)(c0 + 32 * u) * V);
        }
      }
#pragma unroll
      for (int i = 0; i < J; ++i) {
        if (!kept[i]) continue;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (c0 + 32 * u < packs) {
#pragma unroll
            for (int v = 0; v < V; ++v) acc[u][v] = fmaf(w[i], Wide<T>::up(in[i][u].v[v]), acc[u][v]);
          }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (c0 + 32 * u < packs) {
      if (r) {
#pragma unroll
        for (int v = 0; v < V; ++v) acc[u][v] += Wide<T>::up(res[u].v[v]);
      }
      store_pack<T, V>(y + (int64_t)t * ldy + (int64_t)(c0 + 32 * u) * V, round_pack<T, V>(acc[u]));
    }
}

// Gradient of combine.  blockDim.y tokens per CTA, blockDim.x threads on a token's row (whole warps).
// The dot products of J slots are kept at a time and added up over lanes, then over the row's warps,
// in a fixed order.
template <typename T, int V, int J>
__global__ void __launch_bounds__(kRowThreads)
route_combine_grad_kernel(const T* __restrict__ dy, int64_t lddy, const T* ys, int64_t ldys,
                          const float* __restrict__ weights, T* dys, int64_t lddys, float* __restrict__ dweights,
                          const int32_t* __restrict__ position, int tokens, int topk, int packs, int rows) {
  __shared__ float part[kRowThreads / 32][J];
  const int t = (int)blockIdx.x * (int)blockDim.y + (int)threadIdx.y;
  const int lane = threadIdx.x & 31;
  const int warps = (int)blockDim.x >> 5, row_warp0 = (int)threadIdx.y * warps, my_warp = row_warp0 + ((int)threadIdx.x >> 5);
  for (int j0 = 0; j0 < topk; j0 += J) {
    int p[J];
    float w[J], dot[J];
#pragma unroll
    for (int i = 0; i < J; ++i) {
      const bool in = t < tokens && j0 + i < topk;
      p[i] = in ? position[(int64_t)t * topk + j0 + i] : -1;
      w[i] = in && weights ? weights[(int64_t)t * topk + j0 + i] : 1.f;
      dot[i] = 0.f;
    }
    if (t < tokens) {
      for (int c = (int)threadIdx.x; c < packs; c += (int)blockDim.x) {
        const Pack<T, V> g = load_pack<T, V>(dy + (int64_t)t * lddy + (int64_t)c * V);
        Pack<T, V> in[J];
        if (dweights) {
#pragma unroll
          for (int i = 0; i < J; ++i)
            if ((unsigned)p[i] < (unsigned)rows) in[i] = load_pack<T, V>(ys + (int64_t)p[i] * ldys + (int64_t)c * V);
        }
#pragma unroll
        for (int i = 0; i < J; ++i) {
          if ((unsigned)p[i] >= (unsigned)rows) continue;
          float out[V];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float gv = Wide<T>::up(g.v[v]);
            if (dweights) dot[i] = fmaf(gv, Wide<T>::up(in[i].v[v]), dot[i]);
            out[v] = w[i] * gv;
          }
          if (dys) store_pack<T, V>(dys + (int64_t)p[i] * lddys + (int64_t)c * V, round_pack<T, V>(out));
        }
      }
    }
    if (!dweights) continue;
#pragma unroll
    for (int i = 0; i < J; ++i)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot[i] += __shfl_xor_sync(0xffffffffu, dot[i], o);
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < J; ++i) part[my_warp][i] = dot[i];
    }
    __syncthreads();
    if (t < tokens && (int)threadIdx.x < J && j0 + (int)threadIdx.x < topk) {
      float sum = 0.f;
      for (int k = 0; k < warps; ++k) sum += part[row_warp0 + k][threadIdx.x];
      dweights[(int64_t)t * topk + j0 + threadIdx.x] = sum;
    }
    __syncthreads();
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

int sort_blocks(alphasparseHandle_t h) { return impl(h)->sm_count; }

template <typename Id>
alphasparseStatus_t run_sort(alphasparseHandle_t h, alphasparseRoutingDescr_t r, void* buffer) {
  const int slots = (int)(r->tokens * r->topk), experts = (int)r->experts;
  const Id* ids = (const Id*)r->expert_ids;
  const size_t smem = sizeof(int) * ((size_t)kSortWarps * experts + 2 * (size_t)experts + kSortWarps);
  if (slots <= kSortClusterSlots) {
    if (smem > 48 * 1024)
      ASP_CUDA(cudaFuncSetAttribute(route_sort_cluster_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)(sizeof(int) * ((kSortWarps + 2) * ALPHASPARSE_MAX_EXPERTS + kSortWarps))));
    // a CTA per 2,048 slots (four rounds of its warps' lanes): few slots need no cluster
    int ctas = 1;
    while (ctas < kSortCluster && ctas * 2048 < slots) ctas *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = h->stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    ASP_CUDA(cudaLaunchKernelEx(&cfg, route_sort_cluster_kernel<Id>, ids, slots, experts, r->expert_offsets, r->position));
    ++impl(h)->launches;
    return ALPHA_SPARSE_STATUS_SUCCESS;
  }
  if (!buffer) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  int* base = reinterpret_cast<int*>((reinterpret_cast<uintptr_t>(buffer) + 15) & ~(uintptr_t)15);
  const int blocks = sort_blocks(h);
  const int most = (int)(sizeof(int) * (kSortWarps + 2) * ALPHASPARSE_MAX_EXPERTS);
  ASP_CUDA(cudaFuncSetAttribute(route_sort_pass_kernel<Id, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
  ASP_CUDA(cudaFuncSetAttribute(route_sort_pass_kernel<Id, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
  const size_t pass_smem = sizeof(int) * (size_t)(kSortWarps + 1) * experts;
  route_sort_pass_kernel<Id, false><<<blocks, kSortThreads, pass_smem, h->stream>>>(ids, slots, experts, base, nullptr);
  ASP_CUDA(cudaGetLastError());
  route_sort_scan_kernel<<<1, kSortThreads, 0, h->stream>>>(base, blocks, experts, r->expert_offsets);
  ASP_CUDA(cudaGetLastError());
  route_sort_pass_kernel<Id, true><<<blocks, kSortThreads, pass_smem, h->stream>>>(ids, slots, experts, base, r->position);
  ASP_CUDA(cudaGetLastError());
  impl(h)->launches += 3;
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

// Warps for tokens x stretches, as a grid; 0 when there is nothing to do.
int64_t row_blocks(int64_t tokens, int64_t stretches) { return (tokens * stretches * 32 + kRowThreads - 1) / kRowThreads; }

template <typename T, int V>
alphasparseStatus_t run_dispatch(alphasparseHandle_t h, alphasparseRoutingDescr_t r, alphasparseDnMatDescr_t x,
                                 alphasparseDnMatDescr_t xs) {
  constexpr int U = 4;
  const int64_t packs = x->cols / V, stretches = (packs + 32 * U - 1) / (32 * U);
  const int64_t blocks = row_blocks(r->tokens, stretches);
  if (blocks >= (int64_t(1) << 31)) return ALPHA_SPARSE_STATUS_INVALID_SIZE;
  route_dispatch_kernel<T, V, U><<<(unsigned)blocks, kRowThreads, 0, h->stream>>>(
      (const T*)x->values, x->ld, (T*)xs->values, xs->ld, r->position, (int)r->tokens, (int)r->topk, (int)packs,
      (int)stretches, (int)xs->rows);
  ASP_CUDA(cudaGetLastError());
  ++impl(h)->launches;
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

template <typename T, int V>
alphasparseStatus_t run_combine(alphasparseHandle_t h, alphasparseRoutingDescr_t r, alphasparseDnMatDescr_t ys,
                                const float* weights, alphasparseDnMatDescr_t res, alphasparseDnMatDescr_t y) {
  constexpr int U = V == 1 ? 4 : 1;
  const int64_t packs = y->cols / V, stretches = (packs + 32 * U - 1) / (32 * U);
  const int64_t blocks = row_blocks(r->tokens, stretches);
  if (blocks >= (int64_t(1) << 31)) return ALPHA_SPARSE_STATUS_INVALID_SIZE;
  route_combine_kernel<T, V, U, 4><<<(unsigned)blocks, kRowThreads, 0, h->stream>>>(
      (const T*)ys->values, ys->ld, weights, res ? (const T*)res->values : nullptr, res ? res->ld : 0, (T*)y->values,
      y->ld, r->position, (int)r->tokens, (int)r->topk, (int)packs, (int)stretches, (int)ys->rows);
  ASP_CUDA(cudaGetLastError());
  ++impl(h)->launches;
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

template <typename T, int V>
alphasparseStatus_t run_combine_grad(alphasparseHandle_t h, alphasparseRoutingDescr_t r, alphasparseDnMatDescr_t dy,
                                     alphasparseDnMatDescr_t ys, const float* weights, alphasparseDnMatDescr_t dys,
                                     float* dweights, int64_t rows) {
  const int64_t packs = dy->cols / V;
  int x = 32;
  while (x < kRowThreads && x < packs) x *= 2;
  const int y = kRowThreads / x;
  const int64_t blocks = (r->tokens + y - 1) / y;
  route_combine_grad_kernel<T, V, 8><<<(unsigned)blocks, dim3(x, y), 0, h->stream>>>(
      (const T*)dy->values, dy->ld, ys ? (const T*)ys->values : nullptr, ys ? ys->ld : 0, weights,
      dys ? (T*)dys->values : nullptr, dys ? dys->ld : 0, dweights, r->position, (int)r->tokens, (int)r->topk, (int)packs,
      (int)rows);
  ASP_CUDA(cudaGetLastError());
  ++impl(h)->launches;
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

}  // namespace
}  // namespace asp

using namespace asp;

extern "C" {

alphasparseStatus_t alphasparseRoutingSort_bufferSize(alphasparseHandle_t h, alphasparseRoutingDescr_t r, size_t* size) {
  if (!size) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  const alphasparseStatus_t s = check_routing(h, r);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  *size = r->tokens * r->topk <= kSortClusterSlots ? 0 : sizeof(int) * (size_t)sort_blocks(h) * r->experts + 16;
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
  const bool wide = packs_of_16(x) && packs_of_16(xs);
  return by_type(x->data_type, [&](auto t) {
    using T = decltype(t);
    return wide ? run_dispatch<T, 16 / sizeof(T)>(h, r, x, xs) : run_dispatch<T, 1>(h, r, x, xs);
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
  const bool wide = packs_of_16(ys) && packs_of_16(res) && packs_of_16(y);
  return by_type(y->data_type, [&](auto t) {
    using T = decltype(t);
    return wide ? run_combine<T, 16 / sizeof(T)>(h, r, ys, weights, res, y) : run_combine<T, 1>(h, r, ys, weights, res, y);
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
  const bool wide = packs_of_16(dy) && packs_of_16(ys) && packs_of_16(dys);
  return by_type(dy->data_type, [&](auto t) {
    using T = decltype(t);
    return wide ? run_combine_grad<T, 16 / sizeof(T)>(h, r, dy, ys, weights, dys, dweights, rows)
                : run_combine_grad<T, 1>(h, r, dy, ys, weights, dys, dweights, rows);
  });
}

}  // extern "C"
