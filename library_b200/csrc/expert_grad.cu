// Gradient of the experts' epilogue:  dZ = dY * act'(Z),  dBias[e] = column sums of the unrounded dZ over segment e.
//
// One pass over dY and Z.  A CTA takes a chunk of 8 x R rows and a stretch of columns, each of its warps R consecutive rows: the warp
// walks the segments that meet its rows with the column sums in registers.  A segment that lies inside the warp's rows goes to dBias
// at once; the pieces at both ends of the warp's rows go to shared memory, where they are joined in warp order after one barrier, and
// what reaches past the chunk goes to the workspace: slot 0 of the chunk for a segment that began before it, slot 1 for one that
// goes on after it.  A second kernel adds up the pieces of such segments in chunk order and zeroes the rows of empty
// segments.  No atomics: the sums do not depend on the order of the CTAs.
#include "expert_act.h"
#include "expert_launch.h"
#include "expert_vec.h"

namespace asp {
namespace {

constexpr int kActThreads = 256;
constexpr int kActWarps = kActThreads / 32;
constexpr int kActBatch = 4;  // rows in flight per warp

__device__ __forceinline__ int clamp_row(const int32_t* off, int e, int segments, int rows) {
  if (!off) return e == 0 ? 0 : rows;
  const int v = off[e];
  return v < 0 ? 0 : v > rows ? rows : v;
}

// The last segment that begins at or before row r (0 if none does).  Whole warp.
__device__ __forceinline__ int segment_of(const int32_t* off, int segments, int rows, int r) {
  const int lane = threadIdx.x & 31, per = (segments + 31) / 32;
  const unsigned hi = __ballot_sync(0xffffffffu, lane * per < segments && clamp_row(off, lane * per, segments, rows) <= r);
  if (hi == 0) return 0;
  const int blk = (31 - __clz(hi)) * per;
  const unsigned lo = __ballot_sync(0xffffffffu, lane < per && blk + lane < segments && clamp_row(off, blk + lane, segments, rows) <= r);
  return lo == 0 ? 0 : blk + 31 - __clz(lo);
}

template <typename T, int V, int U, int ACT>
__global__ void __launch_bounds__(kActThreads, 3)
expert_act_grad_kernel(const T* dy, int64_t lddy, const T* z, int64_t ldz, T* dz, int64_t lddz,
                       float* __restrict__ dbias, int64_t lddb, const int32_t* off, int segments, int rows,
                       int cols, int strips, int warp_rows, float* __restrict__ pieces) {
  constexpr int kStrip = 32 * V * U;
  __shared__ float head[kActWarps][kStrip], tail[kActWarps][kStrip];
  __shared__ int head_e[kActWarps], head_ends[kActWarps], tail_e[kActWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int chunk = (int)(blockIdx.x / (unsigned)strips), c_strip = (int)(blockIdx.x % (unsigned)strips) * kStrip;
  dependency_wait();
  dependents_go();
  const int64_t first = ((int64_t)chunk * kActWarps + warp) * warp_rows;
  const int w0 = (int)(first < rows ? first : rows), w1 = (int)(first + warp_rows < rows ? first + warp_rows : rows);
  int my_head = -1, my_ends = 0, my_tail = -1;
  for (int r = w0, e = w0 < w1 ? segment_of(off, segments, rows, w0) : segments; r < w1 && e < segments; ++e) {
    const int b = clamp_row(off, e, segments, rows), d = clamp_row(off, e + 1, segments, rows);
    if (b >= w1) break;
    const int lo = b > r ? b : r, hi = d < w1 ? d : w1;
    if (lo >= hi) continue;
    float sum[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int v = 0; v < V; ++v) sum[u][v] = 0.f;
    // kActBatch rows are read before the first is written: dZ may be dY or Z, so the compiler cannot reorder them
    for (int q = lo; q < hi; q += kActBatch) {
      Pack<T, V> g[kActBatch][U], a[kActBatch][U];
#pragma unroll
      for (int i = 0; i < kActBatch; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = c_strip + (32 * u + lane) * V;
          if (q + i >= hi || c >= cols) continue;
          g[i][u] = load_pack<T, V>(dy + (int64_t)(q + i) * lddy + c);
          if constexpr (ACT != ALPHASPARSE_ACT_NONE) a[i][u] = load_pack<T, V>(z + (int64_t)(q + i) * ldz + c);
        }
#pragma unroll
      for (int i = 0; i < kActBatch; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = c_strip + (32 * u + lane) * V;
          if (q + i >= hi || c >= cols) continue;
          float f[V];
#pragma unroll
          // (an explicit product: the sum takes the same value whether or not dZ is stored)
          for (int v = 0; v < V; ++v) {
            f[v] = g[i][u].at(v);
            if constexpr (ACT != ALPHASPARSE_ACT_NONE) f[v] = __fmul_rn(f[v], act_slope<ACT>(a[i][u].at(v)));
            sum[u][v] += f[v];
          }
          if (dz) store_pack<T, V>(dz + (int64_t)(q + i) * lddz + c, round_pack<T, V>(f));
        }
    }
    r = hi;
    if (!dbias) continue;
    const bool before = b < w0, ends = hi == d;
    float* out = before ? head[warp] : tail[warp];
    if (before) {
      my_head = e;
      my_ends = ends;
    } else if (!ends) {
      my_tail = e;
    } else {
      out = nullptr;  // the whole segment
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = (32 * u + lane) * V + v;
        if (out) out[i] = sum[u][v];
        else if (c_strip + i < cols) dbias[(int64_t)e * lddb + c_strip + i] = sum[u][v];
      }
  }
  if (!dbias) return;
  if (lane == 0) {
    head_e[warp] = my_head;
    head_ends[warp] = my_ends;
    tail_e[warp] = my_tail;
  }
  __syncthreads();
  for (int i = tid; i < kStrip && c_strip + i < cols; i += kActThreads) {
    float run = 0.f;
    int open = -1;         // the segment that goes on into the next warp's rows
    bool earlier = false;  // it began before the chunk
    for (int w = 0; w < kActWarps; ++w) {
      if (head_e[w] >= 0) {
        if (open != head_e[w]) {
          open = head_e[w];
          earlier = true;
          run = 0.f;
        }
        run += head[w][i];
        if (head_ends[w]) {
          if (earlier) pieces[(int64_t)(2 * chunk) * cols + c_strip + i] = run;
          else dbias[(int64_t)open * lddb + c_strip + i] = run;
          open = -1;
        }
      }
      if (tail_e[w] >= 0) {
        open = tail_e[w];
        earlier = false;
        run = tail[w][i];
      }
    }
    if (open >= 0) pieces[(int64_t)(2 * chunk + (earlier ? 0 : 1)) * cols + c_strip + i] = run;
  }
}

// 64 columns of one segment's dBias per CTA: quarter q of the CTA adds the pieces of every fourth chunk, then the quarters are joined.
constexpr int kJoinCols = 64, kJoinParts = kActThreads / kJoinCols;
__global__ void __launch_bounds__(kActThreads)
expert_bias_join_kernel(float* __restrict__ dbias, int64_t lddb, const int32_t* off, int segments, int rows,
                        int cols, int strips, int chunk_rows, const float* pieces) {
  __shared__ float part[kJoinParts][kJoinCols];
  dependency_wait();
  dependents_go();
  const int q = threadIdx.x / kJoinCols, i = threadIdx.x % kJoinCols;
  const int e = (int)(blockIdx.x / (unsigned)strips), c = (int)(blockIdx.x % (unsigned)strips) * kJoinCols + i;
  const int b = clamp_row(off, e, segments, rows), d = clamp_row(off, e + 1, segments, rows);
  const int k0 = b / chunk_rows, k1 = d > b ? (d - 1) / chunk_rows : k0;
  if (d > b && k0 == k1) return;  // written by the CTA of that chunk
  float sum = 0.f;
  if (d > b && c < cols) {
#pragma unroll 8
    for (int k = k0 + q; k <= k1; k += kJoinParts)
      sum += pieces[(int64_t)(2 * k + ((int64_t)b < (int64_t)k * chunk_rows ? 0 : 1)) * cols + c];
  }
  part[q][i] = sum;
  __syncthreads();
  if (q == 0 && c < cols) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinParts; ++w) s += part[w][i];
    dbias[(int64_t)e * lddb + c] = s;
  }
}

// Rows per warp: 32, fewer where that would leave some of the device's 148 SMs without a CTA.
int act_warp_rows(int64_t rows, int64_t cols) {
  int r = 32;
  // (256 columns per CTA whatever the operands' alignment: the workspace's size may not depend on it)
  while (r > 4 && (rows + kActWarps * r - 1) / (kActWarps * r) * ((cols + 255) / 256) < 148) r /= 2;
  return r;
}
size_t piece_bytes(int64_t rows, int64_t cols) {
  const int64_t chunk = (int64_t)kActWarps * act_warp_rows(rows, cols);
  return (size_t)((rows + chunk - 1) / chunk) * 2 * (size_t)cols * sizeof(float) + 16;
}

template <typename T, int V, int ACT>
alphasparseStatus_t run_act_grad(alphasparseHandle_t h, int segments, const int32_t* off, alphasparseDnMatDescr_t dy,
                                 alphasparseDnMatDescr_t z, alphasparseDnMatDescr_t dz, alphasparseDnMatDescr_t db,
                                 void* buffer) {
  constexpr int U = V == 1 ? 4 : V == 2 && sizeof(T) == 2 ? 2 : 1;
  const int rows = (int)dy->rows, cols = (int)dy->cols, warp_rows = act_warp_rows(rows, cols), chunk_rows = kActWarps * warp_rows;
  const int64_t chunks = ((int64_t)rows + chunk_rows - 1) / chunk_rows, strips = ((int64_t)cols + 32 * V * U - 1) / (32 * V * U);
  float* pieces = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(buffer) + 15) & ~(uintptr_t)15);
  if (chunks * strips >= (int64_t(1) << 31)) return ALPHA_SPARSE_STATUS_INVALID_SIZE;
  if (chunks > 0) {
    const alphasparseStatus_t s = launch_chained(
        h, expert_act_grad_kernel<T, V, U, ACT>, dim3((unsigned)(chunks * strips)), dim3(kActThreads), 0, 1, (const T*)dy->values, dy->ld,
        z ? (const T*)z->values : nullptr, z ? z->ld : 0, dz ? (T*)dz->values : nullptr, dz ? dz->ld : 0,
        db ? (float*)db->values : nullptr, db ? db->ld : 0, off, segments, rows, cols, (int)strips, warp_rows, pieces);
    if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  }
  if (!db) return ALPHA_SPARSE_STATUS_SUCCESS;
  const int64_t js = ((int64_t)cols + kJoinCols - 1) / kJoinCols;
  if (segments * js >= (int64_t(1) << 31)) return ALPHA_SPARSE_STATUS_INVALID_SIZE;
  return launch_chained(h, expert_bias_join_kernel, dim3((unsigned)(segments * js)), dim3(kActThreads), 0, 1, (float*)db->values, db->ld,
                        off, segments, rows, cols, (int)js, chunk_rows, (const float*)pieces);
}

template <typename T>
alphasparseStatus_t act_grad_t(alphasparseHandle_t h, int segments, const int32_t* off, alphasparseActivation_t act,
                               alphasparseDnMatDescr_t dy, alphasparseDnMatDescr_t z, alphasparseDnMatDescr_t dz,
                               alphasparseDnMatDescr_t db, void* buffer) {
  return by_pack<T>(
      [&](auto v) {
        constexpr int V = decltype(v)::value;
        switch (act) {
          case ALPHASPARSE_ACT_RELU: return run_act_grad<T, V, ALPHASPARSE_ACT_RELU>(h, segments, off, dy, z, dz, db, buffer);
          case ALPHASPARSE_ACT_GELU: return run_act_grad<T, V, ALPHASPARSE_ACT_GELU>(h, segments, off, dy, z, dz, db, buffer);
          case ALPHASPARSE_ACT_SILU: return run_act_grad<T, V, ALPHASPARSE_ACT_SILU>(h, segments, off, dy, z, dz, db, buffer);
          default: return run_act_grad<T, V, ALPHASPARSE_ACT_NONE>(h, segments, off, dy, z, dz, db, buffer);
        }
      },
      dy, z, dz);
}

alphasparseStatus_t check_act_grad(alphasparseHandle_t h, int64_t segments, const int32_t* off,
                                   alphasparseActivation_t act, alphasparseDnMatDescr_t dy, alphasparseDnMatDescr_t db) {
  if (!h) return ALPHA_SPARSE_STATUS_INVALID_HANDLE;
  if (!dy) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  if ((int)act < ALPHASPARSE_ACT_NONE || (int)act > ALPHASPARSE_ACT_SILU) return ALPHA_SPARSE_STATUS_INVALID_VALUE;
  alphasparseStatus_t s = expert_check_segments(segments, off);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (!expert_type(dy->data_type) || (db && db->data_type != ALPHA_R_32F)) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
  if ((s = expert_check_mat(dy, -1, -1)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (db && (s = expert_check_mat(db, segments, dy->cols)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

}  // namespace
}  // namespace asp

using namespace asp;

extern "C" {

alphasparseStatus_t alphasparseExpertActGrad_bufferSize(alphasparseHandle_t h, int64_t segments, const int32_t* off,
                                                        alphasparseActivation_t act, alphasparseDnMatDescr_t dy,
                                                        alphasparseDnMatDescr_t db, size_t* size) {
  if (!size) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  const alphasparseStatus_t s = check_act_grad(h, segments, off, act, dy, db);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  *size = db ? piece_bytes(dy->rows, dy->cols) : 0;
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

alphasparseStatus_t alphasparseExpertActGrad(alphasparseHandle_t h, int64_t segments, const int32_t* off,
                                             alphasparseActivation_t act, alphasparseDnMatDescr_t dy,
                                             alphasparseDnMatDescr_t z, alphasparseDnMatDescr_t dz,
                                             alphasparseDnMatDescr_t db, void* buffer) {
  alphasparseStatus_t s = check_act_grad(h, segments, off, act, dy, db);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (act == ALPHASPARSE_ACT_NONE) z = nullptr;
  else if (!z) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  if ((!dz && !db) || (db && !buffer)) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  if ((z && z->data_type != dy->data_type) || (dz && dz->data_type != dy->data_type)) return ALPHA_SPARSE_STATUS_NOT_SUPPORTED;
  if (z && (s = expert_check_mat(z, dy->rows, dy->cols)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (dz && (s = expert_check_mat(dz, dy->rows, dy->cols)) != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  if (dy->cols == 0 || (dy->rows == 0 && !db)) return ALPHA_SPARSE_STATUS_SUCCESS;
  DeviceScope dev(h->device);
  ASP_CUDA(dev.status);
  switch (dy->data_type) {
    case ALPHA_R_32F: return act_grad_t<float>(h, (int)segments, off, act, dy, z, dz, db, buffer);
    case ALPHA_R_16F: return act_grad_t<__half>(h, (int)segments, off, act, dy, z, dz, db, buffer);
    default: return act_grad_t<__nv_bfloat16>(h, (int)segments, off, act, dy, z, dz, db, buffer);
  }
}

}  // extern "C"
