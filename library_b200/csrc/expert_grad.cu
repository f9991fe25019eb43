// Gradient of the experts' epilogue:  dZ = dY * act'(Z),  dBias[e] = column sums of the unrounded dZ over segment e.
//
// One pass over dY and Z.  A CTA takes a chunk of 256 rows x one stretch of columns and walks the
// segments that meet the chunk; a segment's column sums stay in registers, are joined over the CTA's
// warps through shared memory, and go to dBias at once when the segment lies inside the chunk, else
// (a piece of it) to the workspace: slot 0 of the chunk for a segment that began earlier, slot 1 for
// one that goes on.  A second kernel adds up the pieces of such segments in chunk order and
// zeroes the rows of empty segments.  No atomics: the sums do not depend on the order of the CTAs.
#include "expert_act.h"
#include "expert_launch.h"
#include "expert_vec.h"

namespace asp {
namespace {

constexpr int kActThreads = 256;
constexpr int kActWarps = kActThreads / 32;
constexpr int kActRows = 256;
constexpr int kActBatch = 4;

__device__ __forceinline__ int clamp_row(const int32_t* __restrict__ off, int e, int segments, int rows) {
  if (!off) return e == 0 ? 0 : rows;
  const int v = off[e];
  return v < 0 ? 0 : v > rows ? rows : v;
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kActThreads, 3)
expert_act_grad_kernel(const T* dy, int64_t lddy, const T* z, int64_t ldz, T* dz, int64_t lddz,
                       float* __restrict__ dbias, int64_t lddb, const int32_t* __restrict__ off, int segments, int rows,
                       int cols, int strips, float* __restrict__ pieces) {
  __shared__ float part[kActWarps][32 * V + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int chunk = (int)(blockIdx.x / (unsigned)strips), strip = (int)(blockIdx.x % (unsigned)strips);
  const int r0 = chunk * kActRows, r1 = r0 < rows - kActRows ? r0 + kActRows : rows;
  const int c0 = strip * 32 * V, c = c0 + lane * V;
  dependency_wait();
  dependents_go();
  // the last segment that begins at or before the chunk
  int before = 0;
  for (int i = 0; i <= segments; i += kActThreads)
    before += __syncthreads_count(i + tid <= segments && clamp_row(off, i + tid, segments, rows) <= r0);
  for (int e = before > 0 ? before - 1 : 0; e < segments; ++e) {
    const int b = clamp_row(off, e, segments, rows), d = clamp_row(off, e + 1, segments, rows);
    if (b >= r1) break;
    const int lo = b > r0 ? b : r0, hi = d < r1 ? d : r1;
    if (lo >= hi) continue;
    float sum[V];
#pragma unroll
    for (int v = 0; v < V; ++v) sum[v] = 0.f;
    if (c < cols) {
      // kActBatch rows are read before the first is written: dZ may be dY or Z, so the compiler cannot reorder them
      for (int r = lo + warp; r < hi; r += kActWarps * kActBatch) {
        Pack<T, V> g[kActBatch], a[kActBatch];
#pragma unroll
        for (int i = 0; i < kActBatch; ++i) {
          const int row = r + i * kActWarps;
          if (row >= hi) continue;
          g[i] = load_pack<T, V>(dy + (int64_t)row * lddy + c);
          if constexpr (ACT != ALPHASPARSE_ACT_NONE) a[i] = load_pack<T, V>(z + (int64_t)row * ldz + c);
        }
#pragma unroll
        for (int i = 0; i < kActBatch; ++i) {
          const int row = r + i * kActWarps;
          if (row >= hi) continue;
          float f[V];
#pragma unroll
          // (an explicit product: the sum below takes the same value whether or not dZ is stored)
          for (int v = 0; v < V; ++v) {
            f[v] = g[i].at(v);
            if constexpr (ACT != ALPHASPARSE_ACT_NONE) f[v] = __fmul_rn(f[v], act_slope<ACT>(a[i].at(v)));
            sum[v] += f[v];
          }
          if (dz) store_pack<T, V>(dz + (int64_t)row * lddz + c, round_pack<T, V>(f));
        }
      }
    }
    if (!dbias) continue;
#pragma unroll
    for (int v = 0; v < V; ++v) part[warp][lane * V + v] = sum[v];
    __syncthreads();
    float* out = b >= r0 && d <= r1 ? dbias + (int64_t)e * lddb : pieces + (int64_t)(2 * chunk + (b < r0 ? 0 : 1)) * cols;
    for (int i = tid; i < 32 * V && c0 + i < cols; i += kActThreads) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kActWarps; ++w) s += part[w][i];
      out[c0 + i] = s;
    }
    __syncthreads();
  }
}

// 64 columns of one segment's dBias per CTA: quarter q of the CTA adds the pieces of every fourth chunk, then the quarters are joined.
constexpr int kJoinCols = 64, kJoinParts = kActThreads / kJoinCols;
__global__ void __launch_bounds__(kActThreads)
expert_bias_join_kernel(float* __restrict__ dbias, int64_t lddb, const int32_t* __restrict__ off, int segments, int rows,
                        int cols, int strips, const float* __restrict__ pieces) {
  __shared__ float part[kJoinParts][kJoinCols];
  dependency_wait();
  dependents_go();
  const int q = threadIdx.x / kJoinCols, i = threadIdx.x % kJoinCols;
  const int e = (int)(blockIdx.x / (unsigned)strips), c = (int)(blockIdx.x % (unsigned)strips) * kJoinCols + i;
  const int b = clamp_row(off, e, segments, rows), d = clamp_row(off, e + 1, segments, rows);
  const int k0 = b / kActRows, k1 = d > b ? (d - 1) / kActRows : k0;
  if (d > b && k0 == k1) return;  // written by the CTA of that chunk
  float sum = 0.f;
  if (d > b && c < cols) {
#pragma unroll 8
    for (int k = k0 + q; k <= k1; k += kJoinParts)
      sum += pieces[(int64_t)(2 * k + (b < k * kActRows ? 0 : 1)) * cols + c];
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

size_t piece_bytes(int64_t rows, int64_t cols) {
  return (size_t)((rows + kActRows - 1) / kActRows) * 2 * (size_t)cols * sizeof(float) + 16;
}

template <typename T, int V, int ACT>
alphasparseStatus_t run_act_grad(alphasparseHandle_t h, int segments, const int32_t* off, alphasparseDnMatDescr_t dy,
                                 alphasparseDnMatDescr_t z, alphasparseDnMatDescr_t dz, alphasparseDnMatDescr_t db,
                                 void* buffer) {
  const int rows = (int)dy->rows, cols = (int)dy->cols;
  const int64_t chunks = ((int64_t)rows + kActRows - 1) / kActRows, strips = ((int64_t)cols + 32 * V - 1) / (32 * V);
  float* pieces = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(buffer) + 15) & ~(uintptr_t)15);
  if (chunks * strips >= (int64_t(1) << 31)) return ALPHA_SPARSE_STATUS_INVALID_SIZE;
  if (chunks > 0) {
    const alphasparseStatus_t s = launch_chained(
        h, expert_act_grad_kernel<T, V, ACT>, dim3((unsigned)(chunks * strips)), dim3(kActThreads), 0, 1, (const T*)dy->values, dy->ld,
        z ? (const T*)z->values : nullptr, z ? z->ld : 0, dz ? (T*)dz->values : nullptr, dz ? dz->ld : 0,
        db ? (float*)db->values : nullptr, db ? db->ld : 0, off, segments, rows, cols, (int)strips, pieces);
    if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  }
  if (!db) return ALPHA_SPARSE_STATUS_SUCCESS;
  const int64_t js = ((int64_t)cols + kJoinCols - 1) / kJoinCols;
  if (segments * js >= (int64_t(1) << 31)) return ALPHA_SPARSE_STATUS_INVALID_SIZE;
  return launch_chained(h, expert_bias_join_kernel, dim3((unsigned)(segments * js)), dim3(kActThreads), 0, 1, (float*)db->values, db->ld,
                        off, segments, rows, cols, (int)js, (const float*)pieces);
}

template <typename T>
alphasparseStatus_t act_grad_t(alphasparseHandle_t h, int segments, const int32_t* off, alphasparseActivation_t act,
                               alphasparseDnMatDescr_t dy, alphasparseDnMatDescr_t z, alphasparseDnMatDescr_t dz,
                               alphasparseDnMatDescr_t db, void* buffer) {
  constexpr int W = 16 / sizeof(T);
  const bool wide = packs_of_16(dy) && packs_of_16(z) && packs_of_16(dz);
  switch (act) {
    case ALPHASPARSE_ACT_RELU:
      return wide ? run_act_grad<T, W, ALPHASPARSE_ACT_RELU>(h, segments, off, dy, z, dz, db, buffer)
                  : run_act_grad<T, 1, ALPHASPARSE_ACT_RELU>(h, segments, off, dy, z, dz, db, buffer);
    case ALPHASPARSE_ACT_GELU:
      return wide ? run_act_grad<T, W, ALPHASPARSE_ACT_GELU>(h, segments, off, dy, z, dz, db, buffer)
                  : run_act_grad<T, 1, ALPHASPARSE_ACT_GELU>(h, segments, off, dy, z, dz, db, buffer);
    case ALPHASPARSE_ACT_SILU:
      return wide ? run_act_grad<T, W, ALPHASPARSE_ACT_SILU>(h, segments, off, dy, z, dz, db, buffer)
                  : run_act_grad<T, 1, ALPHASPARSE_ACT_SILU>(h, segments, off, dy, z, dz, db, buffer);
    default:
      return wide ? run_act_grad<T, W, ALPHASPARSE_ACT_NONE>(h, segments, off, dy, z, dz, db, buffer)
                  : run_act_grad<T, 1, ALPHASPARSE_ACT_NONE>(h, segments, off, dy, z, dz, db, buffer);
  }
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
