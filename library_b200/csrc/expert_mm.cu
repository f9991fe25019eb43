// The experts' products: a block-diagonal matrix times a dense one, with bias, activation and residual
// in the epilogue, and the gradient with respect to the blocks.
//   Z[p,n] = sum_k X[p,k] op(W_e)[k,n] + bias[e,n],   Y[p,n] = act(Z[p,n]) + R[p,n]   for p in segment e
//   dW_e   = dZ_e^T X_e  (or its transpose)
// Simple form: 64 x 64 tiles staged in shared memory as fp32, a 4 x 4 block of sums per thread.
#include "expert_act.h"
#include "expert_vec.h"

namespace asp {
namespace {

constexpr int kT = 64, kTK = 16, kMmThreads = 256;

__device__ __forceinline__ int clamp_row(const int32_t* __restrict__ off, int e, int segments, int rows) {
  if (!off) return e == 0 ? 0 : rows;
  const int v = off[e];
  return v < 0 ? 0 : v > rows ? rows : v;
}

// Element types the operands may have beside X's.
__device__ __forceinline__ float load_any(const void* p, int64_t i, alphasparseDataType t) {
  if (t == ALPHA_R_32F) return ((const float*)p)[i];
  return t == ALPHA_R_16F ? __half2float(((const __half*)p)[i]) : __bfloat162float(((const __nv_bfloat16*)p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int64_t i, alphasparseDataType t, float v) {
  if (t == ALPHA_R_32F) ((float*)p)[i] = v;
  else if (t == ALPHA_R_16F) ((__half*)p)[i] = __float2half_rn(v);
  else ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
}

struct Mat {
  void* p;
  int64_t ld;
  alphasparseDataType type;
};
Mat mat(alphasparseDnMatDescr_t m) { return m ? Mat{m->values, m->ld, m->data_type} : Mat{nullptr, 0, ALPHA_R_32F}; }

__device__ __forceinline__ float activate_any(float z, int act) {
  switch (act) {
    case ALPHASPARSE_ACT_RELU: return activate<ALPHASPARSE_ACT_RELU>(z);
    case ALPHASPARSE_ACT_GELU: return activate<ALPHASPARSE_ACT_GELU>(z);
    case ALPHASPARSE_ACT_SILU: return activate<ALPHASPARSE_ACT_SILU>(z);
    default: return z;
  }
}

__global__ void __launch_bounds__(kMmThreads)
expert_mm_kernel(Mat x, Mat w, Mat bias, Mat r, Mat z, Mat y, bool w_nk, int act, const int32_t* __restrict__ off,
                 int segments, int rows, int n, int k) {
  __shared__ float sx[kTK][kT + 1], sw[kTK][kT + 1];
  int tile = (int)blockIdx.y, e = 0, lo = 0, hi = 0;
  for (; e < segments; ++e) {
    lo = clamp_row(off, e, segments, rows);
    hi = clamp_row(off, e + 1, segments, rows);
    const int tiles = hi > lo ? (hi - lo + kT - 1) / kT : 0;
    if (tile < tiles) break;
    tile -= tiles;
  }
  if (e == segments) return;
  const int p0 = lo + tile * kT, n0 = (int)blockIdx.x * kT, tid = threadIdx.x;
  const int ty = tid / 16, tx = tid % 16;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < k; k0 += kTK) {
    for (int i = tid; i < kT * kTK; i += kMmThreads) {
      const int a = i / kTK, c = i % kTK;
      sx[c][a] = p0 + a < hi && k0 + c < k ? load_any(x.p, (int64_t)(p0 + a) * x.ld + k0 + c, x.type) : 0.f;
      float v = 0.f;
      if (n0 + a < n && k0 + c < k)
        v = w_nk ? load_any(w.p, ((int64_t)e * n + n0 + a) * w.ld + k0 + c, w.type)
                 : load_any(w.p, ((int64_t)e * k + k0 + c) * w.ld + n0 + a, w.type);
      sw[c][a] = v;
    }
    __syncthreads();
    for (int c = 0; c < kTK; ++c)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sx[c][ty * 4 + i], sw[c][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int p = p0 + ty * 4 + i, c = n0 + tx + 16 * j;
      if (p >= hi || c >= n) continue;
      float v = acc[i][j];
      if (bias.p) v += load_any(bias.p, (int64_t)e * bias.ld + c, bias.type);
      if (z.p) store_any(z.p, (int64_t)p * z.ld + c, z.type, v);
      v = activate_any(v, act);
      if (r.p) v += load_any(r.p, (int64_t)p * r.ld + c, r.type);
      store_any(y.p, (int64_t)p * y.ld + c, y.type, v);
    }
}

// dW_e[a, b] = sum_p A[p, a] B[p, b]
__global__ void __launch_bounds__(kMmThreads)
expert_mm_grad_kernel(Mat a, Mat b, Mat dw, const int32_t* __restrict__ off, int segments, int rows, int m, int n) {
  __shared__ float sa[kTK][kT + 1], sb[kTK][kT + 1];
  const int e = (int)blockIdx.z, m0 = (int)blockIdx.y * kT, n0 = (int)blockIdx.x * kT, tid = threadIdx.x;
  const int lo = clamp_row(off, e, segments, rows), hi = clamp_row(off, e + 1, segments, rows);
  const int ty = tid / 16, tx = tid % 16;
  float acc[4][4] = {};
  for (int p0 = lo; p0 < hi; p0 += kTK) {
    for (int i = tid; i < kT * kTK; i += kMmThreads) {
      const int p = i / kT, c = i % kT;
      sa[p][c] = p0 + p < hi && m0 + c < m ? load_any(a.p, (int64_t)(p0 + p) * a.ld + m0 + c, a.type) : 0.f;
      sb[p][c] = p0 + p < hi && n0 + c < n ? load_any(b.p, (int64_t)(p0 + p) * b.ld + n0 + c, b.type) : 0.f;
    }
    __syncthreads();
    for (int c = 0; c < kTK; ++c)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[c][ty * 4 + i], sb[c][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int r = m0 + ty * 4 + i, c = n0 + tx + 16 * j;
      if (r < m && c < n) store_any(dw.p, ((int64_t)e * m + r) * dw.ld + c, dw.type, acc[i][j]);
    }
}

bool type16(alphasparseDataType t) { return t == ALPHA_R_16F || t == ALPHA_R_16BF; }

struct MmShape {
  int64_t rows, n, k;
};
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
  *size = 0;
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
  DeviceScope dev(h->device);
  ASP_CUDA(dev.status);
  const dim3 grid((unsigned)((shape.n + kT - 1) / kT), (unsigned)((shape.rows + kT - 1) / kT + segments));
  expert_mm_kernel<<<grid, kMmThreads, 0, h->stream>>>(mat(x), mat(w), mat(bias), mat(r), mat(z), mat(y),
                                                       op == ALPHA_SPARSE_OPERATION_TRANSPOSE, (int)act, off,
                                                       (int)segments, (int)shape.rows, (int)shape.n, (int)shape.k);
  ASP_CUDA(cudaGetLastError());
  ++impl(h)->launches;
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

alphasparseStatus_t alphasparseExpertMM_gradW_bufferSize(alphasparseHandle_t h, alphasparseOperation_t op,
                                                         int64_t segments, const int32_t* off,
                                                         alphasparseDnMatDescr_t x, alphasparseDnMatDescr_t dz,
                                                         alphasparseDnMatDescr_t dw, size_t* size) {
  if (!size) return ALPHA_SPARSE_STATUS_INVALID_POINTER;
  const alphasparseStatus_t s = check_grad_w(h, op, segments, off, x, dz, dw);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  *size = 0;
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

alphasparseStatus_t alphasparseExpertMM_gradW(alphasparseHandle_t h, alphasparseOperation_t op, int64_t segments,
                                              const int32_t* off, alphasparseDnMatDescr_t x, alphasparseDnMatDescr_t dz,
                                              alphasparseDnMatDescr_t dw, void* buffer) {
  const alphasparseStatus_t s = check_grad_w(h, op, segments, off, x, dz, dw);
  if (s != ALPHA_SPARSE_STATUS_SUCCESS) return s;
  const bool nk = op == ALPHA_SPARSE_OPERATION_TRANSPOSE;
  alphasparseDnMatDescr_t a = nk ? dz : x, b = nk ? x : dz;
  if (a->cols == 0 || b->cols == 0) return ALPHA_SPARSE_STATUS_SUCCESS;
  DeviceScope dev(h->device);
  ASP_CUDA(dev.status);
  const dim3 grid((unsigned)((b->cols + kT - 1) / kT), (unsigned)((a->cols + kT - 1) / kT), (unsigned)segments);
  expert_mm_grad_kernel<<<grid, kMmThreads, 0, h->stream>>>(mat(a), mat(b), mat(dw), off, (int)segments, (int)x->rows,
                                                            (int)a->cols, (int)b->cols);
  ASP_CUDA(cudaGetLastError());
  ++impl(h)->launches;
  return ALPHA_SPARSE_STATUS_SUCCESS;
}

}  // extern "C"
