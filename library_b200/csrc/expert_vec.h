// Packs of 16 bytes (or single elements) of fp32, fp16 and bf16, widened to fp32, for the kernels
// that stream rows: V = 16 / sizeof(T) where base and leading dimension are 16-byte aligned, else 1.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "asp_internal.h"

namespace asp {

template <typename T> struct Wide;
template <> struct Wide<float> {
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};
template <> struct Wide<__half> {
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <> struct Wide<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};

template <typename T, int V> struct Pack {
  static_assert(V == 1 || V * sizeof(T) == 16, "a pack is one element or 16 bytes");
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> r;
  if constexpr (V == 1) {
    r.v[0] = *p;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    memcpy(r.v, &u, 16);
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& r) {
  if constexpr (V == 1) {
    *p = r.v[0];
  } else {
    uint4 u;
    memcpy(&u, r.v, 16);
    *reinterpret_cast<uint4*>(p) = u;
  }
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> round_pack(const float (&f)[V]) {
  Pack<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = Wide<T>::down(f[i]);
  return r;
}

// Whether every row of the matrix starts on a 16-byte boundary and its width is whole packs.
inline bool packs_of_16(alphasparseDnMatDescr_t m) {
  if (!m) return true;
  const size_t es = elem_size(m->data_type);
  return (reinterpret_cast<uintptr_t>(m->values) & 15) == 0 && ((size_t)m->ld * es) % 16 == 0 &&
         ((size_t)m->cols * es) % 16 == 0;
}

}  // namespace asp
