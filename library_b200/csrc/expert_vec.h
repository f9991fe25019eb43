// Packs of 16 bytes, 4 bytes or single elements of fp32, fp16 and bf16, widened to fp32, for the kernels
// that stream rows: the widest pack that every row's start and width are multiples of.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

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

// A pack as 32-bit words (16-bit elements stay two to a register until they are used), or one element.
template <typename T, int V> struct Pack {
  static constexpr int kWords = V * (int)sizeof(T) / 4;
  static_assert(kWords == 4 || kWords == 1, "a pack is one element, 4 bytes or 16 bytes");
  uint32_t w[kWords];
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    else return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu)));
  }
};
template <typename T> struct Pack<T, 1> {
  T v;
  __device__ __forceinline__ float at(int) const { return Wide<T>::up(v); }
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> r;
  if constexpr (V == 1) {
    r.v = *p;
  } else if constexpr (Pack<T, V>::kWords == 1) {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    r.w[0] = u.x;
    r.w[1] = u.y;
    r.w[2] = u.z;
    r.w[3] = u.w;
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& r) {
  if constexpr (V == 1) *p = r.v;
  else if constexpr (Pack<T, V>::kWords == 1) *reinterpret_cast<uint32_t*>(p) = r.w[0];
  else *reinterpret_cast<uint4*>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> round_pack(const float (&f)[V]) {
  Pack<T, V> r;
  if constexpr (V == 1) {
    r.v = Wide<T>::down(f[0]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) r.w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        memcpy(&r.w[i], &h, 4);
      } else {
        const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        memcpy(&r.w[i], &h, 4);
      }
    }
  }
  return r;
}

// Bytes of the widest pack that fits every row of the matrix (NULL: any).
inline int pack_bytes(alphasparseDnMatDescr_t m) {
  if (!m) return 16;
  const size_t es = elem_size(m->data_type);
  const size_t all = reinterpret_cast<uintptr_t>(m->values) | (size_t)m->ld * es | (size_t)m->cols * es;
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : (int)es;
}
// f(V) with the number of elements of the widest pack that fits all of the matrices.
template <typename T, typename F, typename... M>
alphasparseStatus_t by_pack(F f, M... m) {
  const int b = std::min({pack_bytes(m)...});
  if (b == 16) return f(std::integral_constant<int, 16 / sizeof(T)>());
  if constexpr (sizeof(T) == 2) {
    if (b == 4) return f(std::integral_constant<int, 2>());
  }
  return f(std::integral_constant<int, 1>());
}
// Packs per lane such that a lane has at least `bytes` of a row on the way, up to eight.
template <typename T, int V> constexpr int packs_per_lane(int bytes) {
  const int n = bytes / (V * (int)sizeof(T));
  return n < 1 ? 1 : n > 8 ? 8 : n;
}

}  // namespace asp
