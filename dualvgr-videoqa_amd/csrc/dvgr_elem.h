// dvgr_elem.h -- element types of the operators that take fp32, bf16 and fp16 tensors (enum dvgr_elem): 16-byte vectors of a
// type to and from floats.  Arithmetic is fp32 throughout; a value is rounded to its tensor's type once, where it is stored.
#pragma once
#include "dvgr_common.h"

namespace dvgr {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> struct Vec16 {
  static constexpr int N = 16 / (int)sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
};

// N = 16 / sizeof(T) consecutive elements at a 16-byte aligned address
template <typename T> __device__ __forceinline__ void load_vec(const T* p, float (&f)[Vec16<T>::N]) {
  const typename Vec16<T>::type v = *reinterpret_cast<const typename Vec16<T>::type*>(p);
#pragma unroll
  for (int i = 0; i < Vec16<T>::N; ++i) f[i] = (float)v[i];
}
template <typename T> __device__ __forceinline__ void store_vec(T* p, const float (&f)[Vec16<T>::N]) {
  typename Vec16<T>::type v;
#pragma unroll
  for (int i = 0; i < Vec16<T>::N; ++i) v[i] = (T)f[i];
  *reinterpret_cast<typename Vec16<T>::type*>(p) = v;
}

// Streams: what is read once, or written for a reader far away, does not push other data out of the caches.  Rows of 64 KB read once:
// 6.6 TB/s, 5.9 with ordinary loads.
template <typename V> __device__ __forceinline__ V stream_load(const V* p) { return __builtin_nontemporal_load(p); }
template <typename V> __device__ __forceinline__ void stream_store(V* p, const V& v) { __builtin_nontemporal_store(v, p); }
template <typename T> __device__ __forceinline__ void stream_store_vec(T* p, const float (&f)[Vec16<T>::N]) {
  typename Vec16<T>::type v;
#pragma unroll
  for (int i = 0; i < Vec16<T>::N; ++i) v[i] = (T)f[i];
  stream_store(reinterpret_cast<typename Vec16<T>::type*>(p), v);
}

__device__ __forceinline__ float load_elem(const void* p, int64_t i, int elem) {
  return elem == DVGR_ELEM_F32 ? reinterpret_cast<const float*>(p)[i]
       : elem == DVGR_ELEM_BF16 ? (float)reinterpret_cast<const bf16_t*>(p)[i] : (float)reinterpret_cast<const f16_t*>(p)[i];
}

inline int elem_size(int elem) { return elem == DVGR_ELEM_F32 ? 4 : elem == DVGR_ELEM_BF16 || elem == DVGR_ELEM_F16 ? 2 : 0; }
inline bool ptr16(const void* p) { return ((uintptr_t)p & 15) == 0; }

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// 2^x on the hardware unit (1 ulp); exp2_fast(-inf) = 0
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace dvgr
