// Element types of the training operators (include/pmg_lm.h): loads to and stores from fp32, several elements
// at a time.  The vectors carry the alignment of their element only: global memory takes 16-byte accesses at any
// element's address here, so rows of odd length and tensors cut from a flat buffer need no path of their own.
#pragma once
#include "pmg_common.h"
#include "../../include/pmg_lm.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T, int N> struct pmg_vec {
  typedef T type __attribute__((ext_vector_type(N)));
  typedef T in_memory __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

template <typename T> __device__ __forceinline__ f32x4 pmg_load4(const T* p) {
  const typename pmg_vec<T, 4>::type v = *reinterpret_cast<const typename pmg_vec<T, 4>::in_memory*>(p);
  return f32x4{(float)v.x, (float)v.y, (float)v.z, (float)v.w};
}
template <typename T> __device__ __forceinline__ void pmg_store4(T* p, f32x4 x) {
  typename pmg_vec<T, 4>::type v;
  v.x = (T)x.x; v.y = (T)x.y; v.z = (T)x.z; v.w = (T)x.w;
  *reinterpret_cast<typename pmg_vec<T, 4>::in_memory*>(p) = v;
}
// `left` elements remain at p (>= 1)
template <typename T> __device__ __forceinline__ f32x4 pmg_load4(const T* p, int64_t left) {
  if (left >= 4) return pmg_load4(p);
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < left) x[j] = (float)p[j];
  return x;
}
template <typename T> __device__ __forceinline__ void pmg_store4(T* p, f32x4 x, int64_t left) {
  if (left >= 4) return pmg_store4(p, x);
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < left) p[j] = (T)x[j];
}
// past the caches: for results that nobody reads soon
template <typename T> __device__ __forceinline__ void pmg_store4_nt(T* p, f32x4 x, int64_t left) {
  if (left < 4) return pmg_store4(p, x, left);
  typename pmg_vec<T, 4>::type v;
  v.x = (T)x.x; v.y = (T)x.y; v.z = (T)x.z; v.w = (T)x.w;
  typedef typename pmg_vec<T, 4>::in_memory mem;
  __builtin_nontemporal_store(v, reinterpret_cast<mem*>(p));
}

// eight elements of which `left` (>= 1) remain
template <typename T> __device__ __forceinline__ void pmg_store8(T* p, f32x4 x, f32x4 y, int64_t left) {
  if (left >= 8) {
    typename pmg_vec<T, 8>::type v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = (T)x[j];
      v[4 + j] = (T)y[j];
    }
    *reinterpret_cast<typename pmg_vec<T, 8>::in_memory*>(p) = v;
    return;
  }
  pmg_store4(p, x, left);
  if (left > 4) pmg_store4(p + 4, y, left - 4);
}

static inline size_t pmg_elem_bytes(int dtype) { return dtype == PMG_F32 ? 4 : 2; }
static inline bool pmg_dtype_ok(int dtype) { return dtype == PMG_F32 || dtype == PMG_BF16 || dtype == PMG_F16; }

// 16 bytes of a row: 4 fp32 or 8 bf16 / fp16 elements.
template <typename T> struct pmg_vec16 {
  static constexpr int N = 16 / sizeof(T);
  typedef typename pmg_vec<T, N>::type vec;
  typedef typename pmg_vec<T, N>::in_memory mem;
  // as they lie in memory: a load whose conversion waits until they are needed; `left` elements remain at p (>= 1)
  static __device__ __forceinline__ vec load(const T* p, int64_t left) {
    if (left >= N) return *reinterpret_cast<const mem*>(p);
    vec v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < left ? p[j] : (T)0.0f;
    return v;
  }
  static __device__ __forceinline__ void store(T* p, const float (&x)[N], int64_t left) {
    if (left >= N) {
      vec v;
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = (T)x[j];
      *reinterpret_cast<mem*>(p) = v;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < left) p[j] = (T)x[j];
    }
  }
};
