// Element types of the training operators (include/pmg_lm.h): loads to and stores from fp32, four
// elements at a time where the address allows it.
#pragma once
#include "pmg_common.h"
#include "../../include/pmg_lm.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> struct pmg_vec4;
template <> struct pmg_vec4<float> { typedef f32x4 type; };
template <> struct pmg_vec4<bf16_t> { typedef __bf16 type __attribute__((ext_vector_type(4))); };
template <> struct pmg_vec4<f16_t> { typedef _Float16 type __attribute__((ext_vector_type(4))); };

template <typename T> __device__ __forceinline__ float pmg_to_f32(T x) { return (float)x; }
template <typename T> __device__ __forceinline__ T pmg_from_f32(float x) { return (T)x; }  // to nearest, ties to even

template <typename T> __device__ __forceinline__ f32x4 pmg_load4(const T* p) {
  const typename pmg_vec4<T>::type v = *reinterpret_cast<const typename pmg_vec4<T>::type*>(p);
  return f32x4{(float)v.x, (float)v.y, (float)v.z, (float)v.w};
}
template <typename T> __device__ __forceinline__ void pmg_store4(T* p, f32x4 x) {
  typename pmg_vec4<T>::type v;
  v.x = (T)x.x; v.y = (T)x.y; v.z = (T)x.z; v.w = (T)x.w;
  *reinterpret_cast<typename pmg_vec4<T>::type*>(p) = v;
}
// `left` elements remain at p (>= 1); aligned: p is a multiple of four elements.
template <typename T> __device__ __forceinline__ f32x4 pmg_load4(const T* p, bool aligned, int64_t left) {
  if (aligned && left >= 4) return pmg_load4(p);
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) x[j] = (float)p[j];
  return x;
}
template <typename T> __device__ __forceinline__ void pmg_store4(T* p, f32x4 x, bool aligned, int64_t left) {
  if (aligned && left >= 4) return pmg_store4(p, x);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) p[j] = (T)x[j];
}
// past the caches: for results that nobody reads soon
template <typename T> __device__ __forceinline__ void pmg_store4_nt(T* p, f32x4 x, bool aligned, int64_t left) {
  if (!aligned || left < 4) return pmg_store4(p, x, aligned, left);
  typename pmg_vec4<T>::type v;
  v.x = (T)x.x; v.y = (T)x.y; v.z = (T)x.z; v.w = (T)x.w;
  __builtin_nontemporal_store(v, reinterpret_cast<typename pmg_vec4<T>::type*>(p));
}
template <typename T> __device__ __forceinline__ bool pmg_aligned4(const T* p) {
  return ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0;
}

static inline size_t pmg_elem_bytes(int dtype) { return dtype == PMG_F32 ? 4 : 2; }
static inline bool pmg_dtype_ok(int dtype) { return dtype == PMG_F32 || dtype == PMG_BF16 || dtype == PMG_F16; }

// 16 bytes of a row: 4 fp32 or 8 bf16 / fp16 elements, in fp32 registers.
template <typename T> struct pmg_vec16 {
  static constexpr int N = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(N)));
  float x[N];
  // the 16 bytes as they lie in memory: a load whose conversion (unpack) waits until they are needed
  static __device__ __forceinline__ vec raw(const T* p, bool aligned, int64_t left) {
    if (aligned && left >= N) return *reinterpret_cast<const vec*>(p);
    vec v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = j < left ? p[j] : (T)0.0f;
    return v;
  }
  // `left` elements remain at p (>= 1); aligned: p is a multiple of 16 bytes
  __device__ __forceinline__ void load(const T* p, bool aligned, int64_t left) {
    if (aligned && left >= N) {
      const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = (float)v[j];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = j < left ? (float)p[j] : 0.0f;
    }
  }
  __device__ __forceinline__ void store(T* p, bool aligned, int64_t left) const {
    if (aligned && left >= N) {
      vec v;
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = (T)x[j];
      *reinterpret_cast<vec*>(p) = v;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < left) p[j] = (T)x[j];
    }
  }
};
template <typename T> __device__ __forceinline__ bool pmg_rows_aligned16(const T* p, int64_t ld) {
  return (((uintptr_t)p | (uintptr_t)(ld * (int64_t)sizeof(T))) & 15) == 0;
}
