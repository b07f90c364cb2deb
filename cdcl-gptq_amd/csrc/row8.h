// Eight neighbouring elements of a row as f32, the unit in which the embedding, clipping and logit kernels move
// their data: 16 bytes a lane of the 16-bit types, 32 of f32. Rows may start at any element: the 16-byte accesses
// of gfx950 need no more alignment than an element's.
#pragma once

#include "mma16.h"

namespace cdclq {

// f32 beside the two 16-bit types of mma16.h.
struct F32 {
  static constexpr int kind = 0;  // CDCLQ_DTYPE_F32
};

template <class T>
struct Row8 {
  typedef uint16_t stored;
  uint16_t v[8];
  __device__ __forceinline__ float get(int i) const { return T::widen(v[i]); }
  __device__ __forceinline__ void set(int i, float x) { v[i] = T::narrow(x); }
};
template <>
struct Row8<F32> {
  typedef float stored;
  float v[8];
  __device__ __forceinline__ float get(int i) const { return v[i]; }
  __device__ __forceinline__ void set(int i, float x) { v[i] = x; }
};

// The first n (1..8 or more: 8) of the elements at p; the others 0.
template <class T>
__device__ __forceinline__ Row8<T> row8_load(const typename Row8<T>::stored* p, long n) {
  Row8<T> r;
  if (n >= 8) {
    __builtin_memcpy(r.v, p, sizeof(r.v));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = i < n ? p[i] : typename Row8<T>::stored(0);
  }
  return r;
}
template <class T>
__device__ __forceinline__ void row8_store(typename Row8<T>::stored* p, long n, const Row8<T>& r) {
  if (n >= 8) {
    __builtin_memcpy(p, r.v, sizeof(r.v));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = r.v[i];
  }
}
template <class T>
__device__ __forceinline__ Row8<T> row8_fill(float x) {
  Row8<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.set(i, x);
  return r;
}

}  // namespace cdclq
