// Eight neighbouring elements of a row as f32, the unit in which the embedding, clipping and logit kernels move
// their data: 16 bytes a lane of the 16-bit types, 32 of f32. Rows may start at any element: the 16-byte accesses
// of gfx950 need no more alignment than an element's. The loops over whole units have no other path for a row's last,
// shorter one: with it beside each access the compiler waits for every load by itself (16384 embedding rows of
// 4096: 68 us, without 40).
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
  static __device__ __forceinline__ float widen(uint16_t x) { return T::widen(x); }
  static __device__ __forceinline__ uint16_t narrow(float x) { return T::narrow(x); }
  __device__ __forceinline__ float get(int i) const { return widen(v[i]); }
  __device__ __forceinline__ void set(int i, float x) { v[i] = narrow(x); }
};
template <>
struct Row8<F32> {
  typedef float stored;
  float v[8];
  static __device__ __forceinline__ float widen(float x) { return x; }
  static __device__ __forceinline__ float narrow(float x) { return x; }
  __device__ __forceinline__ float get(int i) const { return v[i]; }
  __device__ __forceinline__ void set(int i, float x) { v[i] = x; }
};

// LAST: what nobody reads again soon, past the L2 (non-temporal). The rows of an embedding's gradient (32768 x 2048:
// 124 us a step, so 115) and gradients on their second, last reading (2.8 GB: 736 us, so 713); logits rather not (41, 44).
template <class T, bool LAST = false>
__device__ __forceinline__ Row8<T> row8_load(const typename Row8<T>::stored* p) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
  Row8<T> r;
  u4 t[sizeof(r.v) / 16];
#pragma unroll
  for (int i = 0; i < (int)(sizeof(r.v) / 16); ++i) {
    if constexpr (LAST) t[i] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p) + i);
    else t[i] = reinterpret_cast<const u4*>(p)[i];
  }
  __builtin_memcpy(r.v, t, sizeof(r.v));
  return r;
}
// Past the L2 (non-temporal): results that no later workgroup of the launch reads. Written lines that the L2 holds when
// a kernel ends have to leave it then: 16384 rows of 4096 from an embedding 40 us, so 36; gradients clipped into f32
// 82 and 78; logits 48 and 41; 1.05 GB of zeros 174 and 159. FILL: through it, for what is small beside it. f32
// goes through it, too: a lane's 32 bytes are two stores, of half lines each.
template <class T, bool FILL = false>
__device__ __forceinline__ void row8_store(typename Row8<T>::stored* p, const Row8<T>& r) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
  u4 t[sizeof(r.v) / 16];
  __builtin_memcpy(t, r.v, sizeof(r.v));
#pragma unroll
  for (int i = 0; i < (int)(sizeof(r.v) / 16); ++i) {
    if constexpr (FILL || sizeof(r.v) > 16) reinterpret_cast<u4*>(p)[i] = t[i];
    else __builtin_nontemporal_store(t[i], reinterpret_cast<u4*>(p) + i);
  }
}
// The first n < 8 of them, the others 0.
template <class T>
__device__ __forceinline__ Row8<T> row8_load(const typename Row8<T>::stored* p, int n) {
  Row8<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = i < n ? p[i] : typename Row8<T>::stored(0);
  return r;
}
template <class T>
__device__ __forceinline__ void row8_store(typename Row8<T>::stored* p, const Row8<T>& r, int n) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = r.v[i];
}

}  // namespace cdclq
