// 8-bit activation checkpoints: a token's features in blocks of 128, each with one f32 scale.
//
//   s = max |x| / 127    c = rint(x / s), 0 where s = 0    restored value = s c
//
// rint rounds ties to even and the divisions are the correctly rounded ones, so the codes follow from
// the formula alone. |c| <= 127. A block that holds a NaN or an infinity has s = NaN (and codes 0): it
// is restored as NaN, so that an overflow stays visible to the gradient.
//
// Both directions are one pass over memory, which bounds them: 16 lanes take a block, 16 bytes of x and 8 of
// codes each, so that a wavefront's loads are whole lines and the maximum takes four lane exchanges.
// 16384 x 14336 bf16: saved in 185 us on average, 147 at least (4.8 TB/s; with a division for each code 230 and 184),
// restored in 117 and 109 (6.5 TB/s, the codes partly from the last cache), one after the other in 262 (5.4 TB/s);
// 512 x 4096: 4.1 and 3.2 us.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cdclq.h"
#include "kernels.h"
#include "mma16.h"

namespace cdclq {
namespace {

// Largest magnitude of the 16-bit patterns (their order is that of the magnitudes; infinities and NaN
// are the largest), and the pattern of infinity.
template <class T>
constexpr uint32_t inf_bits() {
  return T::kind == Bf16::kind ? 0x7f80u : 0x7c00u;
}

// Where a group of 16 lanes stands: block `blk` of token `row`, block b of all, `step` blocks a move. (A
// division by nb for each would cost as much as the codes.)
struct CkptAt {
  long b, row, total;
  int blk, nb, step, drow, dblk;
  __device__ __forceinline__ CkptAt(long t, int nb_) : total(t * nb_), nb(nb_), step(gridDim.x * 16) {
    const uint32_t b0 = blockIdx.x * 16u + (threadIdx.x >> 4);
    b = b0;
    row = b0 / (uint32_t)nb;
    blk = (int)(b0 - (uint32_t)row * nb);
    drow = step / nb;
    dblk = step - drow * nb;
  }
  __device__ __forceinline__ bool on() const { return b < total; }
  __device__ __forceinline__ void move() {
    b += step;
    row += drow;
    blk += dblk;
    if (blk >= nb) blk -= nb, ++row;
  }
};

// rint of the correctly rounded x / s, as a number whose low byte is the code. r = 1 / s correctly rounded: the
// first correction brings x r within an ulp of the quotient, the second to it (Markstein); s is far from f32's
// smallest. Adding 1.5 2^23 rounds to an integer, ties to even.
__device__ __forceinline__ uint32_t code_of(float x, float s, float r) {
  float q = x * r;
  q = __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
  q = __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
  return __float_as_uint(q + 12582912.0f);
}

template <class T, bool VEC>
__global__ __launch_bounds__(256) void k_ckpt_save(const uint16_t* __restrict__ x, long ldx, long t, int n, int nb,
                                                   int8_t* __restrict__ codes, float* __restrict__ scales) {
  const int i = threadIdx.x & 15;
  for (CkptAt at(t, nb); at.on(); at.move()) {
    const long row = at.row;
    const int c0 = at.blk * 128 + 8 * i;
    uint16_t v[8];
    if constexpr (VEC) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (c0 < n) u = *reinterpret_cast<const uint4*>(x + row * ldx + c0);
      *reinterpret_cast<uint4*>(v) = u;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c0 + j < n ? x[row * ldx + c0 + j] : (uint16_t)0;
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, (uint32_t)(v[j] & 0x7fff));
#pragma unroll
    for (int s = 1; s < 16; s <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, s));
    const bool bad = m >= inf_bits<T>();
    const float scale = bad ? __builtin_nanf("") : T::widen((uint16_t)m) / 127.0f;
    union {
      int8_t c[8];
      uint32_t w[2];
      uint2 u;
    } o;
    if (scale >= 0x1p-90f) {
      const float r = 1.0f / scale;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = code_of(T::widen(v[4 * h + j]), scale, r);
        o.w[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u),
                                       __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), 0x05040100u);
      }
    } else {  // a block of zeros or of the smallest numbers, or with a NaN
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float q = scale > 0.0f ? __builtin_rintf(T::widen(v[j]) / scale) : 0.0f;
        o.c[j] = (int8_t)(int)fminf(fmaxf(q, -127.0f), 127.0f);
      }
    }
    if (i == 0) scales[at.b] = scale;
    int8_t* to = codes + row * n + c0;
    if constexpr (VEC) {
      if (c0 < n) *reinterpret_cast<uint2*>(to) = o.u;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + j < n) to[j] = o.c[j];
    }
  }
}

template <class T, bool VEC>
__global__ __launch_bounds__(256) void k_ckpt_restore(const int8_t* __restrict__ codes,
                                                      const float* __restrict__ scales, long t, int n, int nb,
                                                      uint16_t* __restrict__ out, long ldo) {
  const int i = threadIdx.x & 15;
  for (CkptAt at(t, nb); at.on(); at.move()) {
    const long row = at.row;
    const int c0 = at.blk * 128 + 8 * i;
    const float scale = scales[at.b];
    const int8_t* from = codes + row * n + c0;
    uint16_t* to = out + row * ldo + c0;
    if constexpr (VEC) {
      if (c0 < n) {
        union {
          uint2 u;
          int8_t c[8];
        } v;
        v.u = *reinterpret_cast<const uint2*>(from);
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = narrow2<T>(scale * (float)v.c[2 * j], scale * (float)v.c[2 * j + 1]);
        *reinterpret_cast<uint4*>(to) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + j < n) to[j] = T::narrow(scale * (float)from[j]);
    }
  }
}

inline int grid_for(long blocks) { return (int)std::max(1l, std::min((blocks + 15) / 16, 1l << 16)); }

template <class T>
hipError_t save(hipStream_t st, const uint16_t* x, long ldx, long t, long n, int8_t* codes, float* scales) {
  const int nb = (int)((n + 127) / 128), grid = grid_for(t * nb);
  const bool vec = n % 8 == 0 && ldx % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)codes % 8 == 0;
  if (vec) k_ckpt_save<T, true><<<grid, 256, 0, st>>>(x, ldx, t, (int)n, nb, codes, scales);
  else k_ckpt_save<T, false><<<grid, 256, 0, st>>>(x, ldx, t, (int)n, nb, codes, scales);
  return hipGetLastError();
}
template <class T>
hipError_t restore(hipStream_t st, const int8_t* codes, const float* scales, long t, long n, uint16_t* out, long ldo) {
  const int nb = (int)((n + 127) / 128), grid = grid_for(t * nb);
  const bool vec = n % 8 == 0 && ldo % 8 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)codes % 8 == 0;
  if (vec) k_ckpt_restore<T, true><<<grid, 256, 0, st>>>(codes, scales, t, (int)n, nb, out, ldo);
  else k_ckpt_restore<T, false><<<grid, 256, 0, st>>>(codes, scales, t, (int)n, nb, out, ldo);
  return hipGetLastError();
}

}  // namespace

hipError_t ckpt_save(hipStream_t st, int dtype, const uint16_t* x, long ldx, long t, long n, int8_t* codes,
                     float* scales) {
  return dtype == CDCLQ_DTYPE_BF16 ? save<Bf16>(st, x, ldx, t, n, codes, scales)
                                   : save<F16>(st, x, ldx, t, n, codes, scales);
}
hipError_t ckpt_restore(hipStream_t st, int dtype, const int8_t* codes, const float* scales, long t, long n,
                        uint16_t* out, long ldo) {
  return dtype == CDCLQ_DTYPE_BF16 ? restore<Bf16>(st, codes, scales, t, n, out, ldo)
                                   : restore<F16>(st, codes, scales, t, n, out, ldo);
}

}  // namespace cdclq
