// The layout in which a packed (cdclq-v1) layer is kept for products with activations, and its decoding
// in registers. Built once from the container (packed_layout in k_packed.hip).
//
// Columns become slots: the columns of a group, in the container's (permuted) order, take consecutive
// slots, and a group starts at a multiple of 32 slots, so that the 32 columns of one MFMA step share a
// scale and a zero point. Slots that no column fills hold code 0 and meet an activation of 0. Blocks of
// 128 slots (4 steps) share a code width, the largest of their groups'.
//
// Rows go in tiles of 16. A wavefront reads a tile's block as 64 lanes x 4 width bytes: lane l holds row
// l & 15 at slots 32 s + 8 (l >> 4) + i of step s, i < 8, the k order of a 16x16x32 MFMA operand. The
// codes lie in planes of 4, 2 and 1 bits (width 3 = 2 + 1, 8 = 4 + 4, ...; low bits in the first plane);
// within a plane the codes i = 2 p and 2 p + 1 are 16 bits apart, so that one shift and one mask yield
// the pair at the place of two 16-bit operands:
//   4-bit plane: dword s, bits 4 p        2-bit plane: dword s / 2, bits 8 (s & 1) + 2 p
//   1-bit plane: bits 4 s + p             (+ 16 for odd i)
// Decoding needs no conversion: code q of width b stands in the low mantissa bits of 2^b, i.e. as the
// number 2^b + q, exactly, and 2^b + zero is subtracted after the sum (times the sum of the
// activations). bf16 has 7 mantissa bits: width 8 is two operands, 16 + (q & 15) and 16 (16 + (q >> 4)).
#pragma once

#include "kernels.h"
#include "mma16.h"

namespace cdclq {

__host__ __device__ constexpr int packed_slots(const PackedView& v) { return 128 * v.nkb; }

// A lane's codes of one block.
struct PackedRegs {
  mma_u4 p4[2];
  uint32_t p2[2];
  uint32_t p1;
};

// `blk`: the block's bytes; B: its width, or 0 to take `b`.
template <int B>
__device__ __forceinline__ void packed_load(const uint8_t* blk, int lane, int b, PackedRegs& r) {
  const int w = B ? B : b;
  const uint8_t* at = blk;
  if (w & 12) {
    r.p4[0] = *reinterpret_cast<const mma_u4*>(at + 16 * lane);
    at += 1024;
  }
  if (w == 8) {
    r.p4[1] = *reinterpret_cast<const mma_u4*>(at + 16 * lane);
    return;
  }
  if (w & 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(at + 8 * lane);
    r.p2[0] = u.x;
    r.p2[1] = u.y;
    at += 512;
  }
  if (w & 1) r.p1 = *reinterpret_cast<const uint32_t*>(at + 4 * lane);
}

// (v >> right) << left with right - left known, masked: one shift
template <int RIGHT, int LEFT>
__device__ __forceinline__ uint32_t packed_field(uint32_t v, uint32_t mask) {
  constexpr int by = RIGHT - LEFT;
  const uint32_t s = by >= 0 ? v >> (by >= 0 ? by : 0) : v << (by < 0 ? -by : 0);
  return s & (mask << LEFT);
}

// The pair p of step s as codes, at bits LEFT.. of each half.
template <int B, int LEFT, int S, int P>
__device__ __forceinline__ uint32_t packed_pair(const PackedRegs& r) {
  uint32_t q = 0;
  if constexpr (B & 4) q = packed_field<4 * P, LEFT>(r.p4[0][S], 0x000f000fu);
  if constexpr (B & 2) q |= packed_field<8 * (S & 1) + 2 * P, LEFT + (B & 4)>(r.p2[S / 2], 0x00030003u);
  if constexpr (B & 1) q |= packed_field<4 * S + P, LEFT + (B & 6)>(r.p1, 0x00010001u);
  return q;
}

template <class T>
struct PackedNum {
  static constexpr int mant = T::kind == Bf16::kind ? 7 : 10, bias = T::kind == Bf16::kind ? 127 : 15;
  static constexpr uint32_t two_to(int b) { return (uint32_t)((bias + b) << mant) * 0x00010001u; }
};

// Step S of a block as operands holding 2^B + q (B < 8, or 8 in f16), packed_offset what to take off.
template <class T, int B>
constexpr float packed_offset() {
  return B == 8 && T::kind == Bf16::kind ? 272.0f : (float)(1 << B);
}
template <class T, int B, int S>
__device__ __forceinline__ void packed_step(const PackedRegs& r, typename T::v8& lo, typename T::v8& hi) {
  constexpr int M = PackedNum<T>::mant;
  uint32_t a[4], h[4] = {};
  auto pair = [&](auto pc) {
    constexpr int P = decltype(pc)::value;
    if constexpr (B < 8) {
      a[P] = packed_pair<B, M - B, S, P>(r) | PackedNum<T>::two_to(B);
    } else if constexpr (T::kind == F16::kind) {
      a[P] = packed_field<4 * P, M - 8>(r.p4[0][S], 0x000f000fu) | packed_field<4 * P, M - 4>(r.p4[1][S], 0x000f000fu) |
             PackedNum<T>::two_to(8);
    } else {
      a[P] = packed_field<4 * P, M - 4>(r.p4[0][S], 0x000f000fu) | PackedNum<T>::two_to(4);
      h[P] = packed_field<4 * P, M - 4>(r.p4[1][S], 0x000f000fu) | PackedNum<T>::two_to(8);
    }
  };
  pair(std::integral_constant<int, 0>{});
  pair(std::integral_constant<int, 1>{});
  pair(std::integral_constant<int, 2>{});
  pair(std::integral_constant<int, 3>{});
  lo = __builtin_bit_cast(typename T::v8, mma_u4{a[0], a[1], a[2], a[3]});
  hi = __builtin_bit_cast(typename T::v8, mma_u4{h[0], h[1], h[2], h[3]});
}

// Code i of step s (plain form, for expanding and building).
__device__ __forceinline__ uint32_t packed_code(const PackedRegs& r, int b, int s, int i) {
  const int p = i >> 1, h = 16 * (i & 1);
  if (b == 8) return ((r.p4[0][s] >> (4 * p + h)) & 15u) | (((r.p4[1][s] >> (4 * p + h)) & 15u) << 4);
  uint32_t q = 0;
  if (b & 4) q = (r.p4[0][s] >> (4 * p + h)) & 15u;
  if (b & 2) q |= ((r.p2[s >> 1] >> (8 * (s & 1) + 2 * p + h)) & 3u) << (b & 4);
  if (b & 1) q |= ((r.p1 >> (4 * s + p + h)) & 1u) << (b & 6);
  return q;
}

__device__ __forceinline__ float packed_scale(uint32_t sz) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)sz);
}
__device__ __forceinline__ float packed_zero(uint32_t sz) { return (float)(sz >> 16); }

// W in 16 bits, [tiles * 16][slots]: scale (code - zero), exact in f32, rounded once (the matrix cores
// take both operands in the activations' type; two 16-bit values for each weight would be exact and take twice the
// products). The error of a product over it grows from the output's own rounding to about 1.3 times that (2000
// tokens, 2048 -> 5632, bf16: 0.0022 of its size against 0.0017). By workgroups of 256 threads, b of nb.
template <class T, int U>
__device__ __forceinline__ void packed_expand_by(const PackedView& v, uint16_t* w16, long b, long nb) {
  const int lane = threadIdx.x & 63, q = lane >> 4, ns = packed_slots(v);
  const long total = (long)v.tiles * v.nkb;
  for (long id0 = (b * 4 + (threadIdx.x >> 6)) * U; id0 < total; id0 += nb * 4 * U) {
    PackedRegs r[U];
    uint32_t sz[U][4];
    int width[U];
    uint16_t* out[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long id = id0 + u < total ? id0 + u : total - 1;  // the last one twice, with the same values
      const long tile = id / v.nkb;
      const int kb = (int)(id - tile * v.nkb);
      const uint32_t info = __builtin_amdgcn_readfirstlane(v.kinfo[kb]);
      width[u] = info & 15;
      r[u] = PackedRegs{};
      packed_load<0>(v.codes + tile * v.tile_bytes + 256l * (info >> 8), lane, width[u], r[u]);
      out[u] = w16 + (tile * 16 + (lane & 15)) * ns + kb * 128 + 8 * q;
#pragma unroll
      for (int s = 0; s < 4; ++s) sz[u][s] = v.scl[(tile * v.ng + v.grp[4 * kb + s]) * 16 + (lane & 15)];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const float sc = packed_scale(sz[u][s]), z = packed_zero(sz[u][s]);
        uint32_t o[4];
#pragma unroll
        for (int p = 0; p < 4; ++p)
          o[p] = narrow2<T>(sc * ((float)packed_code(r[u], width[u], s, 2 * p) - z),
                            sc * ((float)packed_code(r[u], width[u], s, 2 * p + 1) - z));
        *reinterpret_cast<uint4*>(out[u] + 32 * s) = make_uint4(o[0], o[1], o[2], o[3]);
      }
  }
}

// Blocks of 128 k whose loads a wavefront issues together: one while that gives every SIMD some to hide each
// other's waits, then more (14336 x 4096 in 4 bits: 54 us with one, 48 with two, 53
// with four; 5632 x 2048 in 3: 15.8 with one, 17.8 with two).
inline __host__ __device__ int packed_expand_unit(const PackedView& v) { return (long)v.tiles * v.nkb > 16384 ? 2 : 1; }
template <class T>
__device__ void packed_expand(const PackedView& v, uint16_t* w16, long b, long nb) {
  if (packed_expand_unit(v) == 1) packed_expand_by<T, 1>(v, w16, b, nb);
  else packed_expand_by<T, 2>(v, w16, b, nb);
}

}  // namespace cdclq
