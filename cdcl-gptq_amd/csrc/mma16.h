// Tiles of 16-bit matrix products (bf16 or f16 in, f32 sums) on the gfx950 matrix cores, shared by
// the vocabulary loss and the packed projection.
//
// C[i][j] = sum_k P(i, k) Q(j, k), i over BP rows of P, j over BQ rows of Q. An operand is stored
// either with k contiguous (rows x ld) or, PS / QS, with the rows contiguous (k x ld). A workgroup of
// WP x WQ wavefronts computes BP x BQ = 16 FP WP x 16 FQ WQ elements, a wavefront FP x FQ blocks of
// v_mfma_f32_16x16x32: lane l supplies rows l & 15 at k = 8 (l >> 4) .. + 7 of both operands, and
// register r of a result is row 4 (l >> 4) + r, column l & 15.
//
// Stages of 64 k are loaded straight into LDS (16 bytes a lane) in two buffers: while a stage is
// multiplied the next one is in flight, one barrier a stage. LDS holds an operand as 16-byte granules,
//   k contiguous:    granule g of row i at position g ^ (i & 7) of the row's 8: the 16 rows that a
//                    16-byte read serves together then start in 8 different places of the banks;
//   rows contiguous: granule g of k-row k at position g ^ 2 s(k), s = (k & 3) + 4 (k >> 3 & 1), of
//                    the row's BP / 8: read by ds_read_b64_tr_b16, which hands lane i of 16 the
//                    column i of a 4 x 16 block, so that a block's rows start in 8 different places.
// What lies past the end of k is taken from a page of zeros, rows past the last one repeat it (their
// results are not used). Requirements, checked on the host: 16-byte aligned operands, ld a multiple of
// 8, and k (k contiguous) or the rows (rows contiguous) padded to a multiple of 8 within ld; with k
// contiguous the padding holds zeros.
#pragma once

#include "cdclq_dev.h"

namespace cdclq {

typedef short mma_s4 __attribute__((ext_vector_type(4)));
typedef float mma_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t mma_u4 __attribute__((ext_vector_type(4)));

// The two 16-bit types: stored as their bit patterns.
struct Bf16 {
  typedef __bf16 scalar;
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static constexpr int kind = 2;  // CDCLQ_DTYPE_BF16
  static __device__ __forceinline__ mma_f4 mfma(v8 a, v8 b, mma_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float widen(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }
  static __device__ __forceinline__ uint16_t narrow(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
};
struct F16 {
  typedef _Float16 scalar;
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static constexpr int kind = 1;  // CDCLQ_DTYPE_F16
  static __device__ __forceinline__ mma_f4 mfma(v8 a, v8 b, mma_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float widen(uint16_t u) { return (float)__builtin_bit_cast(_Float16, u); }
  static __device__ __forceinline__ uint16_t narrow(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};

template <class T>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  return (uint32_t)T::narrow(a) | ((uint32_t)T::narrow(b) << 16);
}

// An operand of C: `rows` rows of k values each, element (i, k) at p[i ld + k] or, rows contiguous, at
// p[k ld + i].
struct MmaOp {
  const uint16_t* p;
  long ld;
  int rows;
};

static __device__ uint4 mma_zero_page[1];  // never written

template <class T, bool PS, bool QS, int FP, int FQ, int WP, int WQ>
struct MmaTile {
  static constexpr int W = WP * WQ, THREADS = 64 * W;
  static constexpr int BP = 16 * FP * WP, BQ = 16 * FQ * WQ, BK = 64;
  static constexpr int STAGE = (BP + BQ) * BK * 2;  // bytes of one stage
  static constexpr int LDS = 2 * STAGE;
  static constexpr int NP = (BP / 8 + W - 1) / W, NQ = (BQ / 8 + W - 1) / W;  // loads per wavefront and stage
  typedef typename T::v8 v8;
  static_assert(!PS || BP >= 128, "the transposed read's swizzle spans 8 pairs of granules");
  static_assert(!QS || BQ >= 128, "the transposed read's swizzle spans 8 pairs of granules");

  // Where granule slot `s` of a stage comes from: its offset in k, and its address at k = k0.
  template <bool S, int B>
  static __device__ __forceinline__ int granule_k(int s) {
    return S ? s / (B / 8) : 8 * ((s & 7) ^ ((s >> 3) & 7));
  }
  template <bool S, int B>
  static __device__ __forceinline__ const uint16_t* granule_at(const MmaOp& o, int r0, int k0, int s) {
    if constexpr (S) {
      const int k = s / (B / 8);
      const int g = (s % (B / 8)) ^ (2 * ((k & 3) | ((k >> 1) & 4)));
      return o.p + (long)(k0 + k) * o.ld + min(r0 + 8 * g, (o.rows - 1) & ~7);
    } else {
      return o.p + (long)min(r0 + (s >> 3), o.rows - 1) * o.ld + k0 + granule_k<S, B>(s);
    }
  }

  static __device__ __forceinline__ v8 read_c(uint32_t at) {
    return *(const __attribute__((address_space(3))) v8*)(uintptr_t)(at);
  }
  template <int B>
  static __device__ __forceinline__ v8 read_s(uint32_t at) {
    typedef __attribute__((address_space(3))) mma_s4* lds_s4;
    mma_s4 h[2];
    h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)at);
    h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)(at + 4 * B * 2));
    return __builtin_bit_cast(v8, h);
  }

  // acc += P[p0 .., kbeg .. kend) Q[q0 .., kbeg .. kend)^T; kbeg is a multiple of 64. lds: the byte
  // offset of LDS bytes of shared memory. All wavefronts of the workgroup call it together.
  static __device__ __forceinline__ void run(uint32_t lds, const MmaOp& P, const MmaOp& Q, int p0, int q0, int kbeg,
                                             int kend, mma_f4 (&acc)[FP][FQ]) {
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wv / WQ, wq = wv % WQ;
    if (kbeg >= kend) return;
    const uint16_t *pp[NP], *pq[NQ];
#pragma unroll
    for (int i = 0; i < NP; ++i) pp[i] = granule_at<PS, BP>(P, p0, kbeg, 64 * (wv + W * i) + lane);
#pragma unroll
    for (int i = 0; i < NQ; ++i) pq[i] = granule_at<QS, BQ>(Q, q0, kbeg, 64 * (wv + W * i) + lane);
    const long sp = PS ? BK * P.ld : BK, sq = QS ? BK * Q.ld : BK;
    const float* const zero = reinterpret_cast<const float*>(&mma_zero_page[0]);

    auto issue = [&](int k0, uint32_t buf) {
      const bool whole = k0 + BK <= kend;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if (BP / 8 % W && wv + W * i >= BP / 8) break;
        const float* src = reinterpret_cast<const float*>(pp[i]);
        if (!whole && k0 + granule_k<PS, BP>(64 * (wv + W * i) + lane) >= kend) src = zero;
        dma16_untracked(src, buf + 1024u * (wv + W * i));
        pp[i] += sp;
      }
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if (BQ / 8 % W && wv + W * i >= BQ / 8) break;
        const float* src = reinterpret_cast<const float*>(pq[i]);
        if (!whole && k0 + granule_k<QS, BQ>(64 * (wv + W * i) + lane) >= kend) src = zero;
        dma16_untracked(src, buf + BP * BK * 2 + 1024u * (wv + W * i));
        pq[i] += sq;
      }
    };

    // read addresses within a stage
    const int r = lane & 15, q = lane >> 4;
    const uint32_t s = ((lane >> 2) & 3) | ((q & 1) << 2);
    uint32_t ap[PS ? FP : 2], aq[QS ? FQ : 2];
    if constexpr (PS) {
#pragma unroll
      for (int f = 0; f < FP; ++f)
        ap[f] = (8 * q + (r >> 2)) * (BP * 2) + 32 * ((uint32_t)(FP * wp + f) ^ s) + 8 * (lane & 3);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) ap[h] = (16 * FP * wp + r) * 128 + 16 * ((4 * h + q) ^ (r & 7));
    }
    if constexpr (QS) {
#pragma unroll
      for (int f = 0; f < FQ; ++f)
        aq[f] = BP * BK * 2 + (8 * q + (r >> 2)) * (BQ * 2) + 32 * ((uint32_t)(FQ * wq + f) ^ s) + 8 * (lane & 3);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        aq[h] = BP * BK * 2 + (16 * FQ * wq + r) * 128 + 16 * ((4 * h + q) ^ (r & 7));
    }

    uint32_t buf = lds, other = lds + STAGE;
    issue(kbeg, buf);
    for (int k0 = kbeg; k0 < kend; k0 += BK) {
      // this wavefront's part of the stage has landed and its reads of the last one are done; the
      // barrier says so of every wavefront
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (k0 + BK < kend) issue(k0 + BK, other);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v8 a[FP], b[FQ];
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
          if constexpr (QS) b[f] = read_s<BQ>(buf + aq[f] + 32 * h * BQ * 2);
          else b[f] = read_c(buf + aq[h] + 2048 * f);
        }
#pragma unroll
        for (int f = 0; f < FP; ++f) {
          if constexpr (PS) a[f] = read_s<BP>(buf + ap[f] + 32 * h * BP * 2);
          else a[f] = read_c(buf + ap[h] + 2048 * f);
        }
#pragma unroll
        for (int f = 0; f < FP; ++f)
#pragma unroll
          for (int g = 0; g < FQ; ++g) acc[f][g] = T::mfma(a[f], b[g], acc[f][g]);
      }
      const uint32_t t = buf;
      buf = other;
      other = t;
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the shared memory is free again
  }
  static __device__ __forceinline__ void clear(mma_f4 (&acc)[FP][FQ]) {
#pragma unroll
    for (int f = 0; f < FP; ++f)
#pragma unroll
      for (int g = 0; g < FQ; ++g) acc[f][g] = mma_f4{};
  }
  // first P row / Q row (result row / column) of this wavefront's block f / g; the lane's own rows are
  // row(f) + 4 (lane >> 4) + r, its column col(g) + (lane & 15)
  static __device__ __forceinline__ int row(int p0, int f) {
    return p0 + 16 * (FP * (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / WQ) + f);
  }
  static __device__ __forceinline__ int col(int q0, int g) {
    return q0 + 16 * (FQ * (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % WQ) + g);
  }
};

// Tile of workgroup `id` of np x nq tiles: each XCD (workgroups go round them) takes a contiguous run
// of tiles, and a run goes through bands of 8 P tiles, so that the 32 tiles of an XCD that run together
// share 8 tiles of P and 4 of Q in its L2.
struct MmaTileAt {
  int p, q;
};
__device__ __forceinline__ MmaTileAt mma_tile_at(int id, int np, int nq) {
  const int total = np * nq, x = id & 7, per = total >> 3, extra = total & 7;
  const int i = x * per + min(x, extra) + (id >> 3);
  const int band = i / (8 * nq), left = i - band * 8 * nq;
  const int wide = min(8, np - 8 * band);
  return {8 * band + left % wide, left / wide};
}

// Tile shapes, by the columns (tokens) there are: 256 rows by 256, 128, 64, 32 or 16. Narrow tiles read
// as many rows of P for fewer columns; they are taken where wide ones would compute columns that
// nobody asked for. f gets a MmaShape; its result is returned.
template <int FP, int FQ, int WP, int WQ>
struct MmaShape {
  static constexpr int fp = FP, fq = FQ, wp = WP, wq = WQ, bp = 16 * FP * WP, bq = 16 * FQ * WQ, threads = 64 * WP * WQ;
};
template <class F>
hipError_t with_mma_shape(long cols, F f) {
  if (cols > 128) return f(MmaShape<8, 4, 2, 4>{});
  if (cols > 64) return f(MmaShape<4, 4, 4, 2>{});
  if (cols > 32) return f(MmaShape<4, 2, 4, 2>{});
  if (cols > 16) return f(MmaShape<2, 2, 8, 1>{});
  return f(MmaShape<2, 1, 8, 1>{});
}

}  // namespace cdclq
