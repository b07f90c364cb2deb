// Tiles of 16-bit matrix products (bf16 or f16 in, f32 sums) on the gfx950 matrix cores, shared by
// the vocabulary loss and the packed projection.
//
// C[i][j] = sum_k P(i, k) Q(j, k), i over BP rows of P, j over BQ rows of Q. An operand is stored
// either with k contiguous (rows x ld) or, PS / QS, with the rows contiguous (k x ld). A workgroup of
// WP x WQ wavefronts computes BP x BQ = 16 FP WP x 16 FQ WQ elements, a wavefront FP x FQ blocks of
// v_mfma_f32_16x16x32: lane l supplies rows l & 15 at k = 8 (l >> 4) .. + 7 of both operands, and
// register r of a result is row 4 (l >> 4) + r, column l & 15.
//
// Stages of 64 k (whole cache lines) are loaded straight into LDS, 16 bytes a lane, in two buffers. The
// operands of the next 32 k are read from LDS between the MFMAs of these: Q's into a second set of
// registers, P's each into its own place after its last use. A stage's buffer is therefore free half a
// stage before its products end, and the loads of the stage after the next go there: they have a whole
// stage's MFMAs to land. One barrier a stage.
// LDS holds an operand as 16-byte granules,
//   k contiguous:    granule g of row i at position g ^ (i >> 1 & 7) of the row's 8: the 16 rows that a
//                    16-byte read serves together then cover all the banks once;
//   rows contiguous: granule g of k-row k at position g ^ 2 s(k), s = (k & 3) + 4 (k >> 3 & 1), of
//                    the row's BP / 8: read by ds_read_b64_tr_b16, which hands lane i of 16 the
//                    column i of a 4 x 16 block, so that a block's rows start in 8 different places.
// What lies past the end of k is taken from a page of zeros, rows past the last one repeat it (their
// results are not used). Requirements, checked on the host: 16-byte aligned operands, ld a multiple of
// 8, and k (k contiguous) or the rows (rows contiguous) padded to a multiple of 8 within ld; with k
// contiguous the padding holds zeros.
//
// What bounds the largest tiles (256 x 256 by 8 wavefronts) is the card's power: 4096 x 128256 results over 4096
// at 1.30-1.33 PF, matrix cores busy 67% at 1.6-1.9 GHz (the library's product: 82% at 1.63 GHz, 1.34-1.40 PF). Loads
// given out at once after the barrier, not one by one between the products: 1.17 PF, busy 54%.
#pragma once

#include <algorithm>

#include "cdclq_dev.h"

namespace cdclq {

typedef short mma_s4 __attribute__((ext_vector_type(4)));
typedef uint16_t mma_us8 __attribute__((ext_vector_type(8)));
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

// By workgroups of 256 threads, b of nb: 16-bit rows of `cols` elements into rows of dp (a multiple of 8), zeros past cols
struct PadJob {
  const uint16_t* src;
  long ld;
  int cols, dp;
  long rows;
  uint16_t* dst;
};
__device__ inline void pad_rows16(const PadJob& j, long b, long nb) {
  const int per = j.dp / 8;
  const long total = j.rows * per;
  for (long i = b * 256 + threadIdx.x; i < total; i += nb * 256) {
    const long r = i / per;
    const int c = 8 * (int)(i - r * per);
    const uint16_t* src = j.src + r * j.ld + c;
    uint16_t v[8];
    if (c + 8 <= j.cols) {
      __builtin_memcpy(v, src, 16);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = c + k < j.cols ? src[k] : (uint16_t)0;
    }
    *reinterpret_cast<uint4*>(j.dst + r * j.dp + c) = *reinterpret_cast<const uint4*>(v);
  }
}

// An operand of C: `rows` rows of k values each, element (i, k) at p[i ld + k] or, rows contiguous, at
// p[k ld + i]. With a list (k contiguous only) row i is row list[i] of p.
struct MmaOp {
  const uint16_t* p;
  long ld;
  int rows;
  const int* list = nullptr;
};

static __device__ uint4 mma_zero_page[1];  // never written

// PU: P has any alignment and no padding (element-wise bounds); its granules go through registers instead of
// straight into LDS, for which there is room in narrow tiles only.
template <class T, bool PS, bool QS, int FP, int FQ, int WP, int WQ, bool PU = false>
struct MmaTile {
  static constexpr int W = WP * WQ, THREADS = 64 * W;
  static constexpr int BP = 16 * FP * WP, BQ = 16 * FQ * WQ, BK = 64;
  static constexpr int STAGE = (BP + BQ) * BK * 2;  // bytes of one stage
  static constexpr int LDS = 2 * STAGE;
  static constexpr int GP = BP / 8, GQ = BQ / 8;  // loads of 64 granules a stage
  static constexpr int NP = (GP + W - 1) / W, NQ = (GQ + W - 1) / W;  // ... of a wavefront, at most
  typedef typename T::v8 v8;
  static_assert(GP % W == 0, "every wavefront loads as much of P");
  static_assert(!PS || BP >= 128, "the transposed read's swizzle spans 8 pairs of granules");
  static_assert(!QS || BQ >= 128, "the transposed read's swizzle spans 8 pairs of granules");

  // Where granule slot `s` of a stage comes from: its offset in k, and its address at k = k0.
  template <bool S, int B>
  static __device__ __forceinline__ int granule_k(int s) {
    return S ? s / (B / 8) : 8 * ((s & 7) ^ ((s >> 4) & 7));
  }
  template <bool S, int B>
  static __device__ __forceinline__ const uint16_t* granule_at(const MmaOp& o, int r0, int k0, int s) {
    if constexpr (S) {
      const int k = s / (B / 8);
      const int g = (s % (B / 8)) ^ (2 * ((k & 3) | ((k >> 1) & 4)));
      return o.p + (long)(k0 + k) * o.ld + min(r0 + 8 * g, (o.rows - 1) & ~7);
    } else {
      int row = min(r0 + (s >> 3), o.rows - 1);
      if (o.list) row = o.list[row];
      return o.p + (long)row * o.ld + k0 + granule_k<S, B>(s);
    }
  }

  // first column of a granule of a stage with the rows contiguous
  static __device__ __forceinline__ int col_of(int s) {
    const int k = s / (BP / 8);
    return 8 * ((s % (BP / 8)) ^ (2 * ((k & 3) | ((k >> 1) & 4))));
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
    const int stages = max(2, (kend - kbeg + BK - 1) / BK);
    const uint16_t *pp[NP], *pq[NQ];
#pragma unroll
    for (int i = 0; i < NP; ++i) pp[i] = granule_at<PS, BP>(P, p0, kbeg, 64 * (wv + W * i) + lane);
#pragma unroll
    for (int i = 0; i < NQ; ++i) pq[i] = granule_at<QS, BQ>(Q, q0, kbeg, 64 * (wv + W * i) + lane);
    const long sp = PS ? BK * P.ld : BK, sq = QS ? BK * Q.ld : BK;
    uint4 held[PU ? NP : 1];  // PU: a stage's granules on their way
    const uint16_t* const zero = reinterpret_cast<const uint16_t*>(&mma_zero_page[0]);
    const bool has_q = GQ % W == 0 || wv < GQ % W;  // takes part in the last load of Q

    // The loads of the next stage to be loaded, one at a time: 0 .. NP - 1 of P, then Q's.
    const uint32_t to = lds + 1024u * wv;
    int kp = kbeg;  // PU: first k of the stage being loaded
    auto load = [&](uint32_t buf, int i) {
      if constexpr (PU) {
        if (i < NP) {
          const int slot = 64 * (wv + W * i) + lane, k = kp + granule_k<PS, BP>(slot);
          const int some = PS ? (k < kend ? P.rows - min(p0 + col_of(slot), (P.rows - 1) & ~7) : 0) : kend - k;
          uint16_t v[8];
          if (some >= 8) {
            __builtin_memcpy(v, pp[i], 16);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < some ? pp[i][e] : (uint16_t)0;
          }
          __builtin_memcpy(&held[i], v, 16);
          pp[i] += sp;
          if (i == NP - 1) kp += BK;
          return;
        }
      }
      if (i < NP) {
        dma16_untracked(reinterpret_cast<const float*>(pp[i]), to + buf + 1024u * W * i);
        pp[i] += sp;
      } else if (i < NP + NQ - 1 || has_q) {
        dma16_untracked(reinterpret_cast<const float*>(pq[i - NP]), to + buf + BP * BK * 2 + 1024u * W * (i - NP));
        pq[i - NP] += sq;
      }
    };
    // PU: the held granules into their places
    auto put = [&](uint32_t buf) {
      if constexpr (PU) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
          *(__attribute__((address_space(3))) mma_u4*)(uintptr_t)(to + buf + 1024u * W * i + 16 * lane) =
              mma_u4{held[i].x, held[i].y, held[i].z, held[i].w};
      }
    };
    // Before the loads of stage s: what lies past the end of k comes from the zeros.
    auto cut = [&](int s) {
      const int k0 = kbeg + s * BK;
      if (k0 + BK <= kend) return;
#pragma unroll
      for (int i = 0; i < (PU ? 0 : NP); ++i)
        if (k0 + granule_k<PS, BP>(64 * (wv + W * i) + lane) >= kend) pp[i] = zero;
#pragma unroll
      for (int i = 0; i < NQ; ++i)
        if (k0 + granule_k<QS, BQ>(64 * (wv + W * i) + lane) >= kend) pq[i] = zero;
    };
    auto issue = [&](int s) {
      cut(s);
#pragma unroll
      for (int i = 0; i < NP + NQ; ++i) load((uint32_t)(s & 1) * STAGE, i);
      put((uint32_t)(s & 1) * STAGE);
    };

    // read addresses within a stage
    const int r = lane & 15, q = lane >> 4;
    const uint32_t sw = ((lane >> 2) & 3) | ((q & 1) << 2);
    uint32_t ap[PS ? FP : 2], aq[QS ? FQ : 2];  // k contiguous: of the stage's halves
    if constexpr (PS) {
#pragma unroll
      for (int f = 0; f < FP; ++f)
        ap[f] = lds + (8 * q + (r >> 2)) * (BP * 2) + 32 * ((uint32_t)(FP * wp + f) ^ sw) + 8 * (lane & 3);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) ap[h] = lds + (16 * FP * wp + r) * 128 + 16 * ((4 * h + q) ^ (r >> 1));
    }
    if constexpr (QS) {
#pragma unroll
      for (int f = 0; f < FQ; ++f)
        aq[f] = lds + BP * BK * 2 + (8 * q + (r >> 2)) * (BQ * 2) + 32 * ((uint32_t)(FQ * wq + f) ^ sw) + 8 * (lane & 3);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        aq[h] = lds + BP * BK * 2 + (16 * FQ * wq + r) * 128 + 16 * ((4 * h + q) ^ (r >> 1));
    }
    // block f of half h of the stage in buffer `buf` (0 or STAGE)
    auto read_p = [&](uint32_t buf, int h, int f) {
      if constexpr (PS) return read_s<BP>(buf + ap[f] + 32 * h * BP * 2);
      else return read_c(buf + ap[h] + 2048 * f);
    };
    auto read_q = [&](uint32_t buf, int h, int f) {
      if constexpr (QS) return read_s<BQ>(buf + aq[f] + 32 * h * BQ * 2);
      else return read_c(buf + aq[h] + 2048 * f);
    };
    v8 a[FP], even[FQ], odd[FQ];
    // Products of 32 k while the operands of half h in `buf` are read; with LOAD the loads of a stage into
    // `into` go out between them (at once they would fill the memory pipe and hold up what follows).
    auto step = [&](uint32_t buf, int h, const v8(&cur)[FQ], v8(&next)[FQ], auto loads, uint32_t into) {
      constexpr bool LOAD = decltype(loads)::value;
      int n = 0;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int f = 0; f < FP; ++f) {
#pragma unroll
        for (int g = 0; g < FQ; ++g) {
          acc[f][g] = T::mfma(a[f], cur[g], acc[f][g]);
          if (f == 0) {
            next[g] = read_q(buf, h, g);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        a[f] = read_p(buf, h, f);
        if constexpr (LOAD) {
#pragma unroll
          for (; n < (NP + NQ) * (f + 1) / FP; ++n) load(into, n);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    constexpr std::true_type with_loads{};
    constexpr std::false_type no_loads{};
    issue(0);
    issue(1);
    if (PU) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    else if (has_q) wait_vmcnt<NP + NQ>();
    else wait_vmcnt<NP + NQ - 1>();
    asm volatile("s_barrier" ::: "memory");
#pragma unroll
    for (int g = 0; g < FQ; ++g) even[g] = read_q(0, 0, g);
#pragma unroll
    for (int f = 0; f < FP; ++f) a[f] = read_p(0, 0, f);
    // this wavefront is done reading a stage and its part of the next one has landed; the barrier says so
    // of every wavefront
    auto turn = [&]() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    uint32_t buf = 0;
    for (int s = 2; s < stages; ++s) {
      step(buf, 1, even, odd, no_loads, 0u);
      if (s > 2) put(buf ^ STAGE);  // stage s - 1, held since the last turn
      turn();
      cut(s);
      step(buf ^ STAGE, 0, odd, even, with_loads, buf);
      buf ^= STAGE;
    }
    step(buf, 1, even, odd, no_loads, 0u);
    if (stages > 2) put(buf ^ STAGE);
    turn();
    step(buf ^ STAGE, 0, odd, even, no_loads, 0u);
    step(buf ^ STAGE, 1, even, odd, no_loads, 0u);
#pragma unroll
    for (int f = 0; f < FP; ++f)
#pragma unroll
      for (int g = 0; g < FQ; ++g) acc[f][g] = T::mfma(a[f], odd[g], acc[f][g]);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the shared memory is free again
  }
  static __device__ __forceinline__ void clear(mma_f4 (&acc)[FP][FQ]) {
#pragma unroll
    for (int f = 0; f < FP; ++f)
#pragma unroll
      for (int g = 0; g < FQ; ++g) acc[f][g] = mma_f4{};
  }
  // out[j][i] = acc in 16 bits for the tile's columns j < qrows and rows i < prows (both counted in the
  // whole result), whole row pieces at a time: through LDS, 16-byte granule g of column j at g ^ (j & 15), so
  // that a wavefront's 16 columns write to different banks and 2 BP contiguous bytes go out together
  // (straight from the registers a column's 32 bytes do). All wavefronts call it together.
  static __device__ __forceinline__ void store(uint32_t lds, const mma_f4 (&acc)[FP][FQ], int p0, int q0, int prows,
                                               int qrows, uint16_t* out, long ld) {
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quad = lane >> 4;
    const int wp = wv / WQ, wq = wv % WQ;
    typedef const __attribute__((address_space(3))) mma_u4* lds16;
#pragma unroll
    for (int g = 0; g < FQ; ++g) {
      const int j = 16 * (FQ * wq + g) + (lane & 15);
#pragma unroll
      for (int f = 0; f < FP; ++f) {
        const mma_f4 c = acc[f][g];
        const int gran = 2 * (FP * wp + f) + (quad >> 1);
        const uint2 v = make_uint2(narrow2<T>(c[0], c[1]), narrow2<T>(c[2], c[3]));
        *(__attribute__((address_space(3))) uint64_t*)(uintptr_t)(lds + j * BP * 2 + 16 * (gran ^ (j & 15)) +
                                                                  8 * (quad & 1)) = (uint64_t)v.y << 32 | v.x;
      }
    }
    __syncthreads();
    constexpr int G = BP / 8;
#pragma unroll 4
    for (int e = threadIdx.x; e < BQ * G; e += THREADS) {
      const int j = e / G, g = e - j * G, i = p0 + 8 * g;
      if (q0 + j >= qrows || i >= prows) continue;
      const mma_u4 v = *(lds16)(uintptr_t)(lds + j * BP * 2 + 16 * (g ^ (j & 15)));
      uint16_t* o = out + (long)(q0 + j) * ld + i;
      if (i + 8 <= prows) {
        __builtin_memcpy(o, &v, 16);
      } else {
        for (int k = 0; k < 8 && i + k < prows; ++k) o[k] = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
      }
    }
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

// Tile shapes. f gets a MmaShape; its result is returned.
template <int FP, int FQ, int WP, int WQ>
struct MmaShape {
  static constexpr int fp = FP, fq = FQ, wp = WP, wq = WQ, bp = 16 * FP * WP, bq = 16 * FQ * WQ, threads = 64 * WP * WQ;
};

// The shapes, by number. Wide tiles read each operand less often; small ones spread few results over more
// CUs, narrow ones compute no columns that nobody asked for. `us`: a tile's stage of 64 k with every CU busy,
// measured on 4096 x 65536 results over k = 4096 (the narrow ones estimated); `per_cu`: the workgroups that
// a CU's LDS holds; `alone`: a stage with few tiles in flight, which the latency of its loads and reads sets,
// measured on 200 x 4096 results over 4096, and (P's rows contiguous) on 100 x 2688 over 6720.
// 256 x 192 beside 256 x 256: where the latter leave CUs idle (2000 x 5632 over 2048: 50 us, 59; but 4096 x 14336
// over 4096: 464, 450).
constexpr int kMmaShapes = 9;
struct MmaShapeTime {
  int bp, bq, per_cu;
  double us, alone, alone_strided;
};
constexpr MmaShapeTime kMmaTimes[kMmaShapes] = {
    {256, 256, 1, 1.66, 0.90, 1.15}, {256, 64, 2, 0.55, 0.51, 0.77},
    {256, 32, 2, 0.40, 0.50, 0.75},  {256, 16, 2, 0.33, 0.50, 0.70},  {128, 128, 2, 0.50, 0.49, 0.69},
    {128, 64, 3, 0.31, 0.43, 0.59},  {128, 32, 4, 0.22, 0.42, 0.55},  {128, 16, 4, 0.18, 0.42, 0.55},
    {256, 192, 1, 1.40, 0.78, 1.00}};
template <class F>
hipError_t with_mma_shape(int pick, F f) {
  switch (pick) {
    case 0: return f(MmaShape<8, 4, 2, 4>{});
    case 1: return f(MmaShape<4, 2, 4, 2>{});
    case 2: return f(MmaShape<2, 2, 8, 1>{});
    case 3: return f(MmaShape<2, 1, 8, 1>{});
    case 4: return f(MmaShape<4, 4, 2, 2>{});
    case 5: return f(MmaShape<4, 2, 2, 2>{});
    case 6: return f(MmaShape<2, 2, 4, 1>{});
    case 7: return f(MmaShape<2, 1, 4, 1>{});
    default: return f(MmaShape<8, 3, 2, 4>{});
  }
}
// Microseconds of a product of `rows` x `cols` results over k, `splits` ways in k: rounds of tiles over 256
// CUs, each so many stages and 4 us more for its first loads and its results. strided: P's rows contiguous
// (their transposed reads cost the smaller tiles a fifth). far: P comes from memory, not from a cache; a stage
// then takes 1 us at least (its loads go out one stage ahead; 218 x 13056 results over 12608).
inline double mma_cost(long rows, long cols, long k, int pick, long splits, bool strided, bool far = false) {
  const MmaShapeTime s = kMmaTimes[pick];
  const long tiles = ((rows + s.bp - 1) / s.bp) * ((cols + s.bq - 1) / s.bq) * splits;
  const long stages = std::max(2l, ((k + splits - 1) / splits + 63) / 64);
  const long rounds = (tiles + 256 * s.per_cu - 1) / (256 * s.per_cu);
  const long shared = std::min<long>(s.per_cu, (tiles + 255) / 256);
  const double busy = s.us * shared * (strided && pick ? 1.2 : 1.0);
  const double alone = std::max(strided ? s.alone_strided : s.alone, far ? 1.0 : 0.0);
  return rounds * (std::max(busy, alone) * stages + 4.0);
}

}  // namespace cdclq
