// Many tokens through a packed projection with low-rank adapters beside it, and the gradient.
//
//   y_t = W x_t + s_q B_q low_t, low_t = A_q x_t          q = request of token t (-1: none)
//   u_t = s_q B_q^T dy_t     dx_t = W^T dy_t + A_q^T u_t
//   dA_q = sum_t u_t x^_t^T  dB_q = s_q sum_t dy_t low_t^T     (x^: the 8-bit checkpoint of x)
//
// W is expanded to 16 bits in the caller's workspace and multiplied by the tiles of mma16.h; it is
// bound by those products. The low-rank terms ride along: `shrink` makes low (or u) with the rank as the
// MFMA rows, and the product's epilogue adds B low (A^T u) to its own registers. Tokens keep their order:
// a fragment of 16 tokens goes through the distinct adapters among them, one in all but the fragments
// where requests meet, and a token takes only its own adapter's result, so that what another adapter
// holds cannot reach it. low and u enter the matrix cores as the sum of two 16-bit values of a vector
// scaled to [0.5, 1): about 16 bits of it are kept.
//
// dA and dB sum over the tokens of an adapter: lists in token order, items of at most `chunk` tokens with
// f32 sums of their own, joined in order (no atomics). dA reads the codes of the checkpoint, exact in
// bf16, the scale of token and block going into u.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cdclq.h"
#include "kernels.h"
#include "packed.h"

namespace cdclq {
namespace {

inline size_t up(size_t x, size_t to) { return (x + to - 1) / to * to; }
inline int blocks_for(long items, int per, int most = 1 << 20) {
  return (int)std::max(1l, std::min((items + per - 1) / per, (long)most));
}

// 16-bit rows of `cols` elements into rows of dp, zeros past cols
__global__ __launch_bounds__(256) void k_pad_rows16(const uint16_t* __restrict__ src, long ld, int cols, int dp,
                                                    long rows, uint16_t* __restrict__ dst) {
  const long total = rows * dp;
  for (long i = blockIdx.x * 256l + threadIdx.x; i < total; i += gridDim.x * 256l) {
    const long r = i / dp;
    const int c = (int)(i - r * dp);
    dst[i] = c < cols ? src[r * ld + c] : (uint16_t)0;
  }
}

// Activations into slot order, zeros in empty slots: R rows at a time through LDS (LDS = 0: straight from
// memory, rows too long for it).
template <int R>
__global__ __launch_bounds__(256) void k_to_slots(PackedView v, const uint16_t* __restrict__ x, long ldx, long t,
                                                  uint16_t* __restrict__ xp, int vec) {
  extern __shared__ __align__(16) uint16_t rows[];
  const long t0 = (long)blockIdx.x * (R ? R : 1);
  const int ns = packed_slots(v), stride = (int)((v.n + 7) & ~7);
  if constexpr (R > 0) {
    for (int r = 0; r < R && t0 + r < t; ++r) {
      const uint16_t* src = x + (t0 + r) * ldx;
      if (vec) {
        for (int c = 8 * threadIdx.x; c < v.n; c += 2048)
          *reinterpret_cast<uint4*>(rows + r * stride + c) = *reinterpret_cast<const uint4*>(src + c);
      } else {
        for (int c = threadIdx.x; c < v.n; c += 256) rows[r * stride + c] = src[c];
      }
    }
    __syncthreads();
  }
  for (int s = 8 * threadIdx.x; s < ns; s += 2048) {
    const int4 c0 = *reinterpret_cast<const int4*>(v.col + s), c1 = *reinterpret_cast<const int4*>(v.col + s + 4);
    const int c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    for (int r = 0; r < (R ? R : 1) && t0 + r < t; ++r) {
      const uint16_t* src = R ? rows + r * stride : x + (t0 + r) * ldx;
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = (c[2 * i] >= 0 ? src[c[2 * i]] : 0u) | ((c[2 * i + 1] >= 0 ? (uint32_t)src[c[2 * i + 1]] : 0u) << 16);
      *reinterpret_cast<uint4*>(xp + (t0 + r) * ns + s) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}
// ... and back to columns
template <int R>
__global__ __launch_bounds__(256) void k_from_slots(PackedView v, const uint16_t* __restrict__ xp, long t,
                                                    uint16_t* __restrict__ x, long ldx, int vec) {
  extern __shared__ __align__(16) uint16_t rows[];
  const long t0 = (long)blockIdx.x * (R ? R : 1);
  const int ns = packed_slots(v), stride = (int)((v.n + 7) & ~7);
  for (int s = 8 * threadIdx.x; s < ns; s += 2048) {
    const int4 c0 = *reinterpret_cast<const int4*>(v.col + s), c1 = *reinterpret_cast<const int4*>(v.col + s + 4);
    const int c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    for (int r = 0; r < (R ? R : 1) && t0 + r < t; ++r) {
      uint16_t in[8];
      *reinterpret_cast<uint4*>(in) = *reinterpret_cast<const uint4*>(xp + (t0 + r) * ns + s);
      uint16_t* dst = R ? rows + r * stride : x + (t0 + r) * ldx;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c[i] >= 0) dst[c[i]] = in[i];
    }
  }
  if constexpr (R > 0) {
    __syncthreads();
    for (int r = 0; r < R && t0 + r < t; ++r) {
      uint16_t* dst = x + (t0 + r) * ldx;
      if (vec) {
        for (int c = 8 * threadIdx.x; c < v.n; c += 2048)
          *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(rows + r * stride + c);
      } else {
        for (int c = threadIdx.x; c < v.n; c += 256) dst[c] = rows[r * stride + c];
      }
    }
  }
}

// bt[adapter][j][i] = b[adapter][i][j], rows padded to mp with zeros
__global__ __launch_bounds__(256) void k_transpose_b(const uint16_t* __restrict__ b, int adapters, int m, int rank,
                                                     int mp, uint16_t* __restrict__ bt) {
  const long total = (long)adapters * mp;
  for (long e = blockIdx.x * 256l + threadIdx.x; e < total; e += gridDim.x * 256l) {
    const long q = e / mp;
    const int i = (int)(e - q * mp);
    const uint16_t* src = b + (q * m + i) * rank;
    uint16_t* dst = bt + q * rank * mp + i;
    for (int j = 0; j < rank; ++j) dst[(long)j * mp] = i < m ? src[j] : (uint16_t)0;
  }
}
// at[adapter][slot][j] = a[adapter][j][column of slot], zeros in empty slots and past the rank
__global__ __launch_bounds__(256) void k_transpose_a(PackedView v, const uint16_t* __restrict__ a, int adapters,
                                                     int rank, int rp, uint16_t* __restrict__ at) {
  const int ns = packed_slots(v);
  const long total = (long)adapters * ns;
  for (long e = blockIdx.x * 256l + threadIdx.x; e < total; e += gridDim.x * 256l) {
    const long q = e / ns;
    const int c = v.col[e - q * ns];
    const uint16_t* src = a + q * rank * v.n + c;
    for (int j = 0; j < rp; j += 8) {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = c >= 0 && j + 2 * i < rank ? src[(long)(j + 2 * i) * v.n] : 0u;
        const uint32_t hi = c >= 0 && j + 2 * i + 1 < rank ? src[(long)(j + 2 * i + 1) * v.n] : 0u;
        o[i] = lo | (hi << 16);
      }
      *reinterpret_cast<uint4*>(at + e * rp + j) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// The next adapter of a fragment's tokens that is not done yet (-1: none left). q: lane's token's adapter
// or -1; `left`: lanes still waiting.
__device__ __forceinline__ int next_adapter(int q, uint64_t& left) {
  if (!left) return -1;
  const int a = __builtin_amdgcn_readlane(q, __builtin_ctzll(left));
  left &= ~__builtin_amdgcn_ballot_w64(q == a);
  return a;
}

// low[t][j] = sum_k a[q][j][k] x[t][k] for 16 tokens a workgroup, the 8 wavefronts taking every 8th step
// of k; out (t x rank) = low, or scaling low with `scaled`; hl[t][2 rp]: low / 2^e as two 16-bit values,
// hscale[t] = scaling 2^e.
template <class T, int RF>
__global__ __launch_bounds__(512) void k_shrink(const uint16_t* __restrict__ x, long ldx, int t, int kk,
                                                const uint16_t* __restrict__ a, long lda, int rank, int rp,
                                                int adapters, const int* __restrict__ request,
                                                const float* __restrict__ scaling, int scaled, float* __restrict__ out,
                                                uint16_t* __restrict__ hl, float* __restrict__ hscale) {
  typedef typename T::v8 v8;
  __shared__ float red[8][16][RF * 16 + 1];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quad = lane >> 4;
  const int tok = blockIdx.x * 16 + (lane & 15);
  int q = tok < t ? request[tok] : -1;
  if (q >= adapters) q = -1;
  mma_f4 keep[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) keep[f] = mma_f4{};
  uint64_t left = __builtin_amdgcn_ballot_w64(q >= 0);
  const uint16_t* xr = x + (long)min(tok, t - 1) * ldx;
  for (int ad = next_adapter(q, left); ad >= 0; ad = next_adapter(q, left)) {
    const uint16_t* ar[RF];
    mma_f4 acc[RF];
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      ar[f] = a + ((long)ad * rank + min(16 * f + (lane & 15), rank - 1)) * lda;
      acc[f] = mma_f4{};
    }
    for (int k0 = 32 * wv; k0 < kk; k0 += 256) {
      const int k = k0 + 8 * quad;
      mma_u4 xv = {}, av[RF] = {};
      if (k < kk) {
        xv = *reinterpret_cast<const mma_u4*>(xr + k);
#pragma unroll
        for (int f = 0; f < RF; ++f) av[f] = *reinterpret_cast<const mma_u4*>(ar[f] + k);
      }
#pragma unroll
      for (int f = 0; f < RF; ++f) acc[f] = T::mfma(__builtin_bit_cast(v8, av[f]), __builtin_bit_cast(v8, xv), acc[f]);
    }
#pragma unroll
    for (int f = 0; f < RF; ++f)
      if (q == ad) keep[f] = acc[f];
  }
#pragma unroll
  for (int f = 0; f < RF; ++f)
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wv][lane & 15][16 * f + 4 * quad + r] = keep[f][r];
  __syncthreads();
  // 32 threads a token
  const int it = threadIdx.x >> 5, jt = threadIdx.x & 31, ot = blockIdx.x * 16 + it;
  float v[(RF + 1) / 2], m = 0.0f;
#pragma unroll
  for (int i = 0; i < (RF + 1) / 2; ++i) {
    const int j = jt + 32 * i;
    v[i] = 0.0f;
    if (j < rank)
      for (int w = 0; w < 8; ++w) v[i] += red[w][it][j];
    m = fmaxf(m, __builtin_fabsf(v[i]));
  }
#pragma unroll
  for (int s = 16; s; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
  if (ot >= t) return;
  const int rq = request[ot];
  const float sc = rq >= 0 && rq < adapters ? scaling[rq] : 0.0f;
  const int e = m > 0.0f && m < __builtin_inff() ? __builtin_amdgcn_frexp_expf(m) : 0;
  if (jt == 0 && hscale) hscale[ot] = ldexpf(sc, e);
#pragma unroll
  for (int i = 0; i < (RF + 1) / 2; ++i) {
    const int j = jt + 32 * i;
    if (j < rank && out) out[(long)ot * rank + j] = scaled ? sc * v[i] : v[i];
    if (j < rp && hl) {
      const float y = ldexpf(v[i], -e);
      const uint16_t hi = T::narrow(y);
      hl[(long)ot * 2 * rp + j] = hi;
      hl[(long)ot * 2 * rp + rp + j] = T::narrow(y - T::widen(hi));
    }
  }
}

struct WideArgs {
  const uint16_t* w;  // expanded weights, [rows of the layer][slots]
  long ldw;
  int rows, k;        // result rows (layer rows, or slots), length of the sums
  const uint16_t* x;  // t x k
  long ldx;
  int t, np, nq;
  const uint16_t* e;  // adapters x rows x rp, null: no adapters
  int rp, adapters;
  const uint16_t* hl;
  const float* hscale;
  const int* request;
  uint16_t* out;  // t x rows
  long ldo;
  int vec;
};

// out[t][i] = sum_k W(i, k) x[t][k] + hscale_t sum_j e[q][i][j] (hl[t][j] + hl[t][rp + j])
template <class T, bool PS, int FP, int FQ, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ, 2) void k_wide(WideArgs a) {
  typedef MmaTile<T, PS, false, FP, FQ, WP, WQ> M;
  typedef typename T::v8 v8;
  __shared__ __align__(1024) uint8_t lds[M::LDS];
  const MmaTileAt at = mma_tile_at(blockIdx.x, a.np, a.nq);
  const int p0 = at.p * M::BP, q0 = at.q * M::BQ;
  mma_f4 acc[FP][FQ];
  M::clear(acc);
  M::run(lds_offset(lds), MmaOp{a.w, a.ldw, a.rows}, MmaOp{a.x, a.ldx, a.t}, p0, q0, 0, a.k, acc);
  const int lane = threadIdx.x & 63, quad = lane >> 4;
#pragma unroll
  for (int g = 0; g < FQ; ++g) {
    const int t = M::col(q0, g) + (lane & 15);
    if (a.e) {
      const int q = t < a.t ? a.request[t] : -1;
      const bool known = q >= 0 && q < a.adapters;
      const float scale = known ? a.hscale[t] : 0.0f;
      uint64_t left = __builtin_amdgcn_ballot_w64(known);
      for (int ad = next_adapter(q, left); ad >= 0; ad = next_adapter(q, left)) {
        mma_f4 d[FP];
#pragma unroll
        for (int f = 0; f < FP; ++f) d[f] = mma_f4{};
        for (int kf = 0; kf < 2 * a.rp; kf += 32) {
          const int k = kf + 8 * quad, c = k < a.rp ? k : k - a.rp;
          const v8 h = __builtin_bit_cast(
              v8, *reinterpret_cast<const mma_u4*>(a.hl + (long)min(t, a.t - 1) * 2 * a.rp + k));
#pragma unroll
          for (int f = 0; f < FP; ++f) {
            const int row = min(M::row(p0, f) + (lane & 15), a.rows - 1);
            const v8 e = __builtin_bit_cast(
                v8, *reinterpret_cast<const mma_u4*>(a.e + ((long)ad * a.rows + row) * a.rp + c));
            d[f] = T::mfma(e, h, d[f]);
          }
        }
#pragma unroll
        for (int f = 0; f < FP; ++f)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (q == ad) acc[f][g][r] = __builtin_fmaf(scale, d[f][r], acc[f][g][r]);
      }
      if (!known && q != -1) {  // no such adapter
#pragma unroll
        for (int f = 0; f < FP; ++f)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[f][g][r] = __builtin_nanf("");
      }
    }
    if (t >= a.t) continue;
#pragma unroll
    for (int f = 0; f < FP; ++f) {
      const int row = M::row(p0, f) + 4 * quad;
      uint16_t* o = a.out + (long)t * a.ldo + row;
      const mma_f4 c = acc[f][g];
      if (a.vec && row + 3 < a.rows) {
        *reinterpret_cast<uint2*>(o) = make_uint2(narrow2<T>(c[0], c[1]), narrow2<T>(c[2], c[3]));
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (row + r < a.rows) o[r] = T::narrow(c[r]);
      }
    }
  }
}

// Tokens of adapter blockIdx.x in order, list[start ..], and its items of at most `chunk` tokens. An
// adapter's items begin at slot start / chunk + adapter, which leaves room for all of them and at most
// one more, marked empty. first[q], count[q]: its items.
__global__ __launch_bounds__(1024) void k_adapter_lists(const int* __restrict__ request, int t, int adapters,
                                                        int chunk, int slots, int* __restrict__ list,
                                                        int4* __restrict__ items, int2* __restrict__ of) {
  __shared__ int wsum[16], below, total;
  const int q = blockIdx.x, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  if (threadIdx.x == 0) below = total = 0;
  __syncthreads();
  int b = 0;
  for (int i = threadIdx.x; i < t; i += 1024) {
    const int r = request[i];
    b += r >= 0 && r < q;
  }
  for (int s = 32; s; s >>= 1) b += __shfl_xor(b, s);
  if (lane == 0) atomicAdd(&below, b);  // a sum of counts: the order does not matter
  __syncthreads();
  const int start = below;
  for (int t0 = 0; t0 < t; t0 += 1024) {
    const int i = t0 + threadIdx.x;
    const bool on = i < t && request[i] == q;
    const uint64_t m = __builtin_amdgcn_ballot_w64(on);
    if (lane == 0) wsum[wv] = __popcll(m);
    __syncthreads();
    int at = start + total + __popcll(m & ((1ull << lane) - 1));
    for (int w = 0; w < wv; ++w) at += wsum[w];
    if (on) list[at] = i;
    __syncthreads();
    if (threadIdx.x == 0)
      for (int w = 0; w < 16; ++w) total += wsum[w];
    __syncthreads();
  }
  const int n = total, first = start / chunk + q;
  const int end = q + 1 < adapters ? (start + n) / chunk + q + 1 : slots;
  for (int s = first + threadIdx.x; s < end; s += 1024) {
    const int at = (s - first) * chunk;
    items[s] = at < n ? make_int4(q, start + at, min(chunk, n - at), 0) : make_int4(-1, 0, 0, 0);
  }
  if (threadIdx.x == 0) of[q] = make_int2(first, (n + chunk - 1) / chunk);
}

// part[slot][j][c] = sum over the item's tokens of l[t][j] X[t][c], j in 16 RF ranks from j0, c in 128
// columns a wavefront. X: 8-bit codes with their scales (I8), or 16-bit values; l times scaling[q] if given.
// A lane reads 8 neighbouring columns of 8 tokens: row i of the f-th MFMA operand is column 8 i + f.
template <class T, bool I8, int RF>
__global__ __launch_bounds__(256) void k_outer(const void* __restrict__ xs, const float* __restrict__ xscale, long ldx,
                                               int cols, const float* __restrict__ l, int rank, int rp,
                                               const float* __restrict__ scaling, const int* __restrict__ list,
                                               const int4* __restrict__ items, float* __restrict__ part, int vec) {
  typedef typename T::v8 v8;
  const int4 it = items[blockIdx.y];
  if (it.x < 0) return;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, quad = lane >> 4;
  const int c0 = (blockIdx.x * 4 + wv) * 128, j0 = blockIdx.z * 16 * RF;
  if (c0 >= cols) return;
  const int c = c0 + 8 * (lane & 15), nb = (cols + 127) / 128;
  const float mul = scaling ? scaling[it.x] : 1.0f;
  mma_f4 acc[8][RF];
#pragma unroll
  for (int f = 0; f < 8; ++f)
#pragma unroll
    for (int g = 0; g < RF; ++g) acc[f][g] = mma_f4{};
  for (int t0 = 0; t0 < it.z; t0 += 32) {
    int tok[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) tok[i] = list[it.y + min(t0 + 8 * quad + i, it.z - 1)];
    uint32_t xv[8][4];  // operand f, pairs of tokens
    if constexpr (I8) {
      uint2 raw[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int8_t* src = static_cast<const int8_t*>(xs) + (long)tok[i] * ldx + c;
        raw[i] = make_uint2(0, 0);
        if (vec) {
          if (c < cols) raw[i] = *reinterpret_cast<const uint2*>(src);
        } else {
          uint8_t v[8];
#pragma unroll
          for (int b = 0; b < 8; ++b) v[b] = c + b < cols ? (uint8_t)src[b] : (uint8_t)0;
          raw[i] = *reinterpret_cast<uint2*>(v);
        }
      }
#pragma unroll
      for (int f = 0; f < 8; ++f)
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const uint32_t a = f < 4 ? raw[2 * p].x : raw[2 * p].y, b = f < 4 ? raw[2 * p + 1].x : raw[2 * p + 1].y;
          xv[f][p] = narrow2<T>((float)(int8_t)(a >> (8 * (f & 3))), (float)(int8_t)(b >> (8 * (f & 3))));
        }
    } else {
      mma_u4 raw[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        raw[i] = mma_u4{};
        if (c < cols) raw[i] = *reinterpret_cast<const mma_u4*>(static_cast<const uint16_t*>(xs) + (long)tok[i] * ldx + c);
      }
#pragma unroll
      for (int f = 0; f < 8; ++f)
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const uint32_t a = raw[2 * p][f >> 1], b = raw[2 * p + 1][f >> 1];
          xv[f][p] = __builtin_amdgcn_perm(b, a, f & 1 ? 0x07060302u : 0x05040100u);
        }
    }
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i] = t0 + 8 * quad + i < it.z ? mul : 0.0f;
      if constexpr (I8) s[i] *= xscale[(long)tok[i] * nb + c0 / 128];
    }
#pragma unroll
    for (int g = 0; g < RF; ++g) {
      const int j = j0 + 16 * g + (lane & 15);
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        float y[2];
        uint16_t h[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          y[i] = j < rank ? s[2 * p + i] * l[(long)tok[2 * p + i] * rank + j] : 0.0f;
          h[i] = T::narrow(y[i]);
        }
        hi[p] = (uint32_t)h[0] | ((uint32_t)h[1] << 16);
        lo[p] = narrow2<T>(y[0] - T::widen(h[0]), y[1] - T::widen(h[1]));
      }
      const v8 vh = __builtin_bit_cast(v8, mma_u4{hi[0], hi[1], hi[2], hi[3]});
      const v8 vl = __builtin_bit_cast(v8, mma_u4{lo[0], lo[1], lo[2], lo[3]});
#pragma unroll
      for (int f = 0; f < 8; ++f) {
        const v8 x = __builtin_bit_cast(v8, mma_u4{xv[f][0], xv[f][1], xv[f][2], xv[f][3]});
        acc[f][g] = T::mfma(x, vh, acc[f][g]);
        acc[f][g] = T::mfma(x, vl, acc[f][g]);
      }
    }
  }
  const long ldp = (long)nb * 128;
#pragma unroll
  for (int g = 0; g < RF; ++g) {
    const int j = j0 + 16 * g + (lane & 15);
    if (j >= rp) continue;
    float* o = part + ((long)blockIdx.y * rp + j) * ldp + c0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 8 * (4 * quad + r);
      *reinterpret_cast<mma_f4*>(o + i) = mma_f4{acc[0][g][r], acc[1][g][r], acc[2][g][r], acc[3][g][r]};
      *reinterpret_cast<mma_f4*>(o + i + 4) = mma_f4{acc[4][g][r], acc[5][g][r], acc[6][g][r], acc[7][g][r]};
    }
  }
}

// Sums of an adapter's items in order, rounded once: da[q][j][c], or with ROWS db[q][c][j].
template <class T, bool ROWS>
__global__ __launch_bounds__(256) void k_outer_join(const float* __restrict__ part, const int2* __restrict__ of,
                                                    int rank, int rp, int cols, long ldp, uint16_t* __restrict__ out) {
  const int q = blockIdx.z, c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  const int2 f = of[q];
  for (int j = blockIdx.y; j < rank; j += gridDim.y) {
    float s = 0.0f;
    for (int i = 0; i < f.y; ++i) s += part[((long)(f.x + i) * rp + j) * ldp + c];
    out[ROWS ? ((long)q * cols + c) * rank + j : ((long)q * rank + j) * cols + c] = T::narrow(s);
  }
}

struct Arena {
  char* base;
  size_t at = 0;
  explicit Arena(void* p) : base(static_cast<char*>(p)) {}
  template <class X>
  X* take(size_t count) {
    X* p = reinterpret_cast<X*>(base + at);
    at += up(count * sizeof(X), 256);
    return p;
  }
};

inline bool aligned16(const void* p, long ld, long cols) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && cols % 8 == 0; }
inline int rank_pad(int rank) { return (int)up(rank, 16); }

hipError_t to_slots(hipStream_t st, const PackedView& v, const uint16_t* x, long ldx, long t, uint16_t* xp) {
  const int vec = aligned16(x, ldx, v.n);
  const size_t row = 2 * up(v.n, 8);
  if (row * 4 <= 65536) k_to_slots<4><<<(int)((t + 3) / 4), 256, 4 * row, st>>>(v, x, ldx, t, xp, vec);
  else if (row <= 65536) k_to_slots<1><<<(int)t, 256, row, st>>>(v, x, ldx, t, xp, vec);
  else k_to_slots<0><<<(int)t, 256, 0, st>>>(v, x, ldx, t, xp, vec);
  return hipGetLastError();
}
hipError_t from_slots(hipStream_t st, const PackedView& v, const uint16_t* xp, long t, uint16_t* x, long ldx) {
  const int vec = aligned16(x, ldx, v.n);
  const size_t row = 2 * up(v.n, 8);
  if (row * 4 <= 65536) k_from_slots<4><<<(int)((t + 3) / 4), 256, 4 * row, st>>>(v, xp, t, x, ldx, vec);
  else if (row <= 65536) k_from_slots<1><<<(int)t, 256, row, st>>>(v, xp, t, x, ldx, vec);
  else k_from_slots<0><<<(int)t, 256, 0, st>>>(v, xp, t, x, ldx, vec);
  return hipGetLastError();
}
hipError_t pad_rows16(hipStream_t st, const uint16_t* src, long ld, long cols, long dp, long rows, uint16_t* dst) {
  k_pad_rows16<<<blocks_for(rows * dp, 256 * 8), 256, 0, st>>>(src, ld, (int)cols, (int)dp, rows, dst);
  return hipGetLastError();
}

template <class T>
hipError_t shrink(hipStream_t st, const uint16_t* x, long ldx, long t, int k, const uint16_t* a, long lda,
                  const AdapterArgs& g, int scaled, float* out, uint16_t* hl, float* hscale) {
  const int grid = (int)((t + 15) / 16), rp = rank_pad(g.rank);
  auto go = [&](auto rf) {
    k_shrink<T, decltype(rf)::value><<<grid, 512, 0, st>>>(x, ldx, (int)t, k, a, lda, g.rank, rp, g.adapters, g.request,
                                                           g.scaling, scaled, out, hl, hscale);
    return hipGetLastError();
  };
  if (rp <= 16) return go(std::integral_constant<int, 1>{});
  if (rp <= 32) return go(std::integral_constant<int, 2>{});
  if (rp <= 64) return go(std::integral_constant<int, 4>{});
  return go(std::integral_constant<int, 8>{});
}

template <class T, bool PS>
hipError_t wide_product(hipStream_t st, WideArgs w) {
  w.vec = w.ldo % 4 == 0 && (uintptr_t)w.out % 8 == 0;
  return with_mma_shape(mma_pick(w.rows, w.t, w.k), [&](auto s) {
    typedef decltype(s) S;
    w.np = (w.rows + S::bp - 1) / S::bp;
    w.nq = (w.t + S::bq - 1) / S::bq;
    k_wide<T, PS, S::fp, S::fq, S::wp, S::wq><<<w.np * w.nq, S::threads, 0, st>>>(w);
    return hipGetLastError();
  });
}

#define STEP(expr)                       \
  do {                                   \
    hipError_t e_ = (expr);              \
    if (e_ != hipSuccess) return e_;     \
  } while (0)

// The workspace's parts are laid out by the same code that runs the steps: with `run` false only the
// size is taken.
template <class T>
hipError_t wide(hipStream_t st, const PackedView& v, const AdapterArgs& a, void* work, bool run, size_t* bytes) {
  const int ns = packed_slots(v), rp = rank_pad(a.rank), n8 = (int)up(v.n, 8);
  const bool low = a.rank > 0;
  const bool pad_x = low && !aligned16(a.x, a.ldx, v.n), pad_a = low && !aligned16(a.a, v.n, v.n);
  const bool pad_b = low && (rp != a.rank || (uintptr_t)a.b % 16);
  Arena m(work);
  uint16_t* w16 = m.take<uint16_t>((size_t)v.tiles * 16 * ns);
  uint16_t* xp = m.take<uint16_t>((size_t)a.t * ns);
  uint16_t* xpad = m.take<uint16_t>(pad_x ? (size_t)a.t * n8 : 0);
  uint16_t* apad = m.take<uint16_t>(pad_a ? (size_t)a.adapters * a.rank * n8 : 0);
  uint16_t* bpad = m.take<uint16_t>(pad_b ? (size_t)a.adapters * v.m * rp : 0);
  uint16_t* hl = m.take<uint16_t>(low ? (size_t)a.t * 2 * rp : 0);
  float* hscale = m.take<float>(low ? a.t : 0);
  *bytes = m.at;
  if (!run) return hipSuccess;
  const int dtype = T::kind;
  STEP(packed_expand(st, dtype, v, w16));
  STEP(to_slots(st, v, a.x, a.ldx, a.t, xp));
  WideArgs w = {};
  if (low) {
    const uint16_t *x = a.x, *aa = a.a, *bb = a.b;
    long ldx = a.ldx, lda = v.n;
    if (pad_x) {
      STEP(pad_rows16(st, a.x, a.ldx, v.n, n8, a.t, xpad));
      x = xpad, ldx = n8;
    }
    if (pad_a) {
      STEP(pad_rows16(st, a.a, v.n, v.n, n8, (long)a.adapters * a.rank, apad));
      aa = apad, lda = n8;
    }
    if (pad_b) {
      STEP(pad_rows16(st, a.b, a.rank, a.rank, rp, (long)a.adapters * v.m, bpad));
      bb = bpad;
    }
    STEP(shrink<T>(st, x, ldx, a.t, n8, aa, lda, a, 0, a.low, hl, hscale));
    w.e = bb;
    w.rp = rp;
    w.adapters = a.adapters;
    w.hl = hl;
    w.hscale = hscale;
    w.request = a.request;
  }
  w.w = w16, w.ldw = ns, w.rows = v.m, w.k = ns;
  w.x = xp, w.ldx = ns, w.t = (int)a.t;
  w.out = a.y, w.ldo = a.ldy;
  return wide_product<T, false>(st, w);
}

template <class T, bool I8>
hipError_t outer(hipStream_t st, const void* x, const float* xscale, long ldx, int cols, const float* l,
                 const AdapterArgs& a, const float* scaling, const int* list, const int4* items, int slots,
                 const int2* of, float* part, int vec, uint16_t* out) {
  const int rp = rank_pad(a.rank), nb = (cols + 127) / 128;
  auto go = [&](auto rf) {
    constexpr int RF = decltype(rf)::value;
    k_outer<std::conditional_t<I8, Bf16, T>, I8, RF><<<dim3((nb + 3) / 4, slots, (rp + 16 * RF - 1) / (16 * RF)), 256, 0, st>>>(
        x, xscale, ldx, cols, l, a.rank, rp, scaling, list, items, part, vec);
    return hipGetLastError();
  };
  if (rp <= 16) STEP(go(std::integral_constant<int, 1>{}));
  else if (rp <= 32) STEP(go(std::integral_constant<int, 2>{}));
  else STEP(go(std::integral_constant<int, 4>{}));
  k_outer_join<T, !I8><<<dim3((cols + 255) / 256, std::min(a.rank, 64), a.adapters), 256, 0, st>>>(part, of, a.rank, rp, cols,
                                                                                       128l * nb, out);
  return hipGetLastError();
}

template <class T>
hipError_t grad(hipStream_t st, const PackedView& v, const AdapterArgs& a, void* work, bool run, size_t* bytes) {
  const int ns = packed_slots(v), rp = rank_pad(a.rank), m8 = (int)up(v.m, 8);
  const bool low = a.rank > 0, pad = !aligned16(a.x, a.ldx, v.m);
  const long widest = std::max(up(v.n, 128), up(v.m, 128));
  // items: enough of them that, with 128 columns a wavefront, the smaller side fills the GPU
  const long narrow = std::min(up(v.n, 128), up(v.m, 128)) / 128;
  const int chunk = (int)std::clamp<long>(up(a.t * narrow / 2048, 32), 256, 1024);
  const int slots = (int)(a.t / chunk) + a.adapters;
  Arena m(work);
  uint16_t* w16 = m.take<uint16_t>((size_t)v.tiles * 16 * ns);
  uint16_t* dxp = m.take<uint16_t>((size_t)a.t * ns);
  uint16_t* dyp = m.take<uint16_t>(pad ? (size_t)a.t * m8 : 0);
  uint16_t* bt = m.take<uint16_t>(low ? (size_t)a.adapters * a.rank * m8 : 0);
  uint16_t* at = m.take<uint16_t>(low ? (size_t)a.adapters * ns * rp : 0);
  float* u = m.take<float>(low ? (size_t)a.t * a.rank : 0);
  uint16_t* hl = m.take<uint16_t>(low ? (size_t)a.t * 2 * rp : 0);
  float* hscale = m.take<float>(low ? a.t : 0);
  int* list = m.take<int>(low ? a.t : 0);
  int4* items = m.take<int4>(low ? slots : 0);
  int2* of = m.take<int2>(low ? a.adapters : 0);
  float* part = m.take<float>(low ? (size_t)slots * rp * widest : 0);
  *bytes = m.at;
  if (!run) return hipSuccess;
  const uint16_t* dy = a.x;
  long lddy = a.ldx;
  WideArgs w = {};
  if (a.t) {
    STEP(packed_expand(st, T::kind, v, w16));
    if (pad) {
      STEP(pad_rows16(st, a.x, a.ldx, v.m, m8, a.t, dyp));
      dy = dyp, lddy = m8;
    }
  }
  if (low) {
    if (a.t) {
      k_transpose_b<<<blocks_for((long)a.adapters * m8, 256), 256, 0, st>>>(a.b, a.adapters, v.m, a.rank, m8, bt);
      k_transpose_a<<<blocks_for((long)a.adapters * ns, 256), 256, 0, st>>>(v, a.a, a.adapters, a.rank, rp, at);
      STEP(shrink<T>(st, dy, lddy, a.t, m8, bt, m8, a, 1, u, hl, hscale));
    }
    k_adapter_lists<<<a.adapters, 1024, 0, st>>>(a.request, (int)a.t, a.adapters, chunk, slots, list, items, of);
    STEP(hipGetLastError());
    STEP((outer<T, true>(st, a.codes, a.scales, v.n, v.n, u, a, nullptr, list, items, slots, of, part,
                         v.n % 8 == 0 && (uintptr_t)a.codes % 8 == 0, a.da)));
    STEP((outer<T, false>(st, dy, nullptr, lddy, v.m, a.low, a, a.scaling, list, items, slots, of, part, 1, a.db)));
    w.e = at;
    w.rp = rp;
    w.adapters = a.adapters;
    w.hl = hl;
    w.hscale = hscale;
    w.request = a.request;
  }
  if (!a.t) return hipSuccess;
  w.w = w16, w.ldw = ns, w.rows = ns, w.k = v.m;
  w.x = dy, w.ldx = lddy, w.t = (int)a.t;
  w.out = dxp, w.ldo = ns;
  STEP((wide_product<T, true>(st, w)));
  return from_slots(st, v, dxp, a.t, a.y, a.ldy);
}

}  // namespace

size_t wide_work_bytes(const PackedView& v, const AdapterArgs& a) {
  size_t n = 0;
  (void)wide<Bf16>(nullptr, v, a, nullptr, false, &n);
  return n;
}
hipError_t adapter_wide(hipStream_t st, int dtype, const PackedView& v, const AdapterArgs& a, void* work) {
  size_t n;
  return dtype == CDCLQ_DTYPE_BF16 ? wide<Bf16>(st, v, a, work, true, &n) : wide<F16>(st, v, a, work, true, &n);
}
size_t grad_work_bytes(const PackedView& v, const AdapterArgs& a) {
  size_t n = 0;
  (void)grad<Bf16>(nullptr, v, a, nullptr, false, &n);
  return n;
}
hipError_t adapter_grad(hipStream_t st, int dtype, const PackedView& v, const AdapterArgs& a, void* work) {
  size_t n;
  return dtype == CDCLQ_DTYPE_BF16 ? grad<Bf16>(st, v, a, work, true, &n) : grad<F16>(st, v, a, work, true, &n);
}

}  // namespace cdclq
