// Many tokens through a packed projection with low-rank adapters beside it, and the gradient.
//
//   y_t = W x_t + s_q B_q low_t, low_t = A_q x_t          q = request of token t (-1: none)
//   u_t = s_q B_q^T dy_t     dx_t = W^T dy_t + A_q^T u_t
//   dA_q = sum_t u_t x^_t^T  dB_q = s_q sum_t dy_t low_t^T     (x^: the 8-bit checkpoint of x)
//
// W is expanded to 16 bits in the caller's workspace and multiplied by the tiles of mma16.h; it is
// bound by those products, split in k where few tiles would leave CUs idle. The low-rank terms ride
// along: `shrink` makes low (or u) with the rank as the MFMA rows, and the product's epilogue adds B low
// (A^T u) to its own registers. Tokens keep their order: a fragment of 16 tokens goes through the distinct
// adapters among them, one in all but the fragments where requests meet, and a token takes only its own
// adapter's result, so that what another adapter holds cannot reach it. low and u enter the matrix cores as
// the sum of two 16-bit values of a vector scaled below 1 (by least_exp): about 16 bits of it are kept.
//
// 4096 tokens, 4096 -> 14336, 4 bits, rank 64, bf16: forward product 425-450 us (1.1 PF, 3.5 rounds of tiles), that
// of the gradient 340-356 (1.4 PF, one round), both bound by power where all CUs work; 2000 tokens, 2048 -> 5632:
// 50 us. Expanding the weights and ordering the activations: 41 us (gradient) and 56 (forward), memory at 3.6 TB/s.
//
// dA and dB sum over the tokens of an adapter: lists in token order, items of some hundred tokens with
// f32 sums of their own, joined in order (no atomics). dA reads the codes of the checkpoint, exact in
// bf16, the scale of token and block going into u.
//
// Everything that waits for nothing runs in one launch (`prepare`), every last step in another (`finish`):
// a small step is bound by launches.
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

// ---- parts of `prepare`, each by workgroups of 256 threads, b of nb

// Activations into slot order, zeros in empty slots: `rows` of them at a time through LDS (0: straight from
// memory, rows too long for it).
struct SlotJob {
  const uint16_t* x;
  long ldx;
  int t, rows, vec;
  uint16_t* xp;
};
__device__ void to_slots(const PackedView& v, const SlotJob& j, uint16_t* lds, long b) {
  const int n = j.rows ? j.rows : 1, ns = packed_slots(v), stride = (v.n + 7) & ~7;
  const long t0 = b * n;
  if (j.rows) {
    for (int r = 0; r < n && t0 + r < j.t; ++r) {
      const uint16_t* src = j.x + (t0 + r) * j.ldx;
      if (j.vec) {
        for (int c = 8 * threadIdx.x; c < v.n; c += 2048)
          *reinterpret_cast<uint4*>(lds + r * stride + c) = *reinterpret_cast<const uint4*>(src + c);
      } else {
        for (int c = threadIdx.x; c < v.n; c += 256) lds[r * stride + c] = src[c];
      }
    }
    __syncthreads();
  }
  for (int s = 8 * threadIdx.x; s < ns; s += 2048) {
    const int4 c0 = *reinterpret_cast<const int4*>(v.col + s), c1 = *reinterpret_cast<const int4*>(v.col + s + 4);
    const int c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    for (int r = 0; r < n && t0 + r < j.t; ++r) {
      const uint16_t* src = j.rows ? lds + r * stride : j.x + (t0 + r) * j.ldx;
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = (c[2 * i] >= 0 ? src[c[2 * i]] : 0u) | ((c[2 * i + 1] >= 0 ? (uint32_t)src[c[2 * i + 1]] : 0u) << 16);
      *reinterpret_cast<uint4*>(j.xp + (t0 + r) * ns + s) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// bt[adapter][j][i] = b[adapter][i][j], rows padded to mp with zeros
__device__ void transpose_b(const uint16_t* src0, int adapters, int m, int rank, int mp, uint16_t* bt, long b, long nb) {
  const int groups = (rank + 7) / 8;
  const long total = (long)adapters * groups * mp;
  for (long e = b * 256 + threadIdx.x; e < total; e += nb * 256) {
    const long qg = e / mp, q = qg / groups;
    const int i = (int)(e - qg * mp), j0 = 8 * (int)(qg - q * groups);
    const uint16_t* src = src0 + (q * m + i) * rank + j0;
    uint16_t* dst = bt + (q * rank + j0) * mp + i;
    uint16_t v[8];
    if (i < m && j0 + 8 <= rank) {
      __builtin_memcpy(v, src, 16);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = i < m && j0 + k < rank ? src[k] : (uint16_t)0;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (j0 + k < rank) dst[(long)k * mp] = v[k];
  }
}
// at[adapter][slot][j] = a[adapter][j][column of slot], zeros in empty slots and past the rank
__device__ void transpose_a(const PackedView& v, const uint16_t* a, int adapters, int rank, int rp, uint16_t* at,
                            long b, long nb) {
  const int ns = packed_slots(v), groups = rp / 8;
  const long total = (long)adapters * groups * ns;
  for (long e = b * 256 + threadIdx.x; e < total; e += nb * 256) {
    const long qg = e / ns, q = qg / groups;
    const int s = (int)(e - qg * ns), j0 = 8 * (int)(qg - q * groups), c = v.col[s];
    const uint16_t* src = a + (q * rank + j0) * v.n + c;
    uint32_t o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = c >= 0 && j0 + k < rank ? src[(long)k * v.n] : 0u;
    *reinterpret_cast<uint4*>(at + (q * ns + s) * rp + j0) =
        make_uint4(o[0] | o[1] << 16, o[2] | o[3] << 16, o[4] | o[5] << 16, o[6] | o[7] << 16);
  }
}

// Tokens of adapter q in order, list[start ..], and its items of at most `chunk` tokens. An adapter's items
// begin at slot start / chunk + q, which leaves room for all of them and at most one more, marked empty.
// of[q]: its first item and their number.
constexpr int kTile = 128;  // tokens of a tile of k_shrink_tiles
constexpr int kItem = 256;  // tokens of an item that lie in LDS at a time; chunk is a multiple of it
struct ListJob {
  const int* request;
  int t, adapters, chunk, slots;
  int* list;
  int4* items;
  int2* of;
  int4* tiles;  // the same for items of kTile tokens, null: not asked for
  int ntiles;
};
__device__ void adapter_lists(const ListJob& k, int q) {
  __shared__ int wsum[4], wbelow[4], total;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int b = 0;
  for (int i = threadIdx.x; i < k.t; i += 256) {
    const int r = k.request[i];
    b += r >= 0 && r < q;
  }
#pragma unroll
  for (int s = 32; s; s >>= 1) b += __shfl_xor(b, s);
  if (lane == 0) wbelow[wv] = b;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  const int start = wbelow[0] + wbelow[1] + wbelow[2] + wbelow[3];
  for (int t0 = 0; t0 < k.t; t0 += 256) {
    const int i = t0 + threadIdx.x;
    const bool on = i < k.t && k.request[i] == q;
    const uint64_t m = __builtin_amdgcn_ballot_w64(on);
    if (lane == 0) wsum[wv] = __popcll(m);
    __syncthreads();
    int at = start + total + __popcll(m & ((1ull << lane) - 1));
    for (int w = 0; w < wv; ++w) at += wsum[w];
    if (on) k.list[at] = i;
    __syncthreads();
    if (threadIdx.x == 0) total += wsum[0] + wsum[1] + wsum[2] + wsum[3];
    __syncthreads();
  }
  const int n = total, first = start / k.chunk + q;
  const int end = q + 1 < k.adapters ? (start + n) / k.chunk + q + 1 : k.slots;
  for (int s = first + threadIdx.x; k.items && s < end; s += 256) {
    const int at = (s - first) * k.chunk;
    k.items[s] = at < n ? make_int4(q, start + at, min(k.chunk, n - at), 0) : make_int4(-1, 0, 0, 0);
  }
  if (k.of && threadIdx.x == 0) k.of[q] = make_int2(first, (n + k.chunk - 1) / k.chunk);
  if (k.tiles) {
    const int first2 = start / kTile + q, end2 = q + 1 < k.adapters ? (start + n) / kTile + q + 1 : k.ntiles;
    for (int s = first2 + threadIdx.x; s < end2; s += 256) {
      const int at = (s - first2) * kTile;
      k.tiles[s] = at < n ? make_int4(q, start + at, min(kTile, n - at), 0) : make_int4(-1, 0, 0, 0);
    }
  }
}

// u of few tokens: scaling B^T dy for 8 ranks of one token, a workgroup each
struct DotJob {
  const uint16_t* dy;
  long ldy;
  int t, m;
  const uint16_t* b;
  int rank, adapters;
  const int* request;
  const float* scaling;
  float* u;  // t x rank
};
template <class T>
__device__ void u_dots(const DotJob& k, int id) {
  __shared__ float red[4][8];
  const int groups = (k.rank + 7) / 8, tok = id / groups, j0 = 8 * (id - tok * groups);
  const int q = k.request[tok], lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  if (q < 0 || q >= k.adapters) {
    if (threadIdx.x < 8 && j0 + (int)threadIdx.x < k.rank) k.u[(long)tok * k.rank + j0 + threadIdx.x] = 0.0f;
    return;
  }
  const uint16_t* b = k.b + (long)q * k.m * k.rank + j0;
  const uint16_t* dy = k.dy + (long)tok * k.ldy;
  float s[8] = {};
  const bool whole = j0 + 8 <= k.rank;
#pragma unroll 4
  for (int i = threadIdx.x; i < k.m; i += 256) {
    uint16_t v[8];
    const float d = T::widen(dy[i]);
    if (whole) {
      __builtin_memcpy(v, b + (long)i * k.rank, 16);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j0 + j < k.rank ? b[(long)i * k.rank + j] : (uint16_t)0;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = __builtin_fmaf(d, T::widen(v[j]), s[j]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int x = 32; x; x >>= 1) s[j] += __shfl_xor(s[j], x);
    if (lane == 0) red[wv][j] = s[j];
  }
  __syncthreads();
  if (threadIdx.x < 8 && j0 + (int)threadIdx.x < k.rank) {
    const int j = threadIdx.x;
    k.u[(long)tok * k.rank + j0 + j] = k.scaling[q] * (red[0][j] + red[1][j] + red[2][j] + red[3][j]);
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

// Ranks jt, jt + 32, ... of token ot, by 32 threads: out (t x rank) = low, or scaling low with `scaled`;
// hl[t][2 rp]: scaling low / 2^e as two 16-bit values, hscale[t] = 2^e. e has a floor, since k_wide divides its
// sums by 2^e. f16: -24, where its smallest values times its largest weights lie under half of its smallest
// result; a sum of f16 products is below 2^54 and stays finite. bf16: 0. Its sums reach f32's largest numbers, and
// its range is f32's: smaller vectors need no scale.
template <class T>
constexpr int least_exp() {
  return T::kind == Bf16::kind ? 0 : -24;
}
constexpr int kMostExp = 120;  // 2^120 and a value of up to 2^8 stay finite
constexpr float kMostScale = 0x1p40f;  // up to here sums divided by 2^e keep what counts of them
template <class T, int N>
__device__ __forceinline__ void low_out(const float (&v)[N], int ot, int t, int rank, int rp, int adapters,
                                        const int* request, const float* scaling, int scaled, float* out, uint16_t* hl,
                                        float* hscale) {
  const int jt = threadIdx.x & 31, rq = request[min(ot, t - 1)];
  const float sc = rq >= 0 && rq < adapters ? scaling[rq] : 0.0f;
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, __builtin_fabsf(sc * v[i]));
#pragma unroll
  for (int s = 16; s; s >>= 1) m = fmaxf(m, __shfl_xor(m, s));
  if (ot >= t) return;
  const int e = m > 0.0f && m < __builtin_inff() ? min(max(least_exp<T>(), __builtin_amdgcn_frexp_expf(m)), kMostExp) : 0;
  if (jt == 0 && hscale) hscale[ot] = ldexpf(1.0f, e);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int j = jt + 32 * i;
    if (j < rank && out) out[(long)ot * rank + j] = scaled ? sc * v[i] : v[i];
    if (j < rp && hl) {
      const float y = ldexpf(sc * v[i], -e);
      const uint16_t hi = T::narrow(y);
      hl[(long)ot * 2 * rp + j] = hi;
      hl[(long)ot * 2 * rp + rp + j] = T::narrow(y - T::widen(hi));
    }
  }
}

// low[t][j] = sum_k a[q][j][k] x[t][k] for 16 tokens a workgroup of NW wavefronts, each taking every NW-th
// step of k.
struct ShrinkJob {
  const uint16_t* x;
  long ldx;
  int t, kk;
  const uint16_t* a;
  long lda;
  int rank, rp, adapters;
  const int* request;
  const float* scaling;
  int scaled;
  float* out;  // as low_out takes them
  uint16_t* hl;
  float* hscale;
};
template <class T, int RF, int NW>
__device__ __forceinline__ void shrink_rows(const ShrinkJob& s, int id) {
  typedef typename T::v8 v8;
  __shared__ float red[NW][16][RF * 16 + 1];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quad = lane >> 4;
  const int tok = id * 16 + (lane & 15);
  int q = tok < s.t ? s.request[tok] : -1;
  if (q >= s.adapters) q = -1;
  mma_f4 keep[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) keep[f] = mma_f4{};
  uint64_t left = __builtin_amdgcn_ballot_w64(q >= 0);
  const uint16_t* xr = s.x + (long)min(tok, s.t - 1) * s.ldx;
  for (int ad = next_adapter(q, left); ad >= 0; ad = next_adapter(q, left)) {
    const uint16_t* ar[RF];
    mma_f4 acc[RF];
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      ar[f] = s.a + ((long)ad * s.rank + min(16 * f + (lane & 15), s.rank - 1)) * s.lda;
      acc[f] = mma_f4{};
    }
    // 64 k a wavefront and step, 16 of a row a lane (whole cache lines; the two operands agree on the order
    // of k, which is all a sum needs); U steps' loads in flight
    constexpr int U = RF > 4 ? 1 : 2, STEP = 64 * NW;
    for (int k0 = 64 * wv; k0 < s.kk; k0 += STEP * U) {
      mma_u4 xv[U][2], av[U][2][RF];
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = k0 + STEP * i + 16 * quad + 8 * h;
          xv[i][h] = mma_u4{};
#pragma unroll
          for (int f = 0; f < RF; ++f) av[i][h][f] = mma_u4{};
          if (k < s.kk) {
            xv[i][h] = *reinterpret_cast<const mma_u4*>(xr + k);
#pragma unroll
            for (int f = 0; f < RF; ++f) av[i][h][f] = *reinterpret_cast<const mma_u4*>(ar[f] + k);
          }
        }
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int f = 0; f < RF; ++f)
            acc[f] = T::mfma(__builtin_bit_cast(v8, av[i][h][f]), __builtin_bit_cast(v8, xv[i][h]), acc[f]);
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
  const int jt = threadIdx.x & 31;
  for (int it = threadIdx.x >> 5; it < 16; it += 2 * NW) {
    float v[(RF + 1) / 2];
#pragma unroll
    for (int i = 0; i < (RF + 1) / 2; ++i) {
      const int j = jt + 32 * i;
      v[i] = 0.0f;
      if (j < s.rank)
        for (int w = 0; w < NW; ++w) v[i] += red[w][it][j];
    }
    low_out<T, (RF + 1) / 2>(v, id * 16 + it, s.t, s.rank, s.rp, s.adapters, s.request, s.scaling, s.scaled, s.out, s.hl,
                             s.hscale);
  }
}
template <class T, int RF>
__global__ __launch_bounds__(512) void k_shrink(ShrinkJob s) {
  shrink_rows<T, RF, 8>(s, blockIdx.x);
}

// Workgroups of each part, in this order; 0: not asked for.
struct PrepareArgs {
  int expand, slots, pad[3], tb, ta, lists, dots, shrink;
  uint16_t* w16;
  SlotJob slot;
  PadJob pads[3];
  const uint16_t *a, *b;
  int adapters, rank, rp, mp;
  uint16_t *bt, *at;
  ListJob list;
  DotJob dot;
  ShrinkJob low;
  int total() const { return expand + slots + pad[0] + pad[1] + pad[2] + tb + ta + lists + dots + shrink; }
};
// RF: of the low-rank vectors that are taken along (0: none)
template <class T, int RF = 0>
__global__ __launch_bounds__(256) void k_prepare(PackedView v, PrepareArgs k) {
  extern __shared__ __align__(16) uint16_t lds[];
  int b = blockIdx.x;
  if constexpr (RF > 0) {
    if (b < k.shrink) return shrink_rows<T, RF, 4>(k.low, b);
    b -= k.shrink;
  }
  if (b < k.lists) return adapter_lists(k.list, b);
  b -= k.lists;
  if (b < k.dots) return u_dots<T>(k.dot, b);
  b -= k.dots;
  if (b < k.slots) return to_slots(v, k.slot, lds, b);
  b -= k.slots;
  if (b < k.expand) return packed_expand<T>(v, k.w16, b, k.expand);
  b -= k.expand;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    if (b < k.pad[i]) return pad_rows16(k.pads[i], b, k.pad[i]);
    b -= k.pad[i];
  }
  if (b < k.tb) return transpose_b(k.b, k.adapters, v.m, k.rank, k.mp, k.bt, b, k.tb);
  b -= k.tb;
  transpose_a(v, k.a, k.adapters, k.rank, k.rp, k.at, b, k.ta);
}

// The same for many tokens: tiles of 128 tokens of one adapter (by list) against its ranks, on the tiles of
// mma16.h, split in k; part[split][token][rp]. The fragment loads of k_shrink touch 16 rows for 256 bytes,
// which bounds it (4096 tokens, k = 14336, rank 64: 82 us); here a load takes 8 rows' whole lines (41 us, and 10
// to sum the splits; k = 4096: 15 and 5).
template <class T, int FP, int FQ, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ, 2) void k_shrink_tiles(const uint16_t* __restrict__ x, long ldx, int kk,
                                                                  const uint16_t* __restrict__ a, long lda, int rank,
                                                                  int rp, const int* __restrict__ list,
                                                                  const int4* __restrict__ tiles, int t, int share,
                                                                  float* __restrict__ part) {
  typedef MmaTile<T, false, false, FP, FQ, WP, WQ> M;
  static_assert(M::BP == kTile, "a tile is an item");
  __shared__ __align__(1024) uint8_t lds[M::LDS];
  const int4 it = tiles[blockIdx.x];
  if (it.x < 0) return;
  mma_f4 acc[FP][FQ];
  M::clear(acc);
  M::run(lds_offset(lds), MmaOp{x, ldx, it.z, list + it.y}, MmaOp{a + (long)it.x * rank * lda, lda, rank}, 0, 0,
         blockIdx.y * share, min(kk, ((int)blockIdx.y + 1) * share), acc);
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int f = 0; f < FP; ++f)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = M::row(0, f) + 4 * (lane >> 4) + r;
      if (i >= it.z) continue;
      float* o = part + ((long)blockIdx.y * t + list[it.y + i]) * rp;
#pragma unroll
      for (int g = 0; g < FQ; ++g) {
        const int j = M::col(0, g) + (lane & 15);
        if (j < rp) o[j] = acc[f][g][r];
      }
    }
}
template <class T>
__global__ __launch_bounds__(256) void k_shrink_sum(const float* __restrict__ part, int splits, int t, int rank, int rp,
                                                    int adapters, const int* __restrict__ request,
                                                    const float* __restrict__ scaling, int scaled,
                                                    float* __restrict__ out, uint16_t* __restrict__ hl,
                                                    float* __restrict__ hscale) {
  const int tok = blockIdx.x * 8 + (threadIdx.x >> 5), jt = threadIdx.x & 31;
  const int q = tok < t ? request[tok] : -1;
  float v[4] = {};
  if (q >= 0 && q < adapters)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = jt + 32 * i;
      if (j < rank)
#pragma unroll 4
        for (int s = 0; s < splits; ++s) v[i] += part[((long)s * t + tok) * rp + j];
    }
  low_out<T, 4>(v, tok, t, rank, rp, adapters, request, scaling, scaled, out, hl, hscale);
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
  int share;  // of k, a split's; the low-rank term goes with the first
  float* parts;       // [split][t][rows rounded up to 4] instead of out, or null
};

// out[t][i] = sum_k W(i, k) x[t][k] + hscale_t sum_j e[q][i][j] (hl[t][j] + hl[t][rp + j])
template <class T, bool PS, int FP, int FQ, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ, 2) void k_wide(WideArgs a) {
  typedef MmaTile<T, PS, false, FP, FQ, WP, WQ> M;
  typedef typename T::v8 v8;
  __shared__ __align__(1024) uint8_t lds[M::LDS];
  const int tiles = a.np * a.nq, split = blockIdx.x / tiles;
  const MmaTileAt at = mma_tile_at(blockIdx.x - split * tiles, a.np, a.nq);
  const int p0 = at.p * M::BP, q0 = at.q * M::BQ;
  mma_f4 acc[FP][FQ];
  M::clear(acc);
  M::run(lds_offset(lds), MmaOp{a.w, a.ldw, a.rows}, MmaOp{a.x, a.ldx, a.t}, p0, q0, split * a.share,
         min(a.k, (split + 1) * a.share), acc);
  const int lane = threadIdx.x & 63, quad = lane >> 4;
  const long ldp = (a.rows + 3) & ~3;
  if (a.e && split == 0) {
    int q[FQ];
    float scale[FQ];
    // alike: every token of the wavefront has one and the same adapter, or none, and 2^e is in range of f32
    int only = -1;
#pragma unroll
    for (int g = 0; g < FQ; ++g) {
      const int t = M::col(q0, g) + (lane & 15);
      q[g] = t < a.t ? a.request[t] : -1;
      scale[g] = q[g] >= 0 && q[g] < a.adapters ? a.hscale[t] : 1.0f;
      const uint64_t some = __builtin_amdgcn_ballot_w64(q[g] != -1);
      if (only == -1 && some) only = __builtin_amdgcn_readlane(q[g], __builtin_ctzll(some));
    }
    bool alike = only >= 0 && only < a.adapters, bare = false;
#pragma unroll
    for (int g = 0; g < FQ; ++g) {
      alike &= __builtin_amdgcn_ballot_w64(q[g] != -1 && !(q[g] == only && scale[g] <= kMostScale)) == 0;
      bare |= __builtin_amdgcn_ballot_w64(q[g] == -1 && M::col(q0, g) + (lane & 15) < a.t) != 0;
    }
    // A token without an adapter takes part with zeros, which infinities and NaN in the adapter's rows would
    // turn into NaN: looked for where there is one.
    const uint16_t* const e = a.e + (alike ? (long)only * a.rows * a.rp : 0);
    if (alike && bare) {
      mma_us8 top = {};
      for (int kf = 0; kf < a.rp; kf += 32) {
        const int k = min(kf + 8 * quad, a.rp - 8);
#pragma unroll
        for (int f = 0; f < FP; ++f) {
          const uint32_t row = min(M::row(p0, f) + (lane & 15), a.rows - 1);
          const mma_us8 v = *reinterpret_cast<const mma_us8*>(e + (row * (uint32_t)a.rp + k));
          top = __builtin_elementwise_max(top, v & (uint16_t)0x7fff);
        }
      }
      bool wild = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) wild |= top[i] >= T::narrow(__builtin_inff());
      alike = __builtin_amdgcn_ballot_w64(wild) == 0;
    }
    // alike: straight onto the sums, which are divided by 2^e meanwhile: no second set of them, so all tokens
    // at once and an adapter's rows read once. (Loops of no passes, not branches: those would copy the sums.)
#pragma unroll
    for (int g = 0; g < FQ; ++g) {
      const float inv = alike ? 1.0f / scale[g] : 1.0f;
#pragma unroll
      for (int f = 0; f < FP; ++f) acc[f][g] *= inv;
    }
    const int kfs = alike ? 2 * a.rp : 0;
    for (int kf = 0; kf < kfs; kf += 32) {
      const int k = kf + 8 * quad, c = k < a.rp ? k : k - a.rp;
      v8 ev[FP], h[FQ];
#pragma unroll
      for (int f = 0; f < FP; ++f) {
        const uint32_t row = min(M::row(p0, f) + (lane & 15), a.rows - 1);
        ev[f] = __builtin_bit_cast(v8, *reinterpret_cast<const mma_u4*>(e + (row * (uint32_t)a.rp + c)));
      }
#pragma unroll
      for (int g = 0; g < FQ; ++g) {
        const uint32_t t = min(M::col(q0, g) + (lane & 15), a.t - 1);
        h[g] = __builtin_bit_cast(v8, *reinterpret_cast<const mma_u4*>(a.hl + (t * (uint32_t)(2 * a.rp) + k)));
      }
#pragma unroll
      for (int f = 0; f < FP; ++f)
#pragma unroll
        for (int g = 0; g < FQ; ++g) acc[f][g] = T::mfma(ev[f], h[g], acc[f][g]);
    }
#pragma unroll
    for (int g = 0; g < FQ; ++g) {
      const float back = alike ? scale[g] : 1.0f;
#pragma unroll
      for (int f = 0; f < FP; ++f) acc[f][g] *= back;
      const int t = M::col(q0, g) + (lane & 15);
      const bool known = q[g] >= 0 && q[g] < a.adapters;
      uint64_t left = alike ? 0 : __builtin_amdgcn_ballot_w64(known);
      // the others' tokens one adapter after another, by the same operations in the same order: a token's
      // result does not depend on its neighbours
      const float inv = scale[g] <= kMostScale ? 1.0f / scale[g] : 0.0f;
      for (int ad = next_adapter(q[g], left); ad >= 0; ad = next_adapter(q[g], left)) {
        mma_f4 d[FP];
#pragma unroll
        for (int f = 0; f < FP; ++f) d[f] = acc[f][g] * inv;
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
            if (q[g] == ad) acc[f][g][r] = __builtin_fmaf(scale[g], d[f][r], inv > 0.0f ? 0.0f : acc[f][g][r]);
      }
      if (!known && q[g] != -1) {  // no such adapter
#pragma unroll
        for (int f = 0; f < FP; ++f)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[f][g][r] = __builtin_nanf("");
      }
    }
  }
#pragma unroll
  for (int g = 0; g < FQ; ++g) {
    const int t = M::col(q0, g) + (lane & 15);
    if (a.parts && t < a.t) {
#pragma unroll
      for (int f = 0; f < FP; ++f) {
        const int row = M::row(p0, f) + 4 * quad;
        if (row < a.rows) *reinterpret_cast<mma_f4*>(a.parts + ((long)split * a.t + t) * ldp + row) = acc[f][g];
      }
    }
  }
  if (!a.parts) M::store(lds_offset(lds), acc, p0, q0, a.rows, a.t, a.out, a.ldo);
}

// part[slot][j][c] = sum over the item's tokens of l[t][j] X[t][c], j in 16 RF ranks from j0, c in 128
// columns a wavefront. X: 8-bit codes with their scales (I8), or 16-bit values; l times scaling[q] if given.
// Two sets of four wavefronts take every other 32 tokens each (one set leaves a SIMD one wavefront, which
// waits for its loads and its own results: rank 64 over 4096 tokens, 4096 + 14336 columns: 77 us; two: 59).
// A lane reads 8 neighbouring columns of 8 tokens, the next ones while these are multiplied: row i of the
// f-th MFMA operand is column 8 i + f. The item's l lies in LDS, its token list beside it; it enters the
// matrix cores as the sum of two 16-bit values, in f16 divided by 2^e to keep it in range (e grows with the
// largest l so far, the sums go along): 2^-15 of an element is lost at most down to 2^-10 of the item's largest,
// below that 2^-25 of the largest.
struct OuterJob {
  const void* x;
  const float* xscale;
  long ldx;
  int cols;
  const float* l;
  const float* scaling;
  float* part;  // [slot][rp][128 * blocks of columns]
};
template <class T, bool I8, bool VEC, int RF>
__device__ __forceinline__ void outer(const OuterJob& k, int colgroup, int rank, int rp, const int* list, int4 it,
                                      int slot, int j0, float (*ll)[16 * RF + 1], int* toks) {
  typedef typename T::v8 v8;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6 & 3, set = threadIdx.x >> 8, quad = lane >> 4;
  const float mul = k.scaling ? k.scaling[it.x] : 1.0f;
  const int c0 = (colgroup * 4 + wv) * 128, nb = (k.cols + 127) / 128;
  // columns past the last take part with another's values: nobody reads their sums
  const int c = c0 + 8 * (lane & 15), cs = VEC ? min(c, ((k.cols + 7) & ~7) - 8) : c, blk = min(c0 / 128, nb - 1);
  mma_f4 acc[8][RF];
#pragma unroll
  for (int f = 0; f < 8; ++f)
#pragma unroll
    for (int g = 0; g < RF; ++g) acc[f][g] = mma_f4{};
  int ex = -126;  // f16: the exponent that ll and the sums are divided by
  __shared__ float wtop[8];
  struct Raw {
    mma_u4 h[I8 ? 1 : 8];
    uint2 b[I8 ? 8 : 1];
    float s[8];
  };
  auto load = [&](int t0, Raw& r) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long tok = toks[t0 + 8 * quad + i];
      if constexpr (I8) {
        const int8_t* src = static_cast<const int8_t*>(k.x) + tok * k.ldx + cs;
        if constexpr (VEC) {
          r.b[i] = *reinterpret_cast<const uint2*>(src);
        } else {
          uint8_t v[8];
#pragma unroll
          for (int b = 0; b < 8; ++b) v[b] = c + b < k.cols ? (uint8_t)src[b] : (uint8_t)0;
          r.b[i] = *reinterpret_cast<uint2*>(v);
        }
        r.s[i] = k.xscale[tok * nb + blk];
      } else {
        r.h[i] = *reinterpret_cast<const mma_u4*>(static_cast<const uint16_t*>(k.x) + tok * k.ldx + cs);
      }
    }
  };
  auto mul_add = [&](int t0, const Raw& r) {
    uint32_t xv[8][4];  // operand f, pairs of tokens
#pragma unroll
    for (int f = 0; f < 8; ++f)
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        if constexpr (I8) {
          const uint32_t a = f < 4 ? r.b[2 * p].x : r.b[2 * p].y, b = f < 4 ? r.b[2 * p + 1].x : r.b[2 * p + 1].y;
          xv[f][p] = narrow2<T>((float)(int8_t)(a >> (8 * (f & 3))), (float)(int8_t)(b >> (8 * (f & 3))));
        } else {
          xv[f][p] = __builtin_amdgcn_perm(r.h[2 * p + 1][f >> 1], r.h[2 * p][f >> 1], f & 1 ? 0x07060302u : 0x05040100u);
        }
      }
#pragma unroll
    for (int g = 0; g < RF; ++g) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        float y[2];
        uint16_t h[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          y[i] = ll[t0 + 8 * quad + 2 * p + i][16 * g + (lane & 15)];
          if constexpr (I8) y[i] *= r.s[2 * p + i];
          if constexpr (T::kind == F16::kind) y[i] = ldexpf(y[i], -ex);
          h[i] = T::narrow(y[i]);
        }
        hi[p] = (uint32_t)h[0] | ((uint32_t)h[1] << 16);
        lo[p] = narrow2<T>(y[0] - T::widen(h[0]), y[1] - T::widen(h[1]));
      }
      const v8 vh = __builtin_bit_cast(v8, mma_u4{hi[0], hi[1], hi[2], hi[3]});
      const v8 vl = __builtin_bit_cast(v8, mma_u4{lo[0], lo[1], lo[2], lo[3]});
#pragma unroll
      for (int f = 0; f < 8; ++f)
        acc[f][g] = T::mfma(__builtin_bit_cast(v8, mma_u4{xv[f][0], xv[f][1], xv[f][2], xv[f][3]}), vh, acc[f][g]);
#pragma unroll
      for (int f = 0; f < 8; ++f)
        acc[f][g] = T::mfma(__builtin_bit_cast(v8, mma_u4{xv[f][0], xv[f][1], xv[f][2], xv[f][3]}), vl, acc[f][g]);
    }
  };
  for (int i0 = 0; i0 < it.z; i0 += kItem) {
    const int n = min(kItem, it.z - i0);
    if (i0) __syncthreads();
    if (threadIdx.x < kItem) toks[threadIdx.x] = list[it.y + i0 + min((int)threadIdx.x, n - 1)];
    __syncthreads();
    Raw now, next;
    if (VEC && c0 < k.cols) load(32 * set, now);
    // l of these tokens, 0 past the last: four ranks a load, half of the thread's loads in flight at once
    constexpr int PER = 4 * RF, BATCH = PER / 2 < 4 ? PER / 2 : 4;
    float top = 0.0f;
    for (int e0 = 0; e0 < kItem * PER; e0 += 512 * BATCH) {
      if (e0 / PER >= ((n + 63) & ~63)) break;
      mma_f4 v[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int e = e0 + 512 * u + threadIdx.x, i = e / PER, j = j0 + 4 * (e - i * PER);
        v[u] = mma_f4{};
        if (i < n) {
          const float* src = k.l + (long)toks[i] * rank + j;
          if (rank % 4 == 0) {
            if (j < rank) v[u] = *reinterpret_cast<const mma_f4*>(src);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (j + r < rank) v[u][r] = src[r];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        const int e = e0 + 512 * u + threadIdx.x, i = e / PER, j = 4 * (e - i * PER);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          ll[i][j + r] = mul * v[u][r];
          const float m = __builtin_fabsf(mul * v[u][r]);
          if (m < __builtin_inff()) top = fmaxf(top, m);
        }
      }
    }
    if constexpr (T::kind == F16::kind) {
#pragma unroll
      for (int s = 32; s; s >>= 1) top = fmaxf(top, __shfl_xor(top, s));
      if (lane == 0) wtop[threadIdx.x >> 6] = top;
    }
    __syncthreads();
    if constexpr (T::kind == F16::kind) {
      top = wtop[0];
#pragma unroll
      for (int w = 1; w < 8; ++w) top = fmaxf(top, wtop[w]);
      const int to = max(ex, top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : -126);
      if (to != ex) {
#pragma unroll
        for (int f = 0; f < 8; ++f)
#pragma unroll
          for (int g = 0; g < RF; ++g)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[f][g][r] = ldexpf(acc[f][g][r], ex - to);
        ex = to;
      }
    }
    if (c0 >= k.cols) continue;
    for (int t0 = 32 * set; t0 < n; t0 += 64) {
      if constexpr (VEC) {
        load(min(t0 + 64, kItem - 32), next);
        mul_add(t0, now);
        now = next;
      } else {
        load(t0, now);
        mul_add(t0, now);
      }
    }
  }
  // the two sets' sums together, half of them at a time
  float* const join = &ll[0][0];
#pragma unroll
  for (int f0 = 0; f0 < 8; f0 += 4) {
    __syncthreads();
    if (set)
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int g = 0; g < RF; ++g)
          *reinterpret_cast<mma_f4*>(join + 4 * ((f * RF + g) * 256 + (threadIdx.x & 255))) = acc[f0 + f][g];
    __syncthreads();
    if (!set)
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int g = 0; g < RF; ++g)
          acc[f0 + f][g] += *reinterpret_cast<const mma_f4*>(join + 4 * ((f * RF + g) * 256 + threadIdx.x));
  }
  if (set || c0 >= k.cols) return;
  if constexpr (T::kind == F16::kind) {
#pragma unroll
    for (int f = 0; f < 8; ++f)
#pragma unroll
      for (int g = 0; g < RF; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[f][g][r] = ldexpf(acc[f][g][r], ex);
  }
  const long ldp = (long)nb * 128;
#pragma unroll
  for (int g = 0; g < RF; ++g) {
    const int j = j0 + 16 * g + (lane & 15);
    if (j >= rp) continue;
    float* o = k.part + ((long)slot * rp + j) * ldp + c0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 8 * (4 * quad + r);
      *reinterpret_cast<mma_f4*>(o + i) = mma_f4{acc[0][g][r], acc[1][g][r], acc[2][g][r], acc[3][g][r]};
      *reinterpret_cast<mma_f4*>(o + i + 4) = mma_f4{acc[4][g][r], acc[5][g][r], acc[6][g][r], acc[7][g][r]};
    }
  }
}
// dB's part (16-bit dy) in the first nb_ workgroups of x, dA's (the checkpoint) in the rest
template <class T, int RF, bool VECA>
__global__ __launch_bounds__(512, 2) void k_outer(OuterJob db, int nb_, OuterJob da, int rank, int rp,
                                                  const int* __restrict__ list, const int4* __restrict__ items) {
  __shared__ __align__(16) float ll[kItem][16 * RF + 1];
  __shared__ int toks[kItem];
  const int4 it = items[blockIdx.y];
  if (it.x < 0) return;
  const int j0 = blockIdx.z * 16 * RF;
  if ((int)blockIdx.x < nb_) outer<T, false, true, RF>(db, blockIdx.x, rank, rp, list, it, blockIdx.y, j0, ll, toks);
  else outer<Bf16, true, VECA, RF>(da, blockIdx.x - nb_, rank, rp, list, it, blockIdx.y, j0, ll, toks);
}

// ---- parts of `finish`

// Sums of an adapter's items in order, rounded once: da[q][j][c]
struct JoinJob {
  const float* part;
  int cols;
  long ldp;
  uint16_t* out;
};
template <class T>
__device__ void join_da(const JoinJob& k, const int2* of, int rank, int rp, int b) {
  const int nc = (k.cols + 255) / 256, qj = b / nc, q = qj / rank, j = qj - q * rank;
  const int c = (b - qj * nc) * 256 + threadIdx.x;
  if (c >= k.cols) return;
  const int2 f = of[q];
  float s = 0.0f;
#pragma unroll 4
  for (int i = 0; i < f.y; ++i) s += k.part[((long)(f.x + i) * rp + j) * k.ldp + c];
  k.out[((long)q * rank + j) * k.cols + c] = T::narrow(s);
}
// ... db[q][c][j], 8 ranks a thread
template <class T>
__device__ void join_db(const JoinJob& k, const int2* of, int rank, int rp, int b) {
  const int nc = (k.cols + 255) / 256, groups = (rank + 7) / 8, qg = b / nc, q = qg / groups, j0 = 8 * (qg - q * groups);
  const int c = (b - qg * nc) * 256 + threadIdx.x;
  if (c >= k.cols) return;
  const int2 f = of[q];
  float s[8] = {};
#pragma unroll 2
  for (int i = 0; i < f.y; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] += k.part[((long)(f.x + i) * rp + j0 + j) * k.ldp + c];
  uint16_t* o = k.out + ((long)q * k.cols + c) * rank + j0;
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = narrow2<T>(s[2 * j], s[2 * j + 1]);
  if (j0 + 8 <= rank) {
    __builtin_memcpy(o, w, 16);  // any alignment
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j0 + j < rank) o[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
  }
}

// 16-bit results in slot order back to columns through LDS (as to_slots)
struct BackJob {
  const uint16_t* xp;
  int t, rows, vec;
  uint16_t* x;
  long ldx;
};
__device__ void from_slots(const PackedView& v, const BackJob& j, uint16_t* lds, long b) {
  const int n = j.rows ? j.rows : 1, ns = packed_slots(v), stride = (v.n + 7) & ~7;
  const long t0 = b * n;
  for (int s = 8 * threadIdx.x; s < ns; s += 2048) {
    const int4 c0 = *reinterpret_cast<const int4*>(v.col + s), c1 = *reinterpret_cast<const int4*>(v.col + s + 4);
    const int c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    for (int r = 0; r < n && t0 + r < j.t; ++r) {
      uint16_t in[8];
      *reinterpret_cast<uint4*>(in) = *reinterpret_cast<const uint4*>(j.xp + (t0 + r) * ns + s);
      uint16_t* dst = j.rows ? lds + r * stride : j.x + (t0 + r) * j.ldx;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c[i] >= 0) dst[c[i]] = in[i];
    }
  }
  if (!j.rows) return;
  __syncthreads();
  for (int r = 0; r < n && t0 + r < j.t; ++r) {
    uint16_t* dst = j.x + (t0 + r) * j.ldx;
    if (j.vec) {
      for (int c = 8 * threadIdx.x; c < v.n; c += 2048)
        *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(lds + r * stride + c);
    } else {
      for (int c = threadIdx.x; c < v.n; c += 256) dst[c] = lds[r * stride + c];
    }
  }
}

// Results from the splits' f32 sums: out[t][c] = sum of parts[split][t][slot of c, or c], rounded once, and
// with `a` (few tokens) A_q^T u_t added in f32 before.
struct SumJob {
  const float* parts;
  int splits, t, cols;
  long ldp;
  const int* slot;  // of each column, null: the identity
  const uint16_t* a;  // adapters x rank x cols
  const float* u;
  int rank, adapters;
  const int* request;
  uint16_t* out;
  long ldo;
};
template <class T>
__device__ void sum_parts(const SumJob& k, int b) {
  const int nc = (k.cols + 255) / 256, t = b / nc, c = (b - t * nc) * 256 + threadIdx.x;
  if (c >= k.cols) return;
  const float* p = k.parts + (long)t * k.ldp + (k.slot ? k.slot[c] : c);
  float s = 0.0f;
#pragma unroll 4
  for (int i = 0; i < k.splits; ++i) s += p[(long)i * k.t * k.ldp];
  if (k.a) {
    const int q = k.request[t];
    if (q >= 0 && q < k.adapters) {
      const uint16_t* a = k.a + (long)q * k.rank * k.cols + c;
      const float* u = k.u + (long)t * k.rank;
#pragma unroll 4
      for (int j = 0; j < k.rank; ++j) s = __builtin_fmaf(T::widen(a[(long)j * k.cols]), u[j], s);
    } else if (q != -1) {
      s = __builtin_nanf("");  // no such adapter
    }
  }
  k.out[(long)t * k.ldo + c] = T::narrow(s);
}

// The same from slot order for many tokens: `rows` tokens at a time through LDS in f32 (a column's gather
// from memory costs four times the bytes: a step of 200 tokens, 4096 -> 4096, 131 us, 135 by it).
template <class T>
__device__ void sum_slots(const PackedView& v, const SumJob& k, int rows, float* lds, int b) {
  const int ns = packed_slots(v), t0 = b * rows;
  for (int r = 0; r < rows && t0 + r < k.t; ++r) {
    const float* p = k.parts + (long)(t0 + r) * k.ldp;
    for (int s = 4 * threadIdx.x; s < ns; s += 1024) {
      const int4 c = *reinterpret_cast<const int4*>(v.col + s);
      mma_f4 x = {};
#pragma unroll 4
      for (int i = 0; i < k.splits; ++i) x += *reinterpret_cast<const mma_f4*>(p + (long)i * k.t * k.ldp + s);
      float* d = lds + r * v.n;
      if (c.x >= 0) d[c.x] = x[0];
      if (c.y >= 0) d[c.y] = x[1];
      if (c.z >= 0) d[c.z] = x[2];
      if (c.w >= 0) d[c.w] = x[3];
    }
  }
  __syncthreads();
  for (int r = 0; r < rows && t0 + r < k.t; ++r)
    for (int c = threadIdx.x; c < v.n; c += 256) k.out[(long)(t0 + r) * k.ldo + c] = T::narrow(lds[r * v.n + c]);
}

// Workgroups of each part; 0: not asked for.
struct FinishArgs {
  int nda, ndb, nback, nsum, sum_rows;  // sum_rows: of sum_slots, 0: sum_parts
  JoinJob da, db;
  const int2* of;
  int rank, rp;
  BackJob back;
  SumJob sum;
  __host__ __device__ int total() const { return nda + ndb + nback + nsum; }
};
template <class T>
__global__ __launch_bounds__(256) void k_finish(PackedView v, FinishArgs k) {
  extern __shared__ __align__(16) uint16_t lds[];
  int b = blockIdx.x + blockIdx.y * gridDim.x;
  if (b >= k.total()) return;
  if (b < k.nback) return from_slots(v, k.back, lds, b);
  b -= k.nback;
  if (b < k.nsum) {
    if (k.sum_rows) return sum_slots<T>(v, k.sum, k.sum_rows, reinterpret_cast<float*>(lds), b);
    return sum_parts<T>(k.sum, b);
  }
  b -= k.nsum;
  if (b < k.ndb) return join_db<T>(k.db, k.of, k.rank, k.rp, b);
  join_da<T>(k.da, k.of, k.rank, k.rp, b - k.ndb);
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

// Rows that to_slots / from_slots pass through 64 KB of LDS at a time, and its bytes.
inline int slot_rows(const PackedView& v) {
  const size_t row = 2 * up(v.n, 8);
  return row * 4 <= 65536 ? 4 : row <= 65536 ? 1 : 0;
}
inline size_t slot_lds(const PackedView& v) { return slot_rows(v) * 2 * up(v.n, 8); }
inline int slot_blocks(const PackedView& v, long t) {
  const int r = std::max(slot_rows(v), 1);
  return (int)((t + r - 1) / r);
}
inline int expand_blocks(const PackedView& v) {
  const long per = 4 * packed_expand_unit(v);
  return (int)std::min(((long)v.tiles * v.nkb + per - 1) / per, 1l << 16);
}
inline int pad_blocks(const PadJob& j) { return blocks_for(j.rows * (j.dp / 8), 256 * 4, 8192); }

#define STEP(expr)                       \
  do {                                   \
    hipError_t e_ = (expr);              \
    if (e_ != hipSuccess) return e_;     \
  } while (0)

// How the low-rank vectors are made: k_shrink in about 82 us per 4096 tokens, 14336 of k and 5 operands of 16
// rows; the tiles and their sum in two launches, worth it from about 20 us on (training steps 4096 -> 14336 of rank 64:
// 1024 tokens 477 us, 581 without the tiles; 4096 tokens 1019 and 1046; 640 tokens of 2048 -> 2048, rank 8, stay
// below: 9 us in one launch).
struct ShrinkPlan {
  bool tiles;
  int ntiles, splits, share;
};
ShrinkPlan shrink_plan(long t, long k, int adapters, int rp) {
  ShrinkPlan p = {};
  p.tiles = t >= 512 && 82.0 / 5 * (t / 4096.0) * (k / 14336.0) * (1 + rp / 16) > 20.0;
  p.ntiles = (int)(t / kTile) + adapters;
  const long n = std::max(1l, std::min(768 / std::max(1l, (t + kTile - 1) / kTile), k / 512));
  p.share = (int)up((k + n - 1) / n, 64);
  p.splits = (int)((k + p.share - 1) / p.share);
  return p;
}
template <class T>
hipError_t shrink(hipStream_t st, const ShrinkPlan& p, const int* list, const int4* tiles, float* part,
                  const uint16_t* x, long ldx, long t, int k, const uint16_t* a, long lda, const AdapterArgs& g,
                  int scaled, float* out, uint16_t* hl, float* hscale) {
  const int grid = (int)((t + 15) / 16), rp = rank_pad(g.rank);
  if (p.tiles) {
    auto go = [&](auto s) {
      typedef decltype(s) S;
      k_shrink_tiles<T, S::fp, S::fq, S::wp, S::wq><<<dim3(p.ntiles, p.splits), S::threads, 0, st>>>(
          x, ldx, k, a, lda, g.rank, rp, list, tiles, (int)t, p.share, part);
      return hipGetLastError();
    };
    if (rp <= 16) STEP(go(MmaShape<2, 1, 4, 1>{}));
    else if (rp <= 32) STEP(go(MmaShape<2, 2, 4, 1>{}));
    else if (rp <= 64) STEP(go(MmaShape<4, 2, 2, 2>{}));
    else STEP(go(MmaShape<4, 4, 2, 2>{}));
    k_shrink_sum<T><<<(int)((t + 7) / 8), 256, 0, st>>>(part, p.splits, (int)t, g.rank, rp, g.adapters, g.request,
                                                        g.scaling, scaled, out, hl, hscale);
    return hipGetLastError();
  }
  auto go = [&](auto rf) {
    k_shrink<T, decltype(rf)::value><<<grid, 512, 0, st>>>(
        {x, ldx, (int)t, k, a, lda, g.rank, rp, g.adapters, g.request, g.scaling, scaled, out, hl, hscale});
    return hipGetLastError();
  };
  if (rp <= 16) return go(std::integral_constant<int, 1>{});
  if (rp <= 32) return go(std::integral_constant<int, 2>{});
  if (rp <= 64) return go(std::integral_constant<int, 4>{});
  return go(std::integral_constant<int, 8>{});
}

// Shape and splits of a product: the f32 parts of a split one are written and read at about 4 TB/s, and
// summing them takes a launch (4 us) unless one is there anyway.
constexpr long kCache = 200l << 20;  // expanded weights up to this many bytes are found in the last cache (256 MB)
struct WidePlan {
  int pick, splits, share;
};
WidePlan wide_plan(long rows, long t, long k, bool strided, bool parts_anyway) {
  const bool far = 2 * rows * k > kCache;
  WidePlan best = {};
  double least = 0;
  for (int i = 0; i < kMmaShapes; ++i)
    for (int n = 1; n == 1 || (n <= 16 && k / n >= 256); n *= 2) {
      if (!strided && kMmaTimes[i].bq == 16) continue;  // the forward product has more tokens
      const bool parts = parts_anyway || n > 1;
      const double c = mma_cost(rows, t, k, i, n, strided, far) + (parts ? n * (8.0 / 4e6) * t * rows : 0.0) +
                       (n > 1 && !parts_anyway ? 4.0 : 0.0);
      if ((i == 0 && n == 1) || c < least) least = c, best.pick = i, best.splits = n;
    }
  best.share = (int)up((k + best.splits - 1) / best.splits, 64);
  best.splits = (int)((k + best.share - 1) / best.share);
  return best;
}

template <class T, bool PS>
hipError_t wide_product(hipStream_t st, const WidePlan& p, WideArgs w) {
  w.share = p.share;
  return with_mma_shape(p.pick, [&](auto s) {
    typedef decltype(s) S;
    if constexpr (PS || S::bq > 16) {
      w.np = (w.rows + S::bp - 1) / S::bp;
      w.nq = (w.t + S::bq - 1) / S::bq;
      k_wide<T, PS, S::fp, S::fq, S::wp, S::wq><<<w.np * w.nq * p.splits, S::threads, 0, st>>>(w);
      return hipGetLastError();
    }
    return hipErrorInvalidConfiguration;
  });
}

// The workspace's parts are laid out by the same code that runs the steps: with `run` false only the
// size is taken.
template <class T>
hipError_t wide(hipStream_t st, const PackedView& v, const AdapterArgs& a, void* work, bool run, size_t* bytes) {
  const int ns = packed_slots(v), rp = rank_pad(a.rank), n8 = (int)up(v.n, 8);
  const bool low = a.rank > 0;
  const bool pad_x = low && !aligned16(a.x, a.ldx, v.n), pad_a = low && !aligned16(a.a, v.n, v.n);
  const bool pad_b = low && (rp != a.rank || (uintptr_t)a.b % 16);
  const WidePlan plan = wide_plan(v.m, a.t, ns, false, false);
  Arena m(work);
  uint16_t* w16 = m.take<uint16_t>((size_t)v.tiles * 16 * ns);
  uint16_t* xp = m.take<uint16_t>((size_t)a.t * ns);
  uint16_t* xpad = m.take<uint16_t>(pad_x ? (size_t)a.t * n8 : 0);
  uint16_t* apad = m.take<uint16_t>(pad_a ? (size_t)a.adapters * a.rank * n8 : 0);
  uint16_t* bpad = m.take<uint16_t>(pad_b ? (size_t)a.adapters * v.m * rp : 0);
  uint16_t* hl = m.take<uint16_t>(low ? (size_t)a.t * 2 * rp : 0);
  float* hscale = m.take<float>(low ? a.t : 0);
  const ShrinkPlan sp = shrink_plan(a.t, n8, a.adapters, rp);
  const bool tiled = low && sp.tiles;
  int* list = m.take<int>(tiled ? a.t : 0);
  int4* tiles = m.take<int4>(tiled ? sp.ntiles : 0);
  float* lowpart = m.take<float>(tiled ? (size_t)sp.splits * a.t * rp : 0);
  float* parts = m.take<float>(plan.splits > 1 ? (size_t)plan.splits * a.t * up(v.m, 4) : 0);
  *bytes = m.at;
  if (!run) return hipSuccess;
  PrepareArgs p = {};
  p.expand = expand_blocks(v);
  p.w16 = w16;
  p.slots = slot_blocks(v, a.t);
  p.slot = {a.x, a.ldx, (int)a.t, slot_rows(v), aligned16(a.x, a.ldx, v.n), xp};
  WideArgs w = {};
  const uint16_t *x = a.x, *aa = a.a, *bb = a.b;
  long ldx = a.ldx, lda = v.n;
  if (pad_x) {
    p.pads[0] = {a.x, a.ldx, v.n, n8, a.t, xpad};
    p.pad[0] = pad_blocks(p.pads[0]);
    x = xpad, ldx = n8;
  }
  if (pad_a) {
    p.pads[1] = {a.a, v.n, v.n, n8, (long)a.adapters * a.rank, apad};
    p.pad[1] = pad_blocks(p.pads[1]);
    aa = apad, lda = n8;
  }
  if (pad_b) {
    p.pads[2] = {a.b, a.rank, a.rank, rp, (long)a.adapters * v.m, bpad};
    p.pad[2] = pad_blocks(p.pads[2]);
    bb = bpad;
  }
  if (tiled) {
    p.lists = a.adapters;
    p.list = {a.request, (int)a.t, a.adapters, kItem, 0, list, nullptr, nullptr, tiles, sp.ntiles};
  }
  // The low-rank vectors of few ranks along with the rest, where they need nothing of it (2000 tokens, 2048 ->
  // 5632: 5 us less than with a launch of their own; 4096 tokens, 4096 -> 4096: 145 us and 152). Of more ranks their registers
  // would leave the other parts few wavefronts.
  const bool along = low && !tiled && !pad_x && !pad_a && rp <= 32;
  if (along) {
    p.shrink = (int)((a.t + 15) / 16);
    p.low = {x, ldx, (int)a.t, n8, aa, lda, a.rank, rp, a.adapters, a.request, a.scaling, 0, a.low, hl, hscale};
  }
  if (!along) k_prepare<T><<<p.total(), 256, slot_lds(v), st>>>(v, p);
  else if (rp <= 16) k_prepare<T, 1><<<p.total(), 256, slot_lds(v), st>>>(v, p);
  else k_prepare<T, 2><<<p.total(), 256, slot_lds(v), st>>>(v, p);
  STEP(hipGetLastError());
  if (low) {
    if (!along) STEP(shrink<T>(st, sp, list, tiles, lowpart, x, ldx, a.t, n8, aa, lda, a, 0, a.low, hl, hscale));
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
  w.parts = plan.splits > 1 ? parts : nullptr;
  STEP((wide_product<T, false>(st, plan, w)));
  if (!w.parts) return hipSuccess;
  FinishArgs f = {};
  f.sum = {parts, plan.splits, (int)a.t, v.m, (long)up(v.m, 4), nullptr, nullptr, nullptr, 0, 0, nullptr, a.y, a.ldy};
  f.nsum = (int)(a.t * ((v.m + 255) / 256));
  k_finish<T><<<launch_grid(f.total()), 256, 0, st>>>(v, f);
  return hipGetLastError();
}

// Tokens of an item: long ones write fewer sums (8 bytes a column and rank, at about 5 TB/s), short ones
// make more workgroups, of which a CU holds one (two up to rank 32); 256 tokens take one about 4 us for every
// 16 ranks (768 tokens of 64 ranks: 59 us with the first loads and the sums' stores).
int outer_chunk(long t, int adapters, int rp, int n, int m) {
  const long groups = ((n + 511) / 512 + (m + 511) / 512) * ((rp + 63) / 64), room = rp > 32 ? 256 : 512;
  int best = 1;
  double least = 0;
  for (int c = 1; c <= 16; ++c) {
    const long items = std::max<long>(adapters, (t + kItem * c - 1) / (kItem * c));
    const double cost = (double)((items * groups + room - 1) / room) * ((1.0 + 0.25 * std::min(rp, 64)) * c + 5.0) + items * rp * (8.0 / 5e6) * (n + m);
    if (c == 1 || cost < least) least = cost, best = c;
  }
  return kItem * best;
}

// The gradient's low-rank terms by dots and sums in f32, or by transposed adapters on the matrix cores: the
// dots take no preparation but go by tokens times ranks. 4096 -> 14336, a step of 64 tokens, rank 128: 320 us
// against 690; 128 tokens, rank 8: 161 and 195, rank 64: 322 and 340; 192 tokens, rank 64: 448 and 383.
inline bool few_grad(const AdapterArgs& a) { return a.t <= 128 && a.t * a.rank <= 8192; }

template <class T>
hipError_t grad(hipStream_t st, const PackedView& v, const AdapterArgs& a, void* work, bool run, size_t* bytes) {
  const int ns = packed_slots(v), rp = rank_pad(a.rank), m8 = (int)up(v.m, 8), t = (int)a.t;
  const bool low = a.rank > 0, pad = !aligned16(a.x, a.ldx, v.m), few = few_grad(a);
  const int nbn = (v.n + 127) / 128, nbm = (v.m + 127) / 128;
  const int chunk = outer_chunk(a.t, a.adapters, rp, v.n, v.m);
  const int slots = (int)(a.t / chunk) + a.adapters;
  const WidePlan plan = wide_plan(ns, a.t, v.m, true, few);
  const bool parts_out = few || plan.splits > 1;
  Arena m(work);
  uint16_t* w16 = m.take<uint16_t>((size_t)v.tiles * 16 * ns);
  uint16_t* dxp = m.take<uint16_t>(parts_out ? 0 : (size_t)a.t * ns);
  float* parts = m.take<float>(parts_out ? (size_t)plan.splits * a.t * ns : 0);
  uint16_t* dyp = m.take<uint16_t>(pad ? (size_t)a.t * m8 : 0);
  uint16_t* bt = m.take<uint16_t>(low && !few ? (size_t)a.adapters * a.rank * m8 : 0);
  uint16_t* at = m.take<uint16_t>(low && !few ? (size_t)a.adapters * ns * rp : 0);
  float* u = m.take<float>(low ? (size_t)a.t * a.rank : 0);
  uint16_t* hl = m.take<uint16_t>(low && !few ? (size_t)a.t * 2 * rp : 0);
  float* hscale = m.take<float>(low && !few ? a.t : 0);
  int* list = m.take<int>(low ? a.t : 0);
  int4* items = m.take<int4>(low ? slots : 0);
  int2* of = m.take<int2>(low ? a.adapters : 0);
  const ShrinkPlan sp = shrink_plan(a.t, m8, a.adapters, rp);
  const bool tiled = low && !few && sp.tiles;
  int4* tiles = m.take<int4>(tiled ? sp.ntiles : 0);
  float* lowpart = m.take<float>(tiled ? (size_t)sp.splits * a.t * rp : 0);
  float* part_a = m.take<float>(low ? (size_t)slots * rp * nbn * 128 : 0);
  float* part_b = m.take<float>(low ? (size_t)slots * rp * nbm * 128 : 0);
  *bytes = m.at;
  if (!run) return hipSuccess;
  const uint16_t* dy = a.x;
  long lddy = a.ldx;
  PrepareArgs p = {};
  if (t) {
    p.expand = expand_blocks(v);
    p.w16 = w16;
    if (pad) {
      p.pads[0] = {a.x, a.ldx, v.m, m8, a.t, dyp};
      p.pad[0] = pad_blocks(p.pads[0]);
      dy = dyp, lddy = m8;
    }
  }
  if (low) {
    p.a = a.a, p.b = a.b, p.adapters = a.adapters, p.rank = a.rank, p.rp = rp, p.mp = m8, p.bt = bt, p.at = at;
    p.lists = a.adapters;
    p.list = {a.request, t, a.adapters, chunk, slots, list, items, of, tiled ? tiles : nullptr, sp.ntiles};
    if (t && few) {
      p.dots = t * ((a.rank + 7) / 8);
      p.dot = {a.x, a.ldx, t, v.m, a.b, a.rank, a.adapters, a.request, a.scaling, u};
    } else if (t) {
      p.tb = blocks_for((long)a.adapters * ((a.rank + 7) / 8) * m8, 256, 8192);
      p.ta = blocks_for((long)a.adapters * (rp / 8) * ns, 256, 8192);
    }
  }
  k_prepare<T><<<p.total(), 256, 0, st>>>(v, p);
  STEP(hipGetLastError());
  WideArgs w = {};
  FinishArgs f = {};
  if (low) {
    if (t && !few) STEP(shrink<T>(st, sp, list, tiles, lowpart, dy, lddy, a.t, m8, bt, m8, a, 1, u, hl, hscale));
    const OuterJob jb = {dy, nullptr, lddy, v.m, a.low, a.scaling, part_b};
    const OuterJob ja = {a.codes, a.scales, v.n, v.n, u, nullptr, part_a};
    const bool vec = v.n % 8 == 0 && (uintptr_t)a.codes % 8 == 0;
    const int gb = (nbm + 3) / 4, ga = (nbn + 3) / 4;
    auto go = [&](auto rf) {
      constexpr int RF = decltype(rf)::value;
      const dim3 grid(gb + ga, slots, (rp + 16 * RF - 1) / (16 * RF));
      if (vec) k_outer<T, RF, true><<<grid, 512, 0, st>>>(jb, gb, ja, a.rank, rp, list, items);
      else k_outer<T, RF, false><<<grid, 512, 0, st>>>(jb, gb, ja, a.rank, rp, list, items);
      return hipGetLastError();
    };
    if (t) {
      if (rp <= 16) STEP(go(std::integral_constant<int, 1>{}));
      else if (rp <= 32) STEP(go(std::integral_constant<int, 2>{}));
      else STEP(go(std::integral_constant<int, 4>{}));
    }
    f.of = of;
    f.rank = a.rank, f.rp = rp;
    f.da = {part_a, v.n, 128l * nbn, a.da};
    f.db = {part_b, v.m, 128l * nbm, a.db};
    f.nda = a.adapters * a.rank * ((v.n + 255) / 256);
    f.ndb = a.adapters * ((a.rank + 7) / 8) * ((v.m + 255) / 256);
    if (!few) {
      w.e = at;
      w.rp = rp;
      w.adapters = a.adapters;
      w.hl = hl;
      w.hscale = hscale;
      w.request = a.request;
    }
  }
  if (t) {
    w.w = w16, w.ldw = ns, w.rows = ns, w.k = v.m;
    w.x = dy, w.ldx = lddy, w.t = t;
    w.out = dxp, w.ldo = ns;
    w.parts = parts_out ? parts : nullptr;
    STEP((wide_product<T, true>(st, plan, w)));
    if (parts_out) {
      const bool add = low && few;
      f.sum = {parts, plan.splits, t, v.n, (long)ns, v.slot, add ? a.a : nullptr, u, a.rank, a.adapters, a.request, a.y, a.ldy};
      f.nsum = t * ((v.n + 255) / 256);
      f.sum_rows = few ? 0 : (int)std::min<size_t>(4, 65536 / (4 * (size_t)v.n));
      if (f.sum_rows) f.nsum = (t + f.sum_rows - 1) / f.sum_rows;
    } else {
      f.back = {dxp, t, slot_rows(v), aligned16(a.y, a.ldy, v.n), a.y, a.ldy};
      f.nback = slot_blocks(v, t);
    }
  }
  const size_t lds = f.nback ? slot_lds(v) : 4 * (size_t)f.sum_rows * v.n;
  k_finish<T><<<launch_grid(f.total()), 256, lds, st>>>(v, f);
  return hipGetLastError();
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
