// Softmax cross entropy of hidden states over a large vocabulary, without the logits in memory.
//
//   l_tv = x_t . w_v    lse_t = log sum_v exp l_tv    loss_t = lse_t - l_t,y(t)
//   d_tv = g_t (exp(l_tv - lse_t) - [v = y(t)])    dx_t = sum_v d_tv w_v    dw_v = sum_t d_tv x_t
//
// The tokens that count (target != ignore) are packed together first: the others cost nothing and
// what they hold reaches no result. Forward: tiles of logits on the matrix cores (mma16.h), P = the
// vocabulary and Q = the tokens, so that a lane holds a token's logits in its registers: maximum and
// sum of exponentials of a tile's rows take two lane exchanges, and a (maximum, sum) pair per token
// and slab of rows is all that is stored; loss_combine joins the slabs. Gradient: pieces of the
// vocabulary; the piece's logits are made again and turned into d (16 bits) in memory, then two
// products give dx (f32 sums over the pieces) and the piece's rows of dw.
//
// d is held in the operands' 16-bit type because the matrix cores need both operands alike. bf16: scaled by
// g_t / max |g|, the largest undone in f32. f16, whose range is short: times 2^15, and where all tokens weigh the same
// without g, which dx and dw take in f32. Where they differ by g_t over its own power of two, so that a token's small
// probabilities are kept however little it weighs beside the others; dx takes the power of two in f32, and dw reads
// x with it (k_loss_weigh), exactly but for what passes f16's smallest number there.
//
// The products bound it, and those by the card's power where they are large (matrix cores busy 65-70% at
// 1.6-1.9 GHz; the library's product: 1.34-1.40 PF). d = 4096, vocabulary 128256, bf16: forward of 2048 tokens
// 1.69 ms (1.27 PF); gradient of 4096 tokens, a tenth ignored, in four pieces: d 842 us, dx 747, dw 759 each (1.15,
// 1.31, 1.29 PF of the tiles' work), joining dx 28 us.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cdclq.h"
#include "kernels.h"
#include "mma16.h"

namespace cdclq {
namespace {

constexpr float LOG2E = 1.4426950408889634f;

// Compact list of the tokens that count, in order; zero loss and lse of the others. One workgroup.
// info: [0] their number; backward only: [1] bits of max |g| over the finite g, [2] whether the g differ, [3] the
// bits of one of them.
__global__ __launch_bounds__(1024) void k_loss_tokens(const int64_t* __restrict__ y, long ignore, int t,
                                                      const float* __restrict__ g, int* __restrict__ idx,
                                                      int* __restrict__ pos, uint32_t* __restrict__ info,
                                                      float* __restrict__ loss, float* __restrict__ lse) {
  __shared__ int base;
  __shared__ int wsum[16];
  __shared__ float wmax[16];
  __shared__ uint32_t wlow[16], whigh[16];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  if (threadIdx.x == 0) base = 0;
  float m = 0.0f;
  uint32_t low = ~0u, high = 0;
  __syncthreads();
  for (int t0 = 0; t0 < t; t0 += 1024) {
    const int i = t0 + threadIdx.x;
    const bool on = i < t && y[i] != ignore;
    const uint64_t b = __builtin_amdgcn_ballot_w64(on);
    if (lane == 0) wsum[wv] = __popcll(b);
    __syncthreads();
    int at = base;
    for (int w = 0; w < wv; ++w) at += wsum[w];
    at += __popcll(b & ((1ull << lane) - 1));
    if (on) idx[at] = i;
    if (i < t) {
      if (pos) pos[i] = on ? at : -1;
      if (!on && loss) loss[i] = 0.0f;
      if (!on && lse) lse[i] = 0.0f;
      if (on && g) {
        const float a = __builtin_fabsf(g[i]);
        if (a < __builtin_inff()) m = fmaxf(m, a);
        low = min(low, __float_as_uint(g[i])), high = max(high, __float_as_uint(g[i]));
      }
    }
    __syncthreads();
    if (threadIdx.x == 0)
      for (int w = 0; w < 16; ++w) base += wsum[w];
    __syncthreads();
  }
  for (int s = 32; s; s >>= 1) {
    m = fmaxf(m, __shfl_xor(m, s));
    low = min(low, (uint32_t)__shfl_xor((int)low, s));
    high = max(high, (uint32_t)__shfl_xor((int)high, s));
  }
  if (lane == 0) wmax[wv] = m, wlow[wv] = low, whigh[wv] = high;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < 16; ++w) m = fmaxf(m, wmax[w]), low = min(low, wlow[w]), high = max(high, whigh[w]);
    info[0] = base;
    info[1] = __float_as_uint(m);
    info[2] = low < high;
    info[3] = high;
  }
}

// What the tiles need of a packed token: its target, and for the gradient lse and the scaled weight.
struct LossTok {
  int target;  // -1: outside the vocabulary
  float lse, weight;
  uint32_t xmax;  // f16, where the weights differ: pattern of its largest finite |x|
};
// f16, weights that differ: the power of two that d leaves out of g, 2^(e - 1) <= |g| < 2^e; that of the largest for
// 0, infinities and NaN
__device__ __forceinline__ int weight_exp(float g, float top) {
  const float a = __builtin_fabsf(g), b = a > 0.0f && a < __builtin_inff() ? a : top;
  return b > 0.0f ? __builtin_amdgcn_frexp_expf(b) : 0;
}
struct GatherArgs {
  const uint16_t* x;
  long ldx;
  int d, dp;
  const int64_t* y;
  int v;
  const float *lse, *g;  // gradient
  int half, weigh;       // gradient: in f16; and dw is asked for
  uint16_t* xc;
  LossTok* tok;
  float* hit;  // forward
};
// Token t as the i-th packed one: its row of x in dp elements, zeros past d, and its LossTok.
__device__ __forceinline__ void gather_token(const GatherArgs& k, int t, int i, float top, bool differ) {
  const uint16_t* src = k.x + (long)t * k.ldx;
  uint16_t* dst = k.xc + (long)i * k.dp;
  uint32_t xmax = 0;
  const bool find = k.weigh && differ;
  for (int c = 8 * threadIdx.x; c < k.dp; c += 2048) {
    uint16_t v[8];
    if (c + 8 <= k.d) {
      __builtin_memcpy(v, src + c, 16);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < k.d ? src[c + j] : (uint16_t)0;
    }
    __builtin_memcpy(__builtin_assume_aligned(dst + c, 16), v, 16);
    if (find)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t a = v[j] & 0x7fffu;
        if (a < 0x7c00u) xmax = max(xmax, a);
      }
  }
  if (find) {
    __shared__ uint32_t wx[4];
#pragma unroll
    for (int s = 32; s; s >>= 1) xmax = max(xmax, (uint32_t)__shfl_xor((int)xmax, s));
    if ((threadIdx.x & 63) == 0) wx[threadIdx.x >> 6] = xmax;
    __syncthreads();
    xmax = max(max(wx[0], wx[1]), max(wx[2], wx[3]));
  }
  if (threadIdx.x == 0) {
    const int64_t y = k.y[t];
    LossTok o;
    o.target = y >= 0 && y < k.v ? (int)y : -1;
    o.lse = k.lse ? k.lse[t] : 0.0f;
    o.weight = 0.0f;
    if (k.g) {
      const float g = k.g[t];
      if (k.half) o.weight = differ ? ldexpf(g, 15 - weight_exp(g, top)) : 0x1p15f;
      else o.weight = top > 0.0f ? g / top : g;
      if (o.target < 0) o.weight = __builtin_nanf("");
    }
    o.xmax = xmax;
    k.tok[i] = o;
    if (k.hit) k.hit[i] = __builtin_nanf("");  // replaced by the tile that holds the target
  }
}
__global__ __launch_bounds__(256) void k_loss_gather(GatherArgs k, const int* __restrict__ idx,
                                                     const uint32_t* __restrict__ info) {
  const int i = blockIdx.x;
  if (i < (int)info[0]) gather_token(k, idx[i], i, __uint_as_float(info[1]), info[2] != 0);
}
// Both of the above in one launch for few tokens: every workgroup (one a token) counts for itself, t / 256
// tokens a thread, which costs less than a launch up to kCountTokens (a forward call over 8000 x 1024: 256 tokens
// 21.6 us, 23.8 in two launches; 2048 tokens 46.7 and 48.6; 4096 tokens 86.7 and 83.4).
constexpr int kCountTokens = 2048;
__global__ __launch_bounds__(256) void k_loss_pack(GatherArgs k, long ignore, int t, int* __restrict__ idx,
                                                   int* __restrict__ pos, uint32_t* __restrict__ info,
                                                   float* __restrict__ loss, float* __restrict__ lse) {
  __shared__ int wbefore[4], wall[4];
  __shared__ float wtop[4];
  __shared__ uint32_t wlow[4], whigh[4];
  const int i = blockIdx.x, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int before = 0, all = 0;
  float top = 0.0f;
  uint32_t low = ~0u, high = 0;
  for (int j = threadIdx.x; j < t; j += 256) {
    if (k.y[j] == ignore) continue;
    ++all;
    before += j < i;
    if (k.g) {
      const float a = __builtin_fabsf(k.g[j]);
      if (a < __builtin_inff()) top = fmaxf(top, a);
      low = min(low, __float_as_uint(k.g[j])), high = max(high, __float_as_uint(k.g[j]));
    }
  }
#pragma unroll
  for (int s = 32; s; s >>= 1) {
    before += __shfl_xor(before, s);
    all += __shfl_xor(all, s);
    top = fmaxf(top, __shfl_xor(top, s));
    low = min(low, (uint32_t)__shfl_xor((int)low, s));
    high = max(high, (uint32_t)__shfl_xor((int)high, s));
  }
  if (lane == 0) wbefore[wv] = before, wall[wv] = all, wtop[wv] = top, wlow[wv] = low, whigh[wv] = high;
  __syncthreads();
  before = wbefore[0] + wbefore[1] + wbefore[2] + wbefore[3];
  all = wall[0] + wall[1] + wall[2] + wall[3];
  top = fmaxf(fmaxf(wtop[0], wtop[1]), fmaxf(wtop[2], wtop[3]));
  low = min(min(wlow[0], wlow[1]), min(wlow[2], wlow[3]));
  high = max(max(whigh[0], whigh[1]), max(whigh[2], whigh[3]));
  if (i == 0 && threadIdx.x == 0) {
    info[0] = all;
    info[1] = __float_as_uint(top);
    info[2] = low < high;
    info[3] = high;
  }
  const bool on = k.y[i] != ignore;
  if (threadIdx.x == 0) {
    if (on) idx[before] = i;
    if (pos) pos[i] = on ? before : -1;
    if (!on && loss) loss[i] = 0.0f;
    if (!on && lse) lse[i] = 0.0f;
  }
  if (on) gather_token(k, i, before, top, low < high);
}

// f16, weights that differ: xg = x 2^(up + e - E) for dw, e and E the exponents of the token's and the largest weight
// and 2^up what brings the largest |x| to f16's upper end: x keeps its bits down to weights of about 2^-20 of the
// largest. info[3] = up.
__global__ __launch_bounds__(256) void k_loss_weigh(const uint16_t* __restrict__ xc, int dp,
                                                    const LossTok* __restrict__ tok, const int* __restrict__ idx,
                                                    const float* __restrict__ g, uint32_t* __restrict__ info,
                                                    uint16_t* __restrict__ xg) {
  __shared__ uint32_t wx[4];
  const int count = (int)info[0];
  if (!info[2]) return;
  uint32_t xmax = 0;
  for (int i = threadIdx.x; i < count; i += 256) xmax = max(xmax, tok[i].xmax);
#pragma unroll
  for (int s = 32; s; s >>= 1) xmax = max(xmax, (uint32_t)__shfl_xor((int)xmax, s));
  if ((threadIdx.x & 63) == 0) wx[threadIdx.x >> 6] = xmax;
  __syncthreads();
  xmax = max(max(wx[0], wx[1]), max(wx[2], wx[3]));
  const int raise = xmax ? 16 - __builtin_amdgcn_frexp_expf(F16::widen((uint16_t)xmax)) : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) info[3] = (uint32_t)raise;
  const float top = __uint_as_float(info[1]);
  const long total = (long)count * (dp / 8);
  for (long e = blockIdx.x * 256l + threadIdx.x; e < total; e += gridDim.x * 256l) {
    const int by = raise + weight_exp(g[idx[e / (dp / 8)]], top) - weight_exp(top, top);
    uint16_t v[8];
    *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(xc + 8 * e);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = F16::narrow(ldexpf(F16::widen(v[j]), by));
    *reinterpret_cast<uint4*>(xg + 8 * e) = *reinterpret_cast<const uint4*>(v);
  }
}

__global__ __launch_bounds__(256) void k_pad16(PadJob j) { pad_rows16(j, blockIdx.x, gridDim.x); }

template <class T, int FP, int FQ, int WP, int WQ, bool U>
__global__ __launch_bounds__(64 * WP * WQ, 2) void k_loss_tiles(const uint16_t* __restrict__ w, long ldw, int v,
                                                                const uint16_t* __restrict__ xc, int dp,
                                                                const uint32_t* __restrict__ info, int np, int nq,
                                                                const LossTok* __restrict__ tok,
                                                                float2* __restrict__ part, int ldpart,
                                                                float* __restrict__ hit, int d) {
  typedef MmaTile<T, false, false, FP, FQ, WP, WQ, U> M;
  __shared__ __align__(1024) uint8_t lds[M::LDS];
  const int id = blockIdx.x + blockIdx.y * gridDim.x;
  if (id >= np * nq) return;
  const MmaTileAt at = mma_tile_at(id, np, nq);
  const int p0 = at.p * M::BP, q0 = at.q * M::BQ, count = (int)info[0];
  if (q0 >= count) return;
  mma_f4 acc[FP][FQ];
  M::clear(acc);
  M::run(lds_offset(lds), MmaOp{w, ldw, v}, MmaOp{xc, dp, count}, p0, q0, 0, U ? d : dp, acc);
  const int lane = threadIdx.x & 63;
  const int slab = M::row(p0, 0) / (16 * FP);
#pragma unroll
  for (int g = 0; g < FQ; ++g) {
    const int t = M::col(q0, g) + (lane & 15);
    const int target = t < count ? tok[t].target : -1;
    float m = -__builtin_inff();
#pragma unroll
    for (int f = 0; f < FP; ++f)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = M::row(p0, f) + 4 * (lane >> 4) + r;
        if (row >= v) acc[f][g][r] = -__builtin_inff();
        if (row == target) hit[t] = acc[f][g][r];
        m = fmaxf(m, acc[f][g][r]);
      }
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    const float top = m > -__builtin_inff() ? m : 0.0f;
    float s = 0.0f;
#pragma unroll
    for (int f = 0; f < FP; ++f)
#pragma unroll
      for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f((acc[f][g][r] - top) * LOG2E);
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (lane < 16 && t < count) part[(long)slab * ldpart + t] = make_float2(m, s);
  }
}

// Joins the slabs of 8 tokens: thread (token, j) takes slabs j, j + 128, ..., eight loads in flight.
__global__ __launch_bounds__(1024) void k_loss_combine(const float2* __restrict__ part, int ldpart, int nslabs,
                                                      const uint32_t* __restrict__ info, const int* __restrict__ idx,
                                                      const float* __restrict__ hit, float* __restrict__ loss,
                                                      float* __restrict__ lse) {
  const int count = (int)info[0], i = blockIdx.x * 8 + (threadIdx.x & 7), j = threadIdx.x >> 3;
  if ((int)blockIdx.x * 8 >= count) return;
  __shared__ float2 red[16][8];
  float m = -__builtin_inff(), s = 0.0f;
  auto join = [&](float m2, float s2) {
    const float n = fmaxf(m, m2);
    if (n > -__builtin_inff()) {
      s = s * __builtin_amdgcn_exp2f((m - n) * LOG2E) + s2 * __builtin_amdgcn_exp2f((m2 - n) * LOG2E);
      m = n;
    } else {
      s += s2;  // nothing yet, or NaN
    }
  };
  const int at = min(i, count - 1);
  for (int k = j; k < nslabs; k += 1024) {
    float2 p[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      p[u] = k + 128 * u < nslabs ? part[(long)(k + 128 * u) * ldpart + at] : make_float2(-__builtin_inff(), 0.0f);
#pragma unroll
    for (int u = 0; u < 8; ++u) join(p[u].x, p[u].y);
  }
#pragma unroll
  for (int x = 8; x < 64; x <<= 1) join(__shfl_xor(m, x), __shfl_xor(s, x));
  if ((threadIdx.x & 63) < 8) red[threadIdx.x >> 6][threadIdx.x & 7] = make_float2(m, s);
  __syncthreads();
  if (j == 0 && i < count) {
#pragma unroll
    for (int w = 1; w < 16; ++w) join(red[w][threadIdx.x].x, red[w][threadIdx.x].y);
    const float l = m + logf(s);
    lse[idx[i]] = l;
    loss[idx[i]] = l - hit[i];
  }
}

// d of vocabulary rows [v0, v0 + 256 np) for every packed token: d[t][v - v0], ld = ldd
template <class T, int FP, int FQ, int WP, int WQ, bool U>
__global__ __launch_bounds__(64 * WP * WQ, 2) void k_loss_d(const uint16_t* __restrict__ w, long ldw, int v, int v0,
                                                            const uint16_t* __restrict__ xc, int dp,
                                                            const uint32_t* __restrict__ info, int np, int nq,
                                                            const LossTok* __restrict__ tok, uint16_t* __restrict__ d,
                                                            long ldd, int dcols) {
  typedef MmaTile<T, false, false, FP, FQ, WP, WQ, U> M;
  __shared__ __align__(1024) uint8_t lds[M::LDS];
  const MmaTileAt at = mma_tile_at(blockIdx.x, np, nq);
  const int p0 = at.p * M::BP, q0 = at.q * M::BQ, count = (int)info[0];
  if (q0 >= count) return;
  mma_f4 acc[FP][FQ];
  M::clear(acc);
  M::run(lds_offset(lds), MmaOp{w + (long)v0 * ldw, ldw, v - v0}, MmaOp{xc, dp, count}, p0, q0, 0, U ? dcols : dp, acc);
  const int lane = threadIdx.x & 63;
  // from the registers: d stays in the caches, and the way through LDS costs the 256-column tiles spills
#pragma unroll
  for (int g = 0; g < FQ; ++g) {
    const int t = M::col(q0, g) + (lane & 15);
    if (t >= count) continue;
    const LossTok k = tok[t];
#pragma unroll
    for (int f = 0; f < FP; ++f) {
      const int row = M::row(p0, f) + 4 * (lane >> 4);
      float o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // the difference first: it is exact where p is near 1 and p - 1 has to be right
        const float p = __builtin_amdgcn_exp2f((acc[f][g][r] - k.lse) * LOG2E);
        o[r] = v0 + row + r < v ? (p - (v0 + row + r == k.target ? 1.0f : 0.0f)) * k.weight : 0.0f;
      }
      *reinterpret_cast<uint2*>(d + (long)t * ldd + row) = make_uint2(narrow2<T>(o[0], o[1]), narrow2<T>(o[2], o[3]));
    }
  }
}

// How a piece's dx is split over the vocabulary: about one round of workgroups for the tiles of the tokens
// that count (the host knows only how many there are at most). Both the product and the sum of its parts go
// by it. share: vocabulary entries a split.
struct DxSplit {
  int nq, splits, share;
};
__device__ __forceinline__ DxSplit dx_split(int count, int np, int bq, int piece, int round) {
  DxSplit s;
  s.nq = (count + bq - 1) / bq;
  const int n = max(1, min(round / max(1, np * s.nq), piece / 512));
  s.share = ((piece + n - 1) / n + 63) & ~63;
  s.splits = (piece + s.share - 1) / s.share;
  return s;
}

// dxacc[split][i][c] (+)= sum over the split's share of the piece's vocabulary of d[i][v] w[v0 + v][c], i the
// packed token, splits nq bq tokens apart
template <class T, int FP, int FQ, int WP, int WQ, bool U>
__global__ __launch_bounds__(64 * WP * WQ, 2) void k_loss_dx(const uint16_t* __restrict__ w, long ldw, int dcols,
                                                             int v0, int kpiece, int piece, int round,
                                                             const uint16_t* __restrict__ d, long ldd,
                                                             const uint32_t* __restrict__ info, int np, int dp,
                                                             int add, float* __restrict__ dxacc) {
  typedef MmaTile<T, true, false, FP, FQ, WP, WQ, U> M;
  __shared__ __align__(1024) uint8_t lds[M::LDS];
  const int count = (int)info[0];
  const DxSplit s = dx_split(count, np, M::BQ, piece, round);
  const int tiles = np * s.nq, split = blockIdx.x / max(1, tiles);
  if (split >= s.splits || count == 0) return;
  const MmaTileAt at = mma_tile_at(blockIdx.x - split * tiles, np, s.nq);
  const int p0 = at.p * M::BP, q0 = at.q * M::BQ;
  mma_f4 acc[FP][FQ];
  M::clear(acc);
  M::run(lds_offset(lds), MmaOp{w + (long)v0 * ldw, ldw, dcols}, MmaOp{d, ldd, count}, p0, q0, split * s.share,
         min(kpiece, (split + 1) * s.share), acc);
  const int lane = threadIdx.x & 63;
  float* out = dxacc + (long)split * s.nq * M::BQ * dp;
#pragma unroll
  for (int g = 0; g < FQ; ++g) {
    const int i = M::col(q0, g) + (lane & 15);
    if (i < count) {
#pragma unroll
      for (int f = 0; f < FP; ++f) {
        const int c = M::row(p0, f) + 4 * (lane >> 4);
        if (c >= dp) continue;
        mma_f4* o = reinterpret_cast<mma_f4*>(out + (long)i * dp + c);
        if (add) *o = *o + acc[f][g];
        else *o = acc[f][g];
      }
    }
  }
}

// dw[v0 + v][c] = sum_t d[t][v] xc[t][c], times what d and x were divided by; in f16 with weights that differ of xg
// (k_loss_weigh)
template <class T, int FP, int FQ, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ, 2) void k_loss_dw(const uint16_t* __restrict__ xc, int dp, int dcols,
                                                             const uint16_t* __restrict__ d, long ldd, int rows,
                                                             const uint32_t* __restrict__ info, int np, int nq,
                                                             const uint16_t* __restrict__ xg,
                                                             uint16_t* __restrict__ dw, long lddw) {
  typedef MmaTile<T, true, true, FP, FQ, WP, WQ> M;
  __shared__ __align__(1024) uint8_t lds[M::LDS];
  const MmaTileAt at = mma_tile_at(blockIdx.x, np, nq);
  const int p0 = at.p * M::BP, q0 = at.q * M::BQ, count = (int)info[0];
  const float top = __uint_as_float(info[1]);
  float k = top > 0.0f ? top : 1.0f;
  if constexpr (T::kind == F16::kind) {
    if (info[2]) xc = xg, k = ldexpf(1.0f, weight_exp(top, top) - 15 - (int)info[3]);
    else k = __uint_as_float(info[3]) * 0x1p-15f;
  }
  mma_f4 acc[FP][FQ];
  M::clear(acc);
  if (count > 0)
    M::run(lds_offset(lds), MmaOp{xc, dp, dp}, MmaOp{d, ldd, (int)ldd}, p0, q0, 0, count, acc);
#pragma unroll
  for (int f = 0; f < FP; ++f)
#pragma unroll
    for (int g = 0; g < FQ; ++g) acc[f][g] *= k;
  M::store(lds_offset(lds), acc, p0, q0, dcols, rows, dw, lddw);
}

// dx[t] = sum over the splits of dxacc at the token's packed place, times what its d was divided by; 0 where it does
// not count
template <class T>
__global__ __launch_bounds__(256) void k_loss_dx_out(const float* __restrict__ dxacc, int np, int bq, int piece, int round,
                                                     int t, int d, int dp,
                                                     const int* __restrict__ pos, const uint32_t* __restrict__ info,
                                                     const float* __restrict__ g, uint16_t* __restrict__ dx,
                                                     long lddx, int vec) {
  const float top = __uint_as_float(info[1]), all = top > 0.0f ? top : 1.0f;
  const DxSplit sp = dx_split((int)info[0], np, bq, piece, round);
  const long total = (long)t * dp / 4, apart = (long)sp.nq * bq * dp;
  for (long e = blockIdx.x * 256l + threadIdx.x; e < total; e += gridDim.x * 256l) {
    const int i = (int)(4 * e / dp), c = (int)(4 * e - (long)i * dp), at = pos[i];
    mma_f4 s = {};
    float k = all;
    if (at >= 0) {
      if constexpr (T::kind == F16::kind) k = info[2] ? ldexpf(1.0f, weight_exp(g[i], top) - 15) : g[i] * 0x1p-15f;
      const float* a = dxacc + (long)at * dp + c;
#pragma unroll 8
      for (int j = 0; j < sp.splits; ++j) s += *reinterpret_cast<const mma_f4*>(a + j * apart);
    }
    s *= k;
    uint16_t* o = dx + (long)i * lddx + c;
    if (vec) {
      *reinterpret_cast<uint2*>(o) = make_uint2(narrow2<T>(s[0], s[1]), narrow2<T>(s[2], s[3]));
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (c + r < d) o[r] = T::narrow(s[r]);
    }
  }
}

inline int blocks_for(long items, int per, int most = 1 << 20) {
  return (int)std::max(1l, std::min((items + per - 1) / per, (long)most));
}

// The shapes whose P may have any alignment: those that leave registers for it, all of up to 64 columns.
inline bool direct_shape(int pick) { return kMmaTimes[pick].bq <= 64; }
constexpr int kDirectTokens = 64;
template <class F>
hipError_t with_loss_shape(int pick, bool direct, F f) {
  return with_mma_shape(pick, [&](auto s) {
    if constexpr (s.bq <= kDirectTokens) {
      if (direct) return f(s, std::true_type{});
    }
    return f(s, std::false_type{});
  });
}

inline size_t up(size_t x, size_t to) { return (x + to - 1) / to * to; }

}  // namespace

// Workspace of the loss and its gradient, and where the parts lie in it.
LossPlan loss_plan(long t, long d, long v, bool pad_w, bool grad) {
  LossPlan p = {};
  t = std::max(t, 1l);  // an empty call still writes a zero dw
  p.dp = (int)up(d, 8);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up(bytes, 256);
    return o;
  };
  p.info = take(16);
  p.idx = take(4 * t);
  p.pos = take(4 * t);
  p.tok = take(sizeof(LossTok) * t);
  p.xc = take(2 * (size_t)t * p.dp);
  // Rows of W that the tiles cannot load straight into LDS: few tokens read them through registers (W is
  // what bounds them), for many a padded copy costs less (both gradients of 64 tokens, 50001 x 1001: 176 us, 203
  // with a copy; 32000 x 4097: 353 and 429).
  p.direct = pad_w && t <= kDirectTokens;
  auto pick_of = [&](long rows, long cols, long k) {
    int best = -1;
    for (int i = 0; i < kMmaShapes; ++i)
      if (!p.direct || direct_shape(i))
        if (best < 0 || mma_cost(rows, cols, k, i, 1, false) < mma_cost(rows, cols, k, best, 1, false)) best = i;
    return best;
  };
  p.wpad = pad_w && !p.direct ? take(2 * (size_t)v * p.dp) : 0;
  if (!grad) {
    p.tiles = pick_of(v, t, p.dp);
    (void)with_mma_shape(p.tiles, [&](auto s) {
      p.slab = 16 * s.fp;
      p.nslabs = (int)(up(v, s.bp) / p.slab);
      return hipSuccess;
    });
    p.hit = take(4 * t);
    p.part = take(sizeof(float2) * (size_t)t * p.nslabs);
  } else {
    // pieces of the vocabulary: d of a piece takes at most 256 MB (about what the last-level cache
    // keeps) and the whole vocabulary where that is less; beyond 2^19 tokens a piece of the least size, 256
    // entries, takes more (2 GB at 2^22)
    const size_t rows = up(v, 256), most = std::max<size_t>(256, ((size_t)128 << 20) / t / 256 * 256);
    p.pieces = (int)((rows + most - 1) / most);
    p.piece = (int)up((rows + p.pieces - 1) / p.pieces, 256);
    p.tiles = pick_of(std::min<long>(p.piece, v), t, p.dp);
    // a small dx is split over the vocabulary (dx_split); its f32 parts are written and read at about 4 TB/s.
    // The transposed reads of P cost small tiles about a third more, narrow ones twice as much.
    double best = -1;
    for (int i = 0; i < kMmaShapes; ++i) {
      if (p.direct && !direct_shape(i)) continue;
      const MmaShapeTime s = kMmaTimes[i];
      const long np = (p.dp + s.bp - 1) / s.bp, nq = (t + s.bq - 1) / s.bq, round = 256 * s.per_cu;
      const long n = std::max(1l, std::min(round / (np * nq), (long)p.piece / 512));
      const double c = mma_cost(p.dp, t, p.piece, i, n, false) * (s.bq <= 64 ? 2.0 : s.bp < 256 ? 1.33 : 1.0) + n * (8.0 / 4e6) * t * p.dp;
      if (best < 0 || c < best) {
        best = c;
        p.dx_tiles = i;
        p.dx_round = (int)round;
        p.dx_bytes = 4 * (size_t)p.dp * std::max<size_t>(up(t, s.bq), (size_t)(round / np) * s.bq);
      }
    }
    // few tokens: dw's stores are what costs, and two small tiles on a CU overlap theirs with each other's loads
    // (62 tokens, 50001 x 1000: 36 us, large tiles 42; 64, 128256 x 4096: 363 and 370; 300: 664 and 580)
    p.dw_tiles = t <= 192 || mma_cost(p.dp, p.piece, t, 4, 1, false) < mma_cost(p.dp, p.piece, t, 0, 1, false) ? 4 : 0;
    p.xg = take(2 * (size_t)t * p.dp);  // f16 alone writes it
    p.d = take(2 * (size_t)t * p.piece);
    p.dxacc = take(p.dx_bytes);
  }
  p.bytes = at;
  return p;
}

namespace {

// The packed tokens, and W where the tiles cannot read it as it is
hipError_t prepare(hipStream_t st, const LossArgs& a, const LossPlan& p, bool half, const uint16_t** w, long* ldw) {
  char* ws = static_cast<char*>(a.work);
  const bool grad = a.dx || a.dw;
  int *idx = reinterpret_cast<int*>(ws + p.idx), *pos = grad ? reinterpret_cast<int*>(ws + p.pos) : nullptr;
  uint32_t* info = reinterpret_cast<uint32_t*>(ws + p.info);
  float *loss = grad ? nullptr : a.loss, *lse = grad ? nullptr : a.lse_out;
  const GatherArgs k = {a.x, a.ldx, (int)a.d, p.dp, a.targets, (int)a.v, a.lse_in, a.dloss,
                        grad && half, grad && half && a.dw, reinterpret_cast<uint16_t*>(ws + p.xc), reinterpret_cast<LossTok*>(ws + p.tok),
                        grad ? nullptr : reinterpret_cast<float*>(ws + p.hit)};
  if (a.t > 0 && a.t <= kCountTokens) {
    k_loss_pack<<<(int)a.t, 256, 0, st>>>(k, a.ignore, (int)a.t, idx, pos, info, loss, lse);
  } else {
    k_loss_tokens<<<1, 1024, 0, st>>>(a.targets, a.ignore, (int)a.t, a.dloss, idx, pos, info, loss, lse);
    if (a.t) k_loss_gather<<<(int)a.t, 256, 0, st>>>(k, idx, info);
  }
  *w = a.w;
  *ldw = a.ldw;
  if (p.wpad) {
    uint16_t* wp = reinterpret_cast<uint16_t*>(ws + p.wpad);
    const PadJob j = {a.w, a.ldw, (int)a.d, p.dp, a.v, wp};
    k_pad16<<<blocks_for(a.v * (p.dp / 8), 256 * 2, 1 << 16), 256, 0, st>>>(j);
    *w = wp;
    *ldw = p.dp;
  }
  return hipGetLastError();
}

template <class T>
hipError_t forward(hipStream_t st, const LossArgs& a, const LossPlan& p) {
  char* ws = static_cast<char*>(a.work);
  const uint16_t* w;
  long ldw;
  hipError_t e = prepare(st, a, p, false, &w, &ldw);
  if (e != hipSuccess) return e;
  e = with_loss_shape(p.tiles, p.direct, [&](auto s, auto u) {
    typedef decltype(s) S;
    const int np = (int)((a.v + S::bp - 1) / S::bp), nq = (int)((a.t + S::bq - 1) / S::bq);
    k_loss_tiles<T, S::fp, S::fq, S::wp, S::wq, decltype(u)::value><<<launch_grid((long)np * nq), S::threads, 0, st>>>(
        w, ldw, (int)a.v, reinterpret_cast<uint16_t*>(ws + p.xc), p.dp, reinterpret_cast<uint32_t*>(ws + p.info), np, nq,
        reinterpret_cast<LossTok*>(ws + p.tok), reinterpret_cast<float2*>(ws + p.part), (int)a.t,
        reinterpret_cast<float*>(ws + p.hit), (int)a.d);
    return hipGetLastError();
  });
  if (e != hipSuccess) return e;
  k_loss_combine<<<(int)((a.t + 7) / 8), 1024, 0, st>>>(
      reinterpret_cast<float2*>(ws + p.part), (int)a.t, p.nslabs, reinterpret_cast<uint32_t*>(ws + p.info),
      reinterpret_cast<int*>(ws + p.idx), reinterpret_cast<float*>(ws + p.hit), a.loss, a.lse_out);
  return hipGetLastError();
}

template <class T>
hipError_t backward(hipStream_t st, const LossArgs& a, const LossPlan& p) {
  char* ws = static_cast<char*>(a.work);
  constexpr bool half = T::kind == F16::kind;
  const uint16_t* w;
  long ldw;
  hipError_t e = prepare(st, a, p, half, &w, &ldw);
  if (e != hipSuccess) return e;
  uint32_t* info = reinterpret_cast<uint32_t*>(ws + p.info);
  uint16_t* xc = reinterpret_cast<uint16_t*>(ws + p.xc);
  uint16_t* d = reinterpret_cast<uint16_t*>(ws + p.d);
  float* dxacc = reinterpret_cast<float*>(ws + p.dxacc);
  LossTok* tok = reinterpret_cast<LossTok*>(ws + p.tok);
  uint16_t* xg = reinterpret_cast<uint16_t*>(ws + p.xg);
  const int t = (int)a.t, v = (int)a.v;
  if (half && a.dw && t) {
    k_loss_weigh<<<blocks_for((long)t * (p.dp / 8), 256 * 4, 512), 256, 0, st>>>(xc, p.dp, tok, reinterpret_cast<int*>(ws + p.idx), a.dloss, info, xg);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  for (int i = 0; i < p.pieces; ++i) {
    const int v0 = i * p.piece;
    if (v0 >= v) break;
    const int rows = std::min(p.piece, v - v0);
    if (t) {
      e = with_loss_shape(p.tiles, p.direct, [&](auto s, auto u) {
        typedef decltype(s) S;
        const int nq = (t + S::bq - 1) / S::bq, np = (rows + S::bp - 1) / S::bp;
        k_loss_d<T, S::fp, S::fq, S::wp, S::wq, decltype(u)::value><<<np * nq, S::threads, 0, st>>>(
            w, ldw, v, v0, xc, p.dp, info, np, nq, tok, d, p.piece, (int)a.d);
        return hipGetLastError();
      });
      if (e != hipSuccess) return e;
      e = with_loss_shape(p.dx_tiles, p.direct, [&](auto s, auto u) {
        typedef decltype(s) S;
        const int nq = (t + S::bq - 1) / S::bq, np = (p.dp + S::bp - 1) / S::bp;
        k_loss_dx<T, S::fp, S::fq, S::wp, S::wq, decltype(u)::value><<<std::max(np * nq, p.dx_round), S::threads, 0, st>>>(
            w, ldw, (int)a.d, v0, rows, p.piece, p.dx_round, d, p.piece, info, np, p.dp, i > 0, dxacc);
        return hipGetLastError();
      });
      if (e != hipSuccess) return e;
    }
    if (a.dw) {
      auto go = [&](auto s) {
        typedef decltype(s) S;
        const int np = (p.dp + S::bp - 1) / S::bp, nq = (rows + S::bq - 1) / S::bq;
        k_loss_dw<T, S::fp, S::fq, S::wp, S::wq><<<np * nq, S::threads, 0, st>>>(
            xc, p.dp, (int)a.d, d, p.piece, rows, info, np, nq, xg, a.dw + (long)v0 * a.lddw, a.lddw);
        return hipGetLastError();
      };
      e = p.dw_tiles == 4 ? go(MmaShape<4, 4, 2, 2>{}) : go(MmaShape<8, 4, 2, 4>{});
      if (e != hipSuccess) return e;
    }
  }
  const int vec = a.lddx % 4 == 0 && a.d % 4 == 0 && p.dp == a.d && (uintptr_t)a.dx % 8 == 0;
  if (t) {
    const MmaShapeTime s = kMmaTimes[p.dx_tiles];
    k_loss_dx_out<T><<<blocks_for((long)t * p.dp, 4 * 256), 256, 0, st>>>(
        dxacc, (p.dp + s.bp - 1) / s.bp, s.bq, p.piece, p.dx_round, t, (int)a.d, p.dp, reinterpret_cast<int*>(ws + p.pos),
        info, a.dloss, a.dx, a.lddx, vec);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t loss_forward(hipStream_t st, int dtype, const LossArgs& a, const LossPlan& p) {
  return dtype == CDCLQ_DTYPE_BF16 ? forward<Bf16>(st, a, p) : forward<F16>(st, a, p);
}
hipError_t loss_backward(hipStream_t st, int dtype, const LossArgs& a, const LossPlan& p) {
  return dtype == CDCLQ_DTYPE_BF16 ? backward<Bf16>(st, a, p) : backward<F16>(st, a, p);
}

}  // namespace cdclq
