// The packed projection for few tokens (a decode step), and the kernels that build and expand the
// layout of packed.h.
//
// y_t = W x_t + scaling_q B_q (A_q x_t), W the packed layer, q the adapter of token t's request.
//
// Few tokens: the packed weights are read once and decoded in registers. A wavefront takes every 8th
// block of 128 slots of RT x 16 rows, all tokens at once (NT fragments of 16 tokens as the columns of
// 16x16x32 MFMAs). Per group run: sum of (2^b + q) x on the matrix cores, exact operands, f32 sums; then
// scale (that - (2^b + zero) sum x) in f32, so that no weight is ever rounded. The wavefronts' sums
// meet in LDS, where the low-rank term is added in f32. What bounds it is the read of the codes, for few rows
// the latency of the first of them: 32 tokens of 32 adapters of rank 16, 4096 -> 14336 in 4 bits: 15.8 us
// (46 MB, 2.9 TB/s); one token, 4096 -> 4096: 5.2 us. Every 64 tokens decode the codes again, and the matrix cores
// and the decoding bound it then: 64 tokens, 4096 -> 14336: 33 us a call, 128: 58, 192: 84. k_few_inputs before it
// takes 4-6 us, of which the launch and the loads' latency are most.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cdclq.h"
#include "kernels.h"
#include "packed.h"

namespace cdclq {
namespace {

// One lane's codes of one block, from the container's bit stream. Once per layer: 14336 x 4096 in 4 bits 239 us.
__global__ __launch_bounds__(64) void k_packed_layout(PackedView v, const uint8_t* __restrict__ qw, long rb,
                                                      const int* __restrict__ slotpos,
                                                      const uint32_t* __restrict__ coff,
                                                      const uint8_t* __restrict__ cwid, uint8_t* __restrict__ codes) {
  const int kb = blockIdx.x, lane = threadIdx.x, q = lane >> 4;
  const long tile = blockIdx.y + (long)blockIdx.z * gridDim.y;
  if (tile >= v.tiles) return;
  const uint32_t info = v.kinfo[kb];
  const int b = info & 15;
  const long row = tile * 16 + (lane & 15);
  uint32_t p4[2][4] = {}, p2[2] = {}, p1 = 0;
  for (int s = 0; s < 4; ++s)
    for (int i = 0; i < 8; ++i) {
      const int j = slotpos[kb * 128 + 32 * s + 8 * q + i];
      if (j < 0 || row >= v.m) continue;
      const uint32_t o = coff[j], at = o >> 3;
      const uint8_t* src = qw + row * rb;
      uint32_t w = src[at];
      if ((long)at + 1 < rb) w |= (uint32_t)src[at + 1] << 8;
      const uint32_t c = (w >> (o & 7)) & ((1u << cwid[j]) - 1);
      const int p = i >> 1, h = 16 * (i & 1);
      if (b == 8) {
        p4[0][s] |= (c & 15) << (4 * p + h);
        p4[1][s] |= (c >> 4) << (4 * p + h);
        continue;
      }
      if (b & 4) p4[0][s] |= (c & 15) << (4 * p + h);
      if (b & 2) p2[s >> 1] |= ((c >> (b & 4)) & 3) << (8 * (s & 1) + 2 * p + h);
      if (b & 1) p1 |= ((c >> (b & 6)) & 1) << (4 * s + p + h);
    }
  uint8_t* at = codes + tile * v.tile_bytes + 256l * (info >> 8);
  if (b & 12) {
    *reinterpret_cast<uint4*>(at + 16 * lane) = make_uint4(p4[0][0], p4[0][1], p4[0][2], p4[0][3]);
    at += 1024;
  }
  if (b == 8) *reinterpret_cast<uint4*>(at + 16 * lane) = make_uint4(p4[1][0], p4[1][1], p4[1][2], p4[1][3]);
  if (b == 8) return;
  if (b & 2) {
    *reinterpret_cast<uint2*>(at + 8 * lane) = make_uint2(p2[0], p2[1]);
    at += 512;
  }
  if (b & 1) *reinterpret_cast<uint32_t*>(at + 4 * lane) = p1;
}

__global__ __launch_bounds__(256) void k_packed_scales(PackedView v, int ng_in, const uint16_t* __restrict__ s16,
                                                       const uint8_t* __restrict__ qz, uint32_t* __restrict__ scl) {
  const long total = (long)v.tiles * v.ng * 16;
  for (long e = blockIdx.x * 256l + threadIdx.x; e < total; e += gridDim.x * 256l) {
    const long row = e / (16l * v.ng) * 16 + (e & 15);
    const int g = (int)(e / 16 % v.ng);
    scl[e] = row < v.m ? (uint32_t)s16[row * ng_in + g] | ((uint32_t)qz[row * ng_in + g] << 16) : 0u;
  }
}

// Activations of few tokens as MFMA operands, xf[step][fragment][lane][8], with the running sums of x
// over a block's steps, sx[step][token]; and low = A x of every token with an adapter (0 without), one
// wavefront per (token, rank). Workgroups below nx do the former.
template <class T>
__global__ __launch_bounds__(256) void k_few_inputs(PackedView v, int nx, int nt, const uint16_t* __restrict__ x,
                                                    long ldx, int t, uint16_t* __restrict__ xf,
                                                    float* __restrict__ sx, const uint16_t* __restrict__ a, int rank,
                                                    int adapters, const int* __restrict__ request,
                                                    float* __restrict__ low, int vec) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  if ((int)blockIdx.x < nx) {  // a block of slots and a fragment of tokens, a step each wavefront
    __shared__ float sums[4][16];
    const int kb = blockIdx.x / nt, g = blockIdx.x - kb * nt, step = 4 * kb + wv;
    const int tok = 16 * g + (lane & 15), q = lane >> 4;
    float part = 0.0f;
    if (tok < t) {
      const int4 c0 = *reinterpret_cast<const int4*>(v.col + 32 * step + 8 * q);
      const int4 c1 = *reinterpret_cast<const int4*>(v.col + 32 * step + 8 * q + 4);
      const int c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
      const uint16_t* src = x + (long)tok * ldx;
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = src[max(c[i], 0)];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (c[i] < 0) o[i] = 0;
        part += T::widen((uint16_t)o[i]);
      }
      *reinterpret_cast<uint4*>(xf + ((long)(step * nt + g) * 64 + lane) * 8) =
          make_uint4(o[0] | o[1] << 16, o[2] | o[3] << 16, o[4] | o[5] << 16, o[6] | o[7] << 16);
    }
    part += __shfl_xor(part, 16);
    part += __shfl_xor(part, 32);
    if (lane < 16) sums[wv][lane] = part;
    __syncthreads();
    if (lane < 16) {
      float sum = sums[0][lane];
      for (int w = 1; w <= wv; ++w) sum += sums[w][lane];
      sx[step * 16 * nt + tok] = sum;
    }
    return;
  }
  const long id = (blockIdx.x - nx) * 4l + wv;
  if (id >= (long)t * rank) return;
  const int tok = (int)(id / rank), j = (int)(id - (long)tok * rank), q = request[tok];
  float s = 0.0f;
  if (q >= 0 && q < adapters) {
    const uint16_t *xr = x + (long)tok * ldx, *ar = a + ((long)q * rank + j) * v.n;
    if (vec) {
      for (int c0 = 8 * lane; c0 < v.n; c0 += 2048) {  // four steps' loads in flight
        uint4 xv[4], av[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = c0 + 512 * u;
          xv[u] = av[u] = make_uint4(0, 0, 0, 0);
          if (c < v.n) {
            xv[u] = *reinterpret_cast<const uint4*>(xr + c);
            av[u] = *reinterpret_cast<const uint4*>(ar + c);
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint16_t *xe = reinterpret_cast<const uint16_t*>(&xv[u]), *ae = reinterpret_cast<const uint16_t*>(&av[u]);
#pragma unroll
          for (int i = 0; i < 8; ++i) s = __builtin_fmaf(T::widen(xe[i]), T::widen(ae[i]), s);
        }
      }
    } else {
      for (int c0 = 8 * lane; c0 < v.n; c0 += 512)  // the same order
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c0 + i < v.n) s = __builtin_fmaf(T::widen(xr[c0 + i]), T::widen(ar[c0 + i]), s);
    }
#pragma unroll
    for (int k = 32; k; k >>= 1) s += __shfl_xor(s, k);
  }
  if (lane == 0) low[id] = s;
}

struct FewArgs {
  const uint16_t* xf;
  const float* sx;
  int t, frags;  // of 16 tokens, in xf and sx
  const uint16_t* b;  // adapters x m x rank, null: none
  const float* scaling;
  int adapters, rank, vec;  // vec: b's rows can be read 8 ranks at a time
  const int* request;
  const float* low;
  uint16_t* y;
  long ldy;
};

template <class T, int B, int RT, int NT, int W>
__global__ __launch_bounds__(64 * W) void k_packed_few(PackedView v, FewArgs k) {
  __shared__ float red[W][RT * 16][16 * NT + 1];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long tile0 = (long)blockIdx.x * RT;
  const int first = 16 * NT * blockIdx.y, nt = k.frags, t = k.t - first;  // this workgroup's tokens
  const int* const request = k.request + first;
  const uint16_t* const xf = k.xf + 512l * NT * blockIdx.y;
  const float* const sx = k.sx + first;
  mma_f4 acc[RT][NT], run[RT][NT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int g = 0; g < NT; ++g) acc[i][g] = run[i][g] = mma_f4{};
  const uint8_t* base[RT];
  const uint32_t* scl[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const long tile = min(tile0 + i, (long)v.tiles - 1);
    base[i] = v.codes + tile * v.tile_bytes;
    scl[i] = v.scl + tile * v.ng * 16 + 4 * (lane >> 4);
  }
  // The first 8 (16) ranks of B for this thread's results are asked for here: they come from HBM
  // while the codes are worked on.
  constexpr int OUT = (RT * 16 * 16 * NT + 64 * W - 1) / (64 * W);
  uint4 early[OUT][2];
  if (k.b && k.vec) {
#pragma unroll
    for (int i = 0; i < OUT; ++i) {
      const int e = threadIdx.x + i * 64 * W, tok = e / (RT * 16);
      const long row = tile0 * 16 + (e - tok * (RT * 16));
      early[i][0] = early[i][1] = make_uint4(0, 0, 0, 0);
      const int q = tok < t ? request[tok] : -1;
      if (q >= 0 && q < k.adapters && row < v.m) {
        const uint16_t* br = k.b + ((long)q * v.m + row) * k.rank;
        early[i][0] = *reinterpret_cast<const uint4*>(br);
        if (k.rank >= 16) early[i][1] = *reinterpret_cast<const uint4*>(br + 8);
      }
    }
  }
  PackedRegs next[RT] = {};
  uint32_t ninfo = 0;
  if (wv < v.nkb) {
    ninfo = __builtin_amdgcn_readfirstlane(v.kinfo[wv]);
#pragma unroll
    for (int i = 0; i < RT; ++i) packed_load<B>(base[i] + 256l * (ninfo >> 8), lane, ninfo & 15, next[i]);
  }
  for (int kb = wv; kb < v.nkb; kb += W) {
    const uint32_t info = ninfo;
    PackedRegs cur[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) cur[i] = next[i];
    typename T::v8 xv[4][NT];
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int g = 0; g < NT; ++g) {
        mma_u4 u = {};
        if (16 * g + (lane & 15) < t)
          u = *reinterpret_cast<const mma_u4*>(xf + ((long)((4 * kb + s) * nt + g) * 64 + lane) * 8);
        xv[s][g] = __builtin_bit_cast(typename T::v8, u);
      }
    // scales and sums at the block's end, where a run always ends
    mma_u4 sz3[RT];
    float sx3[NT];
    const uint32_t g3 = v.grp[4 * kb + 3];
#pragma unroll
    for (int i = 0; i < RT; ++i) sz3[i] = *reinterpret_cast<const mma_u4*>(scl[i] + 16 * g3);
#pragma unroll
    for (int g = 0; g < NT; ++g) sx3[g] = sx[(4 * kb + 3) * 16 * nt + 16 * g + (lane & 15)];
    if (kb + W < v.nkb) {
      ninfo = __builtin_amdgcn_readfirstlane(v.kinfo[kb + W]);
#pragma unroll
      for (int i = 0; i < RT; ++i) packed_load<B>(base[i] + 256l * (ninfo >> 8), lane, ninfo & 15, next[i]);
    }
    float before[NT];
#pragma unroll
    for (int g = 0; g < NT; ++g) before[g] = 0.0f;
    auto block = [&](auto bc) {
      constexpr int BB = decltype(bc)::value;
      auto step = [&](auto sc) {
        constexpr int S = decltype(sc)::value;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          typename T::v8 lo, hi;
          packed_step<T, BB, S>(cur[i], lo, hi);
#pragma unroll
          for (int g = 0; g < NT; ++g) {
            run[i][g] = T::mfma(lo, xv[S][g], run[i][g]);
            if constexpr (BB == 8 && T::kind == Bf16::kind) run[i][g] = T::mfma(hi, xv[S][g], run[i][g]);
          }
        }
        if (S == 3 || (info >> (4 + S)) & 1) {
          mma_u4 sz[RT];
          float sum[NT];
          if constexpr (S == 3) {
#pragma unroll
            for (int i = 0; i < RT; ++i) sz[i] = sz3[i];
#pragma unroll
            for (int g = 0; g < NT; ++g) sum[g] = sx3[g];
          } else {
            const uint32_t gi = v.grp[4 * kb + S];
#pragma unroll
            for (int i = 0; i < RT; ++i) sz[i] = *reinterpret_cast<const mma_u4*>(scl[i] + 16 * gi);
#pragma unroll
            for (int g = 0; g < NT; ++g) sum[g] = sx[(4 * kb + S) * 16 * nt + 16 * g + (lane & 15)];
          }
#pragma unroll
          for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int g = 0; g < NT; ++g) {
              const float x = sum[g] - before[g];
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float part =
                    __builtin_fmaf(-(packed_offset<T, BB>() + packed_zero(sz[i][r])), x, run[i][g][r]);
                acc[i][g][r] = __builtin_fmaf(packed_scale(sz[i][r]), part, acc[i][g][r]);
              }
              run[i][g] = mma_f4{};
            }
#pragma unroll
          for (int g = 0; g < NT; ++g) before[g] = sum[g];
        }
      };
      step(std::integral_constant<int, 0>{});
      step(std::integral_constant<int, 1>{});
      step(std::integral_constant<int, 2>{});
      step(std::integral_constant<int, 3>{});
    };
    if constexpr (B != 0) {
      block(std::integral_constant<int, B>{});
    } else {
      switch (info & 15) {
        case 1: block(std::integral_constant<int, 1>{}); break;
        case 2: block(std::integral_constant<int, 2>{}); break;
        case 3: block(std::integral_constant<int, 3>{}); break;
        case 4: block(std::integral_constant<int, 4>{}); break;
        case 5: block(std::integral_constant<int, 5>{}); break;
        case 6: block(std::integral_constant<int, 6>{}); break;
        case 7: block(std::integral_constant<int, 7>{}); break;
        default: block(std::integral_constant<int, 8>{}); break;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int g = 0; g < NT; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[wv][16 * i + 4 * (lane >> 4) + r][16 * g + (lane & 15)] = acc[i][g][r];
  __syncthreads();
  auto dot8 = [&](const uint4& u, const float* lo) {
    const uint16_t* b = reinterpret_cast<const uint16_t*>(&u);
    float d = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) d = __builtin_fmaf(T::widen(b[j]), lo[j], d);
    return d;
  };
#pragma unroll
  for (int i = 0; i < OUT; ++i) {
    const int e = threadIdx.x + i * 64 * W, tok = e / (RT * 16), r = e - tok * (RT * 16);
    const long row = tile0 * 16 + r;
    if (tok >= t || row >= v.m) continue;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) s += red[w][r][tok];
    if (k.b) {
      const int q = request[tok];
      if (q >= 0 && q < k.adapters) {
        const uint16_t* br = k.b + ((long)q * v.m + row) * k.rank;
        const float* lo = k.low + (long)(first + tok) * k.rank;
        float d = 0.0f;
        if (k.vec) {
          d = dot8(early[i][0], lo);
          if (k.rank >= 16) d += dot8(early[i][1], lo + 8);
          for (int j = 16; j < k.rank; j += 8) d += dot8(*reinterpret_cast<const uint4*>(br + j), lo + j);
        } else {
          int j0 = 0;  // the same order
#pragma unroll 4
          for (; j0 + 8 <= k.rank; j0 += 8) {
            uint4 u;
            __builtin_memcpy(&u, br + j0, 16);
            d += dot8(u, lo + j0);
          }
          float p = 0.0f;
          for (int j = j0; j < k.rank; ++j) p = __builtin_fmaf(T::widen(br[j]), lo[j], p);
          d += p;
        }
        s = __builtin_fmaf(k.scaling[q], d, s);
      } else if (q != -1) {
        s = __builtin_nanf("");  // no such adapter
      }
    }
    k.y[(first + tok) * k.ldy + row] = T::narrow(s);
  }
}

template <class T, int B, int NT>
hipError_t few_tiles(hipStream_t st, const PackedView& v, const FewArgs& k) {
  // Two row tiles share the activations' operands where that leaves two workgroups a CU (14336 rows of
  // 4096, 32 tokens: 16 us with two, 21 with one); few rows take 16 wavefronts each (4096 rows of 4096, a
  // token: 5.3 us, 6.0 with eight; 1001 of 1350: 4.6 and 5.0).
  const int groups = (k.t + 16 * NT - 1) / (16 * NT);
  if (v.tiles >= 512) k_packed_few<T, B, 2, NT, 8><<<dim3((v.tiles + 1) / 2, groups), 512, 0, st>>>(v, k);
  else if (v.tiles <= 256) k_packed_few<T, B, 1, NT, 16><<<dim3(v.tiles, groups), 1024, 0, st>>>(v, k);
  else k_packed_few<T, B, 1, NT, 8><<<dim3(v.tiles, groups), 512, 0, st>>>(v, k);
  return hipGetLastError();
}
template <class T, int B>
hipError_t few_tokens(hipStream_t st, const PackedView& v, const FewArgs& k) {
  if (k.t <= 16) return few_tiles<T, B, 1>(st, v, k);
  if (k.t <= 32) return few_tiles<T, B, 2>(st, v, k);
  return few_tiles<T, B, 4>(st, v, k);
}
inline int few_frags(long t) { return t <= 16 ? 1 : t <= 32 ? 2 : (int)((t + 63) / 64 * 4); }

template <class T>
hipError_t few(hipStream_t st, const PackedView& v, const AdapterArgs& a, void* work) {
  const int nt = few_frags(a.t), steps = 4 * v.nkb;
  uint16_t* xf = static_cast<uint16_t*>(work);
  float* sx = reinterpret_cast<float*>(xf + (size_t)steps * nt * 512);
  float* low = a.low ? a.low : sx + (size_t)steps * nt * 16;
  const int nx = v.nkb * nt;
  const long nlow = a.rank ? ((long)a.t * a.rank + 3) / 4 : 0;
  const int vec = v.n % 8 == 0 && a.ldx % 8 == 0 && (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.a % 16 == 0;
  k_few_inputs<T><<<(int)(nx + nlow), 256, 0, st>>>(v, nx, nt, a.x, a.ldx, (int)a.t, xf, sx, a.a, a.rank, a.adapters,
                                                    a.request, low, vec);
  FewArgs k = {xf, sx, (int)a.t, nt, a.rank ? a.b : nullptr, a.scaling, a.adapters, a.rank,
               a.rank % 8 == 0 && (uintptr_t)a.b % 16 == 0, a.request, low, a.y, a.ldy};
  switch (v.bits) {
    case 2: return few_tokens<T, 2>(st, v, k);
    case 3: return few_tokens<T, 3>(st, v, k);
    case 4: return few_tokens<T, 4>(st, v, k);
    case 8: return few_tokens<T, 8>(st, v, k);
    default: return few_tokens<T, 0>(st, v, k);
  }
}

}  // namespace

hipError_t packed_layout(hipStream_t st, const PackedView& v, int ng_in, const uint8_t* qw, long rb,
                         const uint16_t* s16, const uint8_t* qz, const int* slotpos, const uint32_t* coff,
                         const uint8_t* cwid, uint8_t* codes, uint32_t* scl) {
  const int gy = std::min(v.tiles, 32768), gz = (v.tiles + gy - 1) / gy;
  k_packed_layout<<<dim3(v.nkb, gy, gz), 64, 0, st>>>(v, qw, rb, slotpos, coff, cwid, codes);
  k_packed_scales<<<std::min(4096, (int)(((long)v.tiles * v.ng * 16 + 255) / 256)), 256, 0, st>>>(v, ng_in, s16, qz, scl);
  return hipGetLastError();
}

size_t few_work_bytes(const PackedView& v, long t, long rank) {
  const size_t steps = 4 * (size_t)v.nkb, nt = few_frags(t);
  return steps * nt * 1024 + steps * nt * 64 + 4 * (size_t)t * rank;
}
hipError_t adapter_few(hipStream_t st, int dtype, const PackedView& v, const AdapterArgs& a, void* work) {
  return dtype == CDCLQ_DTYPE_BF16 ? few<Bf16>(st, v, a, work) : few<F16>(st, v, a, work);
}

}  // namespace cdclq
