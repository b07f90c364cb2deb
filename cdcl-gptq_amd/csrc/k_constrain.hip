// Penalties for tokens that a request has had, its biases and its grammar's mask on the logits of a decode step.
//
//   c = how often the request has generated v, s = whether v is in its history (prompt or generated)
//   l1 = s ? (l > 0 ? l / rep : l rep) : l      l2 = l1 - (freq c + (c > 0 ? pres : 0))      l3 = l2 + bias of v
//   out = -inf where the mask's bit of v is 0, else l3
//
// in f32, in this order, rounded once; what nothing applies to keeps its bits. Memory bounds it: the logits are read
// and written once. A workgroup takes a slab of one request's vocabulary. Its logits are asked for first; while they
// come it counts the history's tokens of its slab in LDS, a word a token:
//   bit 31 in the prompt      bits 30..20 the token's bias + 1      bits 19..0 times generated
// (whole numbers: the order of the additions does not matter). Every slab of a request reads the whole history, so
// slabs are as large as leaves enough workgroups, and a request's slabs lie on one XCD, whose L2 then holds its
// history. In place, only what changes is read or written, and tokens that the mask shuts out are not read.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cdclq.h"
#include "kernels.h"
#include "row8.h"

namespace cdclq {
namespace {

constexpr uint32_t kPrompt = 1u << 31, kCount = (1u << 20) - 1, kBias = 2047u << 20;


// LDS: TH * 8 * K words if there is a history or a bias, then the biases' values and places.
template <class T, int TH, int K, bool PLACE>
__global__ __launch_bounds__(TH) void k_constrain(ConstrainArgs a, long rows8, int slabs) {
  extern __shared__ __align__(16) uint32_t word[];
  constexpr int SLAB = TH * 8 * K;
  // workgroup b: XCD b % 8 takes the requests of that remainder, slab by slab
  const long b = blockIdx.x + (long)blockIdx.y * gridDim.x, at = b >> 3;
  const long row = (at / slabs) * 8 + (b & 7);
  if (at >= rows8 * slabs || row >= a.r) return;
  const int slab0 = (int)(at % slabs) * SLAB;  // 8 workgroups later the next slab
  const auto* in = static_cast<const typename Row8<T>::stored*>(a.logits) + row * a.ld + slab0;
  auto* out = static_cast<typename Row8<T>::stored*>(a.out) + row * a.ldo + slab0;
  const int n = (int)min((long)SLAB, a.v - slab0);
  const bool marks = a.history || a.biases;

  Row8<T> x[K];
  if constexpr (!PLACE) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = 8 * (k * TH + (int)threadIdx.x);
      if (i + 8 <= n) x[k] = row8_load<T>(in + i);
    }
  }
  const long mrow = a.mask_rows ? a.mask_rows[row] : a.mask ? row : -1;
  const bool wrong = mrow < -1 || (mrow >= 0 && mrow >= a.masks);  // no such mask
  const uint8_t* mask = mrow < 0 || wrong ? nullptr
                                          : reinterpret_cast<const uint8_t*>(a.mask + mrow * a.ldm) + slab0 / 8;
  uint8_t open[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = k * TH + (int)threadIdx.x;
    open[k] = mask && 8 * i < n ? mask[i] : 0xff;
  }
  float* const bias = reinterpret_cast<float*>(word + SLAB);
  if (marks) {
    int* const place = reinterpret_cast<int*>(bias + a.biases);
#pragma unroll
    for (int k = 0; k < 2 * K; ++k) reinterpret_cast<uint4*>(word)[k * TH + threadIdx.x] = make_uint4(0, 0, 0, 0);
    for (int i = threadIdx.x; i < a.biases; i += TH) {
      const int64_t tok = a.bias_tokens[row * a.biases + i] - slab0;
      place[i] = (uint64_t)tok < (uint64_t)n ? (int)tok : -1;
    }
    __syncthreads();
    if (a.history) {
      const int len = a.lengths ? max(0, min(a.lengths[row], a.width)) : a.width;
      const int prompt = a.prompts ? a.prompts[row] : 0;
      const int64_t* h = a.history + row * a.ldh;
      for (int i0 = threadIdx.x; i0 < len; i0 += 8 * TH) {
        int64_t tok[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) tok[u] = i0 + u * TH < len ? h[i0 + u * TH] - slab0 : -1;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          if ((uint64_t)tok[u] >= (uint64_t)n) continue;
          if (i0 + u * TH < prompt) atomicOr(&word[tok[u]], kPrompt);
          else atomicAdd(&word[tok[u]], 1u);
        }
      }
    }
    // the first of a token's biases carries them all, summed in their order
    for (int i = threadIdx.x; i < a.biases; i += TH) {
      const int p = place[i];
      if (p < 0) continue;
      bool first = true;
      for (int j = 0; j < i; ++j) first = first && place[j] != p;
      if (!first) continue;
      float s = a.bias[row * a.biases + i];
      for (int j = i + 1; j < a.biases; ++j)
        if (place[j] == p) s += a.bias[row * a.biases + j];
      bias[i] = s;
      atomicOr(&word[p], (uint32_t)(i + 1) << 20);
    }
    __syncthreads();
  }
  const float rep = a.repetition ? a.repetition[row] : 1.0f, freq = a.frequency ? a.frequency[row] : 0.0f,
              pres = a.presence ? a.presence[row] : 0.0f;
  auto apply = [&](float l, uint32_t m) {
    const uint32_t c = m & kCount;
    if (m & ~kBias) l = l > 0.0f ? l / rep : l * rep;
    if (c) l -= freq * (float)c + pres;
    if (m & kBias) l += bias[((m & kBias) >> 20) - 1];
    return l;
  };
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = 8 * (k * TH + (int)threadIdx.x);
    if (i + 8 > n) continue;
    uint32_t m[8] = {};
    uint32_t any = 0;
    if (marks) {
      *reinterpret_cast<uint4*>(m) = *reinterpret_cast<const uint4*>(word + i);
      *reinterpret_cast<uint4*>(m + 4) = *reinterpret_cast<const uint4*>(word + i + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) any |= m[j];
    }
    if constexpr (PLACE) {
      if (!any && open[k] == 0xff && !wrong) continue;
      if (open[k]) x[k] = row8_load<T>(in + i);
    }
    if (any)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (m[j]) x[k].set(j, apply(x[k].get(j), m[j]));
    if (open[k] != 0xff)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!(open[k] >> j & 1)) x[k].set(j, -__builtin_inff());
    if (wrong)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[k].set(j, __builtin_nanf(""));
    row8_store<T>(out + i, x[k]);
  }
  const int i = (n & ~7) + (int)threadIdx.x;  // the tokens past the last eight
  if (i < n) {
    auto l = in[i];
    const uint32_t m = marks ? word[i] : 0;
    if (m) l = Row8<T>::narrow(apply(Row8<T>::widen(l), m));
    if (mask && !(mask[i / 8] >> (i & 7) & 1)) l = Row8<T>::narrow(-__builtin_inff());
    if (wrong) l = Row8<T>::narrow(__builtin_nanf(""));
    out[i] = l;
  }
}

template <class T, int TH, int K>
hipError_t launch(hipStream_t st, const ConstrainArgs& a) {
  constexpr int SLAB = TH * 8 * K;
  const int slabs = (int)((a.v + SLAB - 1) / SLAB);
  const long rows8 = (a.r + 7) / 8;
  const size_t lds = a.history || a.biases ? 4 * SLAB + 8 * (size_t)a.biases : 0;
  const dim3 grid = launch_grid(rows8 * slabs * 8);
  if (a.logits == a.out) k_constrain<T, TH, K, true><<<grid, TH, lds, st>>>(a, rows8, slabs);
  else k_constrain<T, TH, K, false><<<grid, TH, lds, st>>>(a, rows8, slabs);
  return hipGetLastError();
}

template <class T>
hipError_t constrain(hipStream_t st, const ConstrainArgs& a) {
  const long tokens = a.r * a.v;
  if (tokens >= 512l * 8192) return launch<T, 512, 2>(st, a);
  if (tokens >= 512l * 4096) return launch<T, 256, 2>(st, a);
  return launch<T, 128, 1>(st, a);
}

}  // namespace

hipError_t constrain_logits(hipStream_t st, int dtype, const ConstrainArgs& a) {
  switch (dtype) {
    case CDCLQ_DTYPE_BF16: return constrain<Bf16>(st, a);
    case CDCLQ_DTYPE_F16: return constrain<F16>(st, a);
    default: return constrain<F32>(st, a);
  }
}

}  // namespace cdclq
