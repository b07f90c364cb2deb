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
// slabs are as large as leaves enough workgroups, and where there are many requests a request's slabs lie on one XCD, whose
// L2 then holds its history; long histories of many requests are sorted by slab in a launch before. In place, only what
// changes is read or written, and tokens that the mask shuts out are not read.
// 256 requests, 128256 bf16 tokens, histories of 6100 on average, 32 biases, half with a mask: 39.6 us, 8 of them the
// sorting; without history, biases and masks 20 (131 MB, part of them in the last cache). What bounds it between the two
// are the instructions for tokens that have been: a wavefront takes them for all its lanes wherever one has such a
// token (the vector units issue 70% of the time). One token's logit made by one thread, in a pass before the copying, took
// 2 us more: its barriers and the gathered logits cost what it saves; slabs of one wavefront, without barriers, 14 more.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cdclq.h"
#include "kernels.h"
#include "row8.h"

namespace cdclq {
namespace {

constexpr uint32_t kPrompt = 1u << 31, kCount = (1u << 20) - 1, kBias = 2047u << 20;

// The histories' tokens by slab: those of request r and slab s at place[start[r][s]] up to start[r][s + 1], each its
// place in the slab, | kPrompt.
struct Binned {
  const uint32_t *start, *place;
};

// A workgroup takes a request: counts, their running sum, and the tokens' places, in any order within a slab.
__global__ __launch_bounds__(1024) void k_constrain_bin(ConstrainArgs a, int log_slab, int slabs,
                                                        uint32_t* __restrict__ start, uint32_t* __restrict__ place) {
  extern __shared__ __align__(16) uint32_t word[];  // a slab's count, then where its next token goes
  constexpr int kOnce = 8192;  // tokens that a round takes, 8 a thread
  __shared__ uint32_t sums[16], sorted[kOnce];
  const long row = blockIdx.x + (long)blockIdx.y * gridDim.x;
  if (row >= a.r) return;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  for (int i = tid; i < slabs; i += 1024) word[i] = 0;
  __syncthreads();
  const int len = a.lengths ? max(0, min(a.lengths[row], a.width)) : a.width, prompt = a.prompts ? a.prompts[row] : 0;
  const int64_t* h = a.history + row * a.ldh;
  int64_t tok[8];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < 8; ++u) tok[u] = i0 + 1024 * u < len ? h[i0 + 1024 * u] : -1;
  };
  auto is = [&](int u) { return (uint64_t)tok[u] < (uint64_t)a.v; };
  // A history of one round's tokens stays in registers with what the counters held.
  uint32_t rank[8];
  for (int i0 = tid; i0 < len; i0 += kOnce) {
    load(i0);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (is(u)) rank[u] = atomicAdd(&word[(uint32_t)tok[u] >> log_slab], 1u);
  }
  __syncthreads();
  uint32_t all = 0;
  for (int s0 = 0; s0 < slabs; s0 += 1024) {
    const uint32_t n = s0 + tid < slabs ? word[s0 + tid] : 0;
    uint32_t sum = n;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const uint32_t up = (uint32_t)__shfl_up((int)sum, k);
      if (lane >= k) sum += up;
    }
    if (lane == 63) sums[wv] = sum;
    __syncthreads();
    sum += all;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      if (w < wv) sum += sums[w];
      all += sums[w];
    }
    if (s0 + tid < slabs) {
      word[s0 + tid] = sum - n;
      start[row * (slabs + 1) + s0 + tid] = (uint32_t)(row * a.width) + sum - n;
    }
    __syncthreads();
  }
  if (tid == 0) start[row * (slabs + 1) + slabs] = (uint32_t)(row * a.width) + all;
  uint32_t* const to = place + row * a.width;
  const uint32_t low = (1u << log_slab) - 1;
  auto value = [&](int u, int i) { return ((uint32_t)tok[u] & low) | (i < prompt ? kPrompt : 0); };
  if (len <= kOnce) {  // sorted in LDS, so that whole lines are written
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (tid < len && is(u)) sorted[word[(uint32_t)tok[u] >> log_slab] + rank[u]] = value(u, tid + 1024 * u);
    __syncthreads();
    for (uint32_t i = tid; i < all; i += 1024) to[i] = sorted[i];
    return;
  }
  for (int i0 = tid; i0 < len; i0 += kOnce) {
    load(i0);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (is(u)) to[atomicAdd(&word[(uint32_t)tok[u] >> log_slab], 1u)] = value(u, i0 + 1024 * u);
  }
}

// LDS: TH * 8 * K words if there is a history or a bias, then the biases' values and places.
template <class T, int TH, int K, bool PLACE>
__global__ __launch_bounds__(TH) void k_constrain(ConstrainArgs a, Binned bins, long rows8, int slabs) {
  extern __shared__ __align__(16) uint32_t word[];
  constexpr int SLAB = TH * 8 * K;
  // Workgroup b of many requests: XCD b % 8 takes those of that remainder, slab by slab. Of few: slabs over all XCDs.
  const long b = blockIdx.x + (long)blockIdx.y * gridDim.x, at = rows8 ? b >> 3 : b;
  const long row = rows8 ? (at / slabs) * 8 + (b & 7) : at / slabs;
  if (row >= a.r) return;
  const int slab = (int)(at % slabs), slab0 = slab * SLAB;
  const auto* in = static_cast<const typename Row8<T>::stored*>(a.logits) + row * a.ld + slab0;
  auto* out = static_cast<typename Row8<T>::stored*>(a.out) + row * a.ldo + slab0;
  const int n = (int)min((long)SLAB, a.v - slab0);
  const bool marks = a.history || a.biases;

  // Loads come back in the order in which they are asked for: the few that the counting waits for, then the logits.
  uint32_t next = ~0u, end = 0;  // the slab's tokens, binned
  int64_t tok[8];                // or the history's
  int len = 0, prompt = 0;
  const int64_t* h = a.history + row * a.ldh;
  auto tokens = [&](int i0) {
#pragma unroll
    for (int u = 0; u < 8; ++u) tok[u] = i0 + u * TH < len ? (int64_t)((uint64_t)h[i0 + u * TH] - slab0) : -1;
  };
  if (bins.start) {
    const uint32_t* s = bins.start + row * (slabs + 1) + slab;
    end = s[1];
    next = s[0] + threadIdx.x;
  } else if (a.history) {
    len = a.lengths ? max(0, min(a.lengths[row], a.width)) : a.width;
    prompt = a.prompts ? a.prompts[row] : 0;
    tokens(threadIdx.x);
  }
  uint32_t place = next < end ? bins.place[next] : 0;
  const long mrow = a.mask_rows ? a.mask_rows[row] : a.mask ? row : -1;
  const bool wrong = mrow < -1 || (mrow >= 0 && mrow >= a.masks);  // no such mask
  const uint8_t* mask = mrow < 0 || wrong ? nullptr
                                          : reinterpret_cast<const uint8_t*>(a.mask + mrow * a.ldm) + slab0 / 8;
  int64_t btok = -1;  // a bias each lane of the first wavefront
  float bval = 0.0f;
  auto biases = [&](int i) {
    btok = i < a.biases ? (int64_t)((uint64_t)a.bias_tokens[row * a.biases + i] - slab0) : -1;
    bval = i < a.biases ? a.bias[row * a.biases + i] : 0.0f;
  };
  if (threadIdx.x < 64) biases(threadIdx.x);
  uint8_t open[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = k * TH + (int)threadIdx.x;
    open[k] = mask && 8 * i < n ? mask[i] : 0xff;
  }
  Row8<T> x[K];
  if constexpr (!PLACE) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = 8 * (k * TH + (int)threadIdx.x);
      if (i + 8 <= n) x[k] = row8_load<T>(in + i);
    }
  }
  const float rep = a.repetition ? a.repetition[row] : 1.0f, freq = a.frequency ? a.frequency[row] : 0.0f,
              pres = a.presence ? a.presence[row] : 0.0f;
  float* const bias = reinterpret_cast<float*>(word + SLAB);
  if (marks) {
#pragma unroll
    for (int k = 0; k < 2 * K; ++k) reinterpret_cast<uint4*>(word)[k * TH + threadIdx.x] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    while (next < end) {
      if (place & kPrompt) atomicOr(&word[place & ~kPrompt], kPrompt);
      else atomicAdd(&word[place], 1u);
      next += TH;
      if (next < end) place = bins.place[next];
    }
    for (int i0 = threadIdx.x; i0 < len;) {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if ((uint64_t)tok[u] >= (uint64_t)n) continue;
        if (i0 + u * TH < prompt) atomicOr(&word[tok[u]], kPrompt);
        else atomicAdd(&word[tok[u]], 1u);
      }
      i0 += 8 * TH;
      if (i0 < len) tokens(i0);
    }
    // The slab's biases: a wavefront lists them in their order; the first of a token's carries them all, summed.
    if (a.biases && threadIdx.x < 64) {
      const int lane = threadIdx.x;
      int* const at = reinterpret_cast<int*>(bias + a.biases);
      int m = 0;
      for (int i0 = 0; i0 < a.biases; i0 += 64) {
        if (i0) biases(i0 + lane);
        const bool here = (uint64_t)btok < (uint64_t)n;
        const unsigned long long on = __ballot(here);
        if (here) {
          const int j = m + __popcll(on & ((1ull << lane) - 1));
          at[j] = (int)btok;
          bias[j] = bval;
        }
        m += __popcll(on);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      for (int i0 = 0; i0 < m; i0 += 64) {
        const int i = i0 + lane, p = i < m ? at[i] : -1;
        bool first = i < m;
        float s = 0.0f;
#pragma unroll 8
        for (int j = 0; j < m; ++j) {
          const bool same = at[j] == p;
          first = first && !(same && j < i);
          if (same) s += bias[j];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (first) {
          bias[i] = s;
          atomicOr(&word[p], (uint32_t)(i + 1) << 20);
        }
      }
    }
    __syncthreads();
  }
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
        if (!(open[k] >> j & 1)) x[k].v[j] = Row8<T>::narrow(-__builtin_inff());
    if (wrong)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[k].v[j] = Row8<T>::narrow(__builtin_nanf(""));
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

// Slabs of 1024 tokens by 128 threads or of 8192 by 512, these from 2^20 logits on: 128256 tokens, histories of 500, half
// of the requests with a mask: one request 4.5 us and 5.3, 16 requests 8.4 and 5.8, 128 requests 21 and 14.5. (4096 by
// 256: 5.2, 6.2 and 14.8.)
bool large_slabs(long r, long v) { return r * v >= 1l << 20; }
long slabs_of(long r, long v) { return large_slabs(r, v) ? (v + 8191) / 8192 : (v + 1023) / 1024; }

// Whether the histories are sorted by slab in a launch before: where a workgroup would take many rounds to look at one,
// or all of them much work. 128256 tokens, histories of 1000 and 8192 at most, sorted and not: one request 7.4 and 4.9
// us, 9.2 and 12.5; 8 requests 8.3 and 5.6, 10.6 and 15.1; 64 requests of 4000 14.1 and 10.8; 256 of 1000 27.8 and
// 26.2, of 2000 28.9 and 28.7.
bool binned(long r, long v, long width) {
  return (width > 32l * (large_slabs(r, v) ? 512 : 128) || r * slabs_of(r, v) * width > 1l << 23) && r * width < 1l << 32;
}

template <class T, int TH, int K>
hipError_t launch(hipStream_t st, const ConstrainArgs& a, void* work) {
  constexpr int SLAB = TH * 8 * K;
  const int slabs = (int)((a.v + SLAB - 1) / SLAB);
  // (of 256 requests 27.6 us by XCD and 28.7 without, of 16 9.1 and 6.6)
  const long rows8 = a.r >= 64 ? (a.r + 7) / 8 : 0;
  Binned bins = {};
  if (a.history && binned(a.r, a.v, a.width)) {
    uint32_t* start = static_cast<uint32_t*>(work);
    uint32_t* place = start + a.r * (slabs + 1);
    k_constrain_bin<<<launch_grid(a.r), 1024, 4 * slabs, st>>>(a, __builtin_ctz(SLAB), slabs, start, place);
    bins = {start, place};
  }
  const size_t lds = a.history || a.biases ? 4 * SLAB + 8 * (size_t)a.biases : 0;
  const dim3 grid = launch_grid((rows8 ? 8 * rows8 : a.r) * slabs);
  if (a.logits == a.out) k_constrain<T, TH, K, true><<<grid, TH, lds, st>>>(a, bins, rows8, slabs);
  else k_constrain<T, TH, K, false><<<grid, TH, lds, st>>>(a, bins, rows8, slabs);
  return hipGetLastError();
}

template <class T>
hipError_t constrain(hipStream_t st, const ConstrainArgs& a, void* work) {
  return large_slabs(a.r, a.v) ? launch<T, 512, 2>(st, a, work) : launch<T, 128, 1>(st, a, work);
}

}  // namespace

size_t constrain_work_bytes(long r, long v, long width) {
  if (!width || !binned(r, v, width)) return 0;
  return (4 * (size_t)(r * (slabs_of(r, v) + 1) + r * width) + 255) / 256 * 256;
}

hipError_t constrain_logits(hipStream_t st, int dtype, const ConstrainArgs& a, void* work) {
  switch (dtype) {
    case CDCLQ_DTYPE_BF16: return constrain<Bf16>(st, a, work);
    case CDCLQ_DTYPE_F16: return constrain<F16>(st, a, work);
    default: return constrain<F32>(st, a, work);
  }
}

}  // namespace cdclq
