// The norm of all gradients of a step, and the gradients clipped to it.
//
//   n_g = sqrt(sum of x^2 over part g of every tensor)      c_g = min(1, max / (n_g + 1e-6))      out = c_g x
//
// g: the adapters of several users that train together, each tensor's first dimension (or one part: all). The
// squares are summed in f64, so that neither 1e-30 nor 1e30 leaves the range; c is made in f64 and rounded to f32,
// its product with x rounded to f32 and to the output's type. 1e-6 keeps c finite, as trainers do it. A norm that
// is NaN or infinite in f32 clips nothing (c = 1): the gradients stay as they are, for the caller to look at.
//
// Both passes are bound by memory. A workgroup takes a chunk of one tensor's part; the tensors' addresses come as the
// launch's arguments, so that a captured call keeps them and none has to be copied to the GPU first. The first pass
// leaves one f64 sum a chunk. Each workgroup of the second sums its part's chunks itself, all in the same order, while
// its first loads are on their way: a launch between the two would cost more. In place nothing is read again where
// c = 1.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cdclq.h"
#include "kernels.h"
#include "row8.h"

namespace cdclq {
namespace {

// Tensors of one launch: their arguments keep below 4 KB.
template <int N, bool OUT>
struct ClipTensors {
  const void* x[N];
  void* out[OUT ? N : 1];
  uint32_t n[N];      // elements of a part
  uint32_t start[N];  // first workgroup
  uint8_t kind[N];    // dtype of x, | 4: out is f32 whatever x is
  int count;
};
typedef ClipTensors<200, false> NormTensors;
typedef ClipTensors<144, true> OutTensors;
static_assert(sizeof(NormTensors) < 3900 && sizeof(OutTensors) < 3900, "a launch's arguments");

// Where a workgroup stands.
struct ClipAt {
  int tensor, part;
  long slot;  // of its part's sums
  long i0, i1;  // elements of the part
};
template <class S>
__device__ __forceinline__ ClipAt clip_at(const S& s, uint32_t b, int parts, int log_chunk, long first) {
  const int lane = threadIdx.x & 63;
  int e = -1;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(s.n) / 4 + 63) / 64; ++i) {
    const int j = 64 * i + lane;
    e += __popcll(__ballot(j < s.count && s.start[min(j, s.count - 1)] <= b));
  }
  e = __builtin_amdgcn_readfirstlane(e);
  const uint32_t n = s.n[e], per = (uint32_t)(((uint64_t)n + (1u << log_chunk) - 1) >> log_chunk);
  const uint32_t in = b - s.start[e], part = in / per, ch = in - part * per;
  ClipAt a;
  a.tensor = e, a.part = (int)part;
  a.slot = first + s.start[e] / (uint32_t)parts + ch;
  a.i0 = (long)ch << log_chunk;
  a.i1 = min((long)n, a.i0 + (1l << log_chunk));
  return a;
}

// Sum of v over 256 threads in a fixed order; all get it.
__device__ __forceinline__ double sum256(double v) {
  __shared__ double part[4];
#pragma unroll
  for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (part[0] + part[1]) + (part[2] + part[3]);
  __syncthreads();
  return v;
}

template <class T>
__device__ __forceinline__ double squares(const void* base, long part, long n, long i0, long i1) {
  const auto* x = static_cast<const typename Row8<T>::stored*>(base) + part * n;
  double s = 0.0;
  auto add = [&](float f) {
    const double v = (double)f;
    s = __builtin_fma(v, v, s);
  };
  for (long i = i0 + 8 * threadIdx.x; i + 8 <= i1; i += 8192) {  // four steps' loads in flight
    Row8<T> r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + 2048 * u + 8 <= i1) r[u] = row8_load<T>(x + i + 2048 * u);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + 2048 * u + 8 <= i1)
#pragma unroll
        for (int k = 0; k < 8; ++k) add(r[u].get(k));
  }
  const long i = i1 - ((i1 - i0) & 7) + threadIdx.x;  // the elements past the last eight
  if (i < i1) add(Row8<T>::widen(x[i]));
  return s;
}

__global__ __launch_bounds__(256) void k_norm_parts(const NormTensors s, uint32_t blocks, int parts, int log_chunk,
                                                    long first, long slots, double* __restrict__ sums) {
  const uint32_t b = blockIdx.x;
  if (b >= blocks) return;
  const ClipAt a = clip_at(s, b, parts, log_chunk, first);
  const void* x = s.x[a.tensor];
  const long n = s.n[a.tensor];
  double v;
  switch (s.kind[a.tensor] & 3) {
    case F32::kind: v = squares<F32>(x, a.part, n, a.i0, a.i1); break;
    case F16::kind: v = squares<F16>(x, a.part, n, a.i0, a.i1); break;
    default: v = squares<Bf16>(x, a.part, n, a.i0, a.i1); break;
  }
  v = sum256(v);
  if (threadIdx.x == 0) sums[a.part * slots + a.slot] = v;
}

// The norm of a part from its chunks' sums, by 256 threads.
__device__ __forceinline__ double norm_of(const double* sums, long slots) {
  double v = 0.0;
#pragma unroll 8
  for (long i = threadIdx.x; i < slots; i += 256) v += sums[i];
  return __builtin_sqrt(sum256(v));
}

__global__ __launch_bounds__(256) void k_norm(const double* __restrict__ sums, long slots, float* __restrict__ norm) {
  const double n = norm_of(sums + blockIdx.x * slots, slots);
  if (threadIdx.x == 0) norm[blockIdx.x] = (float)n;
}

template <class T, class O>
__device__ __forceinline__ void scaled(const void* from, void* to, const ClipAt& a, long n, const double* sums,
                                       long slots, double most, float* norm) {
  const auto* x = static_cast<const typename Row8<T>::stored*>(from) + a.part * n;
  auto* y = static_cast<typename Row8<O>::stored*>(to) + a.part * n;
  const bool place = from == to;
  Row8<T> r[4];
  auto load = [&](long i) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + 2048 * u + 8 <= a.i1) r[u] = row8_load<T>(x + i + 2048 * u);
  };
  long i = a.i0 + 8 * threadIdx.x;
  if (!place) load(i);
  const double got = norm_of(sums, slots);
  if (norm && threadIdx.x == 0) norm[a.part] = (float)got;
  float by = 1.0f;
  if (__builtin_isfinite((float)got)) by = (float)__builtin_fmin(1.0, most / (got + 1e-6));
  if (place) {
    if (by == 1.0f) return;
    load(i);
  }
  while (i + 8 <= a.i1) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i + 2048 * u + 8 > a.i1) continue;
      Row8<O> o;
#pragma unroll
      for (int k = 0; k < 8; ++k) o.set(k, by * r[u].get(k));
      row8_store<O>(y + i + 2048 * u, o);
    }
    i += 8192;
    load(i);
  }
  i = a.i1 - ((a.i1 - a.i0) & 7) + threadIdx.x;  // the elements past the last eight
  if (i < a.i1) y[i] = Row8<O>::narrow(by * Row8<T>::widen(x[i]));
}

__global__ __launch_bounds__(256) void k_clip(const OutTensors s, uint32_t blocks, int parts, int log_chunk, long first,
                                              long slots, const double* __restrict__ sums, double most, float* norm) {
  const uint32_t b = blockIdx.x;
  if (b >= blocks) return;
  const ClipAt a = clip_at(s, b, parts, log_chunk, first);
  const void* x = s.x[a.tensor];
  void* y = s.out[a.tensor];
  const long n = s.n[a.tensor];
  sums += a.part * slots;
  if (a.slot) norm = nullptr;  // a part's first chunk says its norm
  switch (s.kind[a.tensor]) {
    case F32::kind:
    case F32::kind | 4: return scaled<F32, F32>(x, y, a, n, sums, slots, most, norm);
    case F16::kind: return scaled<F16, F16>(x, y, a, n, sums, slots, most, norm);
    case F16::kind | 4: return scaled<F16, F32>(x, y, a, n, sums, slots, most, norm);
    case Bf16::kind: return scaled<Bf16, Bf16>(x, y, a, n, sums, slots, most, norm);
    default: return scaled<Bf16, F32>(x, y, a, n, sums, slots, most, norm);
  }
}

constexpr long kMostPart = 1l << 30;    // elements of a part that one entry of the tables takes
constexpr long kMostBlocks = 1l << 23;  // workgroups of a launch: its work-items keep below 2^32

struct ClipPlan {
  int log_chunk;
  long slots;  // chunks of a part, over all tensors
};
// Chunks of 4096 elements, or as long as leaves about 2048 of them: every workgroup of the second pass reads its part's
// sums.
ClipPlan clip_plan(const GradTensor* g, size_t n, int parts) {
  long total = 0;
  for (size_t i = 0; i < n; ++i) total += g[i].n;
  ClipPlan p = {12, 0};
  while (((total / parts >> p.log_chunk) > 2048 || total >> p.log_chunk > kMostBlocks / 2) && p.log_chunk < 30) ++p.log_chunk;
  const long chunk = 1l << p.log_chunk;
  for (size_t i = 0; i < n; ++i) {
    const long e = g[i].n / parts, whole = e / kMostPart;  // a whole entry's chunks end with it
    p.slots += whole * (kMostPart >> p.log_chunk) + (e - whole * kMostPart + chunk - 1) / chunk;
  }
  return p;
}

// Fills tables of S with the tensors (those of one part only in pieces of kMostPart elements) and hands each to `go`.
template <class S, bool OUT, class F>
hipError_t each_table(const GradTensor* g, size_t n, int parts, const ClipPlan& p, F go) {
  constexpr int N = sizeof(S::n) / 4;
  S s;
  s.count = 0;
  long slot = 0, first = 0;
  uint64_t blocks = 0;
  auto flush = [&]() -> hipError_t {
    if (!s.count) return hipSuccess;
    go(s, (uint32_t)blocks, first);
    first = slot;
    blocks = 0;
    s.count = 0;
    return hipGetLastError();
  };
  for (size_t i = 0; i < n; ++i) {
    const long e = g[i].n / parts;
    const size_t size = g[i].dtype == CDCLQ_DTYPE_F32 ? 4 : 2, out_size = g[i].out_dtype == CDCLQ_DTYPE_F32 ? 4 : 2;
    for (long at = 0; at < e; at += kMostPart) {
      const long len = std::min(kMostPart, e - at), per = (len + (1l << p.log_chunk) - 1) >> p.log_chunk;
      if (s.count == N || blocks + (uint64_t)per * parts > (uint64_t)kMostBlocks) {
        const hipError_t err = flush();
        if (err != hipSuccess) return err;
      }
      const int k = s.count++;
      s.x[k] = static_cast<const char*>(g[i].x) + at * size;
      if constexpr (OUT) s.out[k] = static_cast<char*>(g[i].out) + at * out_size;
      s.n[k] = (uint32_t)len;
      s.start[k] = (uint32_t)blocks;
      s.kind[k] = (uint8_t)(g[i].dtype | (g[i].out_dtype == CDCLQ_DTYPE_F32 ? 4 : 0));
      blocks += (uint64_t)per * parts;
      slot += per;
    }
  }
  return flush();
}

hipError_t parts_of(hipStream_t st, const GradTensor* g, size_t n, int parts, const ClipPlan& p, double* sums) {
  return each_table<NormTensors, false>(g, n, parts, p, [&](const NormTensors& s, uint32_t blocks, long first) {
    k_norm_parts<<<blocks, 256, 0, st>>>(s, blocks, parts, p.log_chunk, first, p.slots, sums);
  });
}

}  // namespace

size_t clip_work_bytes(const GradTensor* g, size_t n, int parts) {
  return (8 * (size_t)clip_plan(g, n, parts).slots * parts + 255) / 256 * 256;
}

hipError_t grad_norm(hipStream_t st, const GradTensor* g, size_t n, int parts, float* norm, void* work) {
  const ClipPlan p = clip_plan(g, n, parts);
  const hipError_t e = parts_of(st, g, n, parts, p, static_cast<double*>(work));
  if (e != hipSuccess) return e;
  k_norm<<<parts, 256, 0, st>>>(static_cast<const double*>(work), p.slots, norm);
  return hipGetLastError();
}

hipError_t clip_grads(hipStream_t st, const GradTensor* g, size_t n, int parts, double most, float* norm, void* work) {
  const ClipPlan p = clip_plan(g, n, parts);
  if (p.slots == 0) return grad_norm(st, g, n, parts, norm, work);  // nothing but norms of 0
  double* sums = static_cast<double*>(work);
  const hipError_t e = parts_of(st, g, n, parts, p, sums);
  if (e != hipSuccess) return e;
  return each_table<OutTensors, true>(g, n, parts, p, [&](const OutTensors& s, uint32_t blocks, long first) {
    k_clip<<<blocks, 256, 0, st>>>(s, blocks, parts, p.log_chunk, first, p.slots, sums, most, norm);
  });
}

}  // namespace cdclq
