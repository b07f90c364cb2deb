// The norm of all gradients of a step, and the gradients clipped to it.
//
//   n_g = sqrt(sum of x^2 over part g of every tensor)      c_g = min(1, max / (n_g + 1e-6))      out = c_g x
//
// g: the adapters of several users that train together, each tensor's first dimension (or one part: all). The
// squares are summed in f64, so that neither 1e-30 nor 1e30 leaves the range; c is made in f64 and rounded to f32 (below
// f32's normal numbers it stays in f64), its product with x rounded to f32 and to the output's type. 1e-6 keeps c finite,
// as trainers do it. A part with a NaN or an infinity is not clipped (c = 1): its gradients stay as they are, for the
// caller to look at. A finite norm above f32's numbers is returned as infinite, and clips.
//
// Both passes are bound by memory. A part's elements, over all tensors, are chunks of 4096; a workgroup takes every
// J-th of a part's, so that a part has J sums whatever its size, and each workgroup of the second pass adds them up
// itself, all in the same order: a launch between the two would cost more. The second pass goes backwards, through what
// the first one left in the last cache. In place nothing is read again where c = 1.
// The tensors' addresses come as a launch's arguments, so that a captured call keeps them and the host has nothing to copy
// or to wait for; sets of more than one launch takes are written to a table in the workspace by small launches first
// (448 tensors, 84 MB into f32: 82 us, as three launches a pass 113). Those today: 60 us, of them 6 the table, 18 the
// norm (4.7 TB/s) and 37 the clipping (6.8 TB/s, its reads from the last cache), in place 50; the host takes 49. 1.4 GB into
// a second set: 688-700 us, 214 (6.5 TB/s) and 466 (6.0).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cdclq.h"
#include "kernels.h"
#include "row8.h"

namespace cdclq {
namespace {

constexpr int kTensors = 150;           // of one launch: its arguments keep below 4 KB
constexpr int kRows = 230;              // of one launch that writes the table
constexpr int kChunk = 4096;            // elements
constexpr long kMostPart = 1l << 30;    // elements of a part that one entry of the tables takes
// Sums of all parts together, where parts have several: 84 MB into f32, 1.4 GB, and 268 MB into f32 as 1, 16 or 512 parts
// 61 us, 700 and 170; with 1024 sums 62, 805 and 202, with 2048 60, 700 and 171, with 8192 71, 693 and 173. (3000 parts
// have one sum each and leave workgroups idle at the end: 393 MB 278, with 8192 258.)
constexpr long kMostSums = 4096;

// One tensor, or a piece of it.
struct ClipEntry {
  const void* x;
  void* out;
  uint32_t n;      // elements of a part
  uint32_t start;  // its first chunk among a part's
  uint32_t kind;   // dtype of x, | 4: out is f32 whatever x is
};

// The tensors as a launch's arguments.
struct ClipArgs {
  const void* x[kTensors];
  void* out[kTensors];
  uint32_t n[kTensors], start[kTensors];
  uint8_t kind[kTensors];
  int count;
};
static_assert(sizeof(ClipArgs) < 3900, "a launch's arguments");
// Some of the tensors as the arguments of a launch that writes the table, 17 bytes each: addresses have 48 bits, and the
// chunks are counted there (448 tensors in two launches; as three, of ClipArgs, 4 us more).
struct ClipRows {
  uint32_t x[kRows], out[kRows], n[kRows];
  uint16_t x_high[kRows], out_high[kRows];
  uint8_t kind[kRows];
  int count;
  uint32_t base, chunk;  // of the first one: its place in the table, and its first chunk
};
static_assert(sizeof(ClipRows) < 3950, "a launch's arguments");
// The tensors in device memory, and the tensor of each chunk.
struct ClipTable {
  const ClipEntry* entries;
  const uint32_t* who;
};

__device__ __forceinline__ ClipEntry entry_of(const ClipArgs& s, uint32_t chunk) {
  const int lane = threadIdx.x & 63;
  int e = -1;
#pragma unroll
  for (int i = 0; i < (kTensors + 63) / 64; ++i) {
    const int j = 64 * i + lane;
    e += __popcll(__ballot(j < s.count && s.start[min(j, s.count - 1)] <= chunk));
  }
  e = __builtin_amdgcn_readfirstlane(e);
  return {s.x[e], s.out[e], s.n[e], s.start[e], s.kind[e]};
}
__device__ __forceinline__ ClipEntry entry_of(const ClipTable& s, uint32_t chunk) { return s.entries[s.who[chunk]]; }

// The workgroups blockIdx.y take tensor blockIdx.x: a large one's chunks are many (a head of 525 M elements: 20 us by one
// workgroup, 5 by 16).
__global__ __launch_bounds__(256) void k_clip_table(const ClipRows s, ClipEntry* __restrict__ entries,
                                                    uint32_t* __restrict__ who) {
  __shared__ uint32_t part[4];
  const int e = blockIdx.x, i = threadIdx.x;
  auto chunks = [&](int of) { return (s.n[of] + kChunk - 1) / kChunk; };
  uint32_t start = i < e ? chunks(i) : 0;  // summed: of the tensors before
#pragma unroll
  for (int k = 32; k; k >>= 1) start += (uint32_t)__shfl_xor((int)start, k);
  if ((i & 63) == 0) part[i >> 6] = start;
  __syncthreads();
  start = s.chunk + part[0] + part[1] + part[2] + part[3];
  for (uint32_t c = 256 * blockIdx.y + i; c < chunks(e); c += 256 * gridDim.y) who[start + c] = s.base + e;
  if (i == 0 && blockIdx.y == 0) {
    const uint64_t x = (uint64_t)s.x_high[e] << 32 | s.x[e], out = (uint64_t)s.out_high[e] << 32 | s.out[e];
    entries[s.base + e] = {reinterpret_cast<const void*>(x), reinterpret_cast<void*>(out), s.n[e], start, s.kind[e]};
  }
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

// The sum of the squares of elements [i0, i1), on to s.
template <class T>
__device__ __forceinline__ double squares(const void* base, long i0, long i1, double s) {
  const auto* x = static_cast<const typename Row8<T>::stored*>(base);
  auto add = [&](float f) {
    const double v = (double)f;
    s = __builtin_fma(v, v, s);
  };
  Row8<T> r[kChunk / 2048];
  const long i = i0 + 8 * threadIdx.x;
#pragma unroll
  for (int u = 0; u < kChunk / 2048; ++u)
    if (i + 2048 * u + 8 <= i1) r[u] = row8_load<T>(x + i + 2048 * u);
#pragma unroll
  for (int u = 0; u < kChunk / 2048; ++u)
    if (i + 2048 * u + 8 <= i1)
#pragma unroll
      for (int k = 0; k < 8; ++k) add(r[u].get(k));
  const long last = i1 - ((i1 - i0) & 7) + threadIdx.x;  // the elements past the last eight
  if (last < i1) add(Row8<T>::widen(x[last]));
  return s;
}

// Workgroup part * each + j: chunks j, j + each, ... of a part.
template <class S>
__global__ __launch_bounds__(256) void k_norm_parts(const S s, uint32_t chunks, uint32_t each, uint32_t sums_all,
                                                    double* __restrict__ sums) {
  const uint32_t b = blockIdx.x + blockIdx.y * gridDim.x;
  if (b >= sums_all) return;
  const uint32_t part = b / each;
  double v = 0.0;
  uint32_t c = b - part * each;
  ClipEntry next;
  if (c < chunks) next = entry_of(s, c);
  for (; c < chunks; c += each) {
    const ClipEntry e = next;
    if (c + each < chunks) next = entry_of(s, c + each);
    const long i0 = part * (long)e.n + (long)(c - e.start) * kChunk, i1 = min(i0 + kChunk, (part + 1) * (long)e.n);
    switch (e.kind & 3) {
      case F32::kind: v = squares<F32>(e.x, i0, i1, v); break;
      case F16::kind: v = squares<F16>(e.x, i0, i1, v); break;
      default: v = squares<Bf16>(e.x, i0, i1, v); break;
    }
  }
  v = sum256(v);
  if (threadIdx.x == 0) sums[b] = v;
}

// The norm of a part from its sums, by 256 threads.
__device__ __forceinline__ double norm_of(const double* sums, uint32_t n) {
  double v = 0.0;
#pragma unroll 8
  for (uint32_t i = threadIdx.x; i < n; i += 256) v += sums[i];
  return __builtin_sqrt(sum256(v));
}

__global__ __launch_bounds__(256) void k_norm(const double* __restrict__ sums, uint32_t each, float* __restrict__ norm) {
  const double n = norm_of(sums + blockIdx.x * (long)each, each);
  if (threadIdx.x == 0) norm[blockIdx.x] = (float)n;
}

// y = by x over elements [i0, i1), 16 bytes of y a lane and store, so that a wavefront's are whole lines (as two stores
// of a lane's 32 bytes each, 84 MB into f32 took 49 us, so 37).
template <class T, class O>
__device__ __forceinline__ void scaled(const void* from, void* to, long i0, long i1, float by) {
  typedef typename Row8<T>::stored X;
  typedef typename Row8<O>::stored Y;
  constexpr int E = 16 / sizeof(Y), U = kChunk / (256 * E);
  typedef X XE __attribute__((ext_vector_type(E), aligned(sizeof(X))));
  typedef Y YE __attribute__((ext_vector_type(E), aligned(sizeof(Y))));
  const X* x = static_cast<const X*>(from);
  Y* y = static_cast<Y*>(to);
  XE r[U];
  const long i = i0 + E * threadIdx.x;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (i + 256 * E * u + E <= i1) r[u] = __builtin_nontemporal_load(reinterpret_cast<const XE*>(x + i + 256 * E * u));
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (i + 256 * E * u + E > i1) continue;
    YE o;
#pragma unroll
    for (int k = 0; k < E; ++k) o[k] = Row8<O>::narrow(by * Row8<T>::widen(r[u][k]));
    __builtin_nontemporal_store(o, reinterpret_cast<YE*>(y + i + 256 * E * u));
  }
  const long last = i1 - ((i1 - i0) & (E - 1)) + threadIdx.x;  // the elements past the last E
  if (last < i1) y[last] = Row8<O>::narrow(by * Row8<T>::widen(x[last]));
}

// The same for a factor below f32's normal numbers (gradients of 1e30 held to 1e-9), which f32 would hold in few bits or as
// 0 while the products are ordinary numbers: in f64, element by element.
__device__ __forceinline__ float element(const void* x, long i, uint32_t kind) {
  switch (kind & 3) {
    case F32::kind: return static_cast<const float*>(x)[i];
    case F16::kind: return F16::widen(static_cast<const uint16_t*>(x)[i]);
    default: return Bf16::widen(static_cast<const uint16_t*>(x)[i]);
  }
}
__device__ __forceinline__ void scaled_little(const ClipEntry& e, long i0, long i1, double by) {
  for (long i = i0 + threadIdx.x; i < i1; i += 256) {
    const float y = (float)(by * (double)element(e.x, i, e.kind));
    if ((e.kind & 4) || e.kind == F32::kind) static_cast<float*>(e.out)[i] = y;
    else static_cast<uint16_t*>(e.out)[i] = e.kind == F16::kind ? F16::narrow(y) : Bf16::narrow(y);
  }
}

template <class S>
__global__ __launch_bounds__(256) void k_clip(const S s, uint32_t chunks, uint32_t each, uint32_t sums_all,
                                              const double* __restrict__ sums, double most, float* __restrict__ norm) {
  const uint32_t b = blockIdx.x + blockIdx.y * gridDim.x;
  if (b >= sums_all) return;
  const uint32_t part = b / each, j = b - part * each;
  uint32_t c = j + (chunks - 1 - j) / each * each;  // of those below chunks
  ClipEntry next;
  if (j < chunks) next = entry_of(s, c);
  const double got = norm_of(sums + part * (long)each, each);
  if (j == 0 && threadIdx.x == 0) norm[part] = (float)got;
  double exact = 1.0;
  if (__builtin_isfinite(got)) exact = __builtin_fmin(1.0, most / (got + 1e-6));
  const float by = (float)exact;
  const bool little = exact < 0x1p-126 && exact > 0.0;
  if (j >= chunks) return;
  for (;; c -= each) {
    const ClipEntry e = next;
    if (c >= each) next = entry_of(s, c - each);
    const long i0 = part * (long)e.n + (long)(c - e.start) * kChunk, i1 = min(i0 + kChunk, (part + 1) * (long)e.n);
    if (little) {
      scaled_little(e, i0, i1, exact);
    } else if (e.x != e.out || by != 1.0f) {
      switch (e.kind) {
        case F32::kind:
        case F32::kind | 4: scaled<F32, F32>(e.x, e.out, i0, i1, by); break;
        case F16::kind: scaled<F16, F16>(e.x, e.out, i0, i1, by); break;
        case F16::kind | 4: scaled<F16, F32>(e.x, e.out, i0, i1, by); break;
        case Bf16::kind: scaled<Bf16, Bf16>(e.x, e.out, i0, i1, by); break;
        default: scaled<Bf16, F32>(e.x, e.out, i0, i1, by); break;
      }
    }
    if (c < each) return;
  }
}

// What a call needs, from the tensors' sizes alone.
struct ClipPlan {
  uint32_t entries, chunks;  // chunks of a part
  uint32_t each, sums;       // sums of a part, and of all
  size_t table, who, bytes;  // in the workspace, behind the sums; none where the arguments take all tensors
};
ClipPlan clip_plan(const GradTensor* g, size_t n, int parts) {
  ClipPlan p = {};
  for (size_t i = 0; i < n; ++i)
    for (long e = g[i].n / parts; e > 0; e -= kMostPart) {
      ++p.entries;
      p.chunks += (uint32_t)((std::min(e, kMostPart) + kChunk - 1) / kChunk);
    }
  p.each = (uint32_t)std::max(1l, std::min((long)p.chunks, kMostSums / parts));
  p.sums = p.each * (uint32_t)parts;
  p.bytes = (8 * (size_t)p.sums + 255) / 256 * 256;
  if (p.entries > kTensors) {
    p.table = p.bytes;
    p.who = p.table + ((size_t)p.entries * sizeof(ClipEntry) + 255) / 256 * 256;
    p.bytes = p.who + ((size_t)p.chunks * 4 + 255) / 256 * 256;
  }
  return p;
}

// Hands the tensors to `go`, as arguments or as a table.
template <class F>
hipError_t with_tensors(hipStream_t st, const GradTensor* g, size_t n, int parts, const ClipPlan& p, char* work, F go) {
  auto pieces = [&](auto take) {  // each with its first chunk
    uint32_t chunk = 0;
    for (size_t i = 0; i < n; ++i) {
      const long e = g[i].n / parts;
      const size_t size = g[i].dtype == CDCLQ_DTYPE_F32 ? 4 : 2, out_size = g[i].out_dtype == CDCLQ_DTYPE_F32 ? 4 : 2;
      const uint32_t kind = (uint32_t)g[i].dtype | (g[i].out_dtype == CDCLQ_DTYPE_F32 ? 4 : 0);
      for (long at = 0; at < e; at += kMostPart) {
        const uint32_t len = (uint32_t)std::min(kMostPart, e - at);
        take(ClipEntry{static_cast<const char*>(g[i].x) + at * size, static_cast<char*>(g[i].out) + at * out_size, len,
                       chunk, kind});
        chunk += (len + kChunk - 1) / kChunk;
      }
    }
  };
  if (p.entries <= kTensors) {
    ClipArgs s;
    s.count = 0;
    pieces([&](const ClipEntry& e) {
      const int k = s.count++;
      s.x[k] = e.x, s.out[k] = e.out, s.n[k] = e.n, s.start[k] = e.start, s.kind[k] = (uint8_t)e.kind;
    });
    go(s);
    return hipGetLastError();
  }
  ClipEntry* const entries = reinterpret_cast<ClipEntry*>(work + p.table);
  uint32_t* const who = reinterpret_cast<uint32_t*>(work + p.who);
  ClipRows s;
  s.count = 0, s.base = 0;
  uint64_t high = 0;
  long most = 0;  // chunks of a tensor in this launch
  pieces([&](const ClipEntry& e) { high |= (uint64_t)e.x | (uint64_t)e.out; });
  if (high >> 48) return hipErrorInvalidDevicePointer;
  auto write = [&] {
    k_clip_table<<<dim3(s.count, (unsigned)std::max(1l, std::min(most / 2048, 16l))), 256, 0, st>>>(s, entries, who);
    s.base += (uint32_t)s.count;
    s.count = 0, most = 0;
  };
  pieces([&](const ClipEntry& e) {
    if (s.count == kRows) write();
    const uint64_t x = (uint64_t)e.x, out = (uint64_t)e.out;
    const int k = s.count++;
    if (k == 0) s.chunk = e.start;
    s.x[k] = (uint32_t)x, s.x_high[k] = (uint16_t)(x >> 32);
    s.out[k] = (uint32_t)out, s.out_high[k] = (uint16_t)(out >> 32);
    s.n[k] = e.n, s.kind[k] = (uint8_t)e.kind;
    most = std::max(most, (long)e.n / kChunk);
  });
  write();
  go(ClipTable{entries, who});
  return hipGetLastError();
}

}  // namespace

size_t clip_work_bytes(const GradTensor* g, size_t n, int parts) { return clip_plan(g, n, parts).bytes; }

hipError_t grad_norm(hipStream_t st, const GradTensor* g, size_t n, int parts, float* norm, void* work) {
  const ClipPlan p = clip_plan(g, n, parts);
  double* sums = static_cast<double*>(work);
  return with_tensors(st, g, n, parts, p, static_cast<char*>(work), [&](const auto& s) {
    k_norm_parts<<<launch_grid(p.sums), 256, 0, st>>>(s, p.chunks, p.each, p.sums, sums);
    k_norm<<<parts, 256, 0, st>>>(sums, p.each, norm);
  });
}

hipError_t clip_grads(hipStream_t st, const GradTensor* g, size_t n, int parts, double most, float* norm, void* work) {
  const ClipPlan p = clip_plan(g, n, parts);
  double* sums = static_cast<double*>(work);
  return with_tensors(st, g, n, parts, p, static_cast<char*>(work), [&](const auto& s) {
    k_norm_parts<<<launch_grid(p.sums), 256, 0, st>>>(s, p.chunks, p.each, p.sums, sums);
    k_clip<<<launch_grid(p.sums), 256, 0, st>>>(s, p.chunks, p.each, p.sums, sums, most, norm);
  });
}

}  // namespace cdclq
