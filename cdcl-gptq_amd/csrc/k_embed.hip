// Token embedding and the gradient of its table.
//
//   y_t = scale E[id_t]            dE[v] = scale sum over the tokens t with id_t = v of dy_t
//
// An id equal to the ignored one stands for no token: y_t = 0, and it adds nothing. Any other id outside 0..v
// gives a row of NaN and a gradient that is NaN throughout. Both directions only move memory.
//
// The gradient sums a row's tokens in their order, in f32, with one rounding at the end and no float atomics:
// equal inputs give equal bits. Three forms by the number of tokens:
//   few     one launch. A workgroup takes a token, finds the others of its id by comparing all ids, and leaves
//           unless it is the first of them. Further workgroups clear the rows without tokens.
//   ranked  a token's place among the sorted ones is the number of smaller (id, position) pairs, counted by
//           comparing all pairs of tokens in one launch, which clears the table at the same time. Then chunks
//           of the sorted tokens are summed; runs of equal ids that pass a chunk's end are joined by a third.
//   sorted  the places from a radix sort, 8 or 9 bits a pass, a launch more than the passes.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cdclq.h"
#include "kernels.h"
#include "row8.h"

namespace cdclq {
namespace {

typedef unsigned long long u64;

// Tokens up to which each form is taken.
constexpr long kFewIds = 512, kRankedIds = 8192;
constexpr int kTile = 4096;  // ids of a workgroup of the radix sort

__device__ __forceinline__ long block_id() { return blockIdx.x + (long)blockIdx.y * gridDim.x; }

// An id as a sort key: below v a row, v the ignored one, v + 1 no row.
__device__ __forceinline__ uint32_t id_key(int64_t id, int64_t ignore, uint32_t v) {
  return id == ignore ? v : (uint64_t)id < v ? (uint32_t)id : v + 1;
}

// lanes (a power of two, at most 64) of a wavefront to a row of d elements, eight each and eight times
inline int row_lanes(long d) {
  int l = 1;
  while (l < 64 && l * 8l < d) l *= 2;
  return l;
}

struct EmbedView {
  const int64_t* ids;
  long t, d, v;
  int64_t ignore;
  float scale;
  const uint16_t* dy;
  long lddy;
  void* de;
  long lde;
  int lanes;  // of row_lanes
  int add;
};

template <class T>
__global__ __launch_bounds__(256) void k_embed_rows(const uint16_t* __restrict__ table, long ldt, long v, long d,
                                                    const int64_t* __restrict__ ids, long t, float scale,
                                                    int64_t ignore, uint16_t* __restrict__ out, long ldo, int lanes,
                                                    long parts) {
  const long unit = block_id() * (256 / lanes) + threadIdx.x / lanes;
  if (unit >= t * parts) return;
  const long row = unit / parts, c0 = (unit - row * parts) * lanes * 64 + 8 * (threadIdx.x & (lanes - 1));
  const uint32_t key = id_key(ids[row], ignore, (uint32_t)v);
  uint16_t* to = out + row * ldo;
  if (key >= (uint32_t)v) {
    const Row8<T> f = row8_fill<T>(key == (uint32_t)v ? 0.0f : __builtin_nanf(""));
    for (int k = 0; k < 8; ++k)
      if (c0 + 8l * lanes * k < d) row8_store<T>(to + c0 + 8l * lanes * k, d - c0 - 8l * lanes * k, f);
    return;
  }
  const uint16_t* from = table + key * ldt;
  Row8<T> x[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const long c = c0 + 8l * lanes * k;
    if (c < d) x[k] = row8_load<T>(from + c, d - c);
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const long c = c0 + 8l * lanes * k;
    if (c >= d) continue;
    if (scale != 1.0f)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[k].set(i, scale * x[k].get(i));
    row8_store<T>(to + c, d - c, x[k]);
  }
}

// x in every element of rows [r0, r1) of dE that `skip` (one flag a row, or null) does not name.
template <class O>
__device__ __forceinline__ void fill_rows(const EmbedView& a, long r0, long r1, const uint8_t* skip, float x) {
  auto* de = static_cast<typename Row8<O>::stored*>(a.de);
  const Row8<O> f = row8_fill<O>(x);
  const int per = blockDim.x / a.lanes, l = threadIdx.x & (a.lanes - 1);
  for (long r = r0 + threadIdx.x / a.lanes; r < r1; r += per) {
    if (skip && skip[r - r0]) continue;
    for (long c = 8 * l; c < a.d; c += 8 * a.lanes) row8_store<O>(de + r * a.lde + c, a.d - c, f);
  }
}

// dE = NaN throughout, by all workgroups of a launch (an id outside 0..v).
template <class O>
__device__ void poison(const EmbedView& a, long b, long nb) {
  const long per = (a.v + nb - 1) / nb;
  fill_rows<O>(a, min(a.v, b * per), min(a.v, (b + 1) * per), nullptr, __builtin_nanf(""));
}

// A finished sum of eight columns into dE: the only rounding.
template <class O>
__device__ __forceinline__ void finish8(const EmbedView& a, uint32_t row, long c, const float* sum) {
  auto* p = static_cast<typename Row8<O>::stored*>(a.de) + row * a.lde + c;
  Row8<O> r;
  if (a.add) {
    r = row8_load<O>(p, a.d - c);
#pragma unroll
    for (int i = 0; i < 8; ++i) r.set(i, __builtin_fmaf(a.scale, sum[i], r.get(i)));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.set(i, a.scale * sum[i]);
  }
  row8_store<O>(p, a.d - c, r);
}

// ---------------------------------------------------------------- few tokens
// Workgroups below t slabs: token b / slabs, 8 x 256 columns. The others clear `rows` rows each.
template <class T, class O>
__global__ __launch_bounds__(256) void k_embed_few(EmbedView a, int slabs, long sums, int rows) {
  __shared__ u64 same[kFewIds / 64], bad[kFewIds / 64];
  __shared__ uint8_t has[1024];
  const long b = block_id();
  const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long blocks = sums + (a.add ? 0 : (a.v + rows - 1) / rows);
  if (b >= blocks) return;
  const bool sum = b < sums;
  const int tok = sum ? (int)(b / slabs) : 0;
  const long r0 = sum ? 0 : (b - sums) * rows;
  if (!sum)
    for (int i = threadIdx.x; i < rows; i += 256) has[i] = 0;
  __syncthreads();
  const uint32_t v = (uint32_t)a.v;
  const uint32_t own = sum ? id_key(a.ids[tok], a.ignore, v) : 0;
  for (int w = wv; 64 * w < a.t; w += 4) {
    const int i = 64 * w + lane;
    const uint32_t k = i < a.t ? id_key(a.ids[i], a.ignore, v) : v;
    const u64 s = __ballot(i < a.t && k == own), n = __ballot(k > v);
    if (lane == 0) same[w] = s, bad[w] = n;
    if (!sum && k >= r0 && k < min((long)v, r0 + rows)) has[k - r0] = 1;
  }
  __syncthreads();
  const int words = (int)((a.t + 63) / 64);
  u64 any = 0;
  for (int w = 0; w < words; ++w) any |= bad[w];
  if (any) return poison<O>(a, b, blocks);
  if (!sum) return fill_rows<O>(a, r0, min(a.v, r0 + rows), has, 0.0f);
  if (own >= v) return;
  for (int w = 0; w <= tok / 64; ++w)
    if (same[w] & (w < tok / 64 ? ~0ull : (1ull << (tok & 63)) - 1)) return;  // an earlier token sums them
  const long c = ((b - (long)tok * slabs) * 256 + threadIdx.x) * 8;
  if (c >= a.d) return;
  float acc[8] = {};
  int w = tok / 64;
  u64 left = same[w];
  while (true) {  // eight rows' loads together
    int at[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      while (!left && w + 1 < words) left = same[++w];
      at[k] = left ? 64 * w + __builtin_ctzll(left) : -1;
      left &= left - 1;
    }
    Row8<T> x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (at[k] >= 0) x[k] = row8_load<T>(a.dy + at[k] * a.lddy + c, a.d - c);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (at[k] >= 0)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += x[k].get(i);
    if (at[7] < 0) break;
  }
  finish8<O>(a, own, c, acc);
}

// ---------------------------------------------------------------- places of the sorted tokens
// By workgroups of 1024 threads: 64 tokens, a 16th of all ids each wavefront, from LDS. In front of the
// workgroup's own tokens an equal id counts, behind them it does not. Workgroups from `ranks` on clear dE.
template <class O>
__global__ __launch_bounds__(1024) void k_embed_rank(EmbedView a, long ranks, long fills, uint32_t* __restrict__ keys,
                                                     int* __restrict__ order) {
  __shared__ uint32_t key[kRankedIds];
  __shared__ int part[16][64];
  const long b = block_id();
  if (b >= ranks) {
    const long f = b - ranks, per = (a.v + fills - 1) / fills;
    if (f < fills) fill_rows<O>(a, min(a.v, f * per), min(a.v, (f + 1) * per), nullptr, 0.0f);
    return;
  }
  const int t = (int)a.t, t0 = (int)b * 64, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int seg = (t + 63) / 64 * 4;  // a multiple of 4; 16 of them hold all
  for (int i = threadIdx.x; i < 16 * seg; i += 1024)
    key[i] = i < t ? id_key(a.ids[i], a.ignore, (uint32_t)a.v) : ~0u;
  __syncthreads();
  const uint32_t own = t0 + lane < t ? key[t0 + lane] : ~0u;
  int n = 0;
  const int s0 = wv * seg, s1 = s0 + seg;
  const int before = min(s1, max(s0, t0)), after = min(s1, max(s0, t0 + 64));
#pragma unroll 4
  for (int s = s0; s < before; s += 4) {
    const uint4 k = *reinterpret_cast<const uint4*>(key + s);
    n += k.x <= own, n += k.y <= own, n += k.z <= own, n += k.w <= own;
  }
  for (int s = before; s < after; ++s) n += key[s] < own || (key[s] == own && s < t0 + lane);
#pragma unroll 4
  for (int s = after; s < s1; s += 4) {
    const uint4 k = *reinterpret_cast<const uint4*>(key + s);
    n += k.x < own, n += k.y < own, n += k.z < own, n += k.w < own;
  }
  part[wv][lane] = n;
  __syncthreads();
  if (wv == 0 && t0 + lane < t) {
    int at = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) at += part[w][lane];
    keys[at] = own;
    order[at] = t0 + lane;
  }
}

// Digits of the first pass counted by tile, hist[tile][digit]; the next pass's counts cleared. Workgroups from
// `tiles` on clear dE.
template <class O>
__global__ __launch_bounds__(512) void k_embed_count(EmbedView a, long tiles, long fills, int bits,
                                                     uint32_t* __restrict__ hist, uint32_t* __restrict__ next) {
  __shared__ uint32_t n[512];
  const long b = block_id();
  if (b >= tiles) {
    const long f = b - tiles, per = (a.v + fills - 1) / fills;
    if (f < fills) fill_rows<O>(a, min(a.v, f * per), min(a.v, (f + 1) * per), nullptr, 0.0f);
    return;
  }
  n[threadIdx.x] = 0;
  __syncthreads();
  const int digits = 1 << bits;
  for (int k = 0; k < kTile / 512; ++k) {
    const long i = b * kTile + k * 512 + threadIdx.x;
    if (i < a.t) atomicAdd(&n[id_key(a.ids[i], a.ignore, (uint32_t)a.v) & (digits - 1)], 1u);
  }
  __syncthreads();
  if ((int)threadIdx.x < digits) {
    hist[b * digits + threadIdx.x] = n[threadIdx.x];
    next[b * digits + threadIdx.x] = 0;
  }
}

// One pass of the radix sort, stable: a workgroup of 8 wavefronts moves a tile, each wavefront 512 neighbouring
// ids in 8 rounds of 64. A round's lanes of one digit find each other by a ballot for each bit. The digits' places
// are summed from all tiles' counts by every workgroup (a scan of its own would be a launch more). `next`:
// the next pass's counts, by the places' tiles (whole numbers: any order gives the same), `clear` the ones after.
template <bool FIRST>
__global__ __launch_bounds__(512) void k_embed_sort(EmbedView a, int tiles, int bits, int shift,
                                                    const uint32_t* __restrict__ hist, const uint32_t* __restrict__ keys,
                                                    const int* __restrict__ order, uint32_t* __restrict__ keys_to,
                                                    int* __restrict__ order_to, uint32_t* __restrict__ next,
                                                    uint32_t* __restrict__ clear) {
  __shared__ uint32_t place[8][512];
  __shared__ uint32_t scan[8];
  const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63, digits = 1 << bits;
  const long base = (long)blockIdx.x * kTile + wv * 512;
  uint32_t key[8];
  int tok[8], rank[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const long i = base + 64 * k + lane;
    key[k] = ~0u, tok[k] = 0;
    if (i < a.t) {
      key[k] = FIRST ? id_key(a.ids[i], a.ignore, (uint32_t)a.v) : keys[i];
      tok[k] = FIRST ? (int)i : order[i];
    }
  }
#pragma unroll
  for (int w = 0; w < 8; ++w) place[w][threadIdx.x] = 0;
  __syncthreads();
  volatile uint32_t* mine = place[wv];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const bool on = base + 64 * k + lane < a.t;
    const uint32_t digit = (key[k] >> shift) & (digits - 1);
    u64 peers = __ballot(on);
    for (int j = 0; j < bits; ++j) {
      const u64 ones = __ballot((digit >> j) & 1);
      peers &= (digit >> j) & 1 ? ones : ~ones;
    }
    const int r = __popcll(peers & ((1ull << lane) - 1));
    uint32_t old = 0;
    if (on) old = mine[digit];
    __builtin_amdgcn_wave_barrier();
    if (on && r == 0) mine[digit] = old + (uint32_t)__popcll(peers);
    __builtin_amdgcn_wave_barrier();
    rank[k] = (int)old + r;
  }
  // the digit's tokens in all tiles, and in the tiles before this one
  uint32_t all = 0, before = 0;
  if ((int)threadIdx.x < digits) {
#pragma unroll 8
    for (int i = 0; i < tiles; ++i) {
      const uint32_t c = hist[(long)i * digits + threadIdx.x];
      all += c;
      before += i < (int)blockIdx.x ? c : 0;
    }
    if (clear) clear[(long)blockIdx.x * digits + threadIdx.x] = 0;
  }
  uint32_t sum = all;  // of the digits up to this one
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint32_t up = (uint32_t)__shfl_up((int)sum, s);
    if (lane >= s) sum += up;
  }
  if (lane == 63) scan[wv] = sum;
  __syncthreads();
  uint32_t at = sum - all + before;
  for (int w = 0; w < wv; ++w) at += scan[w];
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const uint32_t c = place[w][threadIdx.x];
    place[w][threadIdx.x] = at;
    at += c;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (base + 64 * k + lane >= a.t) continue;
    const uint32_t to = place[wv][(key[k] >> shift) & (digits - 1)] + rank[k];
    keys_to[to] = key[k];
    order_to[to] = tok[k];
    if (next) atomicAdd(&next[(long)(to / kTile) * digits + ((key[k] >> (shift + bits)) & (digits - 1))], 1u);
  }
}

// ---------------------------------------------------------------- sums of the sorted tokens
// `lanes` lanes take a chunk of the sorted tokens and 8 columns each. A run of equal ids that begins and ends in the
// chunk is finished here; one that came from the chunk before leaves its sum in head[chunk], one that goes on into
// the next in tail[chunk] (head if it came, too).
template <class T, class O>
__global__ __launch_bounds__(256) void k_embed_sums(EmbedView a, const uint32_t* __restrict__ keys,
                                                    const int* __restrict__ order, int chunk, long chunks, long parts,
                                                    float* __restrict__ head, float* __restrict__ tail) {
  const long unit = block_id() * (256 / a.lanes) + threadIdx.x / a.lanes;
  if (unit >= chunks * parts) return;
  const long ch = unit / parts, c = ((unit - ch * parts) * a.lanes + (threadIdx.x & (a.lanes - 1))) * 8;
  if (c >= a.d) return;
  const long p0 = ch * chunk, p1 = min(a.t, p0 + chunk);
  const uint32_t v = (uint32_t)a.v;
  bool came = p0 > 0 && keys[p0 - 1] == keys[p0];
  uint32_t cur = keys[p0];
  float acc[8] = {};
  auto part = [&](float* to) {
    float* p = to + ch * a.d + c;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < a.d) p[i] = acc[i];
  };
  for (long p = p0; p < p1 && cur < v; p += 8) {
    uint32_t k[8];
    Row8<T> x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      k[j] = p + j < p1 ? keys[p + j] : v;
      if (k[j] < v) x[j] = row8_load<T>(a.dy + (long)order[p + j] * a.lddy + c, a.d - c);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (p + j >= p1 || cur >= v) continue;
      if (k[j] != cur) {
        if (came) part(head);
        else finish8<O>(a, cur, c, acc);
        came = false;
        cur = k[j];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
      }
      if (cur < v)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += x[j].get(i);
    }
  }
  if (cur >= v) return;
  if (came) part(head);
  else if (p1 < a.t && keys[p1] == cur) part(tail);
  else finish8<O>(a, cur, c, acc);
}

// A run that passes the end of the chunk where it began: its parts summed in order, a quarter of them each
// wavefront, 256 columns a workgroup.
template <class O>
__global__ __launch_bounds__(256) void k_embed_join(EmbedView a, const uint32_t* __restrict__ keys, int chunk,
                                                    long chunks, long slabs, const float* __restrict__ head,
                                                    const float* __restrict__ tail) {
  __shared__ float red[4][256];
  const long b = block_id(), v = a.v;
  if (keys[a.t - 1] > v) return poison<O>(a, b, (long)gridDim.x * gridDim.y);
  if (b >= chunks * slabs) return;
  const long ch = b / slabs, end = (ch + 1) * chunk;
  if (end >= a.t) return;
  const uint32_t k = keys[end - 1];
  if (k >= v || keys[end] != k) return;
  if (ch > 0 && keys[ch * chunk - 1] == k) return;  // it began before
  const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
  long last = ch + 1;  // the chunk where it ends
  while (true) {
    const long at = (last + lane + 1) * chunk;
    const u64 on = __ballot(at < a.t && keys[at] == k && keys[at - 1] == k);
    if (~on) {
      last += __builtin_ctzll(~on);
      break;
    }
    last += 64;
  }
  const long n = last - ch, c = (b - ch * slabs) * 256 + 4 * lane;
  const long from = ch + 1 + n * wv / 4, to = ch + 1 + n * (wv + 1) / 4;
  float s[4] = {};
#pragma unroll 8
  for (long i = from; i < to; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < a.d) s[j] += head[i * a.d + c + j];
#pragma unroll
  for (int j = 0; j < 4; ++j) red[wv][4 * lane + j] = s[j];
  __syncthreads();
  if (threadIdx.x >= 32) return;
  const long c8 = (b - ch * slabs) * 256 + 8 * threadIdx.x;
  if (c8 >= a.d) return;
  float sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sum[i] = c8 + i < a.d ? tail[ch * a.d + c8 + i] : 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) sum[i] += red[w][8 * threadIdx.x + i];
  }
  finish8<O>(a, k, c8, sum);
}

struct EmbedPlan {
  int chunk, bits, passes;
  long chunks, tiles;
  size_t keys[2], order[2], hist[3], head, tail, bytes;
};
EmbedPlan embed_plan(long t, long d, long v) {
  EmbedPlan p = {};
  if (t <= kFewIds) return p;
  auto take = [&](size_t n) {
    const size_t at = p.bytes;
    p.bytes += (n + 255) / 256 * 256;
    return at;
  };
  const int sets = t <= kRankedIds ? 1 : 2;
  for (int i = 0; i < sets; ++i) p.keys[i] = take(4 * t), p.order[i] = take(4 * t);
  if (sets == 2) {
    int total = 1;
    while ((v + 1) >> total) ++total;
    p.passes = (total + 8) / 9;
    p.bits = (total + p.passes - 1) / p.passes;
    p.tiles = (t + kTile - 1) / kTile;
    for (int i = 0; i < 3; ++i) p.hist[i] = take(4 * p.tiles << p.bits);
  }
  // Chunks as long as leaves 4096 wavefronts (a wavefront reads 8 rows' 16 bytes a lane at once).
  const long waves = (d + 511) / 512 * t;
  p.chunk = 8;
  while (p.chunk < 64 && waves / p.chunk > 8192) p.chunk *= 2;
  while ((t + p.chunk - 1) / p.chunk > 16384) p.chunk *= 2;
  p.chunks = (t + p.chunk - 1) / p.chunk;
  p.head = take(4 * p.chunks * d);
  p.tail = take(4 * p.chunks * d);
  return p;
}

template <class T, class O>
hipError_t backward(hipStream_t st, EmbedView a, void* work) {
  const bool clear = !a.add;
  if (a.t <= kFewIds) {
    const int slabs = (int)((a.d + 2047) / 2048);
    // rows of 128 KB to a clearing workgroup, which looks at all ids once
    const int rows = (int)std::max(1l, std::min(1024l, 65536 / a.d));
    const long sums = a.t * slabs, fills = clear ? (a.v + rows - 1) / rows : 0;
    k_embed_few<T, O><<<launch_grid(std::max(1l, sums + fills)), 256, 0, st>>>(a, slabs, sums, rows);
    return hipGetLastError();
  }
  const EmbedPlan p = embed_plan(a.t, a.d, a.v);
  char* w = static_cast<char*>(work);
  uint32_t *keys[2], *hist[3];
  int* order[2];
  for (int i = 0; i < 2; ++i) {
    keys[i] = reinterpret_cast<uint32_t*>(w + p.keys[i]);
    order[i] = reinterpret_cast<int*>(w + p.order[i]);
  }
  for (int i = 0; i < 3; ++i) hist[i] = reinterpret_cast<uint32_t*>(w + p.hist[i]);
  float *head = reinterpret_cast<float*>(w + p.head), *tail = reinterpret_cast<float*>(w + p.tail);
  int at = 0;
  if (a.t <= kRankedIds) {
    const long ranks = (a.t + 63) / 64, fills = clear ? std::min(a.v, 4096l) : 0;
    k_embed_rank<O><<<launch_grid(ranks + fills), 1024, 0, st>>>(a, ranks, fills, keys[0], order[0]);
  } else {
    const long fills = clear ? std::min(a.v, 4096l) : 0;
    k_embed_count<O><<<launch_grid(p.tiles + fills), 512, 0, st>>>(a, p.tiles, fills, p.bits, hist[0], hist[1]);
    const int tiles = (int)p.tiles;
    uint32_t* next = p.passes > 1 ? hist[1] : nullptr;
    k_embed_sort<true><<<tiles, 512, 0, st>>>(a, tiles, p.bits, 0, hist[0], nullptr, nullptr, keys[0], order[0], next, hist[2]);
    for (int i = 1; i < p.passes; ++i) {
      next = i + 1 < p.passes ? hist[i + 1] : nullptr;
      k_embed_sort<false><<<tiles, 512, 0, st>>>(a, tiles, p.bits, i * p.bits, hist[i], keys[at], order[at], keys[at ^ 1],
                                                 order[at ^ 1], next, nullptr);
      at ^= 1;
    }
  }
  const long parts = (a.d + 8l * a.lanes - 1) / (8l * a.lanes), units = p.chunks * parts, per = 256 / a.lanes;
  k_embed_sums<T, O><<<launch_grid((units + per - 1) / per), 256, 0, st>>>(a, keys[at], order[at], p.chunk, p.chunks, parts, head, tail);
  const long slabs = (a.d + 255) / 256;
  k_embed_join<O><<<launch_grid(p.chunks * slabs), 256, 0, st>>>(a, keys[at], p.chunk, p.chunks, slabs, head, tail);
  return hipGetLastError();
}

}  // namespace

hipError_t embed_rows(hipStream_t st, int dtype, const uint16_t* table, long ldt, long v, long d, const int64_t* ids,
                      long t, float scale, int64_t ignore, uint16_t* out, long ldo) {
  const int lanes = row_lanes(d);
  const long parts = (d + 64l * lanes - 1) / (64l * lanes), per = 256 / lanes;
  const dim3 grid = launch_grid((t * parts + per - 1) / per);
  if (dtype == CDCLQ_DTYPE_BF16) k_embed_rows<Bf16><<<grid, 256, 0, st>>>(table, ldt, v, d, ids, t, scale, ignore, out, ldo, lanes, parts);
  else k_embed_rows<F16><<<grid, 256, 0, st>>>(table, ldt, v, d, ids, t, scale, ignore, out, ldo, lanes, parts);
  return hipGetLastError();
}

size_t embed_work_bytes(long t, long d, long v) { return embed_plan(t, d, v).bytes; }

hipError_t embed_grad(hipStream_t st, int dtype, const uint16_t* dy, long lddy, long t, long d, long v,
                      const int64_t* ids, float scale, int64_t ignore, bool add, void* de, long lde, int de_dtype,
                      void* work) {
  const EmbedView a = {ids, t, d, v, ignore, scale, dy, lddy, de, lde, row_lanes(d), add};
  const bool wide = de_dtype == CDCLQ_DTYPE_F32;
  if (dtype == CDCLQ_DTYPE_BF16) return wide ? backward<Bf16, F32>(st, a, work) : backward<Bf16, Bf16>(st, a, work);
  return wide ? backward<F16, F32>(st, a, work) : backward<F16, F16>(st, a, work);
}

}  // namespace cdclq
