// Token embedding and the gradient of its table.
//
//   y_t = scale E[id_t]            dE[v] = scale sum over the tokens t with id_t = v of dy_t
//
// An id equal to the ignored one stands for no token: y_t = 0, and it adds nothing. Any other id outside 0..v
// gives a row of NaN and a gradient that is NaN throughout. Both directions only move memory: 16384 rows of 4096 of a
// table of 128256 36 us (188 MB, 5.2 TB/s); rows and gradient of 4096 tokens there 180 us, 159 of them the clearing of
// 1.05 GB (6.6 TB/s); of 32768 tokens, 2048 of 32000, 101 us. The last one's launches by themselves, in medians: rows 31,
// sorting and clearing 28, sums 39, runs of chunks 6. Added to a gradient that exists, nothing is cleared beside the ranks
// and the sort: 4096 tokens, 2048 of 32000, 23 us, of them 7 the ranks, 11 the sums and 5 the runs.
//
// The gradient sums a row's tokens in f32, with one rounding at the end and no float atomics: a chunk's in their order, a
// run of chunks in four quarters that are added up. Equal inputs give equal bits. Three forms by the number of tokens:
//   few     one launch: a workgroup takes a token, finds the others of its id by comparing all ids, and leaves unless it
//           is the first of them; other workgroups clear the rows without tokens.
//   ranked  a token's place among the sorted ones is the number of smaller (id, position) pairs, counted by
//           comparing all pairs of tokens in one launch, which clears dE beside it. Then chunks of the sorted tokens
//           are summed; runs of equal ids that pass a chunk's end are joined by a third launch.
//   sorted  the places from a radix sort of 5 to 9 bits a pass, whose launches clear dE beside them.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "cdclq.h"
#include "kernels.h"
#include "row8.h"

namespace cdclq {
namespace {

typedef unsigned long long u64;

// Tokens up to which each form is taken. Rows of 2048 of 32000, added to a gradient that exists: 128 tokens 6.8 us in the
// first and 14.8 in the second, all of one id 25.5 and 14.8 (256: 6.8 and 14.5, 47 and 14.5; into a new gradient 25 and 30);
// 4096 tokens 23 in the second and 36 in the third, 8192 36 and 43, 12000 55 and 53.
constexpr long kFewIds = 128, kRankedIds = 8192;
static_assert(kFewIds <= 256, "64 ids a wavefront of k_embed_few");
// Wavefronts that sum chunks, as long as those have fewer than 64 tokens: 32768 x 2048: 101 us a step, with four times as
// many (chunks of 16, more runs to join) 105.
constexpr long kMostWaves = 2048;
constexpr int kTile = 2048;  // ids of a workgroup of the radix sort

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
  const int lane = threadIdx.x & (lanes - 1);
  const long row = unit / parts, part = unit - row * parts, c0 = part * lanes * 64 + 8 * lane;
  const uint32_t key = id_key(ids[row], ignore, (uint32_t)v);
  const bool is = key < (uint32_t)v;
  const float other = key == (uint32_t)v ? 0.0f : __builtin_nanf("");
  const uint16_t* from = table + (is ? key : 0) * ldt;
  uint16_t* to = out + row * ldo;
  Row8<T> x[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const long c = c0 + 8l * lanes * k;
    if (c + 8 <= d) x[k] = row8_load<T>(from + c);
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const long c = c0 + 8l * lanes * k;
    if (c + 8 > d) continue;
    if (scale != 1.0f || !is)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[k].set(i, is ? scale * x[k].get(i) : other);
    row8_store<T>(to + c, x[k]);
  }
  if (part == parts - 1)  // the elements past the last eight
    for (long c = (d & ~7l) + lane; c < d; c += lanes)
      to[c] = !is ? T::narrow(other) : scale != 1.0f ? T::narrow(scale * T::widen(from[c])) : from[c];
}

// x in every element of share b of nb of dE's elements [e0, e1) in rows of d, counted row by row. KEEP: through the L2,
// which is better for a few rows beside sums (77 tokens, 50001 x 1000: 19.5 us a step, past it 21.3).
template <class O, bool KEEP>
__device__ __forceinline__ void fill(const EmbedView& a, long e0, long e1, long b, long nb, float x) {
  typedef typename Row8<O>::stored E;
  E* const de = static_cast<E*>(a.de);
  const E one = Row8<O>::narrow(x);
  Row8<O> eight;
#pragma unroll
  for (int i = 0; i < 8; ++i) eight.v[i] = one;
  if (a.lde == a.d) {  // one piece of memory
    const long n = e1 - e0, per = ((n + nb - 1) / nb + 7) & ~7l;
    const long from = e0 + min(n, b * per), to = e0 + min(n, (b + 1) * per);
    long i = from + 8 * (long)threadIdx.x;
    for (; i + 8 <= to; i += 8 * blockDim.x) row8_store<O, KEEP>(de + i, eight);
    for (; i < to; ++i) de[i] = one;
    return;
  }
  const long r1 = e1 / a.d;
  for (long r = e0 / a.d + b; r < r1; r += nb) {
    long c = 8 * (long)threadIdx.x;
    for (; c + 8 <= a.d; c += 8 * blockDim.x) row8_store<O, KEEP>(de + r * a.lde + c, eight);
    for (; c < a.d; ++c) de[r * a.lde + c] = one;
  }
}
// Zeros in part `i` of `n` of dE's rows, past the L2 (4096 tokens, 128256 x 4096: 180 us a step, through it 196).
template <class O>
__device__ __forceinline__ void clear(const EmbedView& a, int i, int n, long b, long nb) {
  if (b < nb) fill<O, false>(a, a.v * i / n * a.d, a.v * (i + 1) / n * a.d, b, nb, 0.0f);
}
// dE = NaN throughout, by all workgroups of a launch (an id outside 0..v).
template <class O>
__device__ void poison(const EmbedView& a, long b, long nb) {
  fill<O, true>(a, 0, a.v * a.d, b, nb, __builtin_nanf(""));
}

// A finished sum of eight columns into dE: the only rounding. ALL: all eight are there.
template <class O, bool ALL>
__device__ __forceinline__ void finish8(const EmbedView& a, uint32_t row, long c, const float* sum) {
  auto* p = static_cast<typename Row8<O>::stored*>(a.de) + row * a.lde + c;
  const int n = ALL ? 8 : (int)(a.d - c);
  Row8<O> r;
  if (a.add) {
    if constexpr (ALL) r = row8_load<O>(p);
    else r = row8_load<O>(p, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) r.set(i, __builtin_fmaf(a.scale, sum[i], r.get(i)));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.set(i, a.scale * sum[i]);
  }
  if constexpr (ALL) row8_store<O>(p, r);
  else row8_store<O>(p, r, n);
}
template <class T, bool ALL>
__device__ __forceinline__ Row8<T> load8(const EmbedView& a, long row, long c) {
  const uint16_t* p = a.dy + row * a.lddy + c;
  if constexpr (ALL) return row8_load<T, true>(p);
  else return row8_load<T>(p, (int)(a.d - c));
}

// ---------------------------------------------------------------- few tokens
// Rows that a workgroup clears: 16 KB of them.
inline long few_rows(long d) { return std::max(1l, std::min(8192 / d, 1024l)); }

// Workgroups below t slabs: token b / slabs, 8 x 256 columns. The others clear `rows` rows each, but those of tokens
// (77 tokens, 1000 of 50001: 16.5 us, 6.1 TB/s; with the clearing as a launch before 15.2 + 4.6).
template <class T, class O>
__global__ __launch_bounds__(256) void k_embed_few(EmbedView a, int slabs, int rows) {
  __shared__ u64 same[kFewIds / 64], bad[kFewIds / 64];
  __shared__ uint32_t hits[32];  // a bit for each row to clear that has tokens
  const long b = block_id(), sums = a.t * slabs, blocks = sums + (a.add ? 0 : (a.v + rows - 1) / rows);
  const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (b >= blocks) return;
  const bool clears = b >= sums;
  const int tok = clears ? 0 : (int)(b / slabs), words = (int)((a.t + 63) / 64);
  const long r0 = clears ? (b - sums) * rows : 0, r1 = min(a.v, r0 + rows);
  const uint32_t v = (uint32_t)a.v, own = clears ? 0 : id_key(a.ids[tok], a.ignore, v);
  if (threadIdx.x < 32) hits[threadIdx.x] = 0;
  __syncthreads();
  if (wv < words) {  // `same`: the tokens of this one's id, or those of the rows to clear
    const int i = 64 * wv + lane;
    const uint32_t k = i < a.t ? id_key(a.ids[i], a.ignore, v) : v;
    const bool mine = clears ? k < v && k >= r0 && k < r1 : i < a.t && k == own;
    const u64 s = __ballot(mine), n = __ballot(k > v);
    if (lane == 0) same[wv] = s, bad[wv] = n;
    if (clears && mine) atomicOr(&hits[(k - r0) >> 5], 1u << ((k - r0) & 31));
  }
  __syncthreads();
  u64 any = 0;
  for (int w = 0; w < words; ++w) any |= bad[w];
  if (any) return poison<O>(a, b, blocks);
  if (clears) {  // the rows between those of tokens
    const int n = (int)(r1 - r0);
    for (int i = 0; i < n;) {
      int e = i;
      while (e < n) {
        const uint32_t m = hits[e >> 5] >> (e & 31);
        if (m) {
          e += __builtin_ctz(m);
          break;
        }
        e = (e | 31) + 1;
      }
      e = min(e, n);
      if (e > i) fill<O, true>(a, (r0 + i) * a.d, (r0 + e) * a.d, 0, 1, 0.0f);
      i = e + 1;
    }
    return;
  }
  if (own >= v) return;
  for (int w = 0; w <= tok / 64; ++w)
    if (same[w] & (w < tok / 64 ? ~0ull : (1ull << (tok & 63)) - 1)) return;  // an earlier token sums them
  const long c = ((b - (long)tok * slabs) * 256 + threadIdx.x) * 8;
  if (c >= a.d) return;
  auto sum = [&](auto all) {
    constexpr bool ALL = decltype(all)::value;
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
        if (at[k] >= 0) x[k] = load8<T, ALL>(a, at[k], c);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (at[k] >= 0)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] += x[k].get(i);
      if (at[7] < 0) break;
    }
    finish8<O, ALL>(a, own, c, acc);
  };
  if (c + 8 <= a.d) sum(std::true_type{});
  else sum(std::false_type{});
}

// ---------------------------------------------------------------- places of the sorted tokens
// Ids of one of n shares of t, a multiple of 4.
inline __host__ __device__ int rank_segment(int t, int n) { return (t + 4 * n - 1) / (4 * n) * 4; }
// By workgroups of 1024 threads: 64 / G tokens, each with G lanes of every wavefront, which share all ids between them,
// from LDS (4096 tokens: 20.4 us the gradient with 4 lanes a token, 24.6 with one). In front of the workgroup's own tokens
// an equal id counts, behind them it does not. Workgroups from `ranks` on clear dE.
template <class O, int G>
__global__ __launch_bounds__(1024) void k_embed_rank(EmbedView a, long ranks, long fills, uint32_t* __restrict__ keys,
                                                     int* __restrict__ order, uint32_t* __restrict__ runs) {
  constexpr int NT = 64 / G, SEGS = 16 * G;
  extern __shared__ __align__(16) uint32_t key[];
  __shared__ int part[SEGS][NT];
  const long b = block_id();
  if (b >= ranks) return clear<O>(a, 0, 1, b - ranks, fills);
  if (b == 0 && threadIdx.x == 0) *runs = 0;
  const int t = (int)a.t, lane = threadIdx.x & (NT - 1), sg = threadIdx.x / NT;
  const int t0 = (int)b * NT, seg = rank_segment(t, SEGS);
  for (int i = threadIdx.x; i < SEGS * seg; i += 1024)
    key[i] = i < t ? id_key(a.ids[i], a.ignore, (uint32_t)a.v) : ~0u;
  __syncthreads();
  const uint32_t own = t0 + lane < t ? key[t0 + lane] : ~0u;
  int n = 0;
  const int s0 = sg * seg, s1 = s0 + seg;
  const int before = min(s1, max(s0, t0)), after = min(s1, max(s0, t0 + NT));
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
  part[sg][lane] = n;
  __syncthreads();
  if (threadIdx.x < NT && t0 + lane < t) {
    int at = 0;
#pragma unroll
    for (int w = 0; w < SEGS; ++w) at += part[w][lane];
    keys[at] = own;
    order[at] = t0 + lane;
  }
}
template <class O, int G>
void rank(hipStream_t st, const EmbedView& a, long fills, uint32_t* keys, int* order, uint32_t* runs) {
  const long ranks = (a.t * G + 63) / 64;
  const size_t lds = 4 * (size_t)(16 * G) * rank_segment((int)a.t, 16 * G);
  k_embed_rank<O, G><<<launch_grid(ranks + fills), 1024, lds, st>>>(a, ranks, fills, keys, order, runs);
}

// One pass of the radix sort is two launches. Each clears a share of dE beside it, by the workgroups from `tiles` on.
struct SortPass {
  int tiles, bits, shift;
  int launch, launches;  // for the clearing
  long fills;
  uint32_t* hist;  // [tile][digit]
  const uint32_t* keys;  // null: the ids themselves
  const int* order;
  uint32_t* keys_to;
  int* order_to;
  uint32_t* runs;
};

// The ids of each digit by tile.
template <class O>
__global__ __launch_bounds__(512) void k_embed_count(EmbedView a, SortPass p) {
  __shared__ uint32_t n[512];
  const long b = block_id();
  if (b >= p.tiles) return clear<O>(a, p.launch, p.launches, b - p.tiles, p.fills);
  if (b == 0 && threadIdx.x == 0) *p.runs = 0;
  n[threadIdx.x] = 0;
  __syncthreads();
  const int digits = 1 << p.bits;
#pragma unroll
  for (int k = 0; k < kTile / 512; ++k) {
    const long i = b * kTile + k * 512 + threadIdx.x;
    if (i < a.t) {
      const uint32_t key = p.keys ? p.keys[i] : id_key(a.ids[i], a.ignore, (uint32_t)a.v);
      atomicAdd(&n[(key >> p.shift) & (digits - 1)], 1u);
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < digits) p.hist[b * digits + threadIdx.x] = n[threadIdx.x];
}

// Stable: a workgroup of 8 wavefronts moves a tile, each wavefront 256 neighbouring ids in 4 rounds of 64. A round's
// lanes of one digit find each other by a ballot for each bit. The digits' places are summed from all tiles' counts by
// every workgroup (running sums in a launch of their own: 16384 ids 37.3 us and 37.5, 131072 66 and 72, 2^21 254 and 273).
template <class O>
__global__ __launch_bounds__(512) void k_embed_sort(EmbedView a, SortPass p) {
  __shared__ uint32_t place[8][512];
  __shared__ uint32_t scan[8];
  if (block_id() >= p.tiles) return clear<O>(a, p.launch, p.launches, block_id() - p.tiles, p.fills);
  constexpr int R = kTile / 512;
  const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63, digits = 1 << p.bits;
  const long tile = block_id(), base = tile * kTile + wv * (64 * R);
  uint32_t key[R];
  int tok[R], rank[R];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const long i = base + 64 * k + lane;
    key[k] = ~0u, tok[k] = 0;
    if (i < a.t) {
      key[k] = p.keys ? p.keys[i] : id_key(a.ids[i], a.ignore, (uint32_t)a.v);
      tok[k] = p.keys ? p.order[i] : (int)i;
    }
  }
#pragma unroll
  for (int w = 0; w < 8; ++w) place[w][threadIdx.x] = 0;
  // the digit's tokens in all tiles, and in the tiles before this one
  uint32_t all = 0, before = 0;
  if ((int)threadIdx.x < digits) {
#pragma unroll 16
    for (int i = 0; i < p.tiles; ++i) {
      const uint32_t c = p.hist[(long)i * digits + threadIdx.x];
      all += c;
      before += i < tile ? c : 0;
    }
  }
  __syncthreads();
  volatile uint32_t* mine = place[wv];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const bool on = base + 64 * k + lane < a.t;
    const uint32_t digit = (key[k] >> p.shift) & (digits - 1);
    u64 peers = __ballot(on);
    for (int j = 0; j < p.bits; ++j) {
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
  for (int k = 0; k < R; ++k) {
    if (base + 64 * k + lane >= a.t) continue;
    const uint32_t to = place[wv][(key[k] >> p.shift) & (digits - 1)] + rank[k];
    p.keys_to[to] = key[k];
    p.order_to[to] = tok[k];
  }
}

// ---------------------------------------------------------------- sums of the sorted tokens
// The sorted tokens, and where the sums of runs that pass a chunk's end are kept: rows of dp columns.
struct Sorted {
  const uint32_t* keys;
  const int* order;
  int chunk;
  long chunks, dp;
  float *head, *tail;
  uint32_t *runs, *starts;  // how many such runs, and the chunks where they begin, in any order
};

// `lanes` lanes take a chunk of the sorted tokens and 8 columns each. A run of equal ids that begins and ends in the
// chunk is finished here; one that came from the chunk before leaves its sum in head[chunk], one that goes on into
// the next in tail[chunk] (head if it came, too).
// Rows of more than 256 columns (WAVE): the 64 lanes of a wavefront have a chunk in common, so that its ids and places
// are scalars (loaded as constants: this kernel does not write them) and the runs are told apart by scalar branches; 16
// rows' loads are on their way.
template <class T, class O, bool WAVE>
__global__ __launch_bounds__(256) void k_embed_sums(EmbedView a, Sorted s, long parts) {
  const int lanes = WAVE ? 64 : a.lanes;
  const long unit = WAVE ? block_id() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)
                         : block_id() * (256 / lanes) + threadIdx.x / lanes;
  if (unit >= s.chunks * parts) return;
  const long ch = unit / parts, c = ((unit - ch * parts) * lanes + (threadIdx.x & (lanes - 1))) * 8;
  const long p0 = ch * s.chunk, p1 = min(a.t, p0 + s.chunk);
  const uint32_t v = (uint32_t)a.v;
  typedef const __attribute__((address_space(4))) uint32_t* Keys;
  typedef const __attribute__((address_space(4))) int* Order;
  const std::conditional_t<WAVE, Keys, const uint32_t*> keys = (decltype(keys))(uintptr_t)s.keys;
  const std::conditional_t<WAVE, Order, const int*> order = (decltype(order))(uintptr_t)s.order;
  auto sum = [&](auto all) {
    constexpr bool ALL = decltype(all)::value;
    constexpr int U = 8;
    bool came = p0 > 0 && keys[p0 - 1] == keys[p0];
    uint32_t cur = keys[p0];
    float acc[8] = {};
    auto part = [&](float* to) {
      float* p = to + ch * s.dp + c;
      *reinterpret_cast<float4*>(p) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
    };
    auto add = [&](uint32_t k, const Row8<T>& x) {
      if (k != cur) {
        if (came) part(s.head);
        else finish8<O, ALL>(a, cur, c, acc);
        came = false;
        cur = k;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += x.get(i);
    };
    if constexpr (WAVE) {
      Row8<T> x[2][U];
      auto load = [&](long p, Row8<T>* to) {
#pragma unroll
        for (int j = 0; j < U; ++j) to[j] = load8<T, ALL>(a, order[min(p + j, p1 - 1)], c);
      };
      auto use = [&](long p, const Row8<T>* from) {
#pragma unroll
        for (int j = 0; j < U; ++j)
          if (p + j < p1 && cur < v) add(keys[p + j], from[j]);
      };
      load(p0, x[0]);
      for (long p = p0; p < p1 && cur < v; p += 2 * U) {
        if (p + U < p1) load(p + U, x[1]);
        use(p, x[0]);
        if (p + 2 * U < p1) load(p + 2 * U, x[0]);
        if (p + U < p1) use(p + U, x[1]);
      }
    } else {
      for (long p = p0; p < p1 && cur < v; p += U) {
        uint32_t k[U];
        Row8<T> x[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const long i = min(p + j, p1 - 1);
          k[j] = keys[i];
          x[j] = load8<T, ALL>(a, order[i], c);
        }
#pragma unroll
        for (int j = 0; j < U; ++j)
          if (p + j < p1 && cur < v) add(k[j], x[j]);
      }
    }
    if (cur >= v) return;
    if (came) {
      part(s.head);
    } else if (p1 < a.t && keys[p1] == cur) {
      part(s.tail);
      if (c == 0) s.starts[atomicAdd(s.runs, 1u)] = (uint32_t)ch;
    } else {
      finish8<O, ALL>(a, cur, c, acc);
    }
  };
  if (c + 8 <= a.d) sum(std::true_type{});
  else if (c < a.d) sum(std::false_type{});
}

// The runs that pass the end of the chunk where they began, each by 256 columns a workgroup: their parts summed in
// order, a quarter of them each wavefront.
template <class O>
__global__ __launch_bounds__(256) void k_embed_join(EmbedView a, Sorted s, uint32_t slabs) {
  __shared__ float red[4][256];
  const long b = block_id(), nb = (long)gridDim.x * gridDim.y;
  if (s.keys[a.t - 1] > a.v) return poison<O>(a, b, nb);
  const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long items = (long)*s.runs * slabs;
  for (long it = b; it < items; it += nb) {
    const long run = it / slabs, slab = it - run * slabs, ch = s.starts[run];
    const uint32_t k = s.keys[(ch + 1) * s.chunk];
    long last = ch + 1;  // the chunk where it ends
    while (true) {
      const long at = (last + lane + 1) * s.chunk;
      const u64 on = __ballot(at < a.t && s.keys[at] == k);
      if (~on) {
        last += __builtin_ctzll(~on);
        break;
      }
      last += 64;
    }
    const long n = last - ch, c = slab * 256 + 4 * lane;
    const long from = ch + 1 + n * wv / 4, to = ch + 1 + n * (wv + 1) / 4;
    float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (c < s.dp)
#pragma unroll 8
      for (long i = from; i < to; ++i) {
        const float4 h = *reinterpret_cast<const float4*>(s.head + i * s.dp + c);
        f.x += h.x, f.y += h.y, f.z += h.z, f.w += h.w;
      }
    *reinterpret_cast<float4*>(&red[wv][4 * lane]) = f;
    __syncthreads();
    const long c8 = slab * 256 + 8 * threadIdx.x;
    if (threadIdx.x < 32 && c8 < a.d) {
      float sum[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum[i] = s.tail[ch * s.dp + c8 + i];
#pragma unroll
        for (int w = 0; w < 4; ++w) sum[i] += red[w][8 * threadIdx.x + i];
      }
      if (c8 + 8 <= a.d) finish8<O, true>(a, k, c8, sum);
      else finish8<O, false>(a, k, c8, sum);
    }
    __syncthreads();
  }
}

struct EmbedPlan {
  int chunk, bits, passes, tiles;
  long chunks, dp;
  size_t keys[2], order[2], hist, head, tail, runs, starts, bytes;
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
    p.tiles = (int)((t + kTile - 1) / kTile);
    p.hist = take((size_t)4 * p.tiles << p.bits);
  }
  const long waves = (d + 511) / 512 * t;
  p.chunk = 8;
  while (p.chunk < 64 && waves / p.chunk > kMostWaves) p.chunk *= 2;
  while ((t + p.chunk - 1) / p.chunk > 16384) p.chunk *= 2;
  p.chunks = (t + p.chunk - 1) / p.chunk;
  p.dp = (d + 7) / 8 * 8;
  p.head = take(4 * p.chunks * p.dp);
  p.tail = take(4 * p.chunks * p.dp);
  p.runs = take(4);
  p.starts = take(4 * p.chunks);
  return p;
}

// Workgroups that clear n elements of dE, 16 KB of bf16 each: 4096 tokens, 128256 x 4096: 180 us a step, with 8 KB each
// 193, with 32 KB 195.
long clearing(const EmbedView& a, long n) { return a.add ? 0 : std::max(1l, std::min(n / 8192, 1l << 20)); }

template <class T, class O>
hipError_t backward(hipStream_t st, EmbedView a, void* work) {
  if (a.t <= kFewIds) {
    const int slabs = (int)((a.d + 2047) / 2048), rows = (int)few_rows(a.d);
    const long blocks = a.t * slabs + (a.add ? 0 : (a.v + rows - 1) / rows);
    k_embed_few<T, O><<<launch_grid(blocks), 256, 0, st>>>(a, slabs, rows);
    return hipGetLastError();
  }
  const EmbedPlan p = embed_plan(a.t, a.d, a.v);
  char* w = static_cast<char*>(work);
  uint32_t* keys[2];
  int* order[2];
  for (int i = 0; i < 2; ++i) {
    keys[i] = reinterpret_cast<uint32_t*>(w + p.keys[i]);
    order[i] = reinterpret_cast<int*>(w + p.order[i]);
  }
  uint32_t* const runs = reinterpret_cast<uint32_t*>(w + p.runs);
  int at = 0;
  if (a.t <= kRankedIds) {
    const long fills = clearing(a, a.v * a.d);  // as many lanes a token as give every CU a workgroup
    if (a.t > 4096) rank<O, 2>(st, a, fills, keys[0], order[0], runs);
    else rank<O, 4>(st, a, fills, keys[0], order[0], runs);
  } else {
    const int n = 2 * p.passes;
    const long fills = clearing(a, a.v * a.d / n);
    at = 1;
    for (int i = 0; i < p.passes; ++i) {
      SortPass s = {p.tiles, p.bits, i * p.bits, 2 * i, n, fills, reinterpret_cast<uint32_t*>(w + p.hist),
                    i ? keys[at] : nullptr, order[at], keys[at ^ 1], order[at ^ 1], runs};
      k_embed_count<O><<<launch_grid(p.tiles + fills), 512, 0, st>>>(a, s);
      ++s.launch;
      k_embed_sort<O><<<launch_grid(p.tiles + fills), 512, 0, st>>>(a, s);
      at ^= 1;
    }
  }
  const Sorted s = {keys[at], order[at], p.chunk, p.chunks, p.dp, reinterpret_cast<float*>(w + p.head),
                    reinterpret_cast<float*>(w + p.tail), runs, reinterpret_cast<uint32_t*>(w + p.starts)};
  const long parts = (a.d + 8l * a.lanes - 1) / (8l * a.lanes), units = p.chunks * parts, per = 256 / a.lanes;
  const dim3 grid = launch_grid((units + per - 1) / per);
  if (a.lanes == 64) k_embed_sums<T, O, true><<<grid, 256, 0, st>>>(a, s, parts);
  else k_embed_sums<T, O, false><<<grid, 256, 0, st>>>(a, s, parts);
  const long slabs = (a.d + 255) / 256;
  k_embed_join<O><<<(int)std::min(p.chunks * slabs, 2048l), 256, 0, st>>>(a, s, (uint32_t)slabs);
  return hipGetLastError();
}

}  // namespace

hipError_t embed_rows(hipStream_t st, int dtype, const uint16_t* table, long ldt, long v, long d, const int64_t* ids,
                      long t, float scale, int64_t ignore, uint16_t* out, long ldo) {
  const int lanes = row_lanes(d);
  const long parts = (d + 64l * lanes - 1) / (64l * lanes), per = 256 / lanes;
  const dim3 grid = launch_grid((t * parts + per - 1) / per);
  const auto rows = dtype == CDCLQ_DTYPE_BF16 ? k_embed_rows<Bf16> : k_embed_rows<F16>;
  rows<<<grid, 256, 0, st>>>(table, ldt, v, d, ids, t, scale, ignore, out, ldo, lanes, parts);
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
