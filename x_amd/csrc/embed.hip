// Token embedding: out[i] = scale * table[ids[i]], and its gradient gtable[v] = scale * sum of gout[i] over ids[i] = v.
// An id outside [0, V) is no token (as an event outside the image): its row is zeros and takes no gradient.
//
// Forward: one pass, 16 bytes of a row per lane where widths and addresses allow it.  Rows are stored through the cache:
// past it the 1M x 64 case runs 23 us instead of 44, but the norm that reads the rows next loses 26.
// Gradient: the tokens are sorted by id (a stable radix sort of (id, position), digits of up to 10 bits), so that the
// rows of one id are one run and every sum is taken in the order of the tokens: no atomic adds, the same bits on every
// call however often an id occurs (a hot pixel may own a tenth of a million events).  The sorted positions are cut into
// equal chunks, so a long run is shared by many lanes: a run inside a chunk is written at once, the partial sums of runs
// that cross chunks are joined afterwards, in order.  Sums are fp32, each row is rounded once.
#include "typed.h"
#include "../../include/atl_hip.h"

#include <algorithm>
#include <type_traits>

namespace atlhip {
namespace {

struct Rec { uint32_t key, idx; };

__device__ __forceinline__ int64_t id_at(const void* __restrict__ ids, bool wide, int64_t i) {
  return wide ? ((const int64_t*)ids)[i] : (int64_t)((const int32_t*)ids)[i];
}

template <typename T, typename O, int V>
__global__ void __launch_bounds__(kBlock) k_embed_fwd(const void* __restrict__ ids, bool wide, int64_t N, int64_t vocab,
                                                      const T* __restrict__ table, int64_t st, uint32_t units,
                                                      uint32_t unit_m, float scale, O* __restrict__ out, int rows,
                                                      int64_t first) {
  constexpr int kAhead = 4;                       // pieces in flight: ids, then rows, then stores
  const int64_t r0 = (first + blockIdx.x) * rows;
  const uint32_t items = (uint32_t)min((int64_t)rows, N - r0) * units;
  for (uint32_t e0 = threadIdx.x; e0 < items; e0 += kBlock * kAhead) {
    int64_t id[kAhead];
    uint32_t row[kAhead], c[kAhead];
    Pack<T, V> v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const uint32_t e = min(e0 + k * kBlock, items - 1);
      row[k] = units == 1 ? e : __umulhi(e, unit_m);       // e / units: e and units are below 2^16 + 1
      c[k] = (e - row[k] * units) * V;
      id[k] = id_at(ids, wide, r0 + row[k]);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      v[k] = load_pack<T, V>(table + (id[k] >= 0 && id[k] < vocab ? id[k] : 0) * st + c[k]);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (e0 + k * kBlock >= items) break;
      float f[V];
      const bool token = id[k] >= 0 && id[k] < vocab;
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = token ? (float)v[k].e[j] * scale : 0.f;
      store_f<V>(out + (r0 + row[k]) * (int64_t)units * V + c[k], f);
    }
  }
}

// ------------------------------------------------------------------------------------------- stable radix sort
constexpr int kSortBlock = 1024, kSortItems = 4, kSortTile = kSortBlock * kSortItems, kMaxDigitBits = 10;
constexpr int kSortWaves = kSortBlock / kWave;

// The record at position i: of the first pass from the ids (an id that is no token sorts behind all others).
template <bool FIRST>
__device__ __forceinline__ Rec rec_at(const void* __restrict__ src, bool wide, int64_t vocab, int64_t i) {
  if constexpr (FIRST) {
    const int64_t id = id_at(src, wide, i);
    return Rec{(uint32_t)(id >= 0 && id < vocab ? id : vocab), (uint32_t)i};
  } else {
    return ((const Rec*)src)[i];
  }
}

// Zeros, by 16 bytes, of the given piece of pieces; p is aligned to them.
__device__ __forceinline__ void clear_piece(uint16_t* __restrict__ p, int64_t halves, int64_t piece, int64_t pieces) {
  for (int64_t i = (piece * kSortBlock + threadIdx.x) * 8; i < halves; i += pieces * kSortBlock * 8) {
    if (i + 8 <= halves) *reinterpret_cast<uint4*>(p + i) = make_uint4(0, 0, 0, 0);
    else
      for (int64_t k = i; k < halves; ++k) p[k] = 0;
  }
}

// cnt (blocks, digits): how often each digit occurs in the block's tile.  The workgroups past the tiles clear the
// gradient's rows (of the first pass; most ids may have no token).
template <bool FIRST>
__global__ void __launch_bounds__(kSortBlock) k_sort_count(const void* __restrict__ src, bool wide, int64_t vocab,
                                                           int64_t N, int shift, int bits, int nblk, int* __restrict__ cnt,
                                                           uint16_t* __restrict__ gt, int64_t halves) {
  __shared__ int hist[1 << kMaxDigitBits];
  if ((int)blockIdx.x >= nblk) {
    clear_piece(gt, halves, blockIdx.x - nblk, gridDim.x - nblk);
    return;
  }
  const int nd = 1 << bits;
  for (int d = threadIdx.x; d < nd; d += kSortBlock) hist[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortTile;
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const int64_t i = base + k * kSortBlock + threadIdx.x;
    if (i < N) atomicAdd(&hist[(rec_at<FIRST>(src, wide, vocab, i).key >> shift) & (nd - 1)], 1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < nd; d += kSortBlock) cnt[(int64_t)blockIdx.x * nd + d] = hist[d];
}

// In place, per digit: the count of a block becomes that of the blocks before it; tot (digits): of all.  16 digits a
// workgroup, a stretch of the blocks per 16 threads.
constexpr int kOffDigits = 16, kOffRuns = kSortBlock / kOffDigits;
__global__ void __launch_bounds__(kSortBlock) k_sort_offsets(int* __restrict__ cnt, int nblk, int nd, int* __restrict__ tot) {
  __shared__ int part[kOffRuns][kOffDigits];
  const int ch = threadIdx.x % kOffDigits, r = threadIdx.x / kOffDigits;
  const int d = min((int)blockIdx.x * kOffDigits + ch, nd - 1);       // spare threads repeat the last digit
  const int per = (nblk + kOffRuns - 1) / kOffRuns, b0 = min(r * per, nblk), b1 = min(b0 + per, nblk);
  int sum = 0;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) sum += cnt[(int64_t)b * nd + d];
  part[r][ch] = sum;
  __syncthreads();
  for (int k = 1; k < kOffRuns; k <<= 1) {        // inclusive over the stretches
    const int v = r >= k ? part[r - k][ch] : 0;
    __syncthreads();
    part[r][ch] += v;
    __syncthreads();
  }
  int run = part[r][ch] - sum;
  if ((int)blockIdx.x * kOffDigits + ch >= nd) return;
  if (r == kOffRuns - 1) tot[d] = run + sum;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) {
    const int n = cnt[(int64_t)b * nd + d];
    cnt[(int64_t)b * nd + d] = run;
    run += n;
  }
}

struct SortLds {
  uint16_t at[kSortWaves][1 << kMaxDigitBits];    // a wave's records of a digit so far, then those of the waves before it
  int base[1 << kMaxDigitBits];                   // where the tile's records of a digit go
  int wsum[kSortWaves + 1];
};

// A wave's ranks of its kSortItems x 64 records by digit, in their order: among its lanes of the same digit (found equal
// by a ballot per bit), behind the digit's records of the rounds before.  Leaves the waves' counts in l.at.
__device__ __forceinline__ void rank_records(SortLds& l, const Rec (&rec)[kSortItems], const bool (&live)[kSortItems],
                                             int shift, int bits, int (&rank)[kSortItems]) {
  const int nd = 1 << bits, lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  for (int d = lane; d < nd; d += kWave) l.at[w][d] = 0;
  const uint64_t below = ((uint64_t)1 << lane) - 1;
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const int d = (rec[k].key >> shift) & (nd - 1);
    uint64_t same = __ballot(live[k]);
    for (int b = 0; b < bits; ++b) {
      const uint64_t one = __ballot((d >> b) & 1);
      same &= (d >> b) & 1 ? one : ~one;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");        // LDS accesses of one wave take effect in order
    const int before = live[k] ? l.at[w][d] : 0;
    rank[k] = before + __popcll(same & below);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (live[k] && (same & below) == 0) l.at[w][d] = (uint16_t)(before + __popcll(same));
  }
  __syncthreads();
  for (int d = threadIdx.x; d < nd; d += kSortBlock) {            // the waves' counts into those before each
    int run = 0;
#pragma unroll
    for (int j = 0; j < kSortWaves; ++j) {
      const int n = l.at[j][d];
      l.at[j][d] = (uint16_t)run;
      run += n;
    }
    l.base[d] = run;
  }
  __syncthreads();
}

// off (blocks, digits), tot (digits): as k_sort_offsets leaves them.  The tile's records are put in order in LDS first and
// leave in runs of equal digits: 1M records over 128 digits 9.4 us, 11.4 us each to its place.
template <bool FIRST>
__global__ void __launch_bounds__(kSortBlock) k_sort_scatter(const void* __restrict__ src, bool wide, int64_t vocab,
                                                             int64_t N, int shift, int bits, const int* __restrict__ off,
                                                             const int* __restrict__ tot, Rec* __restrict__ dst) {
  __shared__ SortLds l;
  __shared__ Rec sorted[kSortTile];
  __shared__ int tile_at[1 << kMaxDigitBits];
  const int nd = 1 << bits, lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  const int64_t i0 = (int64_t)blockIdx.x * kSortTile + w * (kWave * kSortItems) + lane;
  Rec rec[kSortItems];
  bool live[kSortItems];
  int rank[kSortItems];
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    live[k] = i0 + k * kWave < N;
    rec[k] = live[k] ? rec_at<FIRST>(src, wide, vocab, i0 + k * kWave) : Rec{0, 0};
  }
  const int t = (int)threadIdx.x < nd ? tot[threadIdx.x] : 0;
  const int o = (int)threadIdx.x < nd ? off[(int64_t)blockIdx.x * nd + threadIdx.x] : 0;
  rank_records(l, rec, live, shift, bits, rank);
  int total;
  const int before = block_exclusive_scan<kSortBlock>(t, l.wsum, total);        // records of smaller digits
  const int c = (int)threadIdx.x < nd ? l.base[threadIdx.x] : 0;
  const int here = block_exclusive_scan<kSortBlock>(c, l.wsum, total);          // those of the tile
  if ((int)threadIdx.x < nd) {
    tile_at[threadIdx.x] = here;
    l.base[threadIdx.x] = before + o - here;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const int d = (rec[k].key >> shift) & (nd - 1);
    if (live[k]) sorted[tile_at[d] + l.at[w][d] + rank[k]] = rec[k];
  }
  __syncthreads();
  const int n = (int)min((int64_t)kSortTile, N - (int64_t)blockIdx.x * kSortTile);
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    const int at = k * kSortBlock + threadIdx.x;
    if (at >= n) break;
    const Rec r = sorted[at];
    dst[l.base[(r.key >> shift) & (nd - 1)] + at] = r;
  }
}

// All passes of up to a tile's tokens in one workgroup; the other workgroups clear the gradient's rows.
__global__ void __launch_bounds__(kSortBlock) k_sort_small(const void* __restrict__ ids, bool wide, int64_t vocab, int64_t N,
                                                           int passes, int bits, Rec* __restrict__ dst,
                                                           uint16_t* __restrict__ gt, int64_t halves) {
  __shared__ SortLds l;
  if (blockIdx.x > 0) {
    clear_piece(gt, halves, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  const int nd = 1 << bits, lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  const int i0 = w * (kWave * kSortItems) + lane;
  Rec rec[kSortItems];
  bool live[kSortItems];
  int rank[kSortItems];
#pragma unroll
  for (int k = 0; k < kSortItems; ++k) {
    live[k] = i0 + k * kWave < N;
    rec[k] = live[k] ? rec_at<true>(ids, wide, vocab, i0 + k * kWave) : Rec{0, 0};
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    rank_records(l, rec, live, shift, bits, rank);
    int total;
    const int n = (int)threadIdx.x < nd ? l.base[threadIdx.x] : 0;
    const int before = block_exclusive_scan<kSortBlock>(n, l.wsum, total);
    if ((int)threadIdx.x < nd) l.base[threadIdx.x] = before;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
      const int d = (rec[k].key >> shift) & (nd - 1);
      if (live[k]) dst[l.base[d] + l.at[w][d] + rank[k]] = rec[k];
    }
    __syncthreads();                              // the workgroup's own stores are seen past this
    if (pass + 1 < passes)
#pragma unroll
      for (int k = 0; k < kSortItems; ++k)
        if (live[k]) rec[k] = dst[i0 + k * kWave];
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------- sums of the runs
constexpr int kAhead = 8;             // rows in flight

struct RunGeo {
  int64_t N, D, sgo, nchunk;
  int chunk;                          // sorted positions of a group of lanes
  uint32_t vocab;
  int cl2;
  float scale;
};

// A workgroup's groups first join the runs that pass from one to the next, in LDS and in order.
// part (workgroups, 2, D): the workgroup's sum of a run that began before it, and of one that goes on after it.
template <typename T, typename O, int V>
__global__ void __launch_bounds__(kBlock) k_embed_runs(RunGeo g, const Rec* __restrict__ rec, const T* __restrict__ go,
                                                       O* __restrict__ gt, float* __restrict__ part) {
  enum { kNone = 0, kEnds = 1, kPasses = 2 };     // a group's run that began before it
  __shared__ float heads[kBlock * V];
  __shared__ uint8_t head_of[kBlock];
  const int lanes = 1 << g.cl2, G = kBlock >> g.cl2, gi = threadIdx.x >> g.cl2;
  const int64_t c = (((int64_t)blockIdx.y << g.cl2) + (threadIdx.x & (lanes - 1))) * V;
  const int64_t p0 = ((int64_t)blockIdx.x * G + gi) * g.chunk, p1 = min(p0 + g.chunk, g.N);
  const bool live = p0 < g.N && c < g.D;
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0.f;
  uint32_t cur = g.vocab;
  bool head = false, goes_on = false;
  int state = kNone;
  auto to_row = [&]() {
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] *= g.scale;
    store_f<V>(gt + cur * g.D + c, acc);
  };
  auto to_heads = [&](int how) {
    state = how;
#pragma unroll
    for (int k = 0; k < V; ++k) heads[threadIdx.x * V + k] = acc[k];
  };
  if (live) {
    cur = rec[p0].key;
    head = p0 > 0 && cur < g.vocab && rec[p0 - 1].key == cur;
    for (int64_t q = p0; q < p1 && cur < g.vocab; q += kAhead) {
      Rec r[kAhead];
      Pack<T, V> v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) r[k] = rec[min(q + k, p1 - 1)];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) v[k] = load_pack<T, V>(go + (int64_t)r[k].idx * g.sgo + c);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (q + k >= p1 || cur >= g.vocab) continue;
        if (r[k].key != cur) {
          if (head) to_heads(kEnds);
          else to_row();
          head = false;
          cur = r[k].key;
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] = 0.f;
          if (cur >= g.vocab) continue;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += (float)v[k].e[j];
      }
    }
    if (cur < g.vocab) {
      goes_on = p1 < g.N && rec[p1].key == cur;
      if (head) to_heads(goes_on ? kPasses : kEnds);
      else if (!goes_on) to_row();
    }
  }
  if ((threadIdx.x & (lanes - 1)) == 0) head_of[gi] = (uint8_t)state;
  __syncthreads();
  const bool first = gi == 0 && state != kNone;   // leads the run that began before the workgroup
  const bool own = goes_on && !head;              // leads its last run on
  auto follow = [&](int how, int slot, bool ends_in_row) {
    int j = gi + 1;
    while (how != kEnds && j < G) {
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += heads[(j * lanes + (threadIdx.x & (lanes - 1))) * V + k];
      how = head_of[j++];
    }
    if (how == kEnds && ends_in_row) to_row();
    else store_f<V>(part + ((int64_t)blockIdx.x * 2 + slot) * g.D + c, acc);
  };
  if (live && own) follow(kPasses, 1, true);
  if (live && first) {
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = heads[threadIdx.x * V + k];
    follow(state, 0, false);
  }
}

// Joins the partial sums of the runs that cross workgroups (chunks here), each by the group of the chunk where the run
// begins: its own share, then those of the chunks after it.  Runs of more than kSerial chunks are added up by the whole workgroup, a
// stretch per group, the stretches joined in order.
constexpr int kSerial = 16;
template <typename O, int V>
__global__ void __launch_bounds__(kBlock) k_embed_join(RunGeo g, const Rec* __restrict__ rec, O* __restrict__ gt,
                                                       const float* __restrict__ part) {
  __shared__ int64_t long_n[kBlock], long_chunk[kBlock];
  __shared__ float lds[kBlock * V];
  const int lanes = 1 << g.cl2, G = kBlock >> g.cl2, gi = threadIdx.x >> g.cl2;
  const int64_t chunk = (int64_t)blockIdx.x * G + gi;
  const int64_t c = (((int64_t)blockIdx.y << g.cl2) + (threadIdx.x & (lanes - 1))) * V;
  const bool live = c < g.D;
  int64_t after = 0;                              // chunks behind this one that share its last run
  uint32_t key = 0;
  const int64_t p0 = chunk * g.chunk, p1 = p0 + g.chunk;
  if (p1 < g.N) {
    key = rec[p1 - 1].key;
    const uint32_t behind = rec[p1].key, after_next = rec[min(p1 + g.chunk, g.N - 1)].key;
    const bool begins = !(p0 > 0 && rec[p0].key == key && rec[p0 - 1].key == key);
    if (key < g.vocab && behind == key && begins) {
      // The first chunk in (lo, hi] that begins with another key: most often the next, else a search by the group's
      // lanes (one probe at a time, a hot token's run of a hundred chunks took 2 us more).
      int lo = (int)chunk + 1, hi = (int)g.nchunk;
      if (lo + 1 < hi && after_next != key) hi = lo + 1;
      const int lane = threadIdx.x & (lanes - 1);
      while (hi - lo > 1) {
        const int step = (hi - lo + lanes) / (lanes + 1), at = lo + step * (lane + 1);
        const uint64_t same = __ballot(at < hi && rec[(int64_t)min(at, hi - 1) * g.chunk].key == key);
        const int n = __popcll(same >> (threadIdx.x & (kWave - 1) & ~(lanes - 1)) & (~(uint64_t)0 >> (kWave - lanes)));
        hi = min(hi, lo + step * (n + 1));
        lo += step * n;
      }
      after = hi - chunk - 1;
    }
  }
  if (after > 0 && after <= kSerial && live) {
    float acc[V];
    load_f<V>(part + (chunk * 2 + 1) * g.D + c, acc);
    for (int64_t j = chunk + 1; j <= chunk + after; ++j) {
      float v[V];
      load_f<V>(part + j * 2 * g.D + c, v);
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += v[k];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] *= g.scale;
    store_f<V>(gt + key * g.D + c, acc);
  }
  if ((threadIdx.x & (lanes - 1)) == 0) {
    long_n[gi] = after > kSerial ? after : 0;
    long_chunk[gi] = chunk;
  }
  if (!__syncthreads_or(after > kSerial)) return;
  for (int run = 0; run < G; ++run) {             // every thread takes the same turns
    const int64_t n = long_n[run];
    if (n == 0) continue;
    const int64_t first = long_chunk[run];
    const int64_t per = (n + G - 1) / G, j0 = first + 1 + gi * per, j1 = min(j0 + per, first + 1 + n);
    float acc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.f;
    if (live) {
      if (gi == 0) load_f<V>(part + (first * 2 + 1) * g.D + c, acc);
      for (int64_t j = j0; j < j1; j += kAhead) {
        Pack<float, V> v[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) v[q] = load_pack<float, V>(part + min(j + q, j1 - 1) * 2 * g.D + c);
#pragma unroll
        for (int q = 0; q < kAhead; ++q)
#pragma unroll
          for (int k = 0; k < V; ++k) acc[k] += j + q < j1 ? v[q].e[k] : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) lds[threadIdx.x * V + k] = acc[k];
    __syncthreads();
    if (gi == 0 && live) {
      for (int o = 1; o < G; ++o)
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += lds[(o * lanes + threadIdx.x) * V + k];
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] *= g.scale;
      store_f<V>(gt + (int64_t)rec[first * g.chunk + g.chunk - 1].key * g.D + c, acc);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------- host
struct SortPlan {
  int passes, bits, nblk, chunk;
  int64_t rec_a, rec_b, cnt, tot, part, bytes;      // workspace offsets in bytes
};

SortPlan sort_plan(int64_t N, int64_t D, int64_t vocab) {
  SortPlan q;
  int total = 1;
  while (((int64_t)1 << total) <= vocab) ++total;          // the keys are [0, vocab]
  q.passes = (total + kMaxDigitBits - 1) / kMaxDigitBits;
  q.bits = (total + q.passes - 1) / q.passes;
  q.nblk = (int)((N + kSortTile - 1) / kSortTile);
  // A chunk is worked off row by row: short ones where there are few tokens, so that more lanes share them (3000 tokens:
  // 22 us with 64 rows a chunk), long ones where partial sums would cost traffic.
  q.chunk = N <= 16 * kSortTile ? 8 : 32;
  const int64_t groups = (N + q.chunk - 1) / q.chunk;
  int64_t at = 0;
  auto take = [&](int64_t bytes) { const int64_t o = at; at += (bytes + 255) / 256 * 256; return o; };
  q.rec_a = take(N * 8);
  q.rec_b = take(N * 8);
  q.cnt = take(((int64_t)q.nblk << q.bits) * 4);
  q.tot = take(((int64_t)1 << q.bits) * 4);
  q.part = take((groups + 3) / 4 * 2 * D * 4);            // a workgroup holds at least four groups
  q.bytes = at;
  return q;
}

bool embed_ok(int64_t N, int64_t vocab, int64_t D) {
  return N >= 0 && N < ((int64_t)1 << 31) - kSortTile && vocab >= 1 && vocab < ((int64_t)1 << 31) - 1 && D >= 1 && D <= 65536;
}

template <typename F>
void by_one(int t, F&& f) {
  if (t == kF32) f(float{});
  else if (t == kBF16) f(bf16_t{});
  else f(f16_t{});
}

template <int V, typename F>
void by_pair(int a, int b, F&& f) {
  by_one(a, [&](auto x) { by_one(b, [&](auto y) { f(x, y, std::integral_constant<int, V>{}); }); });
}

// Vectors of 16 bytes of the first type.
template <typename F>
void by_pair_vec(int a, int b, F&& f) {
  by_one(a, [&](auto x) {
    by_one(b, [&](auto y) { f(x, y, std::integral_constant<int, 16 / (int)sizeof(x)>{}); });
  });
}

}  // namespace
}  // namespace atlhip

using namespace atlhip;

extern "C" {

int atl_embed_fwd(const void* ids, int wide_ids, int64_t N, const void* table, int64_t st, int ttype, int64_t vocab,
                  int64_t D, double scale, void* out, int otype, hipStream_t stream) {
  if (!embed_ok(N, vocab, D) || !dtype_ok(ttype) || !dtype_ok(otype) || st < 0) { set_error("embed_fwd: bad sizes N=%lld V=%lld D=%lld types %d, %d", (long long)N, (long long)vocab, (long long)D, ttype, otype); return 1; }
  if (N == 0) return 0;
  if (!ids || !table || !out) { set_error("embed_fwd: null argument"); return 1; }
  const bool vec = D % 8 == 0 && st % 8 == 0 && aligned_to(table, 16) && aligned_to(out, 16);
  const int V = vec ? 8 : 1;
  const int64_t units = D / V;
  // about 2048 pieces a workgroup, fewer where the call is too small to give every compute unit some
  const int64_t rows = std::max<int64_t>(1, std::min<int64_t>(2048 / units, (N + 1023) / 1024));
  auto go = [&](auto t, auto o, auto v) {
    using T = decltype(t);
    using O = decltype(o);
    in_launches((N + rows - 1) / rows, [&](int64_t first, unsigned n) {
      hipLaunchKernelGGL((k_embed_fwd<T, O, decltype(v)::value>), dim3(n), dim3(kBlock), 0, stream, ids, wide_ids != 0, N, vocab,
                         (const T*)table, st, (uint32_t)units, (uint32_t)((((int64_t)1 << 32) + units - 1) / units), (float)scale,
                         (O*)out, (int)rows, first);
    });
  };
  if (vec) by_pair<8>(ttype, otype, go);
  else by_pair<1>(ttype, otype, go);
  return check_launch("embed_fwd");
}

int64_t atl_embed_bwd_ws_bytes(int64_t N, int64_t vocab, int64_t D) {
  return embed_ok(N, vocab, D) ? sort_plan(N, D, vocab).bytes : -1;
}

int atl_embed_bwd(const void* ids, int wide_ids, int64_t N, const void* gout, int64_t sgo, int otype, int64_t vocab,
                  int64_t D, double scale, void* gtable, int ttype, void* ws, int64_t ws_bytes, hipStream_t stream) {
  if (!embed_ok(N, vocab, D) || !dtype_ok(ttype) || !dtype_ok(otype) || sgo < 0) { set_error("embed_bwd: bad sizes N=%lld V=%lld D=%lld types %d, %d", (long long)N, (long long)vocab, (long long)D, ttype, otype); return 1; }
  if (!gtable || (N > 0 && (!ids || !gout || !ws))) { set_error("embed_bwd: null argument"); return 1; }
  if (!aligned_to(gtable, 16)) { set_error("embed_bwd: gtable must be aligned to 16 bytes"); return 1; }
  const SortPlan q = sort_plan(N, D, vocab);
  if (N > 0 && ws_bytes < q.bytes) { set_error("embed_bwd: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)q.bytes); return 1; }
  const int64_t halves = vocab * D * dtype_size(ttype) / 2;
  const unsigned clear = (unsigned)std::max<int64_t>(1, std::min<int64_t>(2048, (halves + kSortBlock * 8 - 1) / (kSortBlock * 8)));
  char* w = (char*)ws;
  Rec* const rec_a = (Rec*)(w + q.rec_a);
  Rec* const rec_b = (Rec*)(w + q.rec_b);
  int* const cnt = (int*)(w + q.cnt);
  int* const tot = (int*)(w + q.tot);
  const void* src = ids;
  if (q.nblk <= 1) {
    hipLaunchKernelGGL(k_sort_small, dim3(1 + clear), dim3(kSortBlock), 0, stream, ids, wide_ids != 0, vocab, N, q.passes, q.bits,
                       rec_a, (uint16_t*)gtable, halves);
    src = rec_a;
  } else {
    for (int pass = 0; pass < q.passes; ++pass) {
      const int shift = pass * q.bits, nd = 1 << q.bits;
      Rec* const dst = src == rec_a ? rec_b : rec_a;
      if (pass == 0)
        hipLaunchKernelGGL((k_sort_count<true>), dim3(q.nblk + clear), dim3(kSortBlock), 0, stream, src, wide_ids != 0, vocab, N, shift,
                           q.bits, q.nblk, cnt, (uint16_t*)gtable, halves);
      else
        hipLaunchKernelGGL((k_sort_count<false>), dim3(q.nblk), dim3(kSortBlock), 0, stream, src, false, vocab, N, shift, q.bits, q.nblk,
                           cnt, (uint16_t*)gtable, halves);
      hipLaunchKernelGGL(k_sort_offsets, dim3(grid_for(nd, kOffDigits)), dim3(kSortBlock), 0, stream, cnt, q.nblk, nd, tot);
      if (pass == 0)
        hipLaunchKernelGGL((k_sort_scatter<true>), dim3(q.nblk), dim3(kSortBlock), 0, stream, src, wide_ids != 0, vocab, N, shift, q.bits,
                           (const int*)cnt, (const int*)tot, dst);
      else
        hipLaunchKernelGGL((k_sort_scatter<false>), dim3(q.nblk), dim3(kSortBlock), 0, stream, src, false, vocab, N, shift, q.bits,
                           (const int*)cnt, (const int*)tot, dst);
      src = dst;
    }
  }
  if (N == 0) return check_launch("embed_bwd");
  RunGeo g{};
  g.N = N; g.D = D; g.sgo = sgo; g.vocab = (uint32_t)vocab; g.scale = (float)scale;
  g.chunk = q.chunk;
  const bool vec = D % 8 == 0 && sgo % 8 == 0 && aligned_to(gout, 16);
  const int V = vec ? 16 / dtype_size(otype) : 1;
  while ((1 << g.cl2) < kWave && ((int64_t)V << g.cl2) < D) ++g.cl2;
  const int G = kBlock >> g.cl2;
  RunGeo j = g;                                   // the workgroups' sums are the joining kernel's chunks
  j.chunk = q.chunk * G;
  j.nchunk = (N + j.chunk - 1) / j.chunk;
  const unsigned tiles = (unsigned)((D + ((int64_t)V << g.cl2) - 1) / ((int64_t)V << g.cl2));
  auto go = [&](auto o, auto t, auto v) {
    using T = decltype(o);
    using O = decltype(t);
    constexpr int VV = decltype(v)::value;
    hipLaunchKernelGGL((k_embed_runs<T, O, VV>), dim3((unsigned)j.nchunk, tiles), dim3(kBlock), 0, stream, g, (const Rec*)src, (const T*)gout, (O*)gtable, (float*)(w + q.part));
    if (j.nchunk > 1)
      hipLaunchKernelGGL((k_embed_join<O, VV>), dim3(grid_for(j.nchunk, G), tiles), dim3(kBlock), 0, stream, j, (const Rec*)src, (O*)gtable, (const float*)(w + q.part));
  };
  if (vec) by_pair_vec(otype, ttype, go);
  else by_pair<1>(otype, ttype, go);
  return check_launch("embed_bwd");
}

}  // extern "C"
