// Gated linear recurrence over ragged windows of tokens (events in (window, time) order):
//
//   w = sigmoid(g),  z = dt softplus(g),  a = exp(-z),  h_i = a_i h_{i-1} + w_i x_i    per channel,
//
// from h0 (or zero) at each window's first token.  z is the gate's rate times the time gap to the token before (1
// where no gaps are given: then a = 1 - w and h is a running average); tokens of one time stamp (dt = 0) add up.
//
// The recurrence is associative in (Z, U): h_out = exp(-Z) h_in + U.  Tokens are cut into groups of 16 or 8, one thread
// per group and V channels; a workgroup holds as many groups side by side as its threads allow (a chunk).  Forward:
//   1. k_scan_local: every chunk's (Z, U), its groups joined in LDS;
//   2. k_scan_block, k_scan_carry: the states before blocks of chunks, and the chunks' ranges within their block;
//   3. k_scan_apply: decays and inputs once into registers, the groups joined in LDS again, then every group from its
//      own start state: y, the last states, and (for the backward) the start states.
// A call of one chunk needs the third alone.  The backward is the same recurrence from the end, C_i = a_i (gy_i +
// C_{i+1}), in the same three steps, with the group's states recomputed from its saved start state.
//
// A range that holds a window's start is marked: its U alone is its outcome, whatever came before it (an infinity or NaN
// of one window stays there), so chunks need not know about windows.
// States, decays and sums are fp32 whatever the tokens' type; y is rounded once.
#include "typed.h"
#include "../../include/atl_hip.h"

#include <algorithm>
#include <type_traits>

namespace atlhip {
namespace {

// Tokens of a group, and threads of a workgroup.  The forward keeps a decay and an input a token and channel in
// registers, the backward a decay, a weight, a factor and the gradient: it takes half the tokens a thread, so that four
// waves fit a SIMD (1M x 64 bfloat16: 160 us against 174 with 16 tokens and workgroups of 256).
constexpr int kFwdLen = 16, kFwdBlock = 256, kBwdLen = 8, kBwdBlock = 512;
constexpr float kLog2e = 1.44269504088896340736f, kLog2eLow = 1.925962991e-8f, kLn2 = 0.69314718055994530942f;

// The gate's weight w, 1 - w and its rate softplus(g) in units of log 2, from one exp2, one reciprocal and one log2:
// with E = exp(g) and p = 1 + E, w = E / p, 1 - w = 1 / p and softplus = log p, or g itself where E would overflow.
// These kernels are bound by the number of vector instructions next to memory (a transcendental one costs as much as
// two others), hence the form with the fewest.  What p rounds off E is put back into the logarithm: a small rate would
// lose it, and gaps of many time constants multiply it.  What exp2's argument rounds off (up to |g| 2^-24 of E) is put
// back for single precision; a 16-bit gate's own last bit moves E by more.
struct Gate { float w, wc, rate2; };
template <typename T, bool RATE>
__device__ __forceinline__ Gate gate_of(float g) {
  const float arg = g * kLog2e;
  float E = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(arg, 120.f));      // a NaN stays one
  if (sizeof(T) == 4) {
    const float off = fmaf(g, kLog2e, -arg) + g * kLog2eLow;
    E = fmaf(E, fminf(fmaxf(off, -1e-5f), 1e-5f) * kLn2, E);      // the bounds: an infinite gate's off is not a number
  }
  const float p = 1.f + E;
  Gate q;
  q.wc = __builtin_amdgcn_rcpf(p);
  q.w = E * q.wc;
  q.rate2 = 0.f;
  if (RATE) {
    const float l = fmaf((E - (p - 1.f)) * q.wc, kLog2e, __builtin_amdgcn_logf(p));
    q.rate2 = __builtin_elementwise_maximum(l, arg);
  }
  return q;
}

// The decay over a range whose rates (in units of log 2) add up to Z.  Next to 1 the hardware's exp2 errs to one side by
// an eighth of a unit on average, which a state that lives over many ranges would gather: there 1 - x (1 - x / 2 + ...)
// with x = Z log 2 is rounded to nearest (what is cut off is x^6 / 7! < 5e-9).
__device__ __forceinline__ float decay_of(float Z) {
  const float x = Z * kLn2;
  float q = fmaf(x, -1.f / 720, 1.f / 120);
  q = fmaf(x, -q, 1.f / 24);
  q = fmaf(x, -q, 1.f / 6);
  q = fmaf(x, -q, 0.5f);
  q = fmaf(x, -q, 1.f);
  return fabsf(Z) < 0.25f ? fmaf(-x, q, 1.f) : __builtin_amdgcn_exp2f(-Z);
}

// A range of tokens as (Z, U): h_out = decay(Z) h_in + U.  Ranges are joined by adding their Z, so that a decay is
// rounded once however long its range.  Z = kAnew marks a range that holds a window's start: no sum of finite
// rates, whatever the signs of the gaps.
constexpr float kAnew = -__builtin_inff();
__device__ __forceinline__ bool anew(float Z) { return Z == kAnew; }
__device__ __forceinline__ float past(float Z, float U, float h) { return anew(Z) ? U : fmaf(decay_of(Z), h, U); }
__device__ __forceinline__ float joined(float Za, float Zb) { return anew(Za) || anew(Zb) ? kAnew : Za + Zb; }

// The rates behind a decay P = 1 - M, from whichever holds more of it (what 1 - M rounds off is put back).
__device__ __forceinline__ float rate_of(float M, float P) {
  if (M >= 0.5f) return -__builtin_amdgcn_logf(P);
  const float p = 1.f - M;
  return -fmaf(((1.f - p) - M) * __builtin_amdgcn_rcpf(p), kLog2e, __builtin_amdgcn_logf(p));
}

struct ScanGeo {
  int64_t N, D, sx, sg, sgy;          // tokens, channels, row strides in elements
  int64_t nchunk;
  int B;
  int units, G, seg;                  // threads of a row, groups of a workgroup and of a segment of them
  int segs;                           // segments
  uint32_t unit_m, seg_m;             // multipliers of divisions by units and by seg (see over())
};

// n / d for n < 1024 and d < 1024 by the multiplier ceil(2^20 / d): what the multiplier is too large by, n times, stays
// below 2^20.
__device__ __forceinline__ int over(int n, uint32_t m) { return (int)((uint32_t)n * m >> 20); }
inline uint32_t over_multiplier(int d) { return ((1u << 20) + d - 1) / d; }

// Number of entries of start[0, B) below i (start ascends), by the whole wave: 64 probes a step.
__device__ __forceinline__ int count_below(const int64_t* __restrict__ start, int B, int64_t i) {
  const int lane = threadIdx.x & (kWave - 1);
  int lo = 0, n = B;
  while (n > kWave) {
    const int step = (n + kWave - 1) / kWave;
    const int k = lane * step;
    const int c = __popcll(__ballot(k < n && start[lo + (k < n ? k : 0)] < i));
    if (c == 0) return lo;
    lo += (c - 1) * step + 1;
    n = min(step - 1, n - (c - 1) * step - 1);
  }
  return lo + __popcll(__ballot(lane < n && start[lo + (lane < n ? lane : 0)] < i));
}

// The last window from b on that starts before token i (those up to b do).  Steps double until they pass the place and
// halve back to it: windows without tokens may stand there by the million, a window with some is the next one.
__device__ __forceinline__ int last_before(const int64_t* __restrict__ start, int B, int b, int64_t i) {
  uint32_t step = 1;
  for (; step < (uint32_t)B - (uint32_t)b && start[b + (int)step] < i; step <<= 1) b += (int)step;
  for (step >>= 1; step > 0; step >>= 1)
    if (step < (uint32_t)B - (uint32_t)b && start[b + (int)step] < i) b += (int)step;
  return b;
}
// The last window below b that starts at or before token i (b and those behind it start after it), or window 0.
__device__ __forceinline__ int last_upto(const int64_t* __restrict__ start, int b, int64_t i) {
  uint32_t step = 1;
  for (; step < (uint32_t)b && start[b - (int)step] > i; step <<= 1) b -= (int)step;
  for (step >>= 1; step > 0; step >>= 1)
    if (step < (uint32_t)b && start[b - (int)step] > i) b -= (int)step;
  return b - 1;
}

// Where a thread works: its channels, its group and the group's n tokens from i0 on.
struct Place {
  int64_t c, i0;
  int gi, n;
  bool live;                          // has channels and tokens
};
template <int LEN, int V>
__device__ __forceinline__ Place place_of(const ScanGeo& s, int64_t chunk) {
  Place p;
  p.gi = over(threadIdx.x, s.unit_m);
  const int un = threadIdx.x - p.gi * s.units;
  p.c = ((int64_t)blockIdx.y * s.units + un) * V;
  p.i0 = (chunk * s.G + p.gi) * LEN;
  p.live = p.gi < s.G && p.c < s.D && p.i0 < s.N;
  p.n = p.live ? (int)min((int64_t)LEN, s.N - p.i0) : 0;
  return p;
}

template <int BYTES>
using Word = std::conditional_t<BYTES == 2, uint16_t, std::conditional_t<BYTES == 4, uint32_t, uint64_t>>;

// A thread's row pieces of one (tokens, channels) array: the chunk's address, the same for all threads, and a 32-bit
// offset, which steps from token to token (the host sees to it that a chunk spans less than 4 GB).
template <typename T, int LEN>
struct Rows {
  T* base;
  uint32_t off, step;                 // in bytes
  __device__ __forceinline__ Rows(const ScanGeo& s, const Place& p, T* array, int64_t stride, int64_t chunk) {
    base = array + chunk * s.G * LEN * stride;
    step = (uint32_t)stride * (uint32_t)sizeof(T);
    off = (uint32_t)(p.gi * LEN) * step + (uint32_t)p.c * (uint32_t)sizeof(T);
  }
  // Token t's piece (PLAIN: the address steps with the base, which all threads share).
  template <bool PLAIN>
  __device__ __forceinline__ T* at(uint32_t t) const {
    return PLAIN ? (T*)((uintptr_t)base + (uint64_t)t * step + off) : (T*)((uintptr_t)base + (uint32_t)(off + t * step));
  }
};

// The first token of the wave's first group.
template <int LEN>
__device__ __forceinline__ int64_t wave_first_token(const ScanGeo& s, int64_t chunk) {
  return (chunk * s.G + over(threadIdx.x & ~(kWave - 1), s.unit_m)) * LEN;
}

// Walks the windows along a group's ascending tokens.  b: the window of the token before (-1 before the first), next:
// how far from the group's first token the window after it starts.
struct Ascend {
  int b, next;
  __device__ __forceinline__ void look(const int64_t* __restrict__ start, int64_t i0) {
    next = (int)min(start[b + 1] - i0, (int64_t)1 << 30);
  }
  __device__ __forceinline__ Ascend(const int64_t* __restrict__ start, int B, int64_t wave_first, const Place& p) {
    b = count_below(start, B, wave_first) - 1;
    look(start, p.i0);
    if (p.live && next < 0 && b + 1 < B) {
      b = last_before(start, B, b, p.i0);
      look(start, p.i0);
    }
  }
  // Whether token i0 + t is the first of a window, which b is then.
  __device__ __forceinline__ bool starts(const int64_t* __restrict__ start, int B, int64_t i0, int t) {
    if (t != next || b + 1 >= B) return false;
    ++b;
    look(start, i0);
    if (next <= t && b + 1 < B) {                 // windows without tokens
      b = last_before(start, B, b, i0 + t + 1);
      look(start, i0);
    }
    return true;
  }
};

// Walks the windows along descending tokens.  b: the window of the present token, first: how far from the group's
// first token it starts, last: whether the present token is its window's last.
struct Descend {
  int b, first;
  bool last;
  __device__ __forceinline__ void look(const int64_t* __restrict__ start, int64_t i0) {
    first = (int)max(start[b] - i0, -((int64_t)1 << 30));
  }
  __device__ __forceinline__ Descend(const int64_t* __restrict__ start, int B, int64_t wave_first, const Place& p) {
    const int64_t behind = p.i0 + p.n;
    b = max(count_below(start, B, wave_first + 1) - 1, 0);         // the last window that starts at or before it
    int64_t end = start[b + 1];
    if (p.live && end < behind && b + 1 < B) {
      b = last_before(start, B, b, behind);
      end = start[b + 1];
    }
    look(start, p.i0);
    last = behind == end;
  }
  __device__ __forceinline__ void step(const int64_t* __restrict__ start, int64_t i0, int t) {      // to token i0 + t
    last = false;
    if (t < first && b > 0) {
      --b;
      look(start, i0);
      if (t < first && b > 0) {                   // windows without tokens
        b = last_upto(start, b, i0 + t);
        look(start, i0);
      }
      last = true;
    }
  }
};

// Whether all of the wave's groups are whole and touch no window's edge, which spares the tests for every token.
template <int LEN>
__device__ __forceinline__ bool plain_wave(const Place& p, const Ascend& win) {
  return __all(!p.live || (p.n == LEN && win.next > LEN));
}
template <int LEN>
__device__ __forceinline__ bool plain_wave(const Place& p, const Descend& win) {
  return __all(!p.live || (p.n == LEN && win.first < 0 && !win.last));
}

// f(true_type) or f(false_type), by a flag that is the same for the whole wave.
template <typename F>
__device__ __forceinline__ void by_flag(bool flag, F&& f) {
  if (flag) f(std::true_type{});
  else f(std::false_type{});
}

// ------------------------------------------------------------------------------------------- joining a chunk's groups
// In LDS: each group's (Z, U), then, per segment of about sqrt(G) groups, their exclusive prefixes and the segment's total.
template <int BLOCK, int V>
struct JoinLds {
  float z[BLOCK * V], u[BLOCK * V];
  float sz[BLOCK * V], su[BLOCK * V];       // (segments, channels)
};

// Called by all threads with their group's (Z, U) (dead ones: an identity).  On return z, u hold what lies before the
// group in the chunk (REV: behind it); the chunk's total goes to its record in cz, cu where given.
template <int BLOCK, int V, bool REV>
__device__ __forceinline__ void join_groups(const ScanGeo& s, JoinLds<BLOCK, V>& l, float (&z)[V], float (&u)[V], int64_t record,
                                            float* __restrict__ cz, float* __restrict__ cu) {
  const int width = s.units * V;
  const int at0 = threadIdx.x * V;               // (group, channel): the groups' rows are width apart
#pragma unroll
  for (int k = 0; k < V; ++k) {
    l.z[at0 + k] = z[k];
    l.u[at0 + k] = u[k];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < s.segs * width; e += BLOCK) {
    const int seg = over(e / V, s.unit_m), ch = e - seg * width;
    float pz = 0.f, pu = 0.f;
    for (int j = seg * s.seg; j < min((seg + 1) * s.seg, s.G); ++j) {
      const int at = (REV ? s.G - 1 - j : j) * width + ch;
      const float gz = l.z[at], gu = l.u[at];
      l.z[at] = pz;
      l.u[at] = pu;
      pu = past(gz, gu, pu);
      pz = joined(pz, gz);
    }
    l.sz[e] = pz;
    l.su[e] = pu;
  }
  __syncthreads();
  if (s.segs > 1 || cz) {
    for (int ch = threadIdx.x; ch < width; ch += BLOCK) {
      float pz = 0.f, pu = 0.f;
      for (int seg = 0; seg < s.segs; ++seg) {
        const int at = seg * width + ch;
        const float gz = l.sz[at], gu = l.su[at];
        l.sz[at] = pz;
        l.su[at] = pu;
        pu = past(gz, gu, pu);
        pz = joined(pz, gz);
      }
      const int64_t c = (int64_t)blockIdx.y * width + ch;
      if (cz && c < s.D) {
        cz[record * s.D + c] = pz;
        cu[record * s.D + c] = pu;
      }
    }
    if (cz) return;
    __syncthreads();
  }
  const int gi = over(threadIdx.x, s.unit_m);
  if (gi >= s.G) return;
  const int seg = over(REV ? s.G - 1 - gi : gi, s.seg_m), ch0 = at0 - gi * width;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    z[k] = l.z[at0 + k];
    u[k] = l.u[at0 + k];
    if (s.segs > 1) {
      u[k] = past(z[k], u[k], l.su[seg * width + ch0 + k]);
      z[k] = joined(l.sz[seg * width + ch0 + k], z[k]);
    }
  }
}

// A group's decay so far, from its tokens' rates, or without gaps from their decays: one minus the product and the product.
template <int V, bool DT>
struct Decay {
  float z[V], p[V];
  __device__ __forceinline__ Decay() {
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = 0.f, p[k] = 1.f;
  }
  __device__ __forceinline__ void add(int k, const Gate& q, float rate, float a) {
    if (DT) {
      z[k] += rate;
    } else {
      z[k] = fmaf(q.w, 1.f - z[k], z[k]);
      p[k] *= a;
    }
  }
  __device__ __forceinline__ float rate(int k, bool reset) const {
    return reset ? kAnew : DT ? z[k] : rate_of(z[k], p[k]);
  }
};

template <int V>
__device__ __forceinline__ void load_or_zero(const float* __restrict__ p, int64_t at, float (&v)[V]) {
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = p ? p[at + k] : 0.f;
}

// ------------------------------------------------------------------------------------------- forward
constexpr int kAhead = 8;             // tokens whose loads are in flight together

template <typename T, int V, bool DT>
__global__ void __launch_bounds__(kFwdBlock) k_scan_local(ScanGeo s, const T* __restrict__ x, const T* __restrict__ g,
                                                           const int64_t* __restrict__ start,
                                                           const float* __restrict__ dt, const float* __restrict__ h0,
                                                           float* __restrict__ cz, float* __restrict__ cu) {
  __shared__ JoinLds<kFwdBlock, V> lds;
  const Place p = place_of<kFwdLen, V>(s, blockIdx.x);
  const Rows<const T, kFwdLen> rx(s, p, x, s.sx, blockIdx.x);
  const Rows<const T, kFwdLen> rg(s, p, g, s.sg, blockIdx.x);
  Rows<const float, kFwdLen> rd(s, p, dt, 1, blockIdx.x);
  rd.off = p.gi * kFwdLen * 4;
  Ascend win(start, s.B, wave_first_token<kFwdLen>(s, blockIdx.x), p);
  Decay<V, DT> decay;
  float U[V], Z[V];
#pragma unroll
  for (int k = 0; k < V; ++k) U[k] = 0.f;
  bool reset = false;
  if (p.live) by_flag(plain_wave<kFwdLen>(p, win), [&](auto flag) {
    constexpr bool PLAIN = decltype(flag)::value;
#pragma unroll
    for (int q0 = 0; q0 < kFwdLen; q0 += kAhead) {
      if (!PLAIN && q0 >= p.n) continue;
      Pack<T, V> xr[kAhead], gr[kAhead];
      float d[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const uint32_t i = PLAIN ? q0 + j : min(q0 + j, p.n - 1);
        xr[j] = load_pack<T, V>(rx.template at<PLAIN>(i));
        gr[j] = load_pack<T, V>(rg.template at<PLAIN>(i));
        d[j] = DT ? *rd.template at<PLAIN>(i) : 1.f;
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int t = q0 + j;
        if (!PLAIN && t >= p.n) continue;
        if (!PLAIN && win.starts(start, s.B, p.i0, t)) {
          reset = true;
          load_or_zero<V>(h0, win.b * s.D + p.c, U);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const Gate q = gate_of<T, DT>((float)gr[j].e[k]);
          const float z = q.rate2 * d[j];
          const float a = DT ? __builtin_amdgcn_exp2f(-z) : q.wc;
          U[k] = fmaf(a, U[k], q.w * (float)xr[j].e[k]);
          decay.add(k, q, z, a);
        }
      }
    }
  });
#pragma unroll
  for (int k = 0; k < V; ++k) Z[k] = decay.rate(k, reset);
  join_groups<kFwdBlock, V, false>(s, lds, Z, U, blockIdx.x, cz, cu);
}

// Joins the records of up to kBlockChunks chunks (in the order of the recurrence) per channel: each becomes what lies
// before its chunk in the block, the block's total goes to bz, bu.  Records lie chunk by chunk, as their workgroups write
// them: written channel by channel, a line per value, they cost the local kernels a third of their time.
constexpr int kBlockChunks = 32, kBlockSubs = 4;
__global__ void __launch_bounds__(kWave* kBlockSubs) k_scan_block(int64_t nchunk, int64_t D, float* __restrict__ cz,
                                                                  float* __restrict__ cu, float* __restrict__ bz,
                                                                  float* __restrict__ bu) {
  constexpr int kPer = kBlockChunks / kBlockSubs;
  __shared__ float lz[kBlockSubs][kWave], lu[kBlockSubs][kWave];
  const int lane = threadIdx.x & (kWave - 1), sub = threadIdx.x / kWave;
  const int64_t c = min((int64_t)blockIdx.y * kWave + lane, D - 1);              // spare lanes repeat the last channel
  const int64_t j0 = (int64_t)blockIdx.x * kBlockChunks + sub * kPer;
  float z[kPer], u[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int64_t at = min(j0 + k, nchunk - 1) * D + c;
    z[k] = cz[at];
    u[k] = cu[at];
  }
  float tz = 0.f, tu = 0.f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const float gz = j0 + k < nchunk ? z[k] : 0.f, gu = j0 + k < nchunk ? u[k] : 0.f;
    z[k] = tz;
    u[k] = tu;
    tu = past(gz, gu, tu);
    tz = joined(tz, gz);
  }
  lz[sub][lane] = tz;
  lu[sub][lane] = tu;
  __syncthreads();
  float pz = 0.f, pu = 0.f;                       // before the sub
  for (int k = 0; k < sub; ++k) {
    pu = past(lz[k][lane], lu[k][lane], pu);
    pz = joined(pz, lz[k][lane]);
  }
  if ((int64_t)blockIdx.y * kWave + lane >= D) return;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (j0 + k >= nchunk) break;
    cz[(j0 + k) * D + c] = joined(pz, z[k]);
    cu[(j0 + k) * D + c] = past(z[k], u[k], pu);
  }
  if (sub == kBlockSubs - 1) {
    bz[blockIdx.x * D + c] = joined(pz, tz);
    bu[blockIdx.x * D + c] = past(tz, tu, pu);
  }
}

// The state before each block of chunks: 16 channels a workgroup, a stretch of the blocks' records per thread, joined
// across the wave and then across the waves.
constexpr int kCarryBlock = 1024, kCarryChannels = 16, kCarrySegs = kCarryBlock / kCarryChannels;
__global__ void __launch_bounds__(kCarryBlock) k_scan_carry(int64_t n, int64_t D, const float* __restrict__ bz,
                                                            const float* __restrict__ bu, float* __restrict__ carry) {
  __shared__ float wz[kCarryBlock / kWave][kCarryChannels], wu[kCarryBlock / kWave][kCarryChannels];
  const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
  const int ch = threadIdx.x % kCarryChannels, seg = threadIdx.x / kCarryChannels;
  const int64_t c = min((int64_t)blockIdx.x * kCarryChannels + ch, D - 1);       // spare threads repeat the last channel
  const int64_t per = (n + kCarrySegs - 1) / kCarrySegs;
  const int64_t j0 = min(seg * per, n), j1 = min(j0 + per, n);
  float tz = 0.f, tu = 0.f;
#pragma unroll 4
  for (int64_t j = j0; j < j1; ++j) {
    const float z = bz[j * D + c], u = bu[j * D + c];
    tu = past(z, u, tu);
    tz = joined(tz, z);
  }
#pragma unroll
  for (int d = kCarryChannels; d < kWave; d <<= 1) {      // inclusive over the wave's stretches
    const float oz = __shfl_up(tz, d, kWave), ou = __shfl_up(tu, d, kWave);
    if (lane >= d) {
      tu = past(tz, tu, ou);
      tz = joined(oz, tz);
    }
  }
  if (lane >= kWave - kCarryChannels) wz[wid][ch] = tz, wu[wid][ch] = tu;
  __syncthreads();
  float h = 0.f;                                  // the state before the wave's, then the thread's stretch
  for (int w = 0; w < wid; ++w) h = past(wz[w][ch], wu[w][ch], h);
  const float pz = __shfl_up(tz, kCarryChannels, kWave), pu = __shfl_up(tu, kCarryChannels, kWave);
  if (lane >= kCarryChannels) h = past(pz, pu, h);
#pragma unroll 4
  for (int64_t j = j0; j < j1; ++j) {
    carry[j * D + c] = h;
    h = past(bz[j * D + c], bu[j * D + c], h);
  }
}

// The chunk records of a call, as the apply kernels read them: what lies before a chunk in its block of chunks, and the
// state before the block (null: one block, from nothing).
struct Carry {
  const float *z, *u, *block;
  // The state before the chunk at the given place in the order; null z: a single chunk.
  __device__ __forceinline__ float before(int64_t record, int64_t D, int64_t c) const {
    if (!z) return 0.f;
    const int64_t at = record * D + c;
    return past(z[at], u[at], block ? block[record / kBlockChunks * D + c] : 0.f);
  }
};

// The empty windows' last states (the backward: the gradients of their first): out[b] = in[b] or zero.
template <int BLOCK>
__device__ __forceinline__ void fill_empty(const int64_t* __restrict__ start, int B, int64_t D, const float* __restrict__ in,
                                           float* __restrict__ out, int64_t block, int64_t blocks) {
  for (int64_t e = block * BLOCK + threadIdx.x; e < (int64_t)B * D; e += blocks * BLOCK) {
    const int64_t b = e / D;
    if (start[b + 1] <= start[b]) out[e] = in ? in[e] : 0.f;
  }
}

// The workgroups past the chunks fill the empty windows' states.
template <typename T, int V, bool DT>
__global__ void __launch_bounds__(kFwdBlock) k_scan_apply(ScanGeo s, const T* __restrict__ x, const T* __restrict__ g,
                                                           const int64_t* __restrict__ start,
                                                           const float* __restrict__ dt, const float* __restrict__ h0,
                                                           Carry carry, T* __restrict__ y,
                                                           float* __restrict__ last, float* __restrict__ states) {
  __shared__ JoinLds<kFwdBlock, V> lds;
  if (blockIdx.x >= s.nchunk) {
    if (blockIdx.y == 0) fill_empty<kFwdBlock>(start, s.B, s.D, h0, last, blockIdx.x - s.nchunk, gridDim.x - s.nchunk);
    return;
  }
  const int64_t chunk = s.nchunk - 1 - blockIdx.x;         // from the end: what the local kernel read last is still cached
  const Place p = place_of<kFwdLen, V>(s, chunk);
  const Rows<const T, kFwdLen> rx(s, p, x, s.sx, chunk);
  const Rows<const T, kFwdLen> rg(s, p, g, s.sg, chunk);
  Rows<const float, kFwdLen> rd(s, p, dt, 1, chunk);
  rd.off = p.gi * kFwdLen * 4;
  const Rows<T, kFwdLen> ro(s, p, y, s.D, chunk);
  Ascend win(start, s.B, wave_first_token<kFwdLen>(s, chunk), p);
  const Ascend begin = win;
  float a[kFwdLen][V], u[kFwdLen][V];
  Decay<V, DT> decay;
  float U[V], Z[V];
#pragma unroll
  for (int k = 0; k < V; ++k) U[k] = 0.f;
  bool reset = false;
  const bool plain = plain_wave<kFwdLen>(p, win);
  if (p.live) by_flag(plain, [&](auto flag) {
    constexpr bool PLAIN = decltype(flag)::value;
    Pack<T, V> xr[kFwdLen], gr[kFwdLen];
    float d[kFwdLen];
#pragma unroll
    for (int t = 0; t < kFwdLen; ++t) {
      const uint32_t i = PLAIN ? t : min(t, p.n - 1);
      xr[t] = load_pack<T, V>(rx.template at<PLAIN>(i));
      gr[t] = load_pack<T, V>(rg.template at<PLAIN>(i));
      d[t] = DT ? *rd.template at<PLAIN>(i) : 1.f;
    }
#pragma unroll
    for (int t = 0; t < kFwdLen; ++t) {
      if (!PLAIN && win.starts(start, s.B, p.i0, t)) {
        reset = true;
        load_or_zero<V>(h0, win.b * s.D + p.c, U);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const Gate q = gate_of<T, DT>((float)gr[t].e[k]);
        const float z = q.rate2 * d[t];
        a[t][k] = DT ? __builtin_amdgcn_exp2f(-z) : q.wc;
        u[t][k] = q.w * (float)xr[t].e[k];
        U[k] = fmaf(a[t][k], U[k], u[t][k]);
        decay.add(k, q, z, a[t][k]);
      }
    }
  });
#pragma unroll
  for (int k = 0; k < V; ++k) Z[k] = decay.rate(k, reset);
  join_groups<kFwdBlock, V, false>(s, lds, Z, U, chunk, nullptr, nullptr);
  if (!p.live) return;
  win = begin;
  float h[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    h[k] = past(Z[k], U[k], carry.before(chunk, s.D, p.c + k));
  }
  by_flag(plain, [&](auto flag) {
    constexpr bool PLAIN = decltype(flag)::value;
#pragma unroll
    for (int t = 0; t < kFwdLen; ++t) {
      if (!PLAIN && t >= p.n) continue;
      if (t % kBwdLen == 0 && states)
#pragma unroll
        for (int k = 0; k < V; ++k) states[(p.i0 + t) / kBwdLen * s.D + p.c + k] = h[k];
      if (!PLAIN && win.starts(start, s.B, p.i0, t)) load_or_zero<V>(h0, win.b * s.D + p.c, h);
#pragma unroll
      for (int k = 0; k < V; ++k) h[k] = fmaf(a[t][k], h[k], u[t][k]);
      store_f<V>(ro.template at<PLAIN>(t), h);
      if (!PLAIN && t + 1 == win.next && win.b >= 0)
#pragma unroll
        for (int k = 0; k < V; ++k) last[win.b * s.D + p.c + k] = h[k];
    }
  });
}

// ------------------------------------------------------------------------------------------- backward
template <typename T, int V, bool DT, bool GY>
__global__ void __launch_bounds__(kBwdBlock) k_scan_bwd_local(ScanGeo s, const T* __restrict__ g,
                                                               const int64_t* __restrict__ start,
                                                               const float* __restrict__ dt, const T* __restrict__ gy,
                                                               const float* __restrict__ glast, float* __restrict__ cz,
                                                               float* __restrict__ cu) {
  __shared__ JoinLds<kBwdBlock, V> lds;
  const Place p = place_of<kBwdLen, V>(s, blockIdx.x);
  const Rows<const T, kBwdLen> rg(s, p, g, s.sg, blockIdx.x);
  const Rows<const T, kBwdLen> ry(s, p, gy, s.sgy, blockIdx.x);
  Rows<const float, kBwdLen> rd(s, p, dt, 1, blockIdx.x);
  rd.off = p.gi * kBwdLen * 4;
  Descend win(start, s.B, wave_first_token<kBwdLen>(s, blockIdx.x), p);
  Decay<V, DT> decay;
  float U[V], Z[V];
#pragma unroll
  for (int k = 0; k < V; ++k) U[k] = 0.f;
  bool reset = false;
  if (p.live) by_flag(plain_wave<kBwdLen>(p, win), [&](auto flag) {
    constexpr bool PLAIN = decltype(flag)::value;
#pragma unroll
    for (int q0 = kBwdLen - kAhead; q0 >= 0; q0 -= kAhead) {
      if (!PLAIN && q0 >= p.n) continue;
      Pack<T, V> gr[kAhead], yr[kAhead];
      float d[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const uint32_t i = PLAIN ? q0 + j : min(q0 + j, p.n - 1);
        gr[j] = load_pack<T, V>(rg.template at<PLAIN>(i));
        if (GY) yr[j] = load_pack<T, V>(ry.template at<PLAIN>(i));
        d[j] = DT ? *rd.template at<PLAIN>(i) : 1.f;
      }
#pragma unroll
      for (int j = kAhead - 1; j >= 0; --j) {
        const int t = q0 + j;
        if (!PLAIN && t >= p.n) continue;
        if (!PLAIN && t < p.n - 1) win.step(start, p.i0, t);
        if (!PLAIN && win.last) {
          reset = true;
          load_or_zero<V>(glast, win.b * s.D + p.c, U);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const Gate q = gate_of<T, DT>((float)gr[j].e[k]);
          const float z = q.rate2 * d[j];
          const float a = DT ? __builtin_amdgcn_exp2f(-z) : q.wc;
          U[k] = a * ((GY ? (float)yr[j].e[k] : 0.f) + U[k]);
          decay.add(k, q, z, a);
        }
      }
    }
  });
#pragma unroll
  for (int k = 0; k < V; ++k) Z[k] = decay.rate(k, reset);
  join_groups<kBwdBlock, V, true>(s, lds, Z, U, s.nchunk - 1 - blockIdx.x, cz, cu);
}

// gx = H w, gg = H w (x (1 - w) - dt a h_{i-1}) with H_i = gy_i + C_{i+1}; gh0 = C at a window's first token.
template <typename T, int V, bool DT, bool GY>
__global__ void __launch_bounds__(kBwdBlock) k_scan_bwd_apply(ScanGeo s, const T* __restrict__ x, const T* __restrict__ g,
                                                               const int64_t* __restrict__ start,
                                                               const float* __restrict__ dt, const float* __restrict__ h0,
                                                               const float* __restrict__ states,
                                                               const T* __restrict__ gy, const float* __restrict__ glast,
                                                               Carry carry, T* __restrict__ gx,
                                                               T* __restrict__ gg, float* __restrict__ gh0) {
  __shared__ JoinLds<kBwdBlock, V> lds;
  if (blockIdx.x >= s.nchunk) {
    if (blockIdx.y == 0) fill_empty<kBwdBlock>(start, s.B, s.D, glast, gh0, blockIdx.x - s.nchunk, gridDim.x - s.nchunk);
    return;
  }
  const int64_t chunk = s.nchunk - 1 - blockIdx.x;         // from the end: what the local kernel read last is still cached
  const Place p = place_of<kBwdLen, V>(s, chunk);
  const Rows<const T, kBwdLen> rx(s, p, x, s.sx, chunk);
  const Rows<const T, kBwdLen> rg(s, p, g, s.sg, chunk);
  const Rows<const T, kBwdLen> ry(s, p, gy, s.sgy, chunk);
  Rows<const float, kBwdLen> rd(s, p, dt, 1, chunk);
  rd.off = p.gi * kBwdLen * 4;
  const Rows<T, kBwdLen> rox(s, p, gx, s.D, chunk), rog(s, p, gg, s.D, chunk);
  const int64_t wf = wave_first_token<kBwdLen>(s, chunk);
  Descend win(start, s.B, wf, p);
  const Descend begin = win;
  float a[kBwdLen][V], w[kBwdLen][V], f[kBwdLen][V];      // f: gg = H f
  Pack<T, V> yr[kBwdLen];
  Decay<V, DT> decay;
  float U[V], Z[V];
#pragma unroll
  for (int k = 0; k < V; ++k) U[k] = 0.f;
  bool reset = false;
  const bool plain = plain_wave<kBwdLen>(p, win);
  Ascend up(start, s.B, wf, p);
  if (p.live) by_flag(plain, [&](auto flag) {
    constexpr bool PLAIN = decltype(flag)::value;
    Pack<T, V> xr[kBwdLen], gr[kBwdLen];
    float d[kBwdLen], h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = states[p.i0 / kBwdLen * s.D + p.c + k];
#pragma unroll
    for (int t = 0; t < kBwdLen; ++t) {
      const uint32_t i = PLAIN ? t : min(t, p.n - 1);
      xr[t] = load_pack<T, V>(rx.template at<PLAIN>(i));
      gr[t] = load_pack<T, V>(rg.template at<PLAIN>(i));
      if (GY) yr[t] = load_pack<T, V>(ry.template at<PLAIN>(i));
      d[t] = DT ? *rd.template at<PLAIN>(i) : 1.f;
    }
#pragma unroll
    for (int t = 0; t < kBwdLen; ++t) {
      if (!PLAIN && up.starts(start, s.B, p.i0, t)) load_or_zero<V>(h0, up.b * s.D + p.c, h);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const Gate q = gate_of<T, DT>((float)gr[t].e[k]);
        const float z = q.rate2 * d[t], xv = (float)xr[t].e[k];
        a[t][k] = DT ? __builtin_amdgcn_exp2f(-z) : q.wc;
        w[t][k] = q.w;
        f[t][k] = q.w * fmaf(xv, q.wc, -(d[t] * a[t][k]) * h[k]);
        h[k] = fmaf(a[t][k], h[k], q.w * xv);
        asm volatile("" : "+v"(a[t][k]), "+v"(w[t][k]), "+v"(f[t][k]));      // kept: not what they are made of
        if (PLAIN || t < p.n) decay.add(k, q, z, a[t][k]);
      }
    }
#pragma unroll
    for (int t = kBwdLen - 1; t >= 0; --t) {
      if (!PLAIN && t >= p.n) continue;
      if (!PLAIN && t < p.n - 1) win.step(start, p.i0, t);
      if (!PLAIN && win.last) {
        reset = true;
        load_or_zero<V>(glast, win.b * s.D + p.c, U);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) U[k] = a[t][k] * ((GY ? (float)yr[t].e[k] : 0.f) + U[k]);
    }
  });
#pragma unroll
  for (int k = 0; k < V; ++k) Z[k] = decay.rate(k, reset);
  join_groups<kBwdBlock, V, true>(s, lds, Z, U, chunk, nullptr, nullptr);
  if (!p.live) return;
  win = begin;
#pragma unroll
  for (int t = 0; t < kBwdLen; ++t)
    if (GY) asm volatile("" : "+v"(*(Word<sizeof(T) * V>*)&yr[t]));      // as loaded, not widened
  float C[V];
#pragma unroll
  for (int k = 0; k < V; ++k) C[k] = past(Z[k], U[k], carry.before(s.nchunk - 1 - chunk, s.D, p.c + k));
  by_flag(plain, [&](auto flag) {
    constexpr bool PLAIN = decltype(flag)::value;
#pragma unroll
    for (int t = kBwdLen - 1; t >= 0; --t) {
      if (!PLAIN && t >= p.n) continue;
      if (!PLAIN && t < p.n - 1) win.step(start, p.i0, t);
      if (!PLAIN && win.last) load_or_zero<V>(glast, win.b * s.D + p.c, C);
      float ox[V], og[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float H = (GY ? (float)yr[t].e[k] : 0.f) + C[k];
        C[k] = a[t][k] * H;
        ox[k] = H * w[t][k];
        og[k] = H * f[t][k];
      }
      store_f<V>(rox.template at<PLAIN>(t), ox);
      store_f<V>(rog.template at<PLAIN>(t), og);
      if (!PLAIN && gh0 && t == win.first)
#pragma unroll
        for (int k = 0; k < V; ++k) gh0[win.b * s.D + p.c + k] = C[k];
    }
  });
}

// One token of every stream: 4 bytes of state in and out per channel, bound by the launch.
template <typename T, bool DT>
__global__ void __launch_bounds__(kBlock) k_scan_step(int64_t first, int64_t N, int64_t D, int64_t sx, int64_t sg,
                                                      const T* __restrict__ x, const T* __restrict__ g,
                                                      const float* __restrict__ dt, float* __restrict__ h,
                                                      T* __restrict__ y) {
  const int64_t e = (first + blockIdx.x) * kBlock + threadIdx.x;
  if (e >= N * D) return;
  const int64_t i = e / D, c = e - i * D;
  const Gate q = gate_of<T, DT>((float)g[i * sg + c]);
  const float a = DT ? decay_of(q.rate2 * dt[i]) : q.w < 0.5f ? 1.f - q.w : q.wc;
  const float v = fmaf(a, h[e], q.w * (float)x[i * sx + c]);
  h[e] = v;
  y[e] = (T)v;
}

// ------------------------------------------------------------------------------------------- host
struct ScanPlan {
  ScanGeo s;
  int V;
  unsigned tiles;
  int64_t blocks;                                // of chunks
  int64_t cz, cu, bz, bu, carry, bytes;          // workspace offsets in floats, and its size in bytes
};

// Two channels a thread where widths, strides and addresses allow it, else one: a thread keeps the decays, weights and
// factors of a group's tokens of its channels in registers.
int scan_vector(int dtype, int64_t D, int64_t strides, const void* const* ptrs, int n) {
  if (D % 2 || strides % 2) return 1;
  for (int k = 0; k < n; ++k)
    if (!aligned_to(ptrs[k], 2 * dtype_size(dtype))) return 1;
  return 2;
}

// A row's threads: its channels over V, in equal parts of at most half a workgroup.  The states the
// backward starts from lie kBwdLen tokens apart whatever V is.
template <int LEN, int BLOCK>
ScanPlan scan_plan(int64_t N, int64_t D, int V) {
  ScanPlan q;
  q.V = V;
  q.s.N = N;
  q.s.D = D;
  const int64_t all = (D + V - 1) / V;
  q.tiles = (unsigned)((all + BLOCK / 2 - 1) / (BLOCK / 2));
  q.s.units = (int)((all + q.tiles - 1) / q.tiles);
  q.s.G = BLOCK / q.s.units;
  q.s.seg = q.s.G <= 4 ? q.s.G : q.s.G <= 16 ? 4 : q.s.G <= 64 ? 8 : 16;
  q.s.segs = (q.s.G + q.s.seg - 1) / q.s.seg;
  q.s.unit_m = over_multiplier(q.s.units);
  q.s.seg_m = over_multiplier(q.s.seg);
  const int64_t chunk = (int64_t)q.s.G * LEN;
  q.s.nchunk = (N + chunk - 1) / chunk;
  q.blocks = (q.s.nchunk + kBlockChunks - 1) / kBlockChunks;
  q.cz = 0;
  q.cu = q.s.nchunk * D;
  q.bz = 2 * q.cu;
  q.bu = q.bz + q.blocks * D;
  q.carry = q.bu + q.blocks * D;
  q.bytes = q.s.nchunk > 1 ? (q.carry + q.blocks * D) * 4 : 0;
  return q;
}

bool scan_sizes_ok(int64_t N, int64_t D, int64_t B, int dtype) {
  return N >= 0 && N < ((int64_t)1 << 31) && D >= 1 && D <= 65536 && B >= 0 && B < ((int64_t)1 << 31) && (B > 0 || N == 0) &&
         dtype_ok(dtype);
}

// Whether a chunk's rows at this stride lie within a 32-bit offset.
bool scan_span_ok(const ScanPlan& q, int len, int64_t stride, int dtype) {
  return stride < ((int64_t)1 << 32) / dtype_size(dtype) / len / q.s.G - q.s.D;
}

// Joins the chunk records that the local kernels wrote.
Carry scan_join(const ScanPlan& q, float* w, hipStream_t stream) {
  const int64_t D = q.s.D;
  hipLaunchKernelGGL(k_scan_block, dim3((unsigned)q.blocks, grid_for(D, kWave)), dim3(kWave * kBlockSubs), 0, stream,
                     q.s.nchunk, D, w + q.cz, w + q.cu, w + q.bz, w + q.bu);
  if (q.blocks > 1)
    hipLaunchKernelGGL(k_scan_carry, dim3(grid_for(D, kCarryChannels)), dim3(kCarryBlock), 0, stream, q.blocks, D,
                       (const float*)(w + q.bz), (const float*)(w + q.bu), w + q.carry);
  return Carry{w + q.cz, w + q.cu, q.blocks > 1 ? w + q.carry : nullptr};
}

// Workgroups that fill the empty windows' states.
unsigned scan_fill_blocks(int64_t B, int64_t D) { return (unsigned)std::min<int64_t>(256, (B * D + 511) / 512); }

// Whether the workgroups fit a launch (fewer than 2^32 threads; calls of more do not fit the memory but for rows that
// repeat).
bool scan_grid_ok(const ScanPlan& q, unsigned fill, int block) { return (q.s.nchunk + fill) * block < (int64_t)1 << 32; }

template <typename F>
void by_type(int dtype, bool vec, bool dt, F&& f) {
  auto inner = [&](auto t, auto v) {
    if (dt) f(t, v, std::true_type{});
    else f(t, v, std::false_type{});
  };
  if (dtype == kF32) {
    if (vec) inner(float{}, std::integral_constant<int, 2>{});
    else inner(float{}, std::integral_constant<int, 1>{});
  } else if (dtype == kBF16) {
    if (vec) inner(bf16_t{}, std::integral_constant<int, 2>{});
    else inner(bf16_t{}, std::integral_constant<int, 1>{});
  } else {
    if (vec) inner(f16_t{}, std::integral_constant<int, 2>{});
    else inner(f16_t{}, std::integral_constant<int, 1>{});
  }
}

}  // namespace
}  // namespace atlhip

using namespace atlhip;

extern "C" {

int64_t atl_gated_scan_groups(int64_t N) { return N < 0 ? -1 : (N + kBwdLen - 1) / kBwdLen; }

int64_t atl_gated_scan_ws_bytes(int64_t N, int64_t D, int dtype) {
  if (!scan_sizes_ok(N, D, 1, dtype)) return -1;
  int64_t bytes = 256;
  for (int V = 1; V <= 2; ++V)
    bytes = std::max(bytes, std::max(scan_plan<kFwdLen, kFwdBlock>(N, D, V).bytes, scan_plan<kBwdLen, kBwdBlock>(N, D, V).bytes));
  return bytes;
}

int atl_gated_scan_fwd(const void* x, int64_t sx, const void* gate, int64_t sg, int dtype, int64_t N, int64_t D,
                       const int64_t* start, int64_t B, const float* dt, const float* h0, void* y, float* last,
                       float* states, void* ws, int64_t ws_bytes, hipStream_t stream) {
  if (!scan_sizes_ok(N, D, B, dtype) || (N > 0 && (sx < 0 || sg < 0))) { set_error("gated_scan_fwd: bad sizes N=%lld D=%lld B=%lld type %d", (long long)N, (long long)D, (long long)B, dtype); return 1; }
  if (B == 0) return 0;
  const int64_t need = atl_gated_scan_ws_bytes(N, D, dtype);
  if (!start || !last || (N > 0 && (!x || !gate || !y)) || (need > 0 && !ws)) { set_error("gated_scan_fwd: null argument"); return 1; }
  if (ws_bytes < need) { set_error("gated_scan_fwd: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)need); return 1; }
  const void* ptrs[] = {x, gate, y};
  ScanPlan q = scan_plan<kFwdLen, kFwdBlock>(N, D, scan_vector(dtype, D, sx | sg, ptrs, 3));
  if (!scan_span_ok(q, kFwdLen, std::max(sx, sg), dtype)) { set_error("gated_scan_fwd: row strides %lld, %lld too large", (long long)sx, (long long)sg); return 1; }
  q.s.sx = sx; q.s.sg = sg; q.s.sgy = 0; q.s.B = (int)B;
  const unsigned fill = scan_fill_blocks(B, D);
  if (!scan_grid_ok(q, fill, kFwdBlock)) { set_error("gated_scan_fwd: too many tokens, N=%lld D=%lld", (long long)N, (long long)D); return 1; }
  float* w = (float*)ws;
  const bool many = q.s.nchunk > 1;
  Carry carry{};
  by_type(dtype, q.V > 1, dt != nullptr, [&](auto t, auto v, auto d) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    constexpr bool DT = decltype(d)::value;
    if (many) {
      hipLaunchKernelGGL((k_scan_local<T, V, DT>), dim3((unsigned)q.s.nchunk, q.tiles), dim3(kFwdBlock), 0, stream, q.s,
                         (const T*)x, (const T*)gate, start, dt, h0, w + q.cz, w + q.cu);
      carry = scan_join(q, w, stream);
    }
    hipLaunchKernelGGL((k_scan_apply<T, V, DT>), dim3((unsigned)q.s.nchunk + fill, q.tiles), dim3(kFwdBlock), 0,
                       stream, q.s, (const T*)x, (const T*)gate, start, dt, h0, carry,
                       (T*)y, last, states);
  });
  return check_launch("gated_scan_fwd");
}

int atl_gated_scan_bwd(const void* x, int64_t sx, const void* gate, int64_t sg, int dtype, int64_t N, int64_t D,
                       const int64_t* start, int64_t B, const float* dt, const float* h0, const float* states,
                       const void* gy, int64_t sgy, const float* glast, void* gx, void* ggate, float* gh0, void* ws,
                       int64_t ws_bytes, hipStream_t stream) {
  if (!scan_sizes_ok(N, D, B, dtype) || (N > 0 && (sx < 0 || sg < 0 || sgy < 0))) { set_error("gated_scan_bwd: bad sizes N=%lld D=%lld B=%lld type %d", (long long)N, (long long)D, (long long)B, dtype); return 1; }
  if (B == 0) return 0;
  const int64_t need = atl_gated_scan_ws_bytes(N, D, dtype);
  if (!start || (N > 0 && (!x || !gate || !states || !gx || !ggate)) || (need > 0 && !ws)) { set_error("gated_scan_bwd: null argument"); return 1; }
  if (ws_bytes < need) { set_error("gated_scan_bwd: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)need); return 1; }
  const void* ptrs[] = {x, gate, gx, ggate, gy};
  ScanPlan q = scan_plan<kBwdLen, kBwdBlock>(N, D, scan_vector(dtype, D, sx | sg | (gy ? sgy : 0), ptrs, 5));
  if (!scan_span_ok(q, kBwdLen, std::max(sx, std::max(sg, gy ? sgy : 0)), dtype)) { set_error("gated_scan_bwd: row strides too large"); return 1; }
  q.s.sx = sx; q.s.sg = sg; q.s.sgy = sgy; q.s.B = (int)B;
  float* w = (float*)ws;
  const bool many = q.s.nchunk > 1;
  Carry carry{};
  const unsigned fill = gh0 ? scan_fill_blocks(B, D) : 0;
  if (!scan_grid_ok(q, fill, kBwdBlock)) { set_error("gated_scan_bwd: too many tokens, N=%lld D=%lld", (long long)N, (long long)D); return 1; }
  if (q.s.nchunk + fill == 0) return 0;
  auto go = [&](auto t, auto v, auto d, auto y) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    constexpr bool DT = decltype(d)::value, GY = decltype(y)::value;
    if (many) {
      hipLaunchKernelGGL((k_scan_bwd_local<T, V, DT, GY>), dim3((unsigned)q.s.nchunk, q.tiles), dim3(kBwdBlock), 0, stream, q.s,
                         (const T*)gate, start, dt, (const T*)gy, glast, w + q.cz, w + q.cu);
      carry = scan_join(q, w, stream);
    }
    hipLaunchKernelGGL((k_scan_bwd_apply<T, V, DT, GY>), dim3((unsigned)q.s.nchunk + fill, q.tiles), dim3(kBwdBlock), 0, stream, q.s,
                       (const T*)x, (const T*)gate, start, dt, h0, states, (const T*)gy, glast,
                       carry, (T*)gx, (T*)ggate, gh0);
  };
  by_type(dtype, q.V > 1, dt != nullptr, [&](auto t, auto v, auto d) {
    if (gy) go(t, v, d, std::true_type{});
    else go(t, v, d, std::false_type{});
  });
  return check_launch("gated_scan_bwd");
}

int atl_gated_scan_step(const void* x, int64_t sx, const void* gate, int64_t sg, int dtype, int64_t N, int64_t D,
                        const float* dt, float* state, void* y, hipStream_t stream) {
  if (!scan_sizes_ok(N, D, 1, dtype) || sx < 0 || sg < 0) { set_error("gated_scan_step: bad sizes N=%lld D=%lld type %d", (long long)N, (long long)D, dtype); return 1; }
  if (N == 0) return 0;
  if (!x || !gate || !state || !y) { set_error("gated_scan_step: null argument"); return 1; }
  by_type(dtype, false, dt != nullptr, [&](auto t, auto, auto d) {
    using T = decltype(t);
    in_launches((N * D + kBlock - 1) / kBlock, [&](int64_t first, unsigned n) {
      hipLaunchKernelGGL((k_scan_step<T, decltype(d)::value>), dim3(n), dim3(kBlock), 0, stream, first, N, D, sx, sg, (const T*)x,
                         (const T*)gate, dt, state, (T*)y);
    });
  });
  return check_launch("gated_scan_step");
}

}  // extern "C"
