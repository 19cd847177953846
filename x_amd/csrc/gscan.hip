// Gated linear recurrence over ragged windows of tokens (events in (window, time) order):
//
//   w = sigmoid(g),  z = dt softplus(g),  a = exp(-z),  h_i = a_i h_{i-1} + w_i x_i    per channel,
//
// from h0 (or zero) at each window's first token.  z is the gate's rate times the time gap to the token before (1
// where no gaps are given: then a = 1 - w and h is a running average); tokens of one time stamp (dt = 0) add up.
//
// The recurrence is associative in (Z, U): h_out = exp(-Z) h_in + U.  Tokens are cut into groups of kLen, a workgroup
// holds 256 / lanes groups (a chunk); lanes run over the channels, V each.  Forward:
//   1. k_scan_local: every group's (Z, U) and their exclusive prefixes within the chunk, and the chunk's (Z, U);
//   2. k_scan_carry: the state before every chunk;
//   3. k_scan_apply: every group again from its own start state: y, the last states, and (for the backward) the
//      start states.
// The backward is the same recurrence from the end, C_i = a_i (gy_i + C_{i+1}), with the group's states recomputed
// from its saved start state.  A range that holds a window's start is marked: its U alone is its outcome, whatever came
// before it (an infinity or NaN of one window stays there), so chunks need not know about windows.
// States, decays and sums are fp32 whatever the tokens' type; y is rounded once.
#include "typed.h"
#include "../../include/atl_hip.h"

#include <algorithm>
#include <type_traits>

namespace atlhip {
namespace {

constexpr int kLen = 16;              // tokens of a group
constexpr float kLog2e = 1.44269504088896340736f, kLog2eLow = 1.925962991e-8f, kLn2 = 0.69314718055994530942f;

// The gate's weight w, 1 - w and its rate softplus(g) in units of log 2, from one exp2, one reciprocal and one log2:
// with e = exp(-|g|), p = 1 + e: w or 1 - w is 1 / p, the other e / p, and softplus = max(g, 0) + log p.  What p
// rounded off e enters as (e - (p - 1)) / p, so that small rates keep their relative precision (they are multiplied
// by gaps and summed over up to a million tokens).  exp2's argument rounds off up to |g| 2^-24 of e; for single
// precision tokens that is put back.
struct Gate { float w, wc, rate2; };
template <typename T, bool RATE>
__device__ __forceinline__ Gate gate_of(float g) {
  const float arg = -fabsf(g) * kLog2e;
  float e = __builtin_amdgcn_exp2f(arg);
  if (sizeof(T) == 4) {
    const float off = fmaf(-fabsf(g), kLog2e, -arg) - fabsf(g) * kLog2eLow;
    e = fmaf(e, fmaxf(off, -1.f) * kLn2, e);       // the maximum: an infinite gate's off is not a number
  }
  const float p = 1.f + e;
  const float rp = __builtin_amdgcn_rcpf(p);
  const float ep = e * rp;
  const bool pos = g >= 0.f;
  Gate q;
  q.w = pos ? rp : ep;
  q.wc = pos ? ep : rp;
  q.rate2 = RATE ? fmaf(fmaxf(g, 0.f) + (e - (p - 1.f)) * rp, kLog2e, __builtin_amdgcn_logf(p)) : 0.f;
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
  return Z < 0.25f ? fmaf(-x, q, 1.f) : __builtin_amdgcn_exp2f(-Z);
}

// A range of tokens as (Z, U): h_out = decay(Z) h_in + U.  Ranges are joined by adding their Z, so that a decay is
// rounded once however long its range.  Z = kAnew marks a range that holds a window's start.
constexpr float kAnew = -1.f;
__device__ __forceinline__ bool anew(float Z) { return Z < 0.f; }
__device__ __forceinline__ float past(float Z, float U, float h) { return anew(Z) ? U : fmaf(decay_of(Z), h, U); }
__device__ __forceinline__ float joined(float Za, float Zb) { return anew(Za) || anew(Zb) ? kAnew : Za + Zb; }

// The rates behind a decay P = 1 - M, from whichever holds more of it.
__device__ __forceinline__ float rate_of(float M, float P) {
  return M < 0.5f ? -log1pf(-M) * kLog2e : -__builtin_amdgcn_logf(P);
}

struct ScanGeo {
  int64_t N, D, sx, sg, sgy;          // tokens, channels, row strides in elements
  int64_t nchunk;
  int B;
  int cl2;                            // log2 of the lanes of a row
};

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

// Where a thread works: its channels, its group and the group's tokens [i0, i1).
struct Place {
  int64_t c, group, i0, i1;
  int gi, G;
  bool live;                          // has channels
};
template <int V>
__device__ __forceinline__ Place place_of(const ScanGeo& s) {
  Place p;
  const int cl = threadIdx.x & ((1 << s.cl2) - 1);
  p.gi = threadIdx.x >> s.cl2;
  p.G = kBlock >> s.cl2;
  p.c = (((int64_t)blockIdx.y << s.cl2) + cl) * V;
  p.group = (int64_t)blockIdx.x * p.G + p.gi;
  p.i0 = p.group * kLen;
  p.i1 = min(p.i0 + kLen, s.N);
  p.live = p.c < s.D;
  return p;
}

// Walks the windows along ascending tokens.  b: the window of the token before (-1 before the first), next: where the
// window after it starts.
struct Ascend {
  int b;
  int64_t next;
  __device__ __forceinline__ Ascend(const int64_t* __restrict__ start, int B, int64_t wave_first, int64_t i0) {
    b = count_below(start, B, wave_first) - 1;
    while (b + 1 < B && start[b + 1] < i0) ++b;
    next = start[b + 1];
  }
  // Whether token i is the first of a window, which b is then.
  __device__ __forceinline__ bool starts(const int64_t* __restrict__ start, int B, int64_t i) {
    if (i != next || b + 1 >= B) return false;
    do { ++b; next = start[b + 1]; } while (next <= i && b + 1 < B);
    return true;
  }
};

__device__ __forceinline__ int64_t wave_first_token(const ScanGeo& s) {
  const int G = kBlock >> s.cl2;
  return ((int64_t)blockIdx.x * G + ((threadIdx.x & ~(kWave - 1)) >> s.cl2)) * kLen;
}

// The groups' (Z, U) of a chunk through LDS: each group's exclusive prefix (in the order of the recurrence, from
// group 0 up or, REV, from the last down) into pZ, pU, the chunk's total into cZ, cU.  Called by all threads.
template <int V, bool REV>
__device__ __forceinline__ void chunk_prefix(const ScanGeo& s, const Place& p, float (&Z)[V], float (&U)[V],
                                             float* lds, float* __restrict__ pZ, float* __restrict__ pU,
                                             float* __restrict__ cZ, float* __restrict__ cU) {
  float* lZ = lds;
  float* lU = lds + kBlock * V;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    lZ[threadIdx.x * V + k] = Z[k];
    lU[threadIdx.x * V + k] = U[k];
  }
  __syncthreads();
  const int width = V << s.cl2;                  // channels of the block
  for (int ch = threadIdx.x; ch < width; ch += kBlock) {
    float z = 0.f, u = 0.f;
    for (int j = 0; j < p.G; ++j) {
      const int at = (REV ? p.G - 1 - j : j) * width + ch;
      const float gz = lZ[at], gu = lU[at];
      lZ[at] = z;
      lU[at] = u;
      u = past(gz, gu, u);
      z = joined(z, gz);
    }
    const int64_t c = (int64_t)blockIdx.y * width + ch;
    if (c < s.D) {
      cZ[blockIdx.x * s.D + c] = z;
      cU[blockIdx.x * s.D + c] = u;
    }
  }
  __syncthreads();
  if (p.live && p.i0 < s.N) {
    const int64_t at = p.group * s.D + p.c;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      pZ[at + k] = lZ[threadIdx.x * V + k];
      pU[at + k] = lU[threadIdx.x * V + k];
    }
  }
}

template <typename T, int V, bool DT>
__global__ void __launch_bounds__(kBlock) k_scan_local(ScanGeo s, const T* __restrict__ x, const T* __restrict__ g,
                                                       const int64_t* __restrict__ start, const float* __restrict__ dt,
                                                       const float* __restrict__ h0, float* __restrict__ pZ,
                                                       float* __restrict__ pU, float* __restrict__ cZ,
                                                       float* __restrict__ cU) {
  __shared__ float lds[2 * kBlock * V];
  const Place p = place_of<V>(s);
  Ascend win(start, s.B, wave_first_token(s), p.i0);
  float Z[V], U[V], P[V];           // Z: the sum of rates, or without gaps 1 - the decay, and P the decay
#pragma unroll
  for (int k = 0; k < V; ++k) Z[k] = U[k] = 0.f, P[k] = 1.f;
  bool reset = false;
  if (p.live)
    for (int64_t i = p.i0; i < p.i1; ++i) {
      float xv[V], gv[V];
      load_f<V>(x + i * s.sx + p.c, xv);
      load_f<V>(g + i * s.sg + p.c, gv);
      const float d = DT ? dt[i] : 1.f;
      if (win.starts(start, s.B, i)) {
        reset = true;
#pragma unroll
        for (int k = 0; k < V; ++k) U[k] = h0 ? h0[win.b * s.D + p.c + k] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const Gate q = gate_of<T, DT>(gv[k]);
        const float z = q.rate2 * d;
        const float a = DT ? __builtin_amdgcn_exp2f(-z) : q.wc;
        U[k] = fmaf(a, U[k], q.w * xv[k]);
        Z[k] = DT ? Z[k] + z : fmaf(q.w, 1.f - Z[k], Z[k]);
        if (!DT) P[k] *= a;
      }
    }
#pragma unroll
  for (int k = 0; k < V; ++k) Z[k] = reset ? kAnew : DT ? Z[k] : rate_of(Z[k], P[k]);
  chunk_prefix<V, false>(s, p, Z, U, lds, pZ, pU, cZ, cU);
}

// The state before each chunk (REV: after it, from the last chunk down), and the empty windows' last states (the
// backward: their gradients): out[b] = in[b] or zero.
constexpr int kCarryChannels = 16, kCarrySegments = 64, kCarryBlock = kCarryChannels * kCarrySegments;
template <bool REV>
__global__ void __launch_bounds__(kCarryBlock) k_scan_carry(int64_t nchunk, int64_t D, const float* __restrict__ cZ,
                                                            const float* __restrict__ cU, float* __restrict__ carry,
                                                            const int64_t* __restrict__ start, int B,
                                                            const float* __restrict__ in, float* __restrict__ out,
                                                            unsigned carry_blocks) {
  if (blockIdx.x >= carry_blocks) {
    const int64_t stride = (int64_t)(gridDim.x - carry_blocks) * kCarryBlock;
    for (int64_t e = (int64_t)(blockIdx.x - carry_blocks) * kCarryBlock + threadIdx.x; e < (int64_t)B * D; e += stride) {
      const int64_t b = e / D;
      if (start[b + 1] <= start[b]) out[e] = in ? in[e] : 0.f;
    }
    return;
  }
  __shared__ float sZ[kCarryBlock], sU[kCarryBlock];
  const int ch = threadIdx.x % kCarryChannels, seg = threadIdx.x / kCarryChannels;
  const int64_t c = (int64_t)blockIdx.x * kCarryChannels + ch;
  const int64_t per = (nchunk + kCarrySegments - 1) / kCarrySegments;
  const int64_t j0 = min(seg * per, nchunk), j1 = min(j0 + per, nchunk);
  const bool live = c < D;
  float z = 0.f, u = 0.f;
  if (live)
    for (int64_t j = j0; j < j1; ++j) {
      const int64_t at = (REV ? nchunk - 1 - j : j) * D + c;
      const float gz = cZ[at];
      u = past(gz, cU[at], u);
      z = joined(z, gz);
    }
  sZ[threadIdx.x] = z;
  sU[threadIdx.x] = u;
  __syncthreads();
  if (seg == 0) {
    float h = 0.f;
    for (int k = 0; k < kCarrySegments; ++k) {
      const int at = k * kCarryChannels + ch;
      const float gz = sZ[at], gu = sU[at];
      sU[at] = h;
      h = past(gz, gu, h);
    }
  }
  __syncthreads();
  float h = sU[threadIdx.x];
  if (live)
    for (int64_t j = j0; j < j1; ++j) {
      const int64_t at = (REV ? nchunk - 1 - j : j) * D + c;
      carry[at] = h;
      h = past(cZ[at], cU[at], h);
    }
}

// pU: the groups' prefixes in, their start states out (read by the backward).
template <typename T, int V, bool DT>
__global__ void __launch_bounds__(kBlock) k_scan_apply(ScanGeo s, const T* __restrict__ x, const T* __restrict__ g,
                                                       const int64_t* __restrict__ start, const float* __restrict__ dt,
                                                       const float* __restrict__ h0, const float* __restrict__ pZ,
                                                       float* __restrict__ pU, const float* __restrict__ carry,
                                                       T* __restrict__ y, float* __restrict__ last, bool save) {
  const Place p = place_of<V>(s);
  Ascend win(start, s.B, wave_first_token(s), p.i0);
  if (!p.live || p.i0 >= s.N) return;
  float h[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int64_t at = p.group * s.D + p.c + k;
    h[k] = past(pZ[at], pU[at], carry[blockIdx.x * s.D + p.c + k]);
    if (save) pU[at] = h[k];
  }
  for (int64_t i = p.i0; i < p.i1; ++i) {
    float xv[V], gv[V];
    load_f<V>(x + i * s.sx + p.c, xv);
    load_f<V>(g + i * s.sg + p.c, gv);
    const float d = DT ? dt[i] : 1.f;
    if (win.starts(start, s.B, i))
#pragma unroll
      for (int k = 0; k < V; ++k) h[k] = h0 ? h0[win.b * s.D + p.c + k] : 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const Gate q = gate_of<T, DT>(gv[k]);
      h[k] = fmaf(DT ? __builtin_amdgcn_exp2f(-q.rate2 * d) : q.wc, h[k], q.w * xv[k]);
    }
    store_f<V>(y + i * s.D + p.c, h);
    if (i + 1 == win.next && win.b >= 0)
#pragma unroll
      for (int k = 0; k < V; ++k) last[win.b * s.D + p.c + k] = h[k];
  }
}

// Walks the windows along descending tokens.  b: the window of the present token, first: where it starts.
struct Descend {
  int b;
  int64_t first;
  bool last;                          // the present token is its window's last
  __device__ __forceinline__ Descend(const int64_t* __restrict__ start, int B, int64_t wave_first, int64_t i) {
    b = count_below(start, B, wave_first + 1) - 1;                 // the last window that starts at or before it
    while (b + 1 < B && start[b + 1] <= i) ++b;
    b = max(b, 0);
    first = start[b];
    last = i + 1 == start[b + 1];
  }
  __device__ __forceinline__ void step(const int64_t* __restrict__ start, int64_t i) {      // to token i
    last = false;
    if (i < first && b > 0) {
      do { --b; } while (b > 0 && start[b] > i);
      first = start[b];
      last = true;
    }
  }
};

template <typename T, int V, bool DT>
__global__ void __launch_bounds__(kBlock) k_scan_bwd_local(ScanGeo s, const T* __restrict__ g,
                                                           const int64_t* __restrict__ start,
                                                           const float* __restrict__ dt, const T* __restrict__ gy,
                                                           const float* __restrict__ glast, float* __restrict__ pZ,
                                                           float* __restrict__ pU, float* __restrict__ cZ,
                                                           float* __restrict__ cU) {
  __shared__ float lds[2 * kBlock * V];
  const Place p = place_of<V>(s);
  Descend win(start, s.B, wave_first_token(s), p.i1 - 1);
  float Z[V], U[V], P[V];           // Z: the sum of rates, or without gaps 1 - the decay, and P the decay
#pragma unroll
  for (int k = 0; k < V; ++k) Z[k] = U[k] = 0.f, P[k] = 1.f;
  bool reset = false;
  if (p.live)
    for (int64_t i = p.i1 - 1; i >= p.i0; --i) {
      float gv[V], yv[V];
      load_f<V>(g + i * s.sg + p.c, gv);
      if (gy)
        load_f<V>(gy + i * s.sgy + p.c, yv);
      else
#pragma unroll
        for (int k = 0; k < V; ++k) yv[k] = 0.f;
      const float d = DT ? dt[i] : 1.f;
      if (i < p.i1 - 1) win.step(start, i);
      if (win.last) {
        reset = true;
#pragma unroll
        for (int k = 0; k < V; ++k) U[k] = glast ? glast[win.b * s.D + p.c + k] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const Gate q = gate_of<T, DT>(gv[k]);
        const float z = q.rate2 * d;
        const float a = DT ? __builtin_amdgcn_exp2f(-z) : q.wc;
        U[k] = a * (yv[k] + U[k]);
        Z[k] = DT ? Z[k] + z : fmaf(q.w, 1.f - Z[k], Z[k]);
        if (!DT) P[k] *= a;
      }
    }
#pragma unroll
  for (int k = 0; k < V; ++k) Z[k] = reset ? kAnew : DT ? Z[k] : rate_of(Z[k], P[k]);
  chunk_prefix<V, true>(s, p, Z, U, lds, pZ, pU, cZ, cU);
}

// gx = H w, gg = H w (x (1 - w) - dt a h_{i-1}) with H_i = gy_i + C_{i+1}; gh0 = C at a window's first token.
template <typename T, int V, bool DT>
__global__ void __launch_bounds__(kBlock) k_scan_bwd_apply(ScanGeo s, const T* __restrict__ x, const T* __restrict__ g,
                                                           const int64_t* __restrict__ start,
                                                           const float* __restrict__ dt, const float* __restrict__ h0,
                                                           const float* __restrict__ hs, const T* __restrict__ gy,
                                                           const float* __restrict__ glast,
                                                           const float* __restrict__ pZ, const float* __restrict__ pU,
                                                           const float* __restrict__ carry, T* __restrict__ gx,
                                                           T* __restrict__ gg, float* __restrict__ gh0) {
  const Place p = place_of<V>(s);
  const int64_t wf = wave_first_token(s);
  Ascend up(start, s.B, wf, p.i0);
  Descend win(start, s.B, wf, p.i1 - 1);
  if (!p.live || p.i0 >= s.N) return;
  const int64_t at = p.group * s.D + p.c;
  const int n = (int)(p.i1 - p.i0);
  float hp[kLen][V];                             // h_{i-1}
  Pack<T, V> xr[kLen], gr[kLen];
  {
    float h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = hs[at + k];
#pragma unroll
    for (int t = 0; t < kLen; ++t) {
      if (t >= n) continue;
      const int64_t i = p.i0 + t;
      xr[t] = load_pack<T, V>(x + i * s.sx + p.c);
      gr[t] = load_pack<T, V>(g + i * s.sg + p.c);
      const float d = DT ? dt[i] : 1.f;
      if (up.starts(start, s.B, i))
#pragma unroll
        for (int k = 0; k < V; ++k) h[k] = h0 ? h0[up.b * s.D + p.c + k] : 0.f;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        hp[t][k] = h[k];
        const Gate q = gate_of<T, DT>((float)gr[t].e[k]);
        h[k] = fmaf(DT ? __builtin_amdgcn_exp2f(-q.rate2 * d) : q.wc, h[k], q.w * (float)xr[t].e[k]);
      }
    }
  }
  float C[V];
#pragma unroll
  for (int k = 0; k < V; ++k) C[k] = past(pZ[at + k], pU[at + k], carry[blockIdx.x * s.D + p.c + k]);
#pragma unroll
  for (int t = kLen - 1; t >= 0; --t) {
    if (t >= n) continue;
    const int64_t i = p.i0 + t;
    float yv[V], ox[V], og[V];
    if (gy)
      load_f<V>(gy + i * s.sgy + p.c, yv);
    else
#pragma unroll
      for (int k = 0; k < V; ++k) yv[k] = 0.f;
    const float d = DT ? dt[i] : 1.f;
    if (t < n - 1) win.step(start, i);
    if (win.last)
#pragma unroll
      for (int k = 0; k < V; ++k) C[k] = glast ? glast[win.b * s.D + p.c + k] : 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const Gate q = gate_of<T, DT>((float)gr[t].e[k]);
      const float a = DT ? __builtin_amdgcn_exp2f(-q.rate2 * d) : q.wc;
      const float H = yv[k] + C[k];
      const float Hw = H * q.w;
      C[k] = a * H;
      ox[k] = Hw;
      og[k] = Hw * fmaf((float)xr[t].e[k], q.wc, -(d * a) * hp[t][k]);
    }
    store_f<V>(gx + i * s.D + p.c, ox);
    store_f<V>(gg + i * s.D + p.c, og);
    if (gh0 && i == win.first)
#pragma unroll
      for (int k = 0; k < V; ++k) gh0[win.b * s.D + p.c + k] = C[k];
  }
}

// One token of every stream: 4 bytes of state in and out per channel, bound by the launch.
template <typename T, bool DT>
__global__ void __launch_bounds__(kBlock) k_scan_step(int64_t N, int64_t D, int64_t sx, int64_t sg,
                                                      const T* __restrict__ x, const T* __restrict__ g,
                                                      const float* __restrict__ dt, float* __restrict__ h,
                                                      T* __restrict__ y) {
  const int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x;
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
  int64_t groups;
  unsigned gx, gy;
  int64_t pZ, pU, cZ, cU, carry, bytes;          // workspace offsets in floats, and its size
};

// 8 bytes a lane where widths, strides and addresses allow it, else single elements: a lane's 16 tokens of 8 bytes are
// what the backward keeps in registers.
int scan_vector(int dtype, int64_t D, int64_t strides, const void* const* ptrs, int n) {
  const int v = 8 / dtype_size(dtype);
  if (D % v || strides % v) return 1;
  for (int k = 0; k < n; ++k)
    if (!aligned_to(ptrs[k], 8)) return 1;
  return v;
}

// A group is kLen tokens whatever V and the lanes are: the backward reads the forward's start states per group.
ScanPlan scan_plan(int64_t N, int64_t D, int V) {
  ScanPlan q;
  q.V = V;
  q.s.N = N;
  q.s.D = D;
  int cl2 = 0;
  while ((1 << cl2) < kWave && ((int64_t)V << cl2) < D) ++cl2;
  q.s.cl2 = cl2;
  const int G = kBlock >> cl2;
  q.groups = (N + kLen - 1) / kLen;
  q.s.nchunk = (q.groups + G - 1) / G;
  q.gx = (unsigned)q.s.nchunk;
  q.gy = (unsigned)((D + ((int64_t)V << cl2) - 1) / ((int64_t)V << cl2));
  const int64_t ng = (q.groups * D + 3) / 4 * 4, nc = (q.s.nchunk * D + 3) / 4 * 4;
  q.pZ = 0;
  q.pU = ng;
  q.cZ = 2 * ng;
  q.cU = q.cZ + nc;
  q.carry = q.cU + nc;
  q.bytes = (q.carry + nc) * 4;
  return q;
}

bool scan_sizes_ok(int64_t N, int64_t D, int64_t B, int dtype) {
  return N >= 0 && N < ((int64_t)1 << 31) && D >= 1 && D <= 65536 && B >= 0 && B < ((int64_t)1 << 31) && (B > 0 || N == 0) &&
         dtype_ok(dtype);
}

template <bool REV>
void launch_carry(const ScanPlan& q, float* ws, const int64_t* start, int64_t B, const float* in, float* out,
                  hipStream_t stream) {
  const unsigned cb = q.s.nchunk ? (unsigned)((q.s.D + kCarryChannels - 1) / kCarryChannels) : 0;
  const unsigned eb = out ? (unsigned)std::min<int64_t>(256, (B * q.s.D + kCarryBlock - 1) / kCarryBlock) : 0;
  if (cb + eb == 0) return;
  hipLaunchKernelGGL((k_scan_carry<REV>), dim3(cb + eb), dim3(kCarryBlock), 0, stream, q.s.nchunk, q.s.D, ws + q.cZ,
                     ws + q.cU, ws + q.carry, start, (int)B, in, out, cb);
}

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
    if (vec) inner(bf16_t{}, std::integral_constant<int, 4>{});
    else inner(bf16_t{}, std::integral_constant<int, 1>{});
  } else {
    if (vec) inner(f16_t{}, std::integral_constant<int, 4>{});
    else inner(f16_t{}, std::integral_constant<int, 1>{});
  }
}

}  // namespace
}  // namespace atlhip

using namespace atlhip;

extern "C" {

int64_t atl_gated_scan_groups(int64_t N) { return N < 0 ? -1 : (N + kLen - 1) / kLen; }

int64_t atl_gated_scan_ws_bytes(int64_t N, int64_t D, int dtype) {
  if (!scan_sizes_ok(N, D, 1, dtype)) return -1;
  return std::max(scan_plan(N, D, 8 / dtype_size(dtype)).bytes, scan_plan(N, D, 1).bytes);
}

int atl_gated_scan_fwd(const void* x, int64_t sx, const void* gate, int64_t sg, int dtype, int64_t N, int64_t D,
                       const int64_t* start, int64_t B, const float* dt, const float* h0, void* y, float* last,
                       float* states, void* ws, int64_t ws_bytes, hipStream_t stream) {
  if (!scan_sizes_ok(N, D, B, dtype) || (N > 0 && (sx < 0 || sg < 0))) { set_error("gated_scan_fwd: bad sizes N=%lld D=%lld B=%lld type %d", (long long)N, (long long)D, (long long)B, dtype); return 1; }
  if (B == 0) return 0;
  if (!start || !last || (N > 0 && (!x || !gate || !y || !ws))) { set_error("gated_scan_fwd: null argument"); return 1; }
  if (N > 0 && ws_bytes < atl_gated_scan_ws_bytes(N, D, dtype)) { set_error("gated_scan_fwd: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)atl_gated_scan_ws_bytes(N, D, dtype)); return 1; }
  const void* ptrs[] = {x, gate, y};
  ScanPlan q = scan_plan(N, D, scan_vector(dtype, D, sx | sg, ptrs, 3));
  q.s.sx = sx; q.s.sg = sg; q.s.sgy = 0; q.s.B = (int)B;
  float* w = (float*)ws;
  float* pU = states ? states : w + q.pU;
  if (N > 0)
    by_type(dtype, q.V > 1, dt != nullptr, [&](auto t, auto v, auto d) {
      using T = decltype(t);
      hipLaunchKernelGGL((k_scan_local<T, decltype(v)::value, decltype(d)::value>), dim3(q.gx, q.gy), dim3(kBlock), 0, stream,
                         q.s, (const T*)x, (const T*)gate, start, dt, h0, w + q.pZ, pU, w + q.cZ, w + q.cU);
    });
  launch_carry<false>(q, w, start, B, h0, last, stream);
  if (N > 0)
    by_type(dtype, q.V > 1, dt != nullptr, [&](auto t, auto v, auto d) {
      using T = decltype(t);
      hipLaunchKernelGGL((k_scan_apply<T, decltype(v)::value, decltype(d)::value>), dim3(q.gx, q.gy), dim3(kBlock), 0, stream,
                         q.s, (const T*)x, (const T*)gate, start, dt, h0, (const float*)(w + q.pZ), pU,
                         (const float*)(w + q.carry), (T*)y, last, states != nullptr);
    });
  return check_launch("gated_scan_fwd");
}

int atl_gated_scan_bwd(const void* x, int64_t sx, const void* gate, int64_t sg, int dtype, int64_t N, int64_t D,
                       const int64_t* start, int64_t B, const float* dt, const float* h0, const float* states,
                       const void* gy, int64_t sgy, const float* glast, void* gx, void* ggate, float* gh0, void* ws,
                       int64_t ws_bytes, hipStream_t stream) {
  if (!scan_sizes_ok(N, D, B, dtype) || (N > 0 && (sx < 0 || sg < 0 || sgy < 0))) { set_error("gated_scan_bwd: bad sizes N=%lld D=%lld B=%lld type %d", (long long)N, (long long)D, (long long)B, dtype); return 1; }
  if (B == 0) return 0;
  if (!start || (N > 0 && (!x || !gate || !states || !gx || !ggate || !ws))) { set_error("gated_scan_bwd: null argument"); return 1; }
  if (N > 0 && ws_bytes < atl_gated_scan_ws_bytes(N, D, dtype)) { set_error("gated_scan_bwd: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)atl_gated_scan_ws_bytes(N, D, dtype)); return 1; }
  const void* ptrs[] = {x, gate, gx, ggate, gy};
  ScanPlan q = scan_plan(N, D, scan_vector(dtype, D, sx | sg | (gy ? sgy : 0), ptrs, 5));
  q.s.sx = sx; q.s.sg = sg; q.s.sgy = sgy; q.s.B = (int)B;
  float* w = (float*)ws;
  if (N > 0)
    by_type(dtype, q.V > 1, dt != nullptr, [&](auto t, auto v, auto d) {
      using T = decltype(t);
      hipLaunchKernelGGL((k_scan_bwd_local<T, decltype(v)::value, decltype(d)::value>), dim3(q.gx, q.gy), dim3(kBlock), 0, stream,
                         q.s, (const T*)gate, start, dt, (const T*)gy, glast, w + q.pZ, w + q.pU, w + q.cZ, w + q.cU);
    });
  launch_carry<true>(q, w, start, B, glast, gh0, stream);
  if (N > 0)
    by_type(dtype, q.V > 1, dt != nullptr, [&](auto t, auto v, auto d) {
      using T = decltype(t);
      hipLaunchKernelGGL((k_scan_bwd_apply<T, decltype(v)::value, decltype(d)::value>), dim3(q.gx, q.gy), dim3(kBlock), 0, stream,
                         q.s, (const T*)x, (const T*)gate, start, dt, h0, states, (const T*)gy, glast,
                         (const float*)(w + q.pZ), (const float*)(w + q.pU), (const float*)(w + q.carry), (T*)gx,
                         (T*)ggate, gh0);
    });
  return check_launch("gated_scan_bwd");
}

int atl_gated_scan_step(const void* x, int64_t sx, const void* gate, int64_t sg, int dtype, int64_t N, int64_t D,
                        const float* dt, float* state, void* y, hipStream_t stream) {
  if (!scan_sizes_ok(N, D, 1, dtype) || sx < 0 || sg < 0) { set_error("gated_scan_step: bad sizes N=%lld D=%lld type %d", (long long)N, (long long)D, dtype); return 1; }
  if (N == 0) return 0;
  if (!x || !gate || !state || !y) { set_error("gated_scan_step: null argument"); return 1; }
  if ((N * D + kBlock - 1) / kBlock >= ((int64_t)1 << 31)) { set_error("gated_scan_step: too large"); return 1; }
  by_type(dtype, false, dt != nullptr, [&](auto t, auto, auto d) {
    using T = decltype(t);
    hipLaunchKernelGGL((k_scan_step<T, decltype(d)::value>), dim3(grid_for(N * D)), dim3(kBlock), 0, stream, N, D, sx, sg,
                       (const T*)x, (const T*)gate, dt, state, (T*)y);
  });
  return check_launch("gated_scan_step");
}

}  // extern "C"
