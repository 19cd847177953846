// Residual addition with dropout and root-mean-square norm, rows of D channels:
//
//   s = residual + m x / (1 - p)  (rounded to the residual's type),  r = 1 / sqrt(mean(s^2) + eps),  y = s r w
//
// m keeps an element where its 16 random bits are >= t = round(65536 p), and 1 - p is (65536 - t) / 65536.  The bits are
// drawn where they are needed, from Philox4x32-10 at counter (row, 2^31 + column / 8, offset) under the seed (the high
// bit of the second word keeps them apart from the event noise's counters), so no mask is stored: the backward draws the
// same bits.  The norm is that of s as it is returned, so the backward needs s alone:
//
//   ds = gs + r (w gy - shat mean(w gy shat)),  shat = s r;  gresidual = ds,  gx = m ds / (1 - p),
//   gw = sum over the rows of gy shat.
//
// A row lies in the registers of a power of two of lanes (a wave at most, or a workgroup for the widest), which read
// 16 bytes each, aligned to them where widths, strides and addresses are: one pass over memory.  Sums are fp32.
#include "philox.h"
#include "typed.h"
#include "../../include/atl_hip.h"

#include <algorithm>
#include <type_traits>

namespace atlhip {
namespace {

constexpr int kMaxWidth = 8192;
constexpr float kFp8Max = 448.f, kFp8Least = 1e-30f;

struct NormGeo {
  int64_t N, D, sx, sr, sgy, sgs;     // rows, channels, row strides in elements
  float eps, inv_d;
  uint32_t t;                         // dropout's threshold (0: none)
  float keep;                         // 1 / (1 - p)
  uint32_t k0, k1, o0, o1;
  int cl2;                            // log2 of the lanes of a row (within a wave)
};

// Dropout of V elements of a row from column c on (a multiple of V).
template <int V>
__device__ __forceinline__ void dropout(const NormGeo& n, int64_t row, int64_t c, float (&v)[V]) {
  const U4 r = philox4x32_10(U4{(uint32_t)row, 0x80000000u | (uint32_t)(c >> 3), n.o0, n.o1}, n.k0, n.k1);
  uint32_t w[V / 2];
  if constexpr (V == 8) {
    w[0] = r.x, w[1] = r.y, w[2] = r.z, w[3] = r.w;
  } else {
    static_assert(V == 4, "pieces of four or eight elements");
    const bool hi = c & 4;
    w[0] = hi ? r.z : r.x, w[1] = hi ? r.w : r.y;
  }
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = ((w[k >> 1] >> ((k & 1) * 16)) & 0xFFFFu) >= n.t ? v[k] * n.keep : 0.f;
}

// Sum over the lanes of a row (all of the workgroup where WIDE), returned to each.
template <bool WIDE>
__device__ __forceinline__ float row_sum(float v, int cl2, float* lds) {
  if constexpr (WIDE) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
  } else {
    for (int d = 1 << cl2 >> 1; d >= 1; d >>= 1) v += __shfl_xor(v, d, kWave);
    return v;
  }
}

// The larger of two; a NaN stays.
__device__ __forceinline__ float top_of(float a, float b) { return (b > a || b != b) ? b : a; }
template <bool WIDE>
__device__ __forceinline__ float row_top(float v, int cl2, float* lds) {
  for (int d = WIDE ? kWave / 2 : 1 << cl2 >> 1; d >= 1; d >>= 1) v = top_of(v, __shfl_xor(v, d, kWave));
  if constexpr (WIDE) {
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    v = top_of(top_of(lds[0], lds[1]), top_of(lds[2], lds[3]));
  }
  return v;
}

template <int V>
__device__ __forceinline__ void store_fp8(uint8_t* p, int64_t n, bool whole, const float (&v)[V]) {
  int w[V / 4];
#pragma unroll
  for (int k = 0; k < V / 4; ++k) {
    w[k] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k], v[4 * k + 1], 0, false);
    w[k] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * k + 2], v[4 * k + 3], w[k], true);
  }
  if (whole) {
    *reinterpret_cast<Pack<int, V / 4>*>(p) = *reinterpret_cast<const Pack<int, V / 4>*>(w);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < n) p[k] = (uint8_t)(w[k / 4] >> (k % 4 * 8));
  }
}

// A piece from column c on of a row of D: aligned and whole, or neither.
template <bool WHOLE, int V, typename T>
__device__ __forceinline__ void load_piece(const T* row, int64_t c, int64_t D, float (&v)[V]) {
  if constexpr (WHOLE) load_f<V>(row + c, v);
  else load_loose<V>(row + c, D - c, v);
}
template <bool WHOLE, int V, typename T>
__device__ __forceinline__ void store_piece(T* row, int64_t c, int64_t D, const float (&v)[V]) {
  if constexpr (WHOLE) store_f<V>(row + c, v);
  else store_loose<V>(row + c, D - c, v);
}

// Q8: y in e4m3 with a scale per row, a / 448 with a = max |y|.
template <typename T, typename R, int V, int NV, bool WIDE, bool WHOLE, bool Q8>
__global__ void __launch_bounds__(kBlock) k_norm_fwd(NormGeo n, const T* __restrict__ x, const R* __restrict__ res,
                                                     const float* __restrict__ w, void* __restrict__ y,
                                                     R* __restrict__ s, float* __restrict__ scale, int64_t first) {
  __shared__ float lds[kBlock / kWave];
  const int lanes = WIDE ? kBlock : 1 << n.cl2;
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t block = first + blockIdx.x;
  const int64_t row = WIDE ? block : block * (kBlock >> n.cl2) + (threadIdx.x >> n.cl2);
  if (!WIDE && row >= n.N) return;
  float v[NV][V];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t c = ((int64_t)j * lanes + lane) * V;
    if (c >= n.D) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[j][k] = 0.f;
      continue;
    }
    load_piece<WHOLE, V>(x + row * n.sx, c, n.D, v[j]);
    if (n.t) dropout<V>(n, row, c, v[j]);
    if (res) {
      float rv[V];
      load_piece<WHOLE, V>(res + row * n.sr, c, n.D, rv);
#pragma unroll
      for (int k = 0; k < V; ++k) v[j][k] = rv[k] + v[j][k];
    }
    if (s) store_piece<WHOLE, V>(s + row * n.D, c, n.D, v[j]);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      v[j][k] = (float)(R)v[j][k];
      ss = fmaf(v[j][k], v[j][k], ss);
    }
  }
  const float inv = rsqrtf(fmaf(row_sum<WIDE>(ss, n.cl2, lds), n.inv_d, n.eps));
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t c = ((int64_t)j * lanes + lane) * V;
    if (c >= n.D) continue;
    float wv[V];
    load_piece<WHOLE, V>(w, c, n.D, wv);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      v[j][k] = v[j][k] * inv * wv[k];
      if (Q8) top = top_of(top, fabsf(v[j][k]));
    }
    if (!Q8) store_piece<WHOLE, V>((T*)y + row * n.D, c, n.D, v[j]);
  }
  if constexpr (Q8) {
    top = top_of(row_top<WIDE>(top, n.cl2, lds), kFp8Least);
    const float to8 = kFp8Max / top;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t c = ((int64_t)j * lanes + lane) * V;
      if (c >= n.D) continue;
#pragma unroll
      for (int k = 0; k < V; ++k) v[j][k] *= to8;
      store_fp8<V>((uint8_t*)y + row * n.D + c, n.D - c, WHOLE, v[j]);
    }
    if (lane == 0) scale[row] = top * (1.f / kFp8Max);
  }
}

// part (gridDim.x, D): the workgroup's share of gw, its rows added in a fixed order.
template <typename T, typename R, int V, int NV, bool WIDE, bool WHOLE>
__global__ void __launch_bounds__(kBlock) k_norm_bwd(NormGeo n, const R* __restrict__ s, const float* __restrict__ w,
                                                     const T* __restrict__ gy, const R* __restrict__ gs,
                                                     T* __restrict__ gx, R* __restrict__ gres,
                                                     float* __restrict__ part) {
  extern __shared__ float dyn[];
  const int lanes = WIDE ? kBlock : 1 << n.cl2;
  const int lane = threadIdx.x & (lanes - 1), gi = WIDE ? 0 : threadIdx.x >> n.cl2;
  const int rows = kBlock / lanes;
  float wv[NV][V], gw[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t c = ((int64_t)j * lanes + lane) * V;
#pragma unroll
    for (int k = 0; k < V; ++k) wv[j][k] = gw[j][k] = 0.f;
    if (c < n.D) load_piece<WHOLE, V>(w, c, n.D, wv[j]);
  }
  for (int64_t row = (int64_t)blockIdx.x * rows + gi; row < n.N; row += (int64_t)gridDim.x * rows) {
    float sv[NV][V], yv[NV][V];
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t c = ((int64_t)j * lanes + lane) * V;
#pragma unroll
      for (int k = 0; k < V; ++k) sv[j][k] = yv[j][k] = 0.f;
      if (c >= n.D) continue;
      load_piece<WHOLE, V>(s + row * n.sr, c, n.D, sv[j]);
      load_piece<WHOLE, V>(gy + row * n.sgy, c, n.D, yv[j]);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        ss = fmaf(sv[j][k], sv[j][k], ss);
        dot = fmaf(wv[j][k] * yv[j][k], sv[j][k], dot);
      }
    }
    const float inv = rsqrtf(fmaf(row_sum<WIDE>(ss, n.cl2, dyn), n.inv_d, n.eps));
    const float mean = row_sum<WIDE>(dot, n.cl2, dyn) * inv * n.inv_d;         // mean(w gy shat)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t c = ((int64_t)j * lanes + lane) * V;
      if (c >= n.D) continue;
      float d[V];
      if (gs)
        load_piece<WHOLE, V>(gs + row * n.sgs, c, n.D, d);
      else
#pragma unroll
        for (int k = 0; k < V; ++k) d[k] = 0.f;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float hat = sv[j][k] * inv;
        gw[j][k] = fmaf(yv[j][k], hat, gw[j][k]);
        d[k] = fmaf(inv, fmaf(wv[j][k], yv[j][k], -hat * mean), d[k]);
      }
      if (gres) store_piece<WHOLE, V>(gres + row * n.D, c, n.D, d);
      if (gx) {
        if (n.t) dropout<V>(n, row, c, d);
        store_piece<WHOLE, V>(gx + row * n.D, c, n.D, d);
      }
    }
  }
  if (!part) return;
  const int width = lanes * NV * V;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < V; ++k) dyn[gi * width + (j * lanes + lane) * V + k] = gw[j][k];
  __syncthreads();
  for (int c = threadIdx.x; c < width && c < n.D; c += kBlock) {
    float sum = 0.f;
    for (int g = 0; g < rows; ++g) sum += dyn[g * width + c];
    part[blockIdx.x * n.D + c] = sum;
  }
}

// The same where the sum alone was used (no gy): ds = gs, and the norm has no part, nor has a root of a row that is not
// finite (zero times it would be no number).  gs null: zeros.
template <typename T, typename R, int V, bool WHOLE>
__global__ void __launch_bounds__(kBlock) k_norm_bwd_sum(NormGeo n, const R* __restrict__ gs, T* __restrict__ gx,
                                                         R* __restrict__ gres) {
  const int rows = kBlock >> n.cl2, lane = threadIdx.x & ((1 << n.cl2) - 1);
  for (int64_t row = (int64_t)blockIdx.x * rows + (threadIdx.x >> n.cl2); row < n.N; row += (int64_t)gridDim.x * rows)
    for (int64_t c = lane * V; c < n.D; c += V << n.cl2) {
      float d[V];
#pragma unroll
      for (int k = 0; k < V; ++k) d[k] = 0.f;
      if (gs) load_piece<WHOLE, V>(gs + row * n.sgs, c, n.D, d);
      if (gres) store_piece<WHOLE, V>(gres + row * n.D, c, n.D, d);
      if (gx) {
        if (n.t) dropout<V>(n, row, c, d);
        store_piece<WHOLE, V>(gx + row * n.D, c, n.D, d);
      }
    }
}

// gw[c] = sum over the workgroups' shares: 16 channels a workgroup, 64 interleaved runs of the shares side by side.
constexpr int kSumChannels = 16, kSumRuns = 64;
__global__ void __launch_bounds__(kSumChannels* kSumRuns) k_norm_gw(const float* __restrict__ part, int nblk, int64_t D,
                                                                    float* __restrict__ gw) {
  __shared__ float lds[kSumRuns][kSumChannels];
  const int ch = threadIdx.x % kSumChannels, run = threadIdx.x / kSumChannels;
  const int64_t c = (int64_t)blockIdx.x * kSumChannels + ch;
  float sum = 0.f;
  if (c < D)
#pragma unroll 4
    for (int b = run; b < nblk; b += kSumRuns) sum += part[b * D + c];
  lds[run][ch] = sum;
  __syncthreads();
  for (int half = kSumRuns / 2; half >= 1; half /= 2) {
    if (run < half) lds[run][ch] += lds[run + half][ch];
    __syncthreads();
  }
  if (run == 0 && c < D) gw[c] = lds[0][ch];
}

// ------------------------------------------------------------------------------------------- host
struct NormPlan {
  int V, NV, cl2;
  bool wide, whole;
};

// V: 16 bytes of x; whole: the width, strides and addresses are multiples of it (else pieces are read as they lie, and a
// row's last one in part: 60007 x 345 single precision forward and backward runs 230 us with single elements instead).
// A row takes as few lanes as hold it with one piece each, then up to four pieces a lane, then a workgroup.
NormPlan norm_plan(int dtype, int64_t D, bool whole) {
  NormPlan q;
  q.V = 16 / dtype_size(dtype);
  q.whole = whole;
  const int64_t units = (D + q.V - 1) / q.V;
  q.cl2 = 0;
  while ((1 << q.cl2) < kWave && (1 << q.cl2) < units) ++q.cl2;
  const int64_t per = (units + (1 << q.cl2) - 1) >> q.cl2;
  q.wide = per > 4;
  q.NV = q.wide ? 32 / q.V : ceil_pow2(per);
  return q;
}

int norm_blocks(int64_t N, const NormPlan& q) {
  const int64_t rows = q.wide ? 1 : kBlock >> q.cl2;
  return (int)std::min<int64_t>((N + rows - 1) / rows, 1024);
}

template <typename F>
void by_types(int dtype, int rtype, F&& f) {
  if (dtype == kF32) f(float{}, float{});
  else if (dtype == kBF16 && rtype == kF32) f(bf16_t{}, float{});
  else if (dtype == kBF16) f(bf16_t{}, bf16_t{});
  else if (rtype == kF32) f(f16_t{}, float{});
  else f(f16_t{}, f16_t{});
}

template <typename T, typename F>
void by_shape(const NormPlan& q, F&& f) {
  constexpr int VM = 16 / sizeof(T);
  using std::integral_constant;
  auto go = [&](auto nv, auto wide) {
    if (q.whole) f(integral_constant<int, VM>{}, nv, wide, std::true_type{});
    else f(integral_constant<int, VM>{}, nv, wide, std::false_type{});
  };
  if (q.wide) go(integral_constant<int, 32 / VM>{}, std::true_type{});
  else if (q.NV == 1) go(integral_constant<int, 1>{}, std::false_type{});
  else if (q.NV == 2) go(integral_constant<int, 2>{}, std::false_type{});
  else go(integral_constant<int, 4>{}, std::false_type{});
}

bool norm_ok(int dtype, int rtype, int64_t N, int64_t D, double eps, double p) {
  return dtype_ok(dtype) && (rtype == dtype || rtype == kF32) && N >= 0 && N < ((int64_t)1 << 31) && D >= 1 &&
         D <= kMaxWidth && eps >= 0 && eps < 1e30 && p >= 0 && p < 1 && (int)(p * 65536 + 0.5) < 65536;
}

NormGeo norm_geo(int64_t N, int64_t D, double eps, double p, uint64_t seed, uint64_t offset) {
  NormGeo n{};
  n.N = N; n.D = D;
  n.eps = (float)eps;
  n.inv_d = 1.f / (float)D;
  n.t = (uint32_t)__builtin_nearbyint(p * 65536);
  n.keep = 65536.f / (float)(65536 - n.t);
  n.k0 = (uint32_t)seed; n.k1 = (uint32_t)(seed >> 32);
  n.o0 = (uint32_t)offset; n.o1 = (uint32_t)(offset >> 32);
  return n;
}

bool norm_whole(int dtype, int64_t D, int64_t strides, const void* const* ptrs, int n) {
  const int v = 16 / dtype_size(dtype);
  if (D % v || strides % v) return false;
  for (int k = 0; k < n; ++k)
    if (!aligned_to(ptrs[k], 16)) return false;
  return true;
}

}  // namespace
}  // namespace atlhip

using namespace atlhip;

extern "C" {

int atl_rms_norm_fwd(const void* x, int64_t sx, int dtype, const void* res, int64_t sr, int rtype, const float* w,
                     int64_t N, int64_t D, double eps, double p, uint64_t seed, uint64_t offset, void* y, void* s,
                     float* scale, hipStream_t stream) {
  if (!norm_ok(dtype, rtype, N, D, eps, p) || (N > 0 && (sx < 0 || sr < 0))) { set_error("rms_norm_fwd: bad sizes or settings N=%lld D=%lld types %d, %d eps=%g p=%g", (long long)N, (long long)D, dtype, rtype, eps, p); return 1; }
  if (N == 0) return 0;
  if (!x || !w || !y) { set_error("rms_norm_fwd: null argument"); return 1; }
  NormGeo n = norm_geo(N, D, eps, p, seed, offset);
  n.sx = sx; n.sr = sr;
  const void* ptrs[] = {x, res, w, y, s};
  const NormPlan q = norm_plan(dtype, D, norm_whole(dtype, D, sx | (res ? sr : 0), ptrs, 5));
  n.cl2 = q.cl2;
  const int64_t blocks = q.wide ? N : grid_for(N, kBlock >> q.cl2);
  by_types(dtype, rtype, [&](auto t, auto r) {
    using T = decltype(t);
    using R = decltype(r);
    by_shape<T>(q, [&](auto v, auto nv, auto wide, auto whole) {
      constexpr int V = decltype(v)::value, NV = decltype(nv)::value;
      constexpr bool W = decltype(wide)::value, H = decltype(whole)::value;
      in_launches(blocks, [&](int64_t first, unsigned count) {
        if (scale)
          hipLaunchKernelGGL((k_norm_fwd<T, R, V, NV, W, H, true>), dim3(count), dim3(kBlock), 0, stream, n, (const T*)x,
                             (const R*)res, w, y, (R*)s, scale, first);
        else
          hipLaunchKernelGGL((k_norm_fwd<T, R, V, NV, W, H, false>), dim3(count), dim3(kBlock), 0, stream, n, (const T*)x,
                             (const R*)res, w, y, (R*)s, scale, first);
      });
    });
  });
  return check_launch("rms_norm_fwd");
}

int64_t atl_rms_norm_bwd_ws_bytes(int64_t N, int64_t D) {
  if (!norm_ok(kF32, kF32, N, D, 0, 0)) return -1;
  return 1024 * D * 4;
}

int atl_rms_norm_bwd(const void* s, int64_t ss, int rtype, const float* w, const void* gy, int64_t sgy, int dtype,
                     const void* gs, int64_t sgs, int64_t N, int64_t D, double eps, double p, uint64_t seed,
                     uint64_t offset, void* gx, void* gres, float* gw, void* ws, int64_t ws_bytes,
                     hipStream_t stream) {
  if (!norm_ok(dtype, rtype, N, D, eps, p) || (N > 0 && (ss < 0 || sgy < 0 || sgs < 0))) { set_error("rms_norm_bwd: bad sizes or settings N=%lld D=%lld types %d, %d eps=%g p=%g", (long long)N, (long long)D, dtype, rtype, eps, p); return 1; }
  if ((N > 0 && (!s || !w)) || (gw && !ws)) { set_error("rms_norm_bwd: null argument"); return 1; }
  if (gw && ws_bytes < atl_rms_norm_bwd_ws_bytes(N, D)) { set_error("rms_norm_bwd: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)atl_rms_norm_bwd_ws_bytes(N, D)); return 1; }
  NormGeo n = norm_geo(N, D, eps, p, seed, offset);
  n.sr = ss; n.sgy = sgy; n.sgs = sgs;
  const void* ptrs[] = {s, w, gy, gs, gx, gres};
  const NormPlan q = norm_plan(dtype, D, norm_whole(dtype, D, ss | (gy ? sgy : 0) | (gs ? sgs : 0), ptrs, 6));
  n.cl2 = q.cl2;
  const int nblk = gy ? norm_blocks(N, q) : 0;    // shares of gw
  if (!gy && N > 0)
    by_types(dtype, rtype, [&](auto t, auto r) {
      using T = decltype(t);
      using R = decltype(r);
      constexpr int V = 16 / sizeof(T);
      const dim3 grid((unsigned)std::min<int64_t>(grid_for(N, kBlock >> q.cl2), 2048));
      if (q.whole)
        hipLaunchKernelGGL((k_norm_bwd_sum<T, R, V, true>), grid, dim3(kBlock), 0, stream, n, (const R*)gs, (T*)gx, (R*)gres);
      else
        hipLaunchKernelGGL((k_norm_bwd_sum<T, R, V, false>), grid, dim3(kBlock), 0, stream, n, (const R*)gs, (T*)gx, (R*)gres);
    });
  if (nblk > 0)
    by_types(dtype, rtype, [&](auto t, auto r) {
      using T = decltype(t);
      using R = decltype(r);
      by_shape<T>(q, [&](auto v, auto nv, auto wide, auto whole) {
        constexpr int V = decltype(v)::value, NV = decltype(nv)::value;
        hipLaunchKernelGGL((k_norm_bwd<T, R, V, NV, decltype(wide)::value, decltype(whole)::value>), dim3(nblk), dim3(kBlock),
                           kBlock * NV * V * 4, stream, n, (const R*)s, w, (const T*)gy, (const R*)gs, (T*)gx,
                           (R*)gres, gw ? (float*)ws : nullptr);
      });
    });
  if (gw)
    hipLaunchKernelGGL(k_norm_gw, dim3(grid_for(D, kSumChannels)), dim3(kSumChannels * kSumRuns), 0, stream, (const float*)ws, nblk,
                       D, gw);
  return check_launch("rms_norm_bwd");
}

}  // extern "C"
