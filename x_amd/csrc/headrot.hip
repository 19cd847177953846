// Root-mean-square norm of every head's queries and keys, and the rotation of their channel pairs by the token's position,
// in one pass:
//
//   xh = x r w,  r = 1 / sqrt(mean(x^2) + eps)      (no norm: xh = x)
//   (y_2p, y_2p+1) = (xh_2p cos t - xh_2p+1 sin t, xh_2p sin t + xh_2p+1 cos t),  t = pos[axis(p)] freq_p,  p < pairs
//
// the channels past the pairs unturned.  Backward, with g = the output's gradient turned back by t:
//
//   gw = sum over tokens and heads of g x r,   gx = r (w g - x r mean(w g x r)).
//
// Angles are taken in turns in 64 bits and reduced to half a turn before they become single precision: a position of a
// million with a frequency near one keeps its angle.  The hardware's sine and cosine take turns, and are off by 1.3e-7 at
// most over the half turn (measured on 2^23 angles).  They are those of all the token's heads, so a group of lanes that
// holds a row (16 bytes a lane) goes through several heads with them.  Bound by memory (a read and a write of the rows
// forward, two reads and a write backward): 100k tokens x (8 + 2) heads of 128 in float16 take 114 us forward, 4.5 TB/s; 1M x
// (2 + 2) heads of 32 in bfloat16 126 us forward and 215 us backward (4.1 and 3.6 TB/s), of which the vector instructions'
// issue is 61 and 88.  Rows off 16 bytes wait longer: 60k x (5 + 5) of 46 in float32 take 74 and 114 us, of which issue, angles
// of three axes among it, is 21 and 30; a row's last piece is read element by element, and 12 lanes of 16 have one (of 48
// channels, from the cache, 41 us forward instead of 47).
#include "shares.h"
#include "typed.h"
#include "../../include/atl_hip.h"

#include <algorithm>
#include <type_traits>

namespace atlhip {
namespace {

constexpr int kMaxHeadWidth = 256, kMaxAxes = 4;

struct HeadRows {
  const void* p;
  int64_t sn, sh;                     // token and head strides in elements
};

struct RotGeo {
  int64_t N;
  int H, Hk, D, A, pairs;             // heads of the queries and keys, channels, axes, turned pairs
  int bound[kMaxAxes];                // first pair behind each axis
  const void* pos;                    // (N, A)
  int doubles;                        // 1: pos is in double precision, 2: freq is
  const void* freq;
  float eps, inv_d;
  int cl2, per, blocks_of;            // log2 of a row's lanes, heads of an item, items of a token
};

// Cosine and sine of the lane's pairs from column c on.
template <int V>
__device__ __forceinline__ void angles(const RotGeo& g, int64_t n, int c, float (&co)[V / 2], float (&si)[V / 2]) {
#pragma unroll
  for (int m = 0; m < V / 2; ++m) {
    const int p = c / 2 + m;
    co[m] = 1.f, si[m] = 0.f;
    if (p >= g.pairs) continue;
    int a = 0;
#pragma unroll
    for (int k = 0; k < kMaxAxes - 1; ++k) a += k < g.A - 1 && p >= g.bound[k];
    const int64_t at = n * g.A + a;
    const double x = g.doubles & 1 ? ((const double*)g.pos)[at] : (double)((const float*)g.pos)[at];
    const double f = g.doubles & 2 ? ((const double*)g.freq)[p] : (double)((const float*)g.freq)[p];
    const double turns = x * (f * 0.15915494309189535);
    const float t = (float)(turns - rint(turns));
    co[m] = __builtin_amdgcn_cosf(t), si[m] = __builtin_amdgcn_sinf(t);
  }
}

// The first `pairs` of the lane's; the others are passed on as they are (turned by zero, a NaN or an infinity would reach its
// neighbour).
template <int V>
__device__ __forceinline__ void turn(float (&v)[V], const float (&co)[V / 2], const float (&si)[V / 2], float sign, int pairs) {
#pragma unroll
  for (int m = 0; m < V / 2; ++m) {
    const float a = v[2 * m], b = v[2 * m + 1], s = sign * si[m];
    v[2 * m] = m < pairs ? fmaf(a, co[m], -b * s) : a;
    v[2 * m + 1] = m < pairs ? fmaf(a, s, b * co[m]) : b;
  }
}

// Sum over a row's lanes, returned to each.
__device__ __forceinline__ float lanes_sum(float v, int cl2) {
  if (cl2 >= 1) v += dppf<0xB1, 0xF>(v);                    // quad_perm [1, 0, 3, 2]
  if (cl2 >= 2) v += dppf<0x4E, 0xF>(v);                    // quad_perm [2, 3, 0, 1]
  if (cl2 >= 3) v += dppf<0x141, 0xF>(v);                   // row_half_mirror
  if (cl2 >= 4) v += dppf<0x140, 0xF>(v);                   // row_mirror
  if (cl2 >= 5) v += __shfl_xor(v, 16, kWave);
  if (cl2 >= 6) v += __shfl_xor(v, 32, kWave);
  return v;
}

// A piece of a row of D channels, from column c < D on; zeros past it.
template <bool WHOLE, int V, typename T>
__device__ __forceinline__ Pack<T, V> fetch_part(const T* row, int c, int D) {
  Pack<T, V> q;
  if constexpr (WHOLE) {
    q = load_pack<T, V>(row + c);
  } else if (D - c >= V) {
    const LoosePack<T, V> z = *reinterpret_cast<const LoosePack<T, V>*>(row + c);
#pragma unroll
    for (int k = 0; k < V; ++k) q.e[k] = z.e[k];
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) q.e[k] = c + k < D ? row[c + k] : (T)0.f;
  }
  return q;
}
template <bool WHOLE, int V, typename T>
__device__ __forceinline__ void load_part(const T* row, int c, int D, float (&v)[V]) {
  const Pack<T, V> q = fetch_part<WHOLE, V>(row, c, D);
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = (float)q.e[k];
}
template <bool WHOLE, int V, typename T>
__device__ __forceinline__ void store_part(T* row, int c, int D, const float (&v)[V]) {
  if constexpr (WHOLE) store_f<V>(row + c, v);
  else store_loose<V>(row + c, D - c, v);
}

constexpr int kBatch = 2;             // rows whose loads are under way together (four: 5% slower, for the registers)

// A row of a token: its head, and whether it is a key's.
struct Row {
  bool key;
  int head;
};
__device__ __forceinline__ Row row_of(const RotGeo& g, int h) { return Row{h >= g.H, h >= g.H ? h - g.H : h}; }

template <typename T, bool WHOLE>
__global__ void __launch_bounds__(kBlock) k_headrot_fwd(RotGeo g, HeadRows q, HeadRows k, const float* __restrict__ wq,
                                                        const float* __restrict__ wk, T* __restrict__ yq, T* __restrict__ yk,
                                                        int64_t first) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & ((1 << g.cl2) - 1), c = lane * V;
  const int64_t block = first + blockIdx.x, tokens = block / g.blocks_of;
  const int64_t n = tokens * (kBlock >> g.cl2) + (threadIdx.x >> g.cl2);
  if (n >= g.N) return;                                     // a whole row's lanes
  const int h0 = (int)(block - tokens * g.blocks_of) * g.per, h1 = min(h0 + g.per, g.H + g.Hk);
  const bool in = c < g.D;
  float co[V / 2], si[V / 2], wv[2][V];
  if (wq && in) {
    load_part<WHOLE, V>(wq, c, g.D, wv[0]);
    load_part<WHOLE, V>(wk, c, g.D, wv[1]);
  }
  for (int h = h0; h < h1; h += kBatch) {
    Pack<T, V> raw[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      raw[b] = Pack<T, V>{};
      if (h + b < h1 && in) {
        const Row w = row_of(g, h + b);
        const HeadRows& r = w.key ? k : q;
        raw[b] = fetch_part<WHOLE, V>((const T*)r.p + n * r.sn + w.head * r.sh, c, g.D);
      }
    }
    if (h == h0) angles<V>(g, n, c, co, si);                // while the rows are on their way
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (h + b >= h1) break;
      const Row w = row_of(g, h + b);
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = (float)raw[b].e[e];
      if (wq) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) ss = fmaf(v[e], v[e], ss);
        const float inv = rsqrtf(fmaf(lanes_sum(ss, g.cl2), g.inv_d, g.eps));
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = v[e] * inv * (w.key ? wv[1][e] : wv[0][e]);
      }
      turn<V>(v, co, si, 1.f, g.pairs - c / 2);
      if (in) store_part<WHOLE, V>((w.key ? yk + (n * g.Hk + w.head) * g.D : yq + (n * g.H + w.head) * g.D), c, g.D, v);
    }
  }
}

// part (gridDim.x, 2, D): the workgroup's share of the weights' gradients, its rows added in a fixed order.  A null gradient
// stands for zeros.  Workgroup b takes the heads' item b % blocks_of of tokens far apart.
template <typename T, bool WHOLE>
__global__ void __launch_bounds__(kBlock) k_headrot_bwd(RotGeo g, HeadRows q, HeadRows k, const float* __restrict__ wq,
                                                        const float* __restrict__ wk, HeadRows gq, HeadRows gk,
                                                        T* __restrict__ dq, T* __restrict__ dk, float* __restrict__ part) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float lds[kBlock * V];
  const int lanes = 1 << g.cl2, lane = threadIdx.x & (lanes - 1), c = lane * V, group = threadIdx.x >> g.cl2;
  const bool in = c < g.D;
  float wv[2][V], gw[2][V];
#pragma unroll
  for (int e = 0; e < V; ++e) wv[0][e] = wv[1][e] = gw[0][e] = gw[1][e] = 0.f;
  if (in && wq) load_part<WHOLE, V>(wq, c, g.D, wv[0]);
  if (in && wk) load_part<WHOLE, V>(wk, c, g.D, wv[1]);
  const int64_t step = (int64_t)(gridDim.x / g.blocks_of) * (kBlock >> g.cl2);
  const int h0 = (int)(blockIdx.x % g.blocks_of) * g.per, h1 = min(h0 + g.per, g.H + g.Hk);
  for (int64_t n = (int64_t)(blockIdx.x / g.blocks_of) * (kBlock >> g.cl2) + group; n < g.N; n += step) {
    float co[V / 2], si[V / 2];
    bool turned = false;
    auto row = [&](int head, auto which) {
      constexpr int K = decltype(which)::value;             // a key's row (the weights and their sums without a choice per element)
      const HeadRows &r = K ? k : q, &gr = K ? gk : gq;
      Pack<T, V> xs{}, ys{};
      if (in && gr.p) ys = fetch_part<WHOLE, V>((const T*)gr.p + n * gr.sn + head * gr.sh, c, g.D);
      if (in && wq) xs = fetch_part<WHOLE, V>((const T*)r.p + n * r.sn + head * r.sh, c, g.D);
      if (!turned) angles<V>(g, n, c, co, si);              // while the rows are on their way
      turned = true;
      float y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = (float)ys.e[e];
      turn<V>(y, co, si, -1.f, g.pairs - c / 2);
      if (wq) {
        float x[V], ss = 0.f, dot = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          x[e] = (float)xs.e[e];
          ss = fmaf(x[e], x[e], ss);
          dot = fmaf(wv[K][e] * y[e], x[e], dot);
        }
        const float inv = rsqrtf(fmaf(lanes_sum(ss, g.cl2), g.inv_d, g.eps));
        const float mean = lanes_sum(dot, g.cl2) * inv * g.inv_d;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float hat = x[e] * inv;
          gw[K][e] = fmaf(y[e], hat, gw[K][e]);
          y[e] = inv * fmaf(wv[K][e], y[e], -hat * mean);
        }
      }
      T* out = K ? dk : dq;
      if (in && out) store_part<WHOLE, V>(out + (n * (K ? g.Hk : g.H) + head) * g.D, c, g.D, y);
    };
    for (int h = h0; h < min(h1, g.H); ++h) row(h, std::integral_constant<int, 0>{});
    for (int h = max(h0, g.H); h < h1; ++h) row(h - g.H, std::integral_constant<int, 1>{});
  }
  if (!part) return;
#pragma unroll
  for (int K = 0; K < 2; ++K) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) lds[group * lanes * V + c + e] = gw[K][e];
    __syncthreads();
    for (int ch = threadIdx.x; ch < g.D; ch += kBlock) {
      float sum = 0.f;
      for (int r = 0; r < kBlock >> g.cl2; ++r) sum += lds[r * lanes * V + ch];
      part[((int64_t)blockIdx.x * 2 + K) * g.D + ch] = sum;
    }
  }
}

// ------------------------------------------------------------------------------------------- host
constexpr int64_t kRotBlocks = 2048;   // shares of the weights' gradients

bool rot_ok(int dtype, int64_t N, int64_t H, int64_t Hk, int64_t D, int64_t A, const int64_t* sections, double eps) {
  if (!dtype_ok(dtype) || N < 0 || N >= ((int64_t)1 << 40) || H < 1 || Hk < 1 || H > 65536 || Hk > 65536 || D < 1 ||
      D > kMaxHeadWidth || A < 1 || A > kMaxAxes || !sections || !(eps >= 0 && eps < 1e30))
    return false;
  int64_t pairs = 0;
  for (int64_t a = 0; a < A; ++a) {
    if (sections[a] < 0 || sections[a] > D) return false;
    pairs += sections[a];
  }
  return 2 * pairs <= D;
}

RotGeo rot_geo(int dtype, int64_t N, int64_t H, int64_t Hk, int64_t D, const void* pos, int doubles, const void* freq, int64_t A,
               const int64_t* sections, double eps) {
  RotGeo g{};
  g.N = N; g.H = (int)H; g.Hk = (int)Hk; g.D = (int)D; g.A = (int)A;
  g.pos = pos; g.doubles = doubles; g.freq = freq;
  g.eps = (float)eps;
  g.inv_d = 1.f / (float)D;
  for (int a = 0; a < (int)A; ++a) g.bound[a] = g.pairs += (int)sections[a];
  const int64_t units = (D * dtype_size(dtype) + 15) / 16;
  while ((1 << g.cl2) < units) ++g.cl2;
  // Heads that share a token's angles: all up to 16, in even parts (100k tokens of 8 + 2 heads of 128: 114 us with ten, 155
  // with eight and two), fewer where that leaves the card without work.
  const int64_t heads = H + Hk;
  g.blocks_of = (int)((heads + 15) / 16);
  while (g.blocks_of < heads && N * g.blocks_of << g.cl2 < 256 * 1024) g.blocks_of = (int)std::min<int64_t>(2 * g.blocks_of, heads);
  g.per = (int)((heads + g.blocks_of - 1) / g.blocks_of);
  g.blocks_of = (int)((heads + g.per - 1) / g.per);
  return g;
}

bool rot_whole(int dtype, int64_t D, int64_t strides, std::initializer_list<const void*> ptrs) {
  const int v = 16 / dtype_size(dtype);
  if (D % v || strides % v) return false;
  for (const void* p : ptrs)
    if (!aligned_to(p, 16)) return false;
  return true;
}

template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == kF32) f(float{});
  else if (dtype == kBF16) f(bf16_t{});
  else f(f16_t{});
}

}  // namespace
}  // namespace atlhip

using namespace atlhip;

extern "C" {

int atl_head_norm_rotary_fwd(const void* q, int64_t sqn, int64_t sqh, const void* k, int64_t skn, int64_t skh, int dtype,
                             const float* wq, const float* wk, const void* pos, int doubles, const void* freqs, int64_t A,
                             const int64_t* sections, int64_t N, int64_t H, int64_t Hk, int64_t D, double eps, void* yq,
                             void* yk, hipStream_t stream) {
  if (!rot_ok(dtype, N, H, Hk, D, A, sections, eps) || (N > 0 && (sqn < 0 || sqh < 0 || skn < 0 || skh < 0))) { set_error("head_norm_rotary_fwd: bad sizes or settings N=%lld H=%lld, %lld D=%lld axes=%lld type %d eps=%g", (long long)N, (long long)H, (long long)Hk, (long long)D, (long long)A, dtype, eps); return 1; }
  if (N == 0) return 0;
  const RotGeo g = rot_geo(dtype, N, H, Hk, D, pos, doubles, freqs, A, sections, eps);
  if (!q || !k || !yq || !yk || (g.pairs && (!pos || !freqs))) { set_error("head_norm_rotary_fwd: null argument"); return 1; }
  const bool whole = rot_whole(dtype, D, sqn | sqh | skn | skh, {q, k, wq, wk, yq, yk});
  const HeadRows rq{q, sqn, sqh}, rk{k, skn, skh};
  const int64_t blocks = (N + (kBlock >> g.cl2) - 1) / (kBlock >> g.cl2) * g.blocks_of;
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    in_launches(blocks, [&](int64_t first, unsigned count) {
      if (whole)
        hipLaunchKernelGGL((k_headrot_fwd<T, true>), dim3(count), dim3(kBlock), 0, stream, g, rq, rk, wq, wk, (T*)yq, (T*)yk, first);
      else
        hipLaunchKernelGGL((k_headrot_fwd<T, false>), dim3(count), dim3(kBlock), 0, stream, g, rq, rk, wq, wk, (T*)yq, (T*)yk, first);
    });
  });
  return check_launch("head_norm_rotary_fwd");
}

int64_t atl_head_norm_rotary_bwd_ws_bytes(int64_t H, int64_t Hk, int64_t D) {
  if (H < 1 || Hk < 1 || H > 65536 || Hk > 65536 || D < 1 || D > kMaxHeadWidth) return -1;
  return std::max(kRotBlocks, H + Hk) * 2 * D * 4;
}

int atl_head_norm_rotary_bwd(const void* q, int64_t sqn, int64_t sqh, const void* k, int64_t skn, int64_t skh, int dtype,
                             const float* wq, const float* wk, const void* pos, int doubles, const void* freqs, int64_t A,
                             const int64_t* sections, int64_t N, int64_t H, int64_t Hk, int64_t D, double eps, const void* gyq,
                             int64_t sgqn, int64_t sgqh, const void* gyk, int64_t sgkn, int64_t sgkh, void* gq, void* gk,
                             float* gw, void* ws, int64_t ws_bytes, hipStream_t stream) {
  if (!rot_ok(dtype, N, H, Hk, D, A, sections, eps) || (N > 0 && (sqn < 0 || sqh < 0 || skn < 0 || skh < 0 || sgqn < 0 || sgqh < 0 || sgkn < 0 || sgkh < 0))) { set_error("head_norm_rotary_bwd: bad sizes or settings N=%lld H=%lld, %lld D=%lld axes=%lld type %d eps=%g", (long long)N, (long long)H, (long long)Hk, (long long)D, (long long)A, dtype, eps); return 1; }
  const RotGeo g = rot_geo(dtype, N, H, Hk, D, pos, doubles, freqs, A, sections, eps);
  if ((N > 0 && ((wq && !q) || (wk && !k) || (g.pairs && (!pos || !freqs)))) || (gw && !ws)) { set_error("head_norm_rotary_bwd: null argument"); return 1; }
  if (gw && ws_bytes < atl_head_norm_rotary_bwd_ws_bytes(H, Hk, D)) { set_error("head_norm_rotary_bwd: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)atl_head_norm_rotary_bwd_ws_bytes(H, Hk, D)); return 1; }
  const bool whole = rot_whole(dtype, D, (wq ? sqn | sqh : 0) | (wk ? skn | skh : 0) | (gyq ? sgqn | sgqh : 0) | (gyk ? sgkn | sgkh : 0),
                               {wq ? q : nullptr, wk ? k : nullptr, wq, wk, gyq, gyk, gq, gk});
  const HeadRows rq{q, sqn, sqh}, rk{k, skn, skh}, rgq{gyq, sgqn, sgqh}, rgk{gyk, sgkn, sgkh};
  const int64_t each = std::max<int64_t>(kRotBlocks / g.blocks_of, 1);
  const int nblk = (int)std::min<int64_t>((N + (kBlock >> g.cl2) - 1) / (kBlock >> g.cl2), each) * g.blocks_of;
  if (nblk > 0)
    by_type(dtype, [&](auto t) {
      using T = decltype(t);
      if (whole)
        hipLaunchKernelGGL((k_headrot_bwd<T, true>), dim3(nblk), dim3(kBlock), 0, stream, g, rq, rk, wq, wk, rgq, rgk, (T*)gq,
                           (T*)gk, gw ? (float*)ws : nullptr);
      else
        hipLaunchKernelGGL((k_headrot_bwd<T, false>), dim3(nblk), dim3(kBlock), 0, stream, g, rq, rk, wq, wk, rgq, rgk, (T*)gq,
                           (T*)gk, gw ? (float*)ws : nullptr);
    });
  if (gw)
    hipLaunchKernelGGL(k_sum_shares, dim3(grid_for(2 * D, kSumChannels)), dim3(kSumChannels * kSumRuns), 0, stream, (const float*)ws,
                       nblk, 2 * D, gw);
  return check_launch("head_norm_rotary_bwd");
}

}  // extern "C"
