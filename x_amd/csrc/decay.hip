// Linear attention with a decay for each head, over windows of tokens.  With a_i = exp(-rate dt_i) and per head
//
//   S_i = a_i S_{i-1} + k_i v_i^T,   y_i = scale q_i S_i                                      (S is D x D)
//
// the gradients have the same form: dq_i = scale S_i gy_i is the recurrence over (gy, v, k) instead of (q, k, v), and with
// G_i = scale q_i gy_i^T + a_{i+1} G_{i+1}, dv_j = k_j G_j and dk_j = G_j v_j are recurrences from the end over (k, q, gy) and
// (v, gy, q).  So there is one sweep, over rows X, Y, W in either direction, with a state M of Y by W channels:
//
//   out_i = ps sum_{j <= i} e^{-(E_i - E_j)} (X_i Y_j) W_j + xs e^{-E_i} X_i M,   M' = e^{-E} M + us sum_j e^{-(E - E_j)} Y_j W_j^T
//
// for a chunk of 64 rows, with E_i the decay from the chunk's begin to row i: up to the row's own gap forward, up to the gap
// before it from the end (a token's gap lies before it).  The products run on the matrix cores.  Decays stay exponents, in
// 64 bits within a chunk, and a factor of the state near one is applied as M + M expm1(-E): a product of many factors just
// below one would lose what each rounds off.  Exponents past 400 (in powers of two: the factor is zero in 32 bits) count as 400,
// so an endless gap forgets what was before it and no difference of infinities appears.
//
// A window is cut into stretches of L tokens; a workgroup follows one stretch of one head.  The state before a stretch comes
// from a pass that sums every stretch but the last on its own (k_decay_local) and one that joins them (k_decay_join); windows
// of one stretch need neither, and both return at once there.
#include "typed.h"
#include "../../include/atl_hip.h"

#include <algorithm>
#include <type_traits>

namespace atlhip {
namespace {

constexpr int kChunk = 64;                 // rows of a chunk: a wave's lanes, and four tiles
constexpr int kMaxHead = 128;
constexpr double kForgotten = 400.0;       // exponents (of two) from which a factor is zero

using F4 = float __attribute__((ext_vector_type(4)));

struct Rows {                              // (N, H, D) with strides in elements
  const void* p;
  int64_t sn, sh;
};

struct DecayGeo {
  const int64_t* start;                    // (B + 1)
  const float *dt, *rate;
  int64_t N, B, L, slots;
  int H, D;
};

// ------------------------------------------------------------------------------------------- fragments
// Eight elements a lane of a 16 x 32 operand of a matrix product: lane l holds index l % 16 of the operand's outer axis, and of
// the axis that is summed over the elements t 16 + 4 (l / 16) + r, t < 2, r < 4.  That order (any is right if both operands have
// it) is the one in which a product's result lies in its lanes, so results go into the next product as they are.
template <typename T>
struct FragOf {
  using type = T __attribute__((ext_vector_type(8)));
};
template <>
struct FragOf<float> {
  struct type {
    float e[8];
    __device__ __forceinline__ float& operator[](int k) { return e[k]; }
    __device__ __forceinline__ float operator[](int k) const { return e[k]; }
  };
};
template <typename T>
using Frag = typename FragOf<T>::type;

__device__ __forceinline__ F4 mma(Frag<bf16_t> a, Frag<bf16_t> b, F4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ F4 mma(Frag<f16_t> a, Frag<f16_t> b, F4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ F4 mma(const Frag<float>& a, const Frag<float>& b, F4 c) {
#pragma unroll
  for (int k = 0; k < 8; ++k) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k], b[k], c, 0, 0, 0);
  return c;
}

// Row `row` of a tile (the lane's own), from column 32 kb on.
template <typename T, int LD>
__device__ __forceinline__ Frag<T> frag_row(const T* tile, int row, int kb) {
  const int g = (threadIdx.x & (kWave - 1)) >> 4;
  const T* p = tile + row * LD + kb * 32 + g * 4;
  const Pack<T, 4> a = load_pack<T, 4>(p), b = load_pack<T, 4>(p + 16);
  Frag<T> f;
#pragma unroll
  for (int r = 0; r < 4; ++r) f[r] = a.e[r], f[4 + r] = b.e[r];
  return f;
}

// Column col0 + l % 16 of a tile, from row 32 kb on.
template <typename T, int LD>
__device__ __forceinline__ Frag<T> frag_col(const T* tile, int col0, int kb) {
  const int l = threadIdx.x & (kWave - 1), g = l >> 4, i = l & 15;
  Frag<T> f;
  if constexpr (sizeof(T) == 2) {
    // The transposed read: 16 lanes name four rows of 16 elements, four to a lane, and each gets a column.
    using S4 = short __attribute__((ext_vector_type(4)));
    using LdsS4 = __attribute__((address_space(3))) S4;
    union { S4 s[2]; Frag<T> f; } u;
    const T* p = tile + (kb * 32 + g * 4 + (i >> 2)) * LD + col0 + 4 * (i & 3);
    u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4*)p);
    u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4*)(p + 16 * LD));
    f = u.f;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = tile[(kb * 32 + (k >> 2) * 16 + g * 4 + (k & 3)) * LD + col0 + i];
  }
  return f;
}

// Values in 32 bits as the sum of NS fragments of T: 8 or 11 more bits of each value with every fragment, so that the
// products' sums are those of values in 24 bits (NS = 3), or within 2^-17 (bfloat16, NS = 2).
template <typename T, int NS>
__device__ __forceinline__ void split(const float (&v)[8], Frag<T> (&f)[NS]) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[0][k] = v[k];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float x = v[k];
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        f[s][k] = (T)x;
        x = s + 1 < NS && fabsf(x) < INFINITY ? x - (float)f[s][k] : 0.f;
      }
    }
  }
}
template <typename T>
constexpr int pieces(int n) {
  return std::is_same<T, float>::value ? 1 : n;
}

// Half precision reaches from 6e-8 to 65504 only: what goes into it is brought to a largest value of 2^14 first.  Returns the
// power of two to multiply by (1 for the other types, and where there is nothing); top: the largest finite magnitude.
__device__ __forceinline__ float finite_top(float top, float v) { return fabsf(v) < INFINITY ? fmaxf(top, fabsf(v)) : top; }
template <typename T>
__device__ __forceinline__ float fit(float top) {
  if constexpr (!std::is_same<T, f16_t>::value) {
    return 1.f;
  } else {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, kWave));
    if (!(top > 0.f)) return 1.f;
    const int e = 14 - ilogbf(top);
    return ldexpf(1.f, e > 126 ? 126 : e < -126 ? -126 : e);
  }
}

// A state's factor e^{-z}: for small z by what it is less than one (else that would lose the factor's own bits).
struct Fade {
  float a;
  int keep;
  __device__ __forceinline__ float operator()(float m) const { return fmaf(m, a, keep ? m : 0.f); }
};
__device__ __forceinline__ Fade fade_of(float z) {
  const bool keep = !(z > 0.5f);
  return Fade{keep ? expm1f(-z) : expf(-z), keep};
}

// ------------------------------------------------------------------------------------------- windows
// Stretch of a slot.  Windows are numbered with the tokens before the first (window -1) and behind the last (window B), which
// are in none; window b begins at slot floor(first token / L) + b + 1, so every window has as many slots as stretches or
// more, and no sum over the windows is needed.
struct Stretch {
  int64_t window, lo, hi;                  // tokens of the stretch
  bool first, last, live;                  // of its window; live: there is one
  int64_t entry;                           // of the states after stretches: unlike for all but windows' last stretches
};

__device__ __forceinline__ int64_t edge_of(const DecayGeo& d, int64_t e) {     // first token of window e - 1
  if (e <= 0) return 0;
  if (e > d.B + 1) return d.N;
  const int64_t s = d.start[e - 1];
  return s < 0 ? 0 : s > d.N ? d.N : s;
}

// Every lane of a wave calls it: 64 windows are looked at in one step.
__device__ __forceinline__ Stretch stretch_of(const DecayGeo& d, int64_t slot) {
  const int lane = threadIdx.x & (kWave - 1);
  int64_t lo = 0, n = d.B + 2;             // the last of n windows from lo on whose first slot is not past this one
  while (n > 1) {
    const int64_t step = (n + kWave - 1) / kWave;
    const int64_t e = lo + lane * step;
    const bool at = lane * step < n && edge_of(d, e) / d.L + e <= slot;
    const int c = __popcll(__ballot(at));
    const int64_t k = c > 0 ? c - 1 : 0;
    lo += k * step;
    n = min(step, n - k * step);
  }
  Stretch s;
  const int64_t begin = edge_of(d, lo), end = max(begin, edge_of(d, lo + 1));
  const int64_t k = slot - (begin / d.L + lo);
  s.window = lo - 1;
  s.entry = begin / d.L + k;
  s.lo = begin + k * d.L;
  s.hi = min(end, s.lo + d.L);
  s.first = k == 0;
  s.last = s.lo + d.L >= end;
  s.live = k == 0 || (k > 0 && s.lo < end);
  return s;
}

// Workgroups of one die (they are dealt out round robin over eight) take neighbouring slots and heads, whose rows share lines.
__device__ __forceinline__ int64_t near_first(int64_t block, int64_t blocks) {
  const int64_t per = (blocks + 7) / 8;
  return (block & 7) * per + (block >> 3);
}

// ------------------------------------------------------------------------------------------- the sweep
template <typename T, int DP, int NW>
struct SweepLds {
  static constexpr int LD = DP + 16 / (int)sizeof(T);       // rows a vector apart: no bank conflicts
  static constexpr int LP = kChunk + 16 / (int)sizeof(T);
  static constexpr int TILE = kChunk * LD, PAIR = kChunk * LP;
  T x[TILE], y[TILE], w[TILE], p[PAIR];
  double e[kChunk];                                         // E_i in powers of two
  float xe[kChunk], we[kChunk];                             // xs e^{-E_i}, us e^{-(E - E_i)}
  Fade fade;                                                // e^{-E}
  float pscale[4][2];                                       // of the pairs' blocks of 16 x 32 (half precision)
};
template <typename T, int DP, int NW>
struct LocalLds {
  static constexpr int LD = DP + 16 / (int)sizeof(T);
  static constexpr int TILE = kChunk * LD;
  T y[TILE], w[TILE];
  double e[kChunk];
  float xe[kChunk], we[kChunk];
  Fade fade;
};

// Pieces of 16 bytes of a chunk's rows, in registers until the chunk's turn.
template <typename T, int DP, int NW>
struct Stage {
  static constexpr int V = 16 / (int)sizeof(T), PER = DP / V, THREADS = NW * kWave, COUNT = kChunk * PER / THREADS;
  static_assert(COUNT * THREADS == kChunk * PER, "whole rounds of pieces");
  Pack<T, V> v[COUNT];

  // Row r of the chunk is token at + r (or at - r where REV); len rows are there, the others zero.
  template <bool REV, bool WHOLE>
  __device__ __forceinline__ void load(const Rows& rows, int64_t head, int64_t at, int len, int D) {
    const T* base = (const T*)rows.p + head * rows.sh;
#pragma unroll
    for (int n = 0; n < COUNT; ++n) {
      const int p = threadIdx.x + n * THREADS, r = p / PER, c = p % PER * V;
      Pack<T, V> q{};
      if (r < len && c < D) {
        const T* from = base + (REV ? at - r : at + r) * rows.sn + c;
        if constexpr (WHOLE) {
          q = load_pack<T, V>(from);
        } else if (c + V <= D) {
          const LoosePack<T, V> z = *reinterpret_cast<const LoosePack<T, V>*>(from);
#pragma unroll
          for (int k = 0; k < V; ++k) q.e[k] = z.e[k];
        } else {
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (c + k < D) q.e[k] = from[k];
        }
      }
      v[n] = q;
    }
  }
  __device__ __forceinline__ void store(T* tile) const {
    constexpr int LD = DP + 16 / (int)sizeof(T);
#pragma unroll
    for (int n = 0; n < COUNT; ++n) {
      const int p = threadIdx.x + n * THREADS, r = p / PER, c = p % PER * V;
      *reinterpret_cast<Pack<T, V>*>(tile + r * LD + c) = v[n];
    }
  }
};

// The chunk's exponents, by one wave: a lane's gap is that of its row.  Returns E.
template <bool REV, typename LDS>
__device__ __forceinline__ double exponents(LDS& s, float gap, float rate, int len, float xs, float us) {
  const int lane = threadIdx.x & (kWave - 1);
  double z = (double)rate * (double)gap * 1.4426950408889634;
  if (z > kForgotten) z = kForgotten;                       // a NaN stays
  if (lane >= len) z = 0;
  double sum = z;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const double o = __shfl_up(sum, d, kWave);
    if (lane >= d) sum += o;
  }
  const double total = __shfl(sum, kWave - 1, kWave);
  const double e = REV ? sum - z : sum;
  s.e[lane] = e;
  s.xe[lane] = xs * exp2f((float)-e);
  s.we[lane] = us * exp2f((float)(e - total));
  if (lane == 0) s.fade = fade_of((float)(total * 0.6931471805599453));
  return total;
}

// M += us sum_j e^{-(E - E_j)} Y_j W_j^T over the chunk; the wave holds the columns (W channels) of its CT tiles.
template <typename T, int DP, int NW, int CT, typename LDS>
__device__ __forceinline__ void add_chunk(LDS& s, F4 (&M)[CT][DP / 16], int c0, const Frag<T> (&wf)[CT][2]) {
  constexpr int LD = LDS::LD, DT = DP / 16, NS = pieces<T>(3);
  const int g = (threadIdx.x & (kWave - 1)) >> 4;
  float wv[CT][2][8];
  float top = 0.f;
#pragma unroll
  for (int kb = 0; kb < 2; ++kb)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float we = s.we[kb * 32 + (k >> 2) * 16 + g * 4 + (k & 3)];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        wv[ct][kb][k] = we * (float)wf[ct][kb][k];
        top = finite_top(top, wv[ct][kb][k]);
      }
    }
  const float up = fit<T>(top), down = 1.f / up;
  Frag<T> b[CT][2][NS];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      if constexpr (std::is_same<T, f16_t>::value)
#pragma unroll
        for (int k = 0; k < 8; ++k) wv[ct][kb][k] *= up;
      split<T, NS>(wv[ct][kb], b[ct][kb]);
    }
  const Fade fade = s.fade;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    F4 u[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        M[ct][dt][r] = fade(M[ct][dt][r]);
        u[ct][r] = 0.f;
      }
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const Frag<T> a = frag_col<T, LD>(s.y, dt * 16, kb);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int n = 0; n < NS; ++n) u[ct] = mma(a, b[ct][kb][n], u[ct]);
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int r = 0; r < 4; ++r) M[ct][dt][r] = fmaf(u[ct][r], down, M[ct][dt][r]);
  }
}

// The lane's elements of a state (D x D at p, rows Y channels, or columns where FLIP), zeros past D.
template <int DP, int CT, bool FLIP>
__device__ __forceinline__ void load_state(const float* p, int D, int c0, F4 (&M)[CT][DP / 16]) {
  const int l = threadIdx.x & (kWave - 1), g = l >> 4, i = l & 15;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int y = dt * 16 + g * 4 + r, w = c0 + ct * 16 + i;
        M[ct][dt][r] = p && y < D && w < D ? p[FLIP ? w * D + y : y * D + w] : 0.f;
      }
}
template <int DP, int CT>
__device__ __forceinline__ void store_state(float* p, int D, int c0, const F4 (&M)[CT][DP / 16]) {
  const int l = threadIdx.x & (kWave - 1), g = l >> 4, i = l & 15;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int y = dt * 16 + g * 4 + r, w = c0 + ct * 16 + i;
        if (y < D && w < D) p[y * D + w] = M[ct][dt][r];
      }
}

struct Sweep {
  Rows x, y, w;
  void* out;                               // (N, H, D)
  const float *carry, *given;              // states after stretches (entries, H, D, D); before the windows (B, H, D, D) or null
  float* end;                              // behind the windows (B, H, D, D), or null
  float ps, xs, us;
};

template <typename T, int DP, int NW, bool REV, bool FLIP, bool WHOLE>
__global__ void __launch_bounds__(NW* kWave) k_decay_sweep(DecayGeo d, Sweep a, int64_t first) {
  using LDS = SweepLds<T, DP, NW>;
  constexpr int LD = LDS::LD, LP = LDS::LP, DT = DP / 16, CT = DT / NW > 0 ? DT / NW : 1, KD = DP / 32;
  constexpr int NS = pieces<T>(2);         // the state within 2^-17 of its values: far below the outputs' own rounding
  __shared__ LDS s;
  const int64_t work = near_first(first + blockIdx.x, d.slots * d.H);
  if (work >= d.slots * d.H) return;
  const int64_t slot = work / d.H;
  const int head = (int)(work - slot * d.H);
  const Stretch st = stretch_of(d, slot);
  if (!st.live) return;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1), g = lane >> 4, i16 = lane & 15;
  const int c0 = wave * CT * 16;
  T* out = (T*)a.out;
  if (st.window < 0 || st.window >= d.B) {                  // tokens of no window
    for (int64_t t = st.lo + wave; t < st.hi; t += NW)
      for (int c = lane; c < d.D; c += kWave) out[(t * d.H + head) * d.D + c] = (T)0.f;
    return;
  }
  const bool begins = REV ? st.last : st.first, ends = REV ? st.first : st.last;
  const int64_t DD = (int64_t)d.D * d.D;
  F4 M[CT][DT];
  load_state<DP, CT, FLIP>(begins ? (a.given ? a.given + (st.window * d.H + head) * DD : nullptr)
                                  : a.carry + ((st.entry + (REV ? 1 : -1)) * d.H + head) * DD,
                           d.D, c0, M);
  const float rate = d.rate[head];
  Stage<T, DP, NW> rx, ry, rw;
  float gap = 1.f;
  auto fetch = [&](int64_t done) {
    const int len = (int)min((int64_t)kChunk, st.hi - st.lo - done);
    const int64_t at = REV ? st.hi - 1 - done : st.lo + done;
    rx.template load<REV, WHOLE>(a.x, head, at, len, d.D);
    ry.template load<REV, WHOLE>(a.y, head, at, len, d.D);
    rw.template load<REV, WHOLE>(a.w, head, at, len, d.D);
    if (d.dt && wave == 0) gap = lane < len ? d.dt[REV ? at - lane : at + lane] : 0.f;
  };
  const int64_t tokens = st.hi - st.lo;
  if (tokens > 0) fetch(0);
  for (int64_t done = 0; done < tokens; done += kChunk) {
    const int len = (int)min((int64_t)kChunk, tokens - done);
    const int64_t at = REV ? st.hi - 1 - done : st.lo + done;
    __syncthreads();
    rx.store(s.x);
    ry.store(s.y);
    rw.store(s.w);
    if (wave == 0) exponents<REV>(s, gap, rate, len, a.xs, a.us);
    __syncthreads();
    if (done + kChunk < tokens) fetch(done + kChunk);

    // Pairs: blocks of 16 rows i by 32 rows j, six that reach below the diagonal, dealt out over the waves.  The product is
    // taken as Y X^T, so a lane holds four neighbouring j of its i.
#pragma unroll
    for (int u = 0; u < 6; ++u) {
      if (u % NW != wave) continue;
      constexpr int kIt[6] = {1, 2, 3, 3, 0, 2}, kKb[6] = {0, 0, 0, 1, 0, 1};
      const int it = kIt[u], kb = kKb[u], i = it * 16 + i16;
      float v[2][4];
      float top = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int jt = kb * 2 + t;
        F4 acc = {0.f, 0.f, 0.f, 0.f};
        if (jt <= it)
#pragma unroll
          for (int k = 0; k < KD; ++k)
            acc = mma(frag_row<T, LD>(s.y, jt * 16 + i16, k), frag_row<T, LD>(s.x, i, k), acc);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = jt * 16 + g * 4 + r;
          v[t][r] = j <= i ? acc[r] * a.ps * __builtin_amdgcn_exp2f((float)(s.e[j] - s.e[i])) : 0.f;
          top = finite_top(top, v[t][r]);
        }
      }
      const float up = fit<T>(top);
      if (std::is_same<T, f16_t>::value && lane == 0) s.pscale[it][kb] = 1.f / up;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        Pack<T, 4> q;
#pragma unroll
        for (int r = 0; r < 4; ++r) q.e[r] = (T)(v[t][r] * up);
        *reinterpret_cast<Pack<T, 4>*>(s.p + i * LP + (kb * 2 + t) * 16 + g * 4) = q;
      }
    }
    Frag<T> wf[CT][2];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) wf[ct][kb] = frag_col<T, LD>(s.w, c0 + ct * 16, kb);
    // The state as an operand.
    Frag<T> sf[CT][KD][NS];
    float top = 0.f;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = finite_top(top, M[ct][dt][r]);
    const float up = fit<T>(top), down = 1.f / up;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = M[ct][k * 2 + (e >> 2)][e & 3] * up;
        split<T, NS>(v, sf[ct][k]);
      }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      if (it * 16 >= len) continue;
      const int i = it * 16 + i16;
      Frag<T> xf[KD], pf[2];
#pragma unroll
      for (int k = 0; k < KD; ++k) xf[k] = frag_row<T, LD>(s.x, i, k);
#pragma unroll
      for (int kb = 0; kb <= it / 2; ++kb) pf[kb] = frag_row<T, LP>(s.p, i, kb);
      const float xe = s.xe[i] * down;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        auto pairs = [&](const Frag<T>(&w)[2]) {
          F4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kb = 0; kb <= it / 2; ++kb) {
            if constexpr (std::is_same<T, f16_t>::value) {
              const F4 z = mma(w[kb], pf[kb], F4{0.f, 0.f, 0.f, 0.f});
              const float ds = s.pscale[it][kb];
#pragma unroll
              for (int r = 0; r < 4; ++r) sum[r] = fmaf(z[r], ds, sum[r]);
            } else {
              sum = mma(w[kb], pf[kb], sum);
            }
          }
          return sum;
        };
        F4 pv = pairs(wf[ct]);
        // Rows past i have weight zero, and zero times an infinity or NaN would be a NaN: where one shows, the product is
        // taken without them, and those of the rows up to i are added.
        if (__any(!(fabsf((pv[0] + pv[1]) + (pv[2] + pv[3])) < INFINITY))) {
          Frag<T> clean[2];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int k = 0; k < 8; ++k) clean[kb][k] = fabsf((float)wf[ct][kb][k]) < INFINITY ? wf[ct][kb][k] : (T)0.f;
          pv = pairs(clean);
          for (int j = 0; j <= i; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float w = (float)s.w[j * LD + c0 + ct * 16 + g * 4 + r];
              if (!(fabsf(w) < INFINITY)) pv[r] = fmaf((float)s.p[i * LP + j], w, pv[r]);
            }
        }
        F4 far = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KD; ++k)
#pragma unroll
          for (int n = 0; n < NS; ++n) far = mma(sf[ct][k][n], xf[k], far);
        if (i < len) {
          const int c = c0 + ct * 16 + g * 4;
          float o[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = fmaf(far[r], xe, pv[r]);
          T* to = out + ((REV ? at - i : at + i) * d.H + head) * d.D + c;
          if constexpr (WHOLE) {
            if (c < d.D) store_f<4>(to, o);
          } else if (c < d.D) {
            store_loose<4>(to, d.D - c, o);
          }
        }
      }
    }
    add_chunk<T, DP, NW, CT>(s, M, c0, wf);
  }
  if (ends && a.end) store_state<DP, CT>(a.end + (st.window * d.H + head) * DD, d.D, c0, M);
}

// A stretch's own sum from nothing (all but the last of a window, in the sweep's direction): carry (entries, H, D, D), and
// its exponent (entries, H).
template <typename T, int DP, int NW, bool REV, bool WHOLE>
__global__ void __launch_bounds__(NW* kWave) k_decay_local(DecayGeo d, Rows y, Rows w, float us, float* __restrict__ carry,
                                                           double* __restrict__ sums, int64_t first) {
  using LDS = LocalLds<T, DP, NW>;
  constexpr int LD = LDS::LD, DT = DP / 16, CT = DT / NW > 0 ? DT / NW : 1;
  __shared__ LDS s;
  const int64_t work = near_first(first + blockIdx.x, d.slots * d.H);
  if (work >= d.slots * d.H) return;
  const int64_t slot = work / d.H;
  const int head = (int)(work - slot * d.H);
  const Stretch st = stretch_of(d, slot);
  if (!st.live || (REV ? st.first : st.last) || st.window < 0 || st.window >= d.B) return;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1), c0 = wave * CT * 16;
  F4 M[CT][DT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) M[ct][dt] = F4{0.f, 0.f, 0.f, 0.f};
  const float rate = d.rate[head];
  Stage<T, DP, NW> ry, rw;
  float gap = 1.f;
  auto fetch = [&](int64_t done) {
    const int len = (int)min((int64_t)kChunk, st.hi - st.lo - done);
    const int64_t at = REV ? st.hi - 1 - done : st.lo + done;
    ry.template load<REV, WHOLE>(y, head, at, len, d.D);
    rw.template load<REV, WHOLE>(w, head, at, len, d.D);
    if (d.dt && wave == 0) gap = lane < len ? d.dt[REV ? at - lane : at + lane] : 0.f;
  };
  const int64_t tokens = st.hi - st.lo;
  double sum = 0;
  if (tokens > 0) fetch(0);
  for (int64_t done = 0; done < tokens; done += kChunk) {
    const int len = (int)min((int64_t)kChunk, tokens - done);
    __syncthreads();
    ry.store(s.y);
    rw.store(s.w);
    if (wave == 0) sum += exponents<REV>(s, gap, rate, len, 1.f, us);
    __syncthreads();
    if (done + kChunk < tokens) fetch(done + kChunk);
    Frag<T> wf[CT][2];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) wf[ct][kb] = frag_col<T, LD>(s.w, c0 + ct * 16, kb);
    add_chunk<T, DP, NW, CT>(s, M, c0, wf);
  }
  store_state<DP, CT>(carry + (st.entry * d.H + head) * (int64_t)d.D * d.D, d.D, c0, M);
  if (threadIdx.x == 0) sums[st.entry * d.H + head] = sum;
}

// The states after the stretches of every window (all but its last) from the stretches' own sums, in place: a thread an
// element.
template <bool REV>
__global__ void __launch_bounds__(kBlock) k_decay_join(DecayGeo d, const float* __restrict__ given, float* __restrict__ carry,
                                                       const double* __restrict__ sums, int64_t first) {
  const int64_t DD = (int64_t)d.D * d.D, per = (DD + kBlock - 1) / kBlock;
  const int64_t block = first + blockIdx.x, bh = block / per;
  const int64_t el = (block - bh * per) * kBlock + threadIdx.x;
  const int64_t b = bh / d.H;
  const int head = (int)(bh - b * d.H);
  const int64_t lo = edge_of(d, b + 1), hi = max(lo, edge_of(d, b + 2));
  const int64_t n = (hi - lo + d.L - 1) / d.L;
  if (n < 2 || el >= DD) return;
  float run = given ? given[bh * DD + el] : 0.f;
  const int64_t at0 = lo / d.L + (REV ? n - 1 : 0), dir = REV ? -1 : 1;
  float* p = carry + (at0 * d.H + head) * DD + el;
  const double* z = sums + at0 * d.H + head;
  const int64_t step = dir * d.H * DD, zstep = dir * d.H;
  constexpr int kAhead = 8;
  for (int64_t k = 0; k < n - 1; k += kAhead) {
    float u[kAhead], f[kAhead];
#pragma unroll
    for (int m = 0; m < kAhead; ++m) {
      const bool on = k + m < n - 1;
      u[m] = on ? p[(k + m) * step] : 0.f;
      f[m] = on ? (float)(z[(k + m) * zstep] * 0.6931471805599453) : 0.f;
    }
#pragma unroll
    for (int m = 0; m < kAhead; ++m) {
      run = fade_of(f[m])(run) + u[m];
      if (k + m < n - 1) p[(k + m) * step] = run;
    }
  }
}

// One token of every stream: M = e^{-z} M + k v^T in place, y = scale q M.  A wave a stream's head: lanes side by side along
// the rows of M, 16 bytes each where they are aligned; bound by reading and writing the states.
template <typename T, int V>
__global__ void __launch_bounds__(kBlock) k_decay_step(Rows q, Rows k, Rows v, const float* __restrict__ rate,
                                                       const float* __restrict__ dt, int64_t N, int H, int D, int cl2, float scale,
                                                       float* __restrict__ state, T* __restrict__ y, int64_t first) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t nh = (first + blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave;
  if (nh >= N * H) return;
  const int64_t n = nh / H;
  const int h = (int)(nh - n * H);
  const Fade fade = fade_of(rate[h] * (dt ? dt[n] : 1.f));
  const T* qp = (const T*)q.p + n * q.sn + h * q.sh;
  const T* kp = (const T*)k.p + n * k.sn + h * k.sh;
  const T* vp = (const T*)v.p + n * v.sn + h * v.sh;
  float* M = state + nh * D * D;
  const int rows = kWave >> cl2, row = lane >> cl2;
  for (int c = (lane & ((1 << cl2) - 1)) * V; c - (lane & ((1 << cl2) - 1)) * V < D; c += V << cl2) {
    const bool in = c < D;
    float vv[V], acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) vv[e] = in ? (float)vp[c + e] : 0.f, acc[e] = 0.f;
#pragma unroll 8
    for (int r = row; r < D; r += rows) {
      if (!in) continue;
      float m[V];
      load_f<V>(M + r * D + c, m);
      const float kr = (float)kp[r], qr = (float)qp[r];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        m[e] = fmaf(kr, vv[e], fade(m[e]));
        acc[e] = fmaf(qr, m[e], acc[e]);
      }
      store_f<V>(M + r * D + c, m);
    }
    for (int s = 1 << cl2; s < kWave; s <<= 1)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += __shfl_xor(acc[e], s, kWave);
    if (row == 0 && in)
#pragma unroll
      for (int e = 0; e < V; ++e) y[nh * D + c + e] = (T)(acc[e] * scale);
  }
}

// ------------------------------------------------------------------------------------------- host
// Tokens of a stretch: as many workgroups as the card holds at a time (four to a compute unit), whole chunks, four at least.
int64_t stretch_len(int64_t N, int64_t H) {
  const int64_t chunks = (N * H / 1024 + kChunk - 1) / kChunk;
  return kChunk * std::min<int64_t>(std::max<int64_t>(chunks, 4), 512);
}

bool decay_ok(int dtype, int64_t N, int64_t B, int64_t H, int64_t D) {
  return dtype_ok(dtype) && N >= 0 && B >= 0 && H >= 1 && D >= 1 && D <= kMaxHead && N < ((int64_t)1 << 40) &&
         B < ((int64_t)1 << 31) && H <= 65536 && N * H < ((int64_t)1 << 46);
}

int64_t decay_entries(int64_t N, int64_t H) { return N / stretch_len(N, H) + 1; }
int64_t decay_sums_bytes(int64_t N, int64_t H) { return (decay_entries(N, H) * H * 8 + 255) / 256 * 256; }

template <typename F>
void by_head(int dtype, int64_t D, F&& f) {
  auto width = [&](auto t) {
    using std::integral_constant;
    constexpr bool wide = sizeof(t) == 4;
    if (D <= 32) f(t, integral_constant<int, 32>{}, integral_constant<int, 2>{});
    else if (D <= 64) f(t, integral_constant<int, 64>{}, integral_constant<int, 4>{});
    else f(t, integral_constant<int, 128>{}, integral_constant<int, wide ? 8 : 4>{});
  };
  if (dtype == kF32) width(float{});
  else if (dtype == kBF16) width(bf16_t{});
  else width(f16_t{});
}

bool rows_whole(const Rows& r, int dtype, int64_t D) {
  const int v = 16 / dtype_size(dtype);
  return D % v == 0 && r.sn % v == 0 && r.sh % v == 0 && aligned_to(r.p, 16);
}

template <bool REV>
void decay_states(const DecayGeo& d, int dtype, const Rows& y, const Rows& w, float us, const float* given, void* ws, float* carry,
                  hipStream_t stream) {
  if (d.N <= d.L) return;                                  // every window is one stretch at most
  const bool whole = rows_whole(y, dtype, d.D) && rows_whole(w, dtype, d.D);
  const int64_t blocks = (d.slots * d.H + 7) / 8 * 8;
  by_head(dtype, d.D, [&](auto t, auto dp, auto nw) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value, NW = decltype(nw)::value;
    in_launches(blocks, [&](int64_t first, unsigned count) {
      if (whole)
        hipLaunchKernelGGL((k_decay_local<T, DP, NW, REV, true>), dim3(count), dim3(NW * kWave), 0, stream, d, y, w, us, carry,
                           (double*)ws, first);
      else
        hipLaunchKernelGGL((k_decay_local<T, DP, NW, REV, false>), dim3(count), dim3(NW * kWave), 0, stream, d, y, w, us, carry,
                           (double*)ws, first);
    });
  });
  const int64_t per = ((int64_t)d.D * d.D + kBlock - 1) / kBlock;
  in_launches(d.B * d.H * per, [&](int64_t first, unsigned count) {
    hipLaunchKernelGGL((k_decay_join<REV>), dim3(count), dim3(kBlock), 0, stream, d, given, carry, (const double*)ws, first);
  });
}

template <bool REV, bool FLIP>
void decay_sweep(const DecayGeo& d, int dtype, const Sweep& a, hipStream_t stream) {
  const bool whole = rows_whole(a.x, dtype, d.D) && rows_whole(a.y, dtype, d.D) && rows_whole(a.w, dtype, d.D) &&
                     aligned_to(a.out, 16);
  const int64_t blocks = (d.slots * d.H + 7) / 8 * 8;
  by_head(dtype, d.D, [&](auto t, auto dp, auto nw) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value, NW = decltype(nw)::value;
    in_launches(blocks, [&](int64_t first, unsigned count) {
      if (whole)
        hipLaunchKernelGGL((k_decay_sweep<T, DP, NW, REV, FLIP, true>), dim3(count), dim3(NW * kWave), 0, stream, d, a, first);
      else
        hipLaunchKernelGGL((k_decay_sweep<T, DP, NW, REV, FLIP, false>), dim3(count), dim3(NW * kWave), 0, stream, d, a, first);
    });
  });
}

DecayGeo decay_geo(int64_t N, int64_t B, int64_t H, int64_t D, const int64_t* start, const float* dt, const float* rate) {
  DecayGeo d{};
  d.start = start; d.dt = dt; d.rate = rate;
  d.N = N; d.B = B; d.L = stretch_len(N, H);
  d.slots = N / d.L + B + 2;
  d.H = (int)H; d.D = (int)D;
  return d;
}

}  // namespace
}  // namespace atlhip

using namespace atlhip;

extern "C" {

int64_t atl_decay_attn_states(int64_t N, int64_t H, int64_t D) {
  if (!decay_ok(kF32, N, 0, H, D)) return -1;
  return N <= stretch_len(N, H) ? 0 : decay_entries(N, H) * H * D * D;
}

int64_t atl_decay_attn_ws_bytes(int64_t N, int64_t H, int64_t D, int backward) {
  const int64_t n = atl_decay_attn_states(N, H, D);
  return n < 0 ? -1 : decay_sums_bytes(N, H) + (backward ? 4 * n : 0);
}

int atl_decay_attn_fwd(const void* q, int64_t sqn, int64_t sqh, const void* k, int64_t skn, int64_t skh, const void* v,
                       int64_t svn, int64_t svh, int dtype, int64_t N, int64_t H, int64_t D, const float* rate,
                       const int64_t* start, int64_t B, const float* dt, const float* h0, double scale, void* y, float* last,
                       float* states, void* ws, int64_t ws_bytes, hipStream_t stream) {
  if (!decay_ok(dtype, N, B, H, D) || (N > 0 && (sqn < 0 || sqh < 0 || skn < 0 || skh < 0 || svn < 0 || svh < 0))) { set_error("decay_attn_fwd: bad sizes N=%lld B=%lld H=%lld D=%lld type %d", (long long)N, (long long)B, (long long)H, (long long)D, dtype); return 1; }
  if (!start || !rate || !ws || (N > 0 && (!q || !k || !v || !y)) || (atl_decay_attn_states(N, H, D) && !states)) { set_error("decay_attn_fwd: null argument"); return 1; }
  if (ws_bytes < atl_decay_attn_ws_bytes(N, H, D, 0)) { set_error("decay_attn_fwd: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)atl_decay_attn_ws_bytes(N, H, D, 0)); return 1; }
  const DecayGeo d = decay_geo(N, B, H, D, start, dt, rate);
  const Rows rq{q, sqn, sqh}, rk{k, skn, skh}, rv{v, svn, svh};
  decay_states<false>(d, dtype, rk, rv, 1.f, h0, ws, states, stream);
  decay_sweep<false, false>(d, dtype, Sweep{rq, rk, rv, y, states, h0, last, (float)scale, (float)scale, 1.f}, stream);
  return check_launch("decay_attn_fwd");
}

int atl_decay_attn_bwd(const void* q, int64_t sqn, int64_t sqh, const void* k, int64_t skn, int64_t skh, const void* v,
                       int64_t svn, int64_t svh, const void* gy, int64_t sgn, int64_t sgh, int dtype, int64_t N, int64_t H,
                       int64_t D, const float* rate, const int64_t* start, int64_t B, const float* dt, const float* h0,
                       const float* glast, double scale, const float* states, void* gq, void* gk, void* gv, float* gh0, void* ws,
                       int64_t ws_bytes, hipStream_t stream) {
  if (!decay_ok(dtype, N, B, H, D) || (N > 0 && (sqn < 0 || sqh < 0 || skn < 0 || skh < 0 || svn < 0 || svh < 0 || sgn < 0 || sgh < 0))) { set_error("decay_attn_bwd: bad sizes N=%lld B=%lld H=%lld D=%lld type %d", (long long)N, (long long)B, (long long)H, (long long)D, dtype); return 1; }
  if (!start || !rate || !ws || (N > 0 && (!q || !k || !v || !gy || !gq || !gk || !gv)) || (atl_decay_attn_states(N, H, D) && !states)) { set_error("decay_attn_bwd: null argument"); return 1; }
  if (ws_bytes < atl_decay_attn_ws_bytes(N, H, D, 1)) { set_error("decay_attn_bwd: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)atl_decay_attn_ws_bytes(N, H, D, 1)); return 1; }
  const DecayGeo d = decay_geo(N, B, H, D, start, dt, rate);
  const Rows rq{q, sqn, sqh}, rk{k, skn, skh}, rv{v, svn, svh}, rg{gy, sgn, sgh};
  const float sc = (float)scale;
  float* carry = (float*)((char*)ws + decay_sums_bytes(N, H));
  decay_states<true>(d, dtype, rq, rg, sc, glast, ws, carry, stream);
  decay_sweep<false, true>(d, dtype, Sweep{rg, rv, rk, gq, states, h0, nullptr, sc, sc, 1.f}, stream);
  decay_sweep<true, false>(d, dtype, Sweep{rk, rq, rg, gv, carry, glast, gh0, sc, 1.f, sc}, stream);
  decay_sweep<true, true>(d, dtype, Sweep{rv, rg, rq, gk, carry, glast, nullptr, sc, 1.f, sc}, stream);
  return check_launch("decay_attn_bwd");
}

int atl_decay_attn_step(const void* q, int64_t sqn, int64_t sqh, const void* k, int64_t skn, int64_t skh, const void* v,
                        int64_t svn, int64_t svh, int dtype, int64_t N, int64_t H, int64_t D, const float* rate, const float* dt,
                        double scale, float* state, void* y, hipStream_t stream) {
  if (!decay_ok(dtype, N, 0, H, D) || (N > 0 && (sqn < 0 || sqh < 0 || skn < 0 || skh < 0 || svn < 0 || svh < 0))) { set_error("decay_attn_step: bad sizes N=%lld H=%lld D=%lld type %d", (long long)N, (long long)H, (long long)D, dtype); return 1; }
  if (N == 0) return 0;
  if (!q || !k || !v || !rate || !state || !y) { set_error("decay_attn_step: null argument"); return 1; }
  const bool vec = D % 4 == 0 && aligned_to(state, 16);
  const int64_t units = vec ? D / 4 : D;
  int cl2 = 0;
  while ((1 << cl2) < kWave && (1 << cl2) < units) ++cl2;
  const Rows rq{q, sqn, sqh}, rk{k, skn, skh}, rv{v, svn, svh};
  auto go = [&](auto t) {
    using T = decltype(t);
    in_launches(grid_for(N * H, kBlock / kWave), [&](int64_t first, unsigned count) {
      if (vec)
        hipLaunchKernelGGL((k_decay_step<T, 4>), dim3(count), dim3(kBlock), 0, stream, rq, rk, rv, rate, dt, N, (int)H, (int)D, cl2,
                           (float)scale, state, (T*)y, first);
      else
        hipLaunchKernelGGL((k_decay_step<T, 1>), dim3(count), dim3(kBlock), 0, stream, rq, rk, rv, rate, dt, N, (int)H, (int)D, cl2,
                           (float)scale, state, (T*)y, first);
    });
  };
  if (dtype == kF32) go(float{});
  else if (dtype == kBF16) go(bf16_t{});
  else go(f16_t{});
  return check_launch("decay_attn_step");
}

}  // extern "C"
