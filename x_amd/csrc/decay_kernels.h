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
// for a chunk of 32 rows, with E_i the decay from the chunk's begin to row i: up to the row's own gap forward, up to the gap
// before it from the end (a token's gap lies before it).  The products run on the matrix cores.  Decays stay exponents, in
// 64 bits within a chunk, and a factor of the state near one is applied as M + M expm1(-E): a product of many factors just
// below one would lose what each rounds off.  Exponents past 400 (in powers of two: the factor is zero in 32 bits) count as 400,
// so an endless gap forgets what was before it and no difference of infinities appears.
//
// A window is cut into stretches of L tokens; a workgroup follows one stretch of one head.  The state before a stretch comes
// from a pass that sums every stretch but the last on its own (k_decay_local) and one that joins them (k_decay_join); windows
// of one stretch need neither, and both return at once there.  Training so moves 18 tensors' worth of rows where 8 would do, each once
// (forward 2 + 4, backward 2 + 4 + 6; 17 with heads of 32 channels, where the backward pass's own sums share a sweep).  What
// bounds it: heads of 32 channels, memory (1M tokens x 2 x 32 in bfloat16: the sweeps move 3.7 to 4.1 TB/s, forward and backward
// take 605 us); wider ones the vector instructions around the products and their latency at two waves a SIMD, whose
// registers hold the states (65k x 8 x 128: a forward sweep takes 215 to 228 us; its vector instructions' issue is 78, its matrix
// instructions' 43 and its traffic at a copy's rate 105); single precision its matrix instructions (251k x 3 x 45: 1140 us).
#pragma once
#include "decay.h"

#include <algorithm>
#include <type_traits>

namespace atlhip {
namespace {

constexpr int kChunk = 32;                 // rows of a chunk: what one step of a matrix instruction sums

constexpr double kForgotten = 400.0;       // exponents (of two) from which a factor is zero

using F4 = float __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------------- fragments
// Eight elements a lane of a 16 x 32 operand of a matrix product: lane l holds index l % 16 of the operand's outer axis, and a
// fourth of the axis that is summed over, in any order that both operands have.  A product's result has its outer axes at
// (4 (l / 16) + r, l % 16), r < 4.  Two orders make results the next product's operands as they lie in their lanes:
//
//   rows (tokens) are summed in the order t 16 + 4 (l / 16) + r, t < 2, of two results' blocks of 16;
//   channels are summed in their order, 8 (l / 16) + 4 t + r, and a state's blocks hold the channels that this asks for:
//   block 2 k + t at 32 k + 8 (m / 4) + 4 t + m % 4, m < 16.
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

// Row `row` of a tile (the lane's own), channels 32 kb to 32 kb + 31.
template <typename T, int LD>
__device__ __forceinline__ Frag<T> frag_row(const T* tile, int row, int kb) {
  const int g = (threadIdx.x & (kWave - 1)) >> 4;
  union { Pack<T, 16 / sizeof(T)> p[sizeof(T) / 2]; Frag<T> f; } u;
#pragma unroll
  for (int k = 0; k < (int)sizeof(T) / 2; ++k) u.p[k] = load_pack<T, 16 / sizeof(T)>(tile + row * LD + kb * 32 + g * 8 + k * 4);
  return u.f;
}

// A channel of a chunk's rows: col0 + l % 16, or where STATE the l % 16-th of a state's block col0 / 16.
template <typename T, int LD, bool STATE>
__device__ __forceinline__ Frag<T> frag_col(const T* tile, int col0) {
  const int l = threadIdx.x & (kWave - 1), g = l >> 4, i = l & 15;
  const int base = STATE ? col0 / 32 * 32 + (col0 / 16 & 1) * 4 : col0, four = STATE ? 8 : 4;
  Frag<T> f;
  if constexpr (sizeof(T) == 2) {
    // The transposed read: 16 lanes name four rows of four times four elements, and each gets a column of four.
    using S4 = short __attribute__((ext_vector_type(4)));
    using LdsS4 = __attribute__((address_space(3))) S4;
    union { S4 s[2]; Frag<T> f; } u;
    const T* p = tile + (g * 4 + (i >> 2)) * LD + base + (i & 3) * four;
    u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4*)p);
    u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4*)(p + 16 * LD));
    f = u.f;
  } else {
    const T* p = tile + g * 4 * LD + base + (i >> 2) * four + (i & 3);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = p[((k >> 2) * 16 + (k & 3)) * LD];
  }
  return f;
}

// Values in 32 bits as the sum of NS fragments of T, each piece the rounded rest of those before: three hold a value's 24 bits, two
// the value within 2^-17 (bfloat16) or 2^-22 (half precision), a 256th of the output's own rounding or less.  The weights of
// tokens in a state go in as three, since states are kept and handed on; the states and pairs' weights that meet a row's
// output as two.  Three there take 2% more of the time at 32 channels, 7% at 64 and 10% at 128 (forward + backward: 1M x 2 x 32
// 605 -> 619 us, 256 windows of 400 x 4 x 64 366 -> 397, 65k x 8 x 128 962 -> 1057); bfloat16 outputs are then 3.8e-5 instead of
// 9.5e-5 from those of a plain form in single precision, and either way 1.66e-3 from the values before they are rounded,
// as the plain form's own are.
template <typename T, int NS>
__device__ __forceinline__ void split(const float (&v)[8], Frag<T> (&f)[NS]) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[0][k] = v[k];
  } else if constexpr (std::is_same<T, bf16_t>::value) {     // two values an instruction, there and back
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = v[k];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      union { uint32_t w[4]; Frag<T> f; } u;
#pragma unroll
      for (int k = 0; k < 8; ++k) u.f[k] = (T)x[k];
      f[s] = u.f;
      if (s + 1 < NS)
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] -= __uint_as_float(k & 1 ? u.w[k / 2] & 0xFFFF0000u : u.w[k / 2] << 16);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float x = v[k];
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        f[s][k] = (T)x;
        x -= (float)f[s][k];
      }
    }
  }
}
template <typename T>
constexpr int pieces(int n) {
  return std::is_same<T, float>::value ? 1 : n;
}

// Half precision reaches from 6e-8 to 65504 only: what goes into it is brought to a largest value of 2^14 to 2^15 first, by
// a power of two: a state column by column, pairs' weights row by row, weighted W column by column.  What lies 2^28 below the
// largest of its column or row keeps fewer bits than the type's own.
struct Fit {
  float up, down;
};
__device__ __forceinline__ float finite_top(float top, float v) { return fabsf(v) < INFINITY ? fmaxf(top, fabsf(v)) : top; }
__device__ __forceinline__ Fit fit_of(float top) {
  const uint32_t e = max(__float_as_uint(top) >> 23, 15u);
  return Fit{__uint_as_float((268u - e) << 23), __uint_as_float((e - 14u) << 23)};
}
// Of the lanes l % 16 alike.
__device__ __forceinline__ float top_of_four(float top) {
  top = fmaxf(top, __shfl_xor(top, 16, kWave));
  return fmaxf(top, __shfl_xor(top, 32, kWave));
}

// A state's factor e^{-z}: for small z by what it is less than one (else that would lose the factor's own bits).
struct Fade {
  float a, keep;                           // m e^{-z} + u = m a + (m keep + u), keep 0 or 1
  __device__ __forceinline__ float operator()(float m, float u) const { return fmaf(m, a, fmaf(m, keep, u)); }
  // Of an infinite m too, of which the two parts would make a NaN.
  __device__ __forceinline__ float any(float m, float u) const { return fabsf(m) < INFINITY ? (*this)(m, u) : fmaf(m, a + keep, u); }
};
__device__ __forceinline__ Fade fade_of(float z) {
  const bool keep = !(z > 0.5f);
  return Fade{keep ? expm1f(-z) : expf(-z), keep ? 1.f : 0.f};
}

// A stretch's exponent (of two) and factor.
struct Span {
  double z;
  Fade fade;
};
// Stretches of a window up to which a sweep adds up their sums by itself: it reads half of them on average, and the join is
// spared.  The sums that the sweeps read grow with the square of a window's stretches: up to 10 instead of 6 took 402 -> 441 us
// (forward + backward of 60k tokens in 40 windows x 8 x 64), up to 16 took 512; up to 4 changed nothing by more than 2%.
constexpr int kFew = 6;

// ------------------------------------------------------------------------------------------- windows
// Stretch of a slot.  Windows are numbered with the tokens before the first (window -1) and behind the last (window B), which
// are in none; window b begins at slot floor(first token / L) + b + 1, so every window has as many slots as stretches or
// more, and no sum over the windows is needed.
struct Stretch {
  int64_t window, lo, hi;                  // tokens of the stretch
  bool first, last, live;                  // of its window; live: there is one
  int64_t entry;                           // of the states after stretches: unlike for all but windows' last stretches
  int64_t index, count;                    // of the window's stretches
};

__device__ __forceinline__ int64_t edge_of(const DecayGeo& d, int64_t e) {     // first token of window e - 1
  if (e <= 0) return 0;
  if (e > d.B + 1) return d.N;
  const int64_t s = d.start[e - 1];
  return s < 0 ? 0 : s > d.N ? d.N : s;
}

// The last of 0..n-1 that holds `at` (which holds for the first ones only, 0 among them).  Every lane of a wave calls it: 64
// are looked at in one step.
template <typename F>
__device__ __forceinline__ int64_t last_of(int64_t n, F&& at) {
  const int lane = threadIdx.x & (kWave - 1);
  int64_t lo = 0;
  while (n > 1) {
    const int64_t step = (n + kWave - 1) / kWave;
    const int c = __popcll(__ballot(lane * step < n && at(lo + lane * step)));
    const int64_t k = c > 0 ? c - 1 : 0;
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}

__device__ __forceinline__ Stretch stretch_of(const DecayGeo& d, int64_t slot) {
  const int64_t lo = last_of(d.B + 2, [&](int64_t e) { return edge_of(d, e) / d.L + e <= slot; });
  Stretch s;
  const int64_t begin = edge_of(d, lo), end = max(begin, edge_of(d, lo + 1));
  const int64_t k = slot - (begin / d.L + lo);
  s.window = lo - 1;
  s.entry = begin / d.L + k;
  s.index = k;
  s.count = (end - begin + d.L - 1) / d.L;
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

// ------------------------------------------------------------------------------------------- a chunk
template <typename T, int DP>
constexpr int tile_ld() { return DP + 16 / (int)sizeof(T); }                // rows a vector apart (bank conflicts: 32 to 54% of LDS cycles)

// The exponents E_i of a chunk (in powers of two) and the factors made of them.  A pair's factor e^{-(E_i - E_j)} is taken from
// the exponents inside a block of 16 rows, and between the two blocks as row_i col_j, from and to the first block's last
// row: a product instead of an exponential.
struct Decays {
  double e[kChunk];
  float row[kChunk], col[kChunk];                           // ps e^{-..}, e^{-..}
  float xe[kChunk], we[kChunk];                             // xs e^{-E_i}, us e^{-(E - E_i)}
  Fade fade;                                                // e^{-E}
  double total;                                             // E
};

template <int CTRL>
__device__ __forceinline__ double dppd(double v) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xF, 0xF, true);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xF, 0xF, true);
  return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double lane_of(double v, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}

// Those of two chunks, by one wave: a lane's gap is that of its row.  Returns E over both.
template <bool REV>
__device__ __forceinline__ double exponents(Decays (&two)[2], float gap, float rate, int len, float ps, float xs, float us) {
  const int lane = threadIdx.x & (kWave - 1), block = lane >> 4;
  double z = (double)rate * (double)gap * 1.4426950408889634;
  if (z > kForgotten) z = kForgotten;                       // a NaN stays
  if (lane >= len) z = 0;
  double sum = z;                                           // within the block of 16, then within the chunk
  sum += dppd<0x111>(sum);
  sum += dppd<0x112>(sum);
  sum += dppd<0x114>(sum);
  sum += dppd<0x118>(sum);
  const double a = lane_of(sum, 15), b = a + lane_of(sum, 31), c = lane_of(sum, 47), d = c + lane_of(sum, 63);
  const double half = block < 2 ? a : c, total = block < 2 ? b : d;
  if (block & 1) sum += half;
  const double e = REV ? sum - z : sum;
  Decays& s = two[block >> 1];
  const int i = lane & (kChunk - 1);
  s.e[i] = e;
  s.row[i] = ps * exp2f((float)(half - e));
  s.col[i] = exp2f((float)(e - half));
  s.xe[i] = xs * exp2f((float)-e);
  s.we[i] = us * exp2f((float)(e - total));
  if (i == 0) {
    s.fade = fade_of((float)(total * 0.6931471805599453));
    s.total = total;
  }
  return b + d;
}

// A chunk's rows as a buffer: its lowest token at p, row r at offset r stride (or (len - 1 - r) stride where REV), so that a row
// that is not there, and a channel past D (kNoChannel), lie outside, where loads give zeros and stores do nothing.  Strides
// are below 2^22 elements, so 32 rows are 2^29 bytes at most.
constexpr uint32_t kNoChannel = 0x80000000u;
using U4v = uint32_t __attribute__((ext_vector_type(4)));
using U2v = uint32_t __attribute__((ext_vector_type(2)));
template <bool REV>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t chunk_buffer(const void* row0, int64_t stride, int len, int width) {
  const char* p = (const char*)row0 - (REV ? (len - 1) * stride : 0);
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (len - 1) * (int)stride + width, 0x00020000);
}
template <bool REV>
__device__ __forceinline__ uint32_t row_offset(int r, int stride, int len) {
  return (uint32_t)((REV ? len - 1 - r : r) * stride);
}

// How rows lie: in pieces of 16 bytes, in words of 32 bits (16 bytes at least), or anyhow.
constexpr int kLoose = 0, kWords = 1, kWhole = 2;

// Pieces of 16 bytes of a chunk's rows, in registers until the chunk's turn.
template <typename T, int DP, int THREADS>
struct Stage {
  static constexpr int V = 16 / (int)sizeof(T), PER = DP / V, COUNT = kChunk * PER / THREADS, STEP = THREADS / PER;
  static_assert(COUNT * THREADS == kChunk * PER && STEP * PER == THREADS, "whole rounds of whole rows");
  Pack<T, V> v[COUNT];

  // Row r of the chunk is token at + r (or at - r where REV); len rows are there, the others zero.
  template <bool REV, int LAY>
  __device__ __forceinline__ void load(const Rows& rows, int64_t head, int64_t at, int len, int D) {
    const T* row0 = (const T*)rows.p + head * rows.sh + at * rows.sn;
    const int r0 = threadIdx.x / PER, c = threadIdx.x % PER * V;
    if constexpr (LAY != kLoose) {                                  // a row's last piece ends with the row, and is moved up when it is stored
      const int stride = (int)rows.sn * (int)sizeof(T);
      const auto buf = chunk_buffer<REV>(row0, stride, len, D * (int)sizeof(T));
      const uint32_t off = row_offset<REV>(r0, stride, len) + (c < D ? (LAY == kWords ? min(c, D - V) : c) * (uint32_t)sizeof(T) : kNoChannel);
#pragma unroll
      for (int n = 0; n < COUNT; ++n) {
        const U4v w = __builtin_amdgcn_raw_buffer_load_b128(buf, off + (uint32_t)((REV ? -n : n) * STEP * stride), 0, 0);
        v[n] = *reinterpret_cast<const Pack<T, V>*>(&w);
      }
    } else {
#pragma unroll
      for (int n = 0; n < COUNT; ++n) {
        const int r = r0 + n * STEP;
        Pack<T, V> q{};
        if (r < len && c < D) {
          const T* from = row0 + (REV ? -r : r) * rows.sn + c;
          if (c + V <= D) {
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
  }
  // Whether some of the lane's elements are not finite: magnitudes, as whole numbers, from the infinity's on.
  __device__ __forceinline__ bool odd() const {
    if constexpr (sizeof(T) == 2) {
      using H2 = uint16_t __attribute__((ext_vector_type(2)));
      H2 top = {0, 0};
#pragma unroll
      for (int n = 0; n < COUNT; ++n) {
        const U4v w = *reinterpret_cast<const U4v*>(&v[n]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t m = w[k] & 0x7FFF7FFFu;
          top = __builtin_elementwise_max(top, *reinterpret_cast<const H2*>(&m));
        }
      }
      return max(top[0], top[1]) >= (std::is_same<T, f16_t>::value ? 0x7C00 : 0x7F80);
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int n = 0; n < COUNT; ++n)
#pragma unroll
        for (int k = 0; k < V; ++k) top = max(top, __float_as_uint(v[n].e[k]) & 0x7FFFFFFFu);
      return top >= 0x7F800000u;
    }
  }
  template <int LAY>
  __device__ __forceinline__ void store(T* tile, int D) {
    if constexpr (LAY == kWords) {
      const int c = threadIdx.x % PER * V, by = (V - D % V) * (int)sizeof(T) / 4;
      const bool last = c < D && c + V > D;
#pragma unroll
      for (int n = 0; n < COUNT; ++n) {
        U4v w = *reinterpret_cast<U4v*>(&v[n]);
        if (by & 1) w = last ? U4v{w[1], w[2], w[3], 0} : w;
        if (by & 2) w = last ? U4v{w[2], w[3], 0, 0} : w;
        v[n] = *reinterpret_cast<Pack<T, V>*>(&w);
      }
    }
    T* to = tile + threadIdx.x / PER * tile_ld<T, DP>() + threadIdx.x % PER * V;
#pragma unroll
    for (int n = 0; n < COUNT; ++n) *reinterpret_cast<Pack<T, V>*>(to + n * STEP * tile_ld<T, DP>()) = v[n];
  }
};

// The Y channel of a lane's element r of block dt of a state.
__device__ __forceinline__ int state_row(int dt, int r) {
  return dt / 2 * 32 + ((threadIdx.x & (kWave - 1)) >> 4) * 8 + (dt & 1) * 4 + r;
}

// M = M e^{-z} + times sum_j weight_j Y_j W_j^T over the chunk; the wave holds the columns (W channels) of its CT tiles.  The
// weighted W go in as three pieces, so a state is as good as one summed in single precision; the chunk's sum is taken
// from zero and added once.
template <typename T, int DP, int CT>
__device__ __forceinline__ void add_chunk(const float* weight, Fade fade, float times, const T* y, F4 (&M)[CT][DP / 16],
                                          const Frag<T> (&wf)[CT]) {
  constexpr int LD = tile_ld<T, DP>(), DT = DP / 16, NS = pieces<T>(3);
  constexpr bool HALF = std::is_same<T, f16_t>::value;
  const int g = (threadIdx.x & (kWave - 1)) >> 4;
  const Pack<float, 4> we[2] = {load_pack<float, 4>(weight + g * 4), load_pack<float, 4>(weight + 16 + g * 4)};
  Frag<T> b[CT][NS];
  float wv[CT][8], down[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      wv[ct][k] = we[k >> 2].e[k & 3] * (float)wf[ct][k];
      if (HALF) top = finite_top(top, wv[ct][k]);
    }
    if (HALF) {
      const Fit f = fit_of(top_of_four(top));
      down[ct] = f.down;
#pragma unroll
      for (int k = 0; k < 8; ++k) wv[ct][k] *= f.up;
    }
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) split<T, NS>(wv[ct], b[ct]);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const Frag<T> a = frag_col<T, LD, true>(y, dt * 16);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      F4 u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NS; ++n) u = mma(a, b[ct][n], u);
#pragma unroll
      for (int r = 0; r < 4; ++r) M[ct][dt][r] = fade(M[ct][dt][r], HALF ? u[r] * (down[ct] * times) : u[r] * times);
    }
  }
}

// W that are not finite are left out of the products: their pieces would be NaNs, and so would weights of zero times them ...
template <typename T, int CT>
__device__ __forceinline__ void leave_out(Frag<T> (&wf)[CT]) {
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int k = 0; k < 8; ++k) wf[ct][k] = fabsf((float)wf[ct][k]) < INFINITY ? wf[ct][k] : (T)0.f;
}
// ... and what they have a part in is marked by a NaN, to be taken again by by_token: their columns of the state (and their
// rows from their own on, where those are stored).
template <typename T, int DP, int CT>
__device__ __forceinline__ void mark(const T* w, int c0, F4 (&M)[CT][DP / 16]) {
#pragma unroll 1
  for (int j = 0; j < kChunk; ++j)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const bool odd = !(fabsf((float)w[j * tile_ld<T, DP>() + c0 + ct * 16 + (threadIdx.x & 15)]) < INFINITY);
      if (!__any(odd)) continue;
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) M[ct][dt][r] = odd ? NAN : M[ct][dt][r];
    }
}

// M = e^{-z} M + the lane's elements of a state (D x D at p, rows Y channels, or columns where flip), zeros past D.
template <int DP, int CT>
__device__ __forceinline__ void add_state(const float* p, bool flip, int D, int c0, Fade fade, F4 (&M)[CT][DP / 16]) {
  const auto buf = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, D * D * 4, 0x00020000);
  const int sy = flip ? 1 : D, sw = flip ? D : 1;
  int y0 = state_row(0, 0);
  asm volatile("" : "+v"(y0));                              // (the elements' places, kept over a loop, would not fit the registers)
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int w = c0 + ct * 16 + (threadIdx.x & 15);
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int y = y0 + dt / 2 * 32 + (dt & 1) * 4 + r;
        const uint32_t off = y < D && w < D ? (uint32_t)(y * sy + w * sw) * 4 : kNoChannel;
        M[ct][dt][r] = fade.any(M[ct][dt][r], __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(buf, off, 0, 0)));
      }
  }
}
// (Where not `all`, over what is there and not finite.)
template <int DP, int CT>
__device__ __forceinline__ void store_state(float* p, int D, int c0, const F4 (&M)[CT][DP / 16], bool all) {
  const int i = threadIdx.x & 15;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int y = state_row(dt, r), w = c0 + ct * 16 + i;
        if (y < D && w < D && (all || !(fabsf(p[y * D + w]) < INFINITY))) p[y * D + w] = M[ct][dt][r];
      }
}
template <int DP, int CT>
__device__ __forceinline__ void clear_state(F4 (&M)[CT][DP / 16]) {
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) M[ct][dt] = F4{0.f, 0.f, 0.f, 0.f};
}
template <int DP, int CT>
__device__ __forceinline__ bool finite_state(const F4 (&M)[CT][DP / 16]) {
  float check = 0.f;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) check = fmaf(M[ct][dt][r], 0.f, check);
  return !__any(check != check);
}

// The recurrence as it is written, token by token in single precision, for a stretch with something in it that is not finite:
// infinities do not come through the matrix products (an infinity's second piece is Inf - Inf, and weights of zero make NaNs of
// them), nor do products past single precision on the way to a smaller result.  Only where the products left no finite result
// is one written.  kAlong and kBack: the sweeps' directions, rows from the stretch's begin or end, with the gap before a row
// taken before it or before the next; kFromEnd: the sum from the end's side, in the order of the tokens.  One wave waits for
// every token's rows, about 2.5 us: 1M tokens x 2 x 32 in bfloat16 with one infinity take 13 ms forward + backward instead of 0.6.
// What the check costs where all is finite, by the cases: 256 windows of 400 x 4 x 64 361 -> 366 us, 1M x 2 x 32 600 -> 606,
// 251k x 3 x 45 in float32 1127 -> 1146, 65k x 8 x 128 960 -> 970, 100k x 8 x 64 in float16 forward 231 -> 235.
enum Way : int { kAlong = 0, kBack = 1, kFromEnd = 2 };
template <typename T, int DP, int CT, int WAY>
__device__ __forceinline__ void by_token(const DecayGeo& d, const Stretch& st, int head, const Rows& x, const Rows& y, const Rows& w,
                                         int c0, float xs, float us, F4 (&M)[CT][DP / 16], T* out) {
  const int lane = threadIdx.x & (kWave - 1), g = lane >> 4, i16 = lane & 15;
  const float rate = d.rate[head];
  __threadfence();                                          // the results so far are read again
  Fade pending{0.f, 1.f};
  double gone = 0;
#pragma unroll 1
  for (int64_t n = st.hi - st.lo; n > 0; --n) {
    const int64_t t = WAY == kBack ? st.lo + n - 1 : st.hi - n;
    double z = (double)rate * (double)(d.dt ? d.dt[t] : 1.f) * 1.4426950408889634;
    if (z > kForgotten) z = kForgotten;                     // a NaN stays
    const Fade own = fade_of((float)(z * 0.6931471805599453));
    gone += z;
    const Fade f = WAY == kAlong ? own : pending;
    if (WAY == kBack) pending = own;
    const float weight = WAY == kFromEnd ? us * exp2f((float)-gone) : us;
    const T* yr = (const T*)y.p + t * y.sn + head * y.sh;
    const T* xr = (const T*)x.p + t * x.sn + head * x.sh;
    const T* wr = (const T*)w.p + t * w.sn + head * w.sh;
    float yv[DP / 16][4], xv[DP / 16][4], wv[CT], sum[CT];
    bool odd[CT];                                           // (read with the rows: one wait a token)
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) {
      const int row = state_row(dt, 0);
      load_loose<4>(yr + row, d.D - row, yv[dt]);
      if (out) load_loose<4>(xr + row, d.D - row, xv[dt]);
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int c = c0 + ct * 16 + i16;
      wv[ct] = c < d.D ? weight * (float)wr[c] : 0.f;
      sum[ct] = 0.f;
      odd[ct] = out && g == ct && c < d.D && !(fabsf((float)out[(t * d.H + head) * d.D + c]) < INFINITY);
    }
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (state_row(dt, r) >= d.D) continue;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          M[ct][dt][r] = f.any(M[ct][dt][r], yv[dt][r] * wv[ct]);
          if (out) sum[ct] = fmaf(xv[dt][r], M[ct][dt][r], sum[ct]);
        }
      }
    if (!out) continue;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      sum[ct] += __shfl_xor(sum[ct], 16, kWave);
      sum[ct] += __shfl_xor(sum[ct], 32, kWave);
      if (odd[ct]) out[(t * d.H + head) * d.D + c0 + ct * 16 + i16] = (T)(xs * sum[ct]);
    }
  }
  if (WAY == kBack)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) M[ct][dt][r] = pending.any(M[ct][dt][r], 0.f);
}

// ------------------------------------------------------------------------------------------- the sweep
constexpr int kLdsBytes = 160 * 1024, kSweepWaves = 2;

template <typename T, int DP, int NT>
struct ChunkLds {
  T tile[NT][kChunk * tile_ld<T, DP>()];
  Decays decay[2][2];                                       // of two chunks and of the next two
  int odd[NT];                                              // done + 1 of the last chunk in which a tile had values that are not finite
};
// Waves to a SIMD that the shared memory leaves room for.
template <typename LDS, int MOST>
constexpr int waves_of(int waves) {
  const int n = (int)(kLdsBytes / sizeof(LDS)) * waves / 4;
  return n < 1 ? 1 : n > MOST ? MOST : n;
}

// What a workgroup's waves do: one recurrence over X, Y, W (rows 0, 1, 2); or two that share their rows (q, k, v, gy: dv over
// (k, q, gy), dk over (v, gy, q)), each by its own waves; or one (dq: gy, v, k, and q) beside the stretch's own sum from its
// end, sum_i e^{-E_i} q_i gy_i^T, which those two begin with (the rows of gy are there already).  That one is for heads of one
// tile of 32 channels: forward + backward of 1M tokens x 2 x 32 took 631 us with a pass over q and gy for those sums and 599
// with them beside dq; 102k x 4 x 64 took 370 and 383, 65k x 8 x 128 1069 and 1113, 251k x 3 x 45 in float32 1191 and 1220:
// the sums' waves have a third of the others' work and hold as many registers.  (Heads of up to 32 channels in float32 and
// float16 were not measured apart.)
enum Work : int { kSweep = 0, kSweepPair = 1, kSweepAndSums = 2 };
struct Sweep {
  Rows rows[4];
  void* out[2];                            // (N, H, D)
  const float* carry;                      // sums of stretches, or in windows of more than kFew the states after them (entries, H, D, D)
  const Span* spans;                       // (entries, H)
  const float* given;                      // states before the windows (B, H, D, D), or null
  float* end;                              // behind the windows (B, H, D, D), or null (the first job's)
  int flip;                                // the states lie transposed (the first job's; the second's the other way)
  float ps, xs, us;
  float* sums;                             // the stretches' sums from their ends, and their spans (kSweepAndSums)
  Span* sum_spans;
};

constexpr int kTiles = 2;                  // blocks of 16 W channels of a wave

// Goes through a stretch's chunks: chunk(done, len, decays) with its rows and exponents in shared memory.  W_TILES: the tiles
// that are looked through for values that are not finite.
template <typename T, int DP, int NT, int W_TILES, int THREADS, bool REV, int LAY, typename Chunk>
__device__ __forceinline__ double follow(ChunkLds<T, DP, NT>& s, const DecayGeo& d, const Stretch& st, const Rows (&rows)[NT],
                                         int head, float ps, float xs, float us, Chunk&& chunk) {
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const float rate = d.rate[head];
  const int tokens = (int)(st.hi - st.lo);
  const int64_t from = REV ? st.hi - 1 : st.lo;             // the token of the stretch's first row
  Stage<T, DP, THREADS> stage[NT];
  auto fetch = [&](int done) {
    if (done >= tokens) return;
#pragma unroll
    for (int n = 0; n < NT; ++n)
      stage[n].template load<REV, LAY>(rows[n], head, REV ? from - done : from + done, min(kChunk, tokens - done), d.D);
  };
  auto put = [&](int done) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      stage[n].template store<LAY>(s.tile[n], d.D);
      if ((W_TILES >> n & 1) && __any(stage[n].odd()) && lane == 0) s.odd[n] = done + 1;
    }
  };
  // The last wave makes the exponents, two chunks at a time and two ahead.
  const bool decays = wave == THREADS / kWave - 1;
  double sum = 0;
  auto gap_of = [&](int done) {
    return d.dt && done + lane < tokens ? d.dt[REV ? from - done - lane : from + done + lane] : 1.f;
  };
  auto make = [&](int done, float gap) {
    sum += exponents<REV>(s.decay[done / kWave & 1], gap, rate, tokens - done, ps, xs, us);
  };
  float gap = 1.f;
  fetch(0);
  if (decays && tokens > 0) {
    make(0, gap_of(0));
    gap = gap_of(kWave);
  }
  if (threadIdx.x < NT) s.odd[threadIdx.x] = 0;
  for (int done = 0; done < tokens; done += kChunk) {
    __syncthreads();
    put(done);
    __syncthreads();
    fetch(done + kChunk);
    if (decays && done % kWave == 0 && done + kWave < tokens) {
      make(done + kWave, gap);
      gap = gap_of(done + 2 * kWave);
    }
    __builtin_amdgcn_sched_barrier(0);
    chunk(done, min(kChunk, tokens - done), s.decay[done / kWave & 1][done / kChunk & 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
  return sum;
}

// Waves of a job: a wave for each 32 columns of the states, but two at most where two jobs share a workgroup; the widest heads'
// columns are two workgroups' there, which share their rows in the cache.  65k x 8 x 128: a pair's sweep 445 us with eight waves
// (as many as a compute unit holds: it waits for its own barriers) and 430 with four, a single one 207 with four and 222
// with two.
template <int DP, int WORK>
constexpr int sweep_waves() { return WORK != kSweep && DP / 32 > 2 ? 2 : DP / 32; }
constexpr int jobs_of(int work) { return work == kSweep ? 1 : 2; }
template <typename T, int DP, int WORK>
constexpr int sweep_threads() { return sweep_waves<DP, WORK>() * jobs_of(WORK) * kWave; }

// What a wave of a sweep goes through: its stretch (if `live`), head, job and columns.
template <int DP, int WORK, bool REV>
struct Part {
  Stretch st;
  int head, job, c0, lane0;                // lane0: the wave's first lane among those of a head's workgroups
  bool live, summing, begins, ends;
  __device__ __forceinline__ Part(const DecayGeo& d, int64_t block) {
    constexpr int NW = sweep_waves<DP, WORK>(), PARTS = DP / 16 / kTiles / NW;         // workgroups of a head
    const int64_t work = near_first(block, d.slots * d.H * PARTS);
    live = work < d.slots * d.H * PARTS;
    if (!live) return;
    const int64_t slot = work / (d.H * PARTS);
    const int place = (int)(work - slot * (d.H * PARTS)), every = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    head = place / PARTS;
    st = stretch_of(d, slot);
    live = st.live;
    job = every / NW;
    const int wave = place % PARTS * NW + every % NW;
    c0 = wave * kTiles * 16;
    lane0 = wave * kWave;
    summing = WORK == kSweepAndSums && job == 1;
    begins = REV ? st.last : st.first, ends = REV ? st.first : st.last;
  }
  // What is before the stretch: its window's given state and the sums of the stretches in between, or their joined state.
  __device__ __forceinline__ void begin(const DecayGeo& d, const Sweep& a, F4 (&M)[kTiles][DP / 16]) const {
    clear_state<DP, kTiles>(M);
    const int64_t DD = (int64_t)d.D * d.D;
    const bool flip = (a.flip != 0) != (job != 0);
    const int64_t dir = REV ? 1 : -1, past = begins ? 0 : st.count > kFew ? 1 : REV ? st.count - 1 - st.index : st.index;
    const bool summed = begins || st.count <= kFew;
#pragma unroll 1
    for (int64_t k = summing ? 0 : past + (summed && a.given); k >= 1; --k) {
      const int64_t e = (st.entry + dir * k) * d.H + head;
      const bool given = k > past;
      const float* p = given ? a.given + (st.window * d.H + head) * DD : a.carry + e * DD;
      add_state<DP, kTiles>(p, flip, d.D, c0, !given && summed ? a.spans[e].fade : Fade{0.f, 1.f}, M);
    }
  }
  // The states behind the stretch that are kept.
  __device__ __forceinline__ void store(const DecayGeo& d, const Sweep& a, const F4 (&M)[kTiles][DP / 16], bool all) const {
    const int64_t DD = (int64_t)d.D * d.D;
    if (ends && a.end && job == 0) store_state<DP, kTiles>(a.end + (st.window * d.H + head) * DD, d.D, c0, M, all);
    if (summing && !st.first) store_state<DP, kTiles>(a.sums + (st.entry * d.H + head) * DD, d.D, c0, M, all);
  }
};

// Waves a SIMD that a sweep is to leave registers for.  Two jobs at 32 channels fit into three waves' registers; 128 channels of
// bfloat16 in loose rows (odd widths) not into two waves': with one, 65k x 8 x 127 forward + backward take 3.12 ms instead of
// 3.50; in float16 3.61 instead of 3.41, so there two it is.
template <typename T, int DP, int WORK, int LAY>
constexpr int wanted_waves() {
  if (DP == 32 && WORK != kSweep && LAY == kWhole) return 3;
  return DP == 128 && LAY == kLoose && std::is_same<T, bf16_t>::value ? 1 : kSweepWaves;
}

template <typename T, int DP, int WORK, bool REV, int LAY>
__global__ void __launch_bounds__((sweep_threads<T, DP, WORK>()), (waves_of<ChunkLds<T, DP, jobs_of(WORK) + 2>, (wanted_waves<T, DP, WORK, LAY>())>(sweep_waves<DP, WORK>() * jobs_of(WORK))))
    k_decay_sweep(DecayGeo d, Sweep a, int64_t first) {
  constexpr int LD = tile_ld<T, DP>(), DT = DP / 16, CT = kTiles, KD = DP / 32, THREADS = sweep_threads<T, DP, WORK>();
  constexpr int NT = jobs_of(WORK) + 2, NS = pieces<T>(2);
  constexpr bool HALF = std::is_same<T, f16_t>::value;
  __shared__ ChunkLds<T, DP, NT> s;
  const Part<DP, WORK, REV> part(d, first + blockIdx.x);
  if (!part.live) return;
  const Stretch& st = part.st;
  const int lane = threadIdx.x & (kWave - 1), g = lane >> 4, i16 = lane & 15;
  const int head = part.head, job = part.job, c0 = part.c0;
  T* out = (T*)a.out[job];
  const bool summing = part.summing;
  if (st.window < 0 || st.window >= d.B) {                  // tokens of no window
    if (summing) return;
    for (int64_t t = st.lo + part.lane0 / kWave; t < st.hi; t += DT / CT)
      for (int c = lane; c < d.D; c += kWave) out[(t * d.H + head) * d.D + c] = (T)0.f;
    return;
  }
  F4 M[CT][DT];
  part.begin(d, a, M);
  // Lanes in which a query or a pair's weight was not finite, of which no channel of its row's output is; what is not finite in Y, W
  // or the state before shows in the state at the end.
  uint64_t check = 0;
  Rows rows[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) rows[n] = a.rows[n];
  const int out_stride = d.H * d.D * (int)sizeof(T);
  const int64_t from = REV ? st.hi - 1 : st.lo;
  constexpr int W_TILES = WORK == kSweep ? 4 : WORK == kSweepPair ? 9 : 5;
  double gone = 0;                                          // exponents of the chunks before, for the sums
  follow<T, DP, NT, W_TILES, THREADS, REV, LAY>(s, d, st, rows, head, a.ps, a.xs, a.us, [&](int done, int len, const Decays& dec) {
    const int wt = WORK != kSweepPair ? (summing ? 0 : 2) : job ? 0 : 3;
    const T* X = s.tile[WORK != kSweepPair ? 0 : job ? 2 : 1];
    const T* Y = s.tile[WORK != kSweepPair ? (summing ? 3 : 1) : job ? 3 : 0];
    const T* W = s.tile[wt];
    const bool odd = __builtin_amdgcn_readfirstlane(s.odd[wt]) == done + 1;
    if (summing) {
      if (st.first) return;                                 // nothing is before it
      const float times = exp2f((float)-gone);
      Frag<T> wf[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) wf[ct] = frag_col<T, LD, false>(W, c0 + ct * 16);
      if (odd) leave_out<T, CT>(wf);
      add_chunk<T, DP, CT>(dec.xe, Fade{0.f, 1.f}, times, Y, M, wf);
      if (odd) mark<T, DP, CT>(W, c0, M);
      gone += dec.total;
      return;
    }
    // What the rows take from the state before the chunk, M^T X^T: a lane holds four neighbouring channels of its row.
    F4 far[2][CT];
#pragma unroll
    for (int it = 0; it < 2; ++it)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) far[it][ct] = F4{0.f, 0.f, 0.f, 0.f};
    Fit fm[CT];                                             // of the lane's column: small channels beside large ones keep their bits
    if (HALF)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float top = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 4; ++r) top = finite_top(top, M[ct][dt][r]);
        fm[ct] = fit_of(top_of_four(top));
      }
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      Frag<T> xf[2], sf[CT][NS];
#pragma unroll
      for (int it = 0; it < 2; ++it) xf[it] = frag_row<T, LD>(X, it * 16 + i16, k);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = HALF ? M[ct][k * 2 + (e >> 2)][e & 3] * fm[ct].up : M[ct][k * 2 + (e >> 2)][e & 3];
        split<T, NS>(v, sf[ct]);
      }
#pragma unroll
      for (int it = 0; it < 2; ++it)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int n = 0; n < NS; ++n) far[it][ct] = mma(sf[ct][n], xf[it], far[it][ct]);
    }
    __builtin_amdgcn_sched_barrier(0);                      // (each part by itself: together they would not fit the registers)
    // The pairs, as Y X^T: a lane holds four neighbouring j of its i, in the order in which the next product sums them.  Their
    // weights go on in two pieces: rounded to T once, they would be as far off as the output's own rounding.
    Frag<T> pf[2][NS];
    Fit fp[2] = {{1.f, 1.f}, {1.f, 1.f}};
    F4 acc[3];                                              // blocks (0, 0), (1, 0), (1, 1)
#pragma unroll
    for (int n = 0; n < 3; ++n) acc[n] = F4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      const Frag<T> y0 = frag_row<T, LD>(Y, i16, k), y1 = frag_row<T, LD>(Y, 16 + i16, k);
      const Frag<T> x0 = frag_row<T, LD>(X, i16, k), x1 = frag_row<T, LD>(X, 16 + i16, k);
      acc[0] = mma(y0, x0, acc[0]);
      acc[1] = mma(y0, x1, acc[1]);
      acc[2] = mma(y1, x1, acc[2]);
    }
    Frag<T> wf[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) wf[ct] = frag_col<T, LD, false>(W, c0 + ct * 16);
    if (odd) leave_out<T, CT>(wf);
    {
      float v[3][4];
      const float row = dec.row[16 + i16];
      const Pack<float, 4> col = load_pack<float, 4>(dec.col + g * 4);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[1][r] = acc[1][r] * row * col.e[r];
#pragma unroll
      for (int it = 0; it < 2; ++it) {
        const double e = dec.e[it * 16 + i16];
#pragma unroll
        for (int r = 0; r < 4; ++r) {                       // (taken for all lanes, without a branch; past i it may overflow)
          const float p = acc[it * 2][r] * a.ps * __builtin_amdgcn_exp2f((float)(dec.e[it * 16 + g * 4 + r] - e));
          v[it * 2][r] = g * 4 + r <= i16 ? p : 0.f;
        }
      }
      if (HALF) {
        float top[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < 3; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) top[n > 0] = finite_top(top[n > 0], v[n][r]);
#pragma unroll
        for (int it = 0; it < 2; ++it) fp[it] = fit_of(top_of_four(top[it]));
#pragma unroll
        for (int n = 0; n < 3; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) v[n][r] *= fp[n > 0].up;
      }
      float p[2][8];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[0][r] = v[0][r], p[0][4 + r] = 0.f;
        p[1][r] = v[1][r], p[1][4 + r] = v[2][r];
      }
#pragma unroll
      for (int it = 0; it < 2; ++it) split<T, NS>(p[it], pf[it]);
    }
    __builtin_amdgcn_sched_barrier(0);
    add_chunk<T, DP, CT>(dec.we, dec.fade, 1.f, Y, M, wf);
    __builtin_amdgcn_sched_barrier(0);
    T* to = out + ((REV ? from - done : from + done) * d.H + head) * d.D;
    int from_lane = g * 4;
    if (HALF) asm volatile("" : "+v"(from_lane));           // (the shuffles' addresses, kept over the loop, would take registers)
    const auto out_buf = chunk_buffer<REV>(to, out_stride, len, d.D * (int)sizeof(T));
#pragma unroll
    for (int it = 0; it < 2; ++it) {
      const int i = it * 16 + i16;
      const float xe = dec.xe[i];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        F4 pv = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NS; ++n) pv = mma(wf[ct], pf[it][n], pv);
        const int c = c0 + ct * 16 + g * 4;
        float o[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          o[r] = HALF ? fmaf(far[it][ct][r] * __shfl(fm[ct].down, from_lane + r, kWave), xe, pv[r] * fp[it].down) : fmaf(far[it][ct][r], xe, pv[r]);
        if (ct == 0) check |= __ballot(!(fabsf(o[0]) < INFINITY));
        if constexpr (LAY != kLoose) {
          const uint32_t at_row = row_offset<REV>(i, out_stride, len) + c * (uint32_t)sizeof(T);
          const uint32_t off = c + 4 <= d.D ? at_row : kNoChannel;
          Pack<T, 4> q;
#pragma unroll
          for (int r = 0; r < 4; ++r) q.e[r] = (T)o[r];
          if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b64(*reinterpret_cast<const U2v*>(&q), out_buf, off, 0, 0);
          else __builtin_amdgcn_raw_buffer_store_b128(*reinterpret_cast<const U4v*>(&q), out_buf, off, 0, 0);
          if constexpr (LAY == kWords)                      // a row's end, word by word
#pragma unroll
            for (int r = 0; r < 4; r += 4 / (int)sizeof(T)) {
              const uint32_t word = *reinterpret_cast<const uint32_t*>(&q.e[r]);
              __builtin_amdgcn_raw_buffer_store_b32(word, out_buf, c + 4 > d.D && c + r < d.D ? at_row + r * (uint32_t)sizeof(T) : kNoChannel, 0, 0);
            }
        } else if (i < len && c < d.D) {
          store_loose<4>(to + (int64_t)(REV ? -i : i) * d.H * d.D + c, d.D - c, o);
        }
      }
    }
    if (odd) {
      mark<T, DP, CT>(W, c0, M);
#pragma unroll 1
      for (int q = 0; q < 2 * CT * 4; ++q) {
        const int i = (q & 1) * 16 + i16, c = c0 + (q >> 3) * 16 + g * 4 + (q >> 1 & 3);
        if (i < len && c < d.D)
#pragma unroll 1
          for (int j = 0; j <= i; ++j)
            if (!(fabsf((float)W[j * LD + c]) < INFINITY)) to[(int64_t)(REV ? -i : i) * d.H * d.D + c] = (T)NAN;
      }
    }
  });
  part.store(d, a, M, true);
  if (summing && !st.first && part.lane0 + lane == 0) a.sum_spans[st.entry * d.H + head] = Span{gone, fade_of((float)(gone * 0.6931471805599453))};
  if (finite_state<DP, CT>(M) && !check) return;
  int64_t block = first + blockIdx.x;
  asm volatile("" : "+s"(block));                           // (all is found anew: kept until here, it would take registers from the sweep)
  const Part<DP, WORK, REV> anew(d, block);
  anew.begin(d, a, M);
  if (anew.summing)
    by_token<T, DP, CT, kFromEnd>(d, anew.st, anew.head, a.rows[0], a.rows[3], a.rows[0], anew.c0, 1.f, a.xs, M, nullptr);
  else
    by_token<T, DP, CT, REV ? kBack : kAlong>(d, anew.st, anew.head, a.rows[WORK != kSweepPair ? 0 : anew.job ? 2 : 1],
                                              a.rows[WORK != kSweepPair ? 1 : anew.job ? 3 : 0],
                                              a.rows[WORK != kSweepPair ? 2 : anew.job ? 0 : 3], anew.c0, a.xs, a.us, M, (T*)a.out[anew.job]);
  anew.store(d, a, M, false);
}

// A stretch's own sum from nothing (all but the last of a window, in the sweep's direction): carry (entries, H, D, D), and
// its exponent and factor (entries, H).
template <typename T, int DP, bool REV, int LAY>
__global__ void __launch_bounds__(DP / 32 * kWave, (waves_of<ChunkLds<T, DP, 2>, LAY != kLoose && DP <= 64 ? 4 : kSweepWaves>(DP / 32)))
    k_decay_local(DecayGeo d, Rows y, Rows w, float us, float* __restrict__ carry, Span* __restrict__ spans, int64_t first) {
  constexpr int LD = tile_ld<T, DP>(), DT = DP / 16, CT = kTiles, NW = DT / CT, THREADS = NW * kWave;
  __shared__ ChunkLds<T, DP, 2> s;
  const int64_t work = near_first(first + blockIdx.x, d.slots * d.H);
  if (work >= d.slots * d.H) return;
  const int64_t slot = work / d.H;
  const int head = (int)(work - slot * d.H);
  const Stretch st = stretch_of(d, slot);
  if (!st.live || (REV ? st.first : st.last) || st.window < 0 || st.window >= d.B) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), c0 = wave * CT * 16;
  F4 M[CT][DT];
  clear_state<DP, CT>(M);
  const Rows rows[2] = {y, w};
  const double sum = follow<T, DP, 2, 2, THREADS, REV, LAY>(s, d, st, rows, head, 1.f, 1.f, us, [&](int done, int, const Decays& dec) {
    Frag<T> wf[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) wf[ct] = frag_col<T, LD, false>(s.tile[1], c0 + ct * 16);
    const bool odd = __builtin_amdgcn_readfirstlane(s.odd[1]) == done + 1;
    if (odd) leave_out<T, CT>(wf);
    add_chunk<T, DP, CT>(dec.we, dec.fade, 1.f, s.tile[0], M, wf);
    if (odd) mark<T, DP, CT>(s.tile[1], c0, M);
  });
  store_state<DP, CT>(carry + (st.entry * d.H + head) * (int64_t)d.D * d.D, d.D, c0, M, true);
  if (threadIdx.x == THREADS - kWave) spans[st.entry * d.H + head] = Span{sum, fade_of((float)(sum * 0.6931471805599453))};
  if (finite_state<DP, CT>(M)) return;
  int64_t anew = first + blockIdx.x;
  asm volatile("" : "+s"(anew));                            // (as in the sweep)
  anew = near_first(anew, d.slots * d.H);
  const Stretch at = stretch_of(d, anew / d.H);
  const int h = (int)(anew % d.H);
  clear_state<DP, CT>(M);
  by_token<T, DP, CT, REV ? kBack : kAlong>(d, at, h, y, y, w, c0, 1.f, us, M, nullptr);
  store_state<DP, CT>(carry + (at.entry * d.H + h) * (int64_t)d.D * d.D, d.D, c0, M, false);
}

// The states after the stretches of every window of more than kFew stretches (all but the last) from the stretches' own sums, in
// place; a sweep adds up fewer sums by itself.  Up to kMany stretches a thread follows an element.  Past that a workgroup has EL
// elements and cuts the stretches into runs: every run's own sum, those joined, every run again from its begin (which the cache
// still holds).  A window is found by the first multiple of kFew L in it, or with fewer windows than multiples by its number.
// Bound by the states' traffic where there are many (65k tokens x 8 x 128: 27 us for 134 MB; with one workgroup a compute unit
// instead of two 32), else by the latency of its searches and runs (1M x 2 x 32: 23 us; 11 where no window is to be joined).
constexpr int kAhead = 8, kMany = 64;
struct Join {
  float* p;                                // the element's sum of the first stretch in the sweep's direction
  const Span* z;
  int64_t n, step, zstep;                  // stretches but the last
  bool in;
};
template <bool WRITE>
__device__ __forceinline__ float join_run(const Join& j, int64_t k0, int64_t k1, float state) {
  for (int64_t k = k0; k < k1; k += kAhead) {
    float u[kAhead];
    Fade f[kAhead];
#pragma unroll
    for (int m = 0; m < kAhead; ++m) {
      const int64_t at = min(k + m, k1 - 1);
      u[m] = j.in ? j.p[at * j.step] : 0.f;
      f[m] = j.z[at * j.zstep].fade;
    }
#pragma unroll
    for (int m = 0; m < kAhead; ++m) {
      if (k + m >= k1) break;
      state = f[m].any(state, u[m]);
      if (WRITE && j.in) j.p[(k + m) * j.step] = state;
    }
  }
  return state;
}
template <bool REV, int EL>
__global__ void __launch_bounds__(1024, EL == kWave ? 8 : 4) k_decay_join(DecayGeo d, const float* __restrict__ given, float* __restrict__ carry,
                                                     const Span* __restrict__ spans, int by_place, int parts, int64_t first) {
  constexpr int RUNS = 1024 / EL;
  __shared__ float end[RUNS][EL];
  __shared__ Fade fade[RUNS];
  const int64_t block = first + blockIdx.x, bh = block / parts, DD = (int64_t)d.D * d.D;
  int64_t b = bh / d.H;
  const int head = (int)(bh - b * d.H);
  if (by_place) {
    const int64_t place = b * kFew * d.L;
    const int64_t e = last_of(d.B + 2, [&](int64_t e) { return edge_of(d, e) <= place; });
    if (e < 1 || e > d.B || edge_of(d, e) + kFew * d.L <= place) return;      // in no window, or not the first multiple in it
    b = e - 1;
  }
  const int64_t lo = edge_of(d, b + 1), hi = max(lo, edge_of(d, b + 2));
  Join j;
  j.n = (hi - lo + d.L - 1) / d.L - 1;
  if (j.n < kFew) return;
  const int e = threadIdx.x % EL, run = EL == kWave ? __builtin_amdgcn_readfirstlane(threadIdx.x / EL) : threadIdx.x / EL;
  const int64_t at = lo / d.L + (REV ? j.n : 0);
  j.z = spans + at * d.H + head;
  j.step = (REV ? -1 : 1) * d.H * DD;
  j.zstep = (REV ? -1 : 1) * d.H;
  if (j.n < kMany) {
    j.in = true;
    for (int64_t el = (block - bh * parts) * 1024 + threadIdx.x; el < DD; el += (int64_t)parts * 1024) {
      j.p = carry + (at * d.H + head) * DD + el;
      join_run<true>(j, 0, j.n, given ? given[(b * d.H + head) * DD + el] : 0.f);
    }
    return;
  }
  const int64_t len = (j.n + RUNS - 1) / RUNS, k0 = min(run * len, j.n), k1 = min(k0 + len, j.n);
  if (threadIdx.x < RUNS) {
    double total = 0;
    for (int64_t k = min(threadIdx.x * len, j.n); k < min((threadIdx.x + 1) * len, j.n); ++k) total += j.z[k * j.zstep].z;
    fade[threadIdx.x] = fade_of((float)(total * 0.6931471805599453));
  }
  for (int64_t el = (block - bh * parts) * EL + e; el - e < DD; el += parts * EL) {
    j.in = el < DD;
    j.p = carry + (at * d.H + head) * DD + el;
    __syncthreads();
    end[run][e] = join_run<false>(j, k0, k1, 0.f);
    __syncthreads();
    float state = given && j.in ? given[(b * d.H + head) * DD + el] : 0.f;
    for (int r = 0; r < run && r * len < j.n; ++r) state = fade[r].any(state, end[r][e]);
    join_run<true>(j, k0, k1, state);
  }
}

// One token of every stream: M = e^{-z} M + k v^T in place, y = scale q M.  A wave a stream's head: lanes side by side along
// the rows of M, 16 bytes each where they are aligned.  Bound by reading and writing the states: 4096 streams x 8 heads of 64
// take 210 us, 5.1 TB/s; 256 x 4 take 12 us.
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
        m[e] = fade.any(m[e], kr * vv[e]);
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

// ------------------------------------------------------------------------------------------- launches
template <typename F>
void by_head(int64_t D, F&& f) {
  if (D <= 32) f(std::integral_constant<int, 32>{});
  else if (D <= 64) f(std::integral_constant<int, 64>{});
  else f(std::integral_constant<int, 128>{});
}

// How rows lie.  Words and pieces are read and written as buffers, loose rows element by element at their ends (251k tokens
// of 3 x 45 in single precision forward + backward: 2079 us loose, 1223 as words; 1107 us of 3 x 48 as pieces).
template <typename T>
int layout(const Rows& r, int64_t D) {
  const int64_t all = (D | r.sn | r.sh) * (int64_t)sizeof(T) | (int64_t)(uintptr_t)r.p;
  return all % 16 == 0 ? kWhole : all % 4 == 0 && D * sizeof(T) >= 16 ? kWords : kLoose;
}
template <typename F>
void by_layout(int lay, F&& f) {
  if (lay == kWhole) f(std::integral_constant<int, kWhole>{});
  else if (lay == kWords) f(std::integral_constant<int, kWords>{});
  else f(std::integral_constant<int, kLoose>{});
}

template <typename T, bool REV>
void run_local(const DecayGeo& d, const Rows& y, const Rows& w, float us, Span* spans, float* carry, hipStream_t stream) {
  if (d.N <= d.L || d.B == 0) return;                      // every window is one stretch at most
  by_head(d.D, [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    by_layout(std::min(layout<T>(y, d.D), layout<T>(w, d.D)), [&](auto l) {
      in_launches((d.slots * d.H + 7) / 8 * 8, [&](int64_t first, unsigned count) {
        hipLaunchKernelGGL((k_decay_local<T, DP, REV, decltype(l)::value>), dim3(count), dim3(DP / 32 * kWave), 0, stream, d, y, w, us,
                           carry, spans, first);
      }, DP / 32 * kWave);
    });
  });
}
template <bool REV>
void run_join(const DecayGeo& d, const float* given, const Span* spans, float* carry, hipStream_t stream) {
  if (d.N <= kFew * d.L || d.B == 0) return;               // no window has more than kFew stretches
  const int64_t DD = (int64_t)d.D * d.D, places = d.N / (kFew * d.L) + 1;
  const int by_place = places < d.B;
  const int64_t of = (by_place ? places : d.B) * d.H;
  auto go = [&](auto el) {                                 // (many find no window to join: as few workgroups as fill the card)
    constexpr int EL = decltype(el)::value;
    const int parts = (int)std::min<int64_t>((DD + EL - 1) / EL, std::max<int64_t>(1024 / of, 1));
    in_launches(of * parts, [&](int64_t first, unsigned count) {
      hipLaunchKernelGGL((k_decay_join<REV, EL>), dim3(count), dim3(1024), 0, stream, d, given, carry, spans, by_place, parts, first);
    }, 1024);
  };
  if (DD * d.H * d.B <= 16384) go(std::integral_constant<int, 16>{});         // few elements: more runs, for as many threads
  else go(std::integral_constant<int, 64>{});
}

template <typename T, int WORK, bool REV>
void run_sweep(const DecayGeo& d, const Sweep& a, hipStream_t stream) {
  int lay = kWhole;
  constexpr int JOBS = jobs_of(WORK);
  for (int n = 0; n < JOBS + 2; ++n) lay = std::min(lay, layout<T>(a.rows[n], d.D));
  for (int n = 0; n < JOBS; ++n)
    if (a.out[n]) lay = std::min(lay, layout<T>(Rows{a.out[n], d.D, d.D}, d.D));
  by_head(d.D, [&](auto dp) {
    constexpr int DP = decltype(dp)::value, THREADS = sweep_threads<T, DP, WORK>();
    if constexpr (DP == 32 || WORK != kSweepAndSums)
      by_layout(lay, [&](auto l) {
        in_launches((d.slots * d.H * (DP / 32 / sweep_waves<DP, WORK>()) + 7) / 8 * 8, [&](int64_t first, unsigned count) {
          hipLaunchKernelGGL((k_decay_sweep<T, DP, WORK, REV, decltype(l)::value>), dim3(count), dim3(THREADS), 0, stream, d, a, first);
        }, THREADS);
      });
  });
}

template <typename T>
void run_fwd(const DecayGeo& d, const DecayFwd& a, hipStream_t stream) {
  Span* spans = (Span*)a.states;
  float* carry = (float*)((char*)a.states + a.span_bytes);
  run_local<T, false>(d, a.k, a.v, 1.f, spans, carry, stream);
  run_join<false>(d, a.h0, spans, carry, stream);
  run_sweep<T, kSweep, false>(d, Sweep{{a.q, a.k, a.v}, {a.y}, carry, spans, a.h0, a.last, 0, a.scale, a.scale, 1.f}, stream);
}
template <typename T>
__global__ void __launch_bounds__(kBlock) k_decay_zeros(T* __restrict__ p, int64_t n, int64_t first) {
  constexpr int V = 16 / sizeof(T);
  const int64_t at = ((first + blockIdx.x) * kBlock + threadIdx.x) * V;
  const float zeros[V] = {};
  store_loose<V>(p + at, n - at, zeros);
}

template <typename T>
void run_bwd(const DecayGeo& d, DecayBwd a, hipStream_t stream) {
  Span* own = (Span*)a.ws;
  float* carry = (float*)((char*)a.ws + a.span_bytes);
  const bool of_states = !a.gy.p;                          // alone: no query has met anything, so gq is zero, and stands for both
  if (of_states) {
    const int64_t n = d.N * d.H * d.D, each = kBlock * 16 / (int64_t)sizeof(T);
    in_launches((n + each - 1) / each, [&](int64_t first, unsigned count) {
      hipLaunchKernelGGL((k_decay_zeros<T>), dim3(count), dim3(kBlock), 0, stream, (T*)a.gq, n, first);
    });
    a.q = a.gy = Rows{a.gq, (int64_t)d.H * d.D, d.D};
  }
  const Sweep dq{{a.gy, a.v, a.k, a.q}, {a.gq}, (const float*)((const char*)a.states + a.span_bytes), (const Span*)a.states, a.h0, nullptr,
                 1, a.scale, a.scale, 1.f, carry, own};
  if (of_states) {
    run_local<T, true>(d, a.q, a.gy, a.scale, own, carry, stream);
  } else if (d.D <= 32 && d.N > d.L) {                     // (a window of more than one stretch may be there)
    run_sweep<T, kSweepAndSums, false>(d, dq, stream);
  } else {
    run_local<T, true>(d, a.q, a.gy, a.scale, own, carry, stream);
    run_sweep<T, kSweep, false>(d, dq, stream);
  }
  run_join<true>(d, a.glast, own, carry, stream);
  run_sweep<T, kSweepPair, true>(d, Sweep{{a.q, a.k, a.v, a.gy}, {a.gv, a.gk}, carry, own, a.glast, a.gh0, 0, a.scale, 1.f, a.scale}, stream);
}
template <typename T>
void run_step(const DecayStep& a, hipStream_t stream) {
  const bool vec = a.D % 4 == 0 && aligned_to(a.state, 16);
  const int64_t units = vec ? a.D / 4 : a.D;
  int cl2 = 0;
  while ((1 << cl2) < kWave && (1 << cl2) < units) ++cl2;
  in_launches((a.N * a.H + kBlock / kWave - 1) / (kBlock / kWave), [&](int64_t first, unsigned count) {
    if (vec)
      hipLaunchKernelGGL((k_decay_step<T, 4>), dim3(count), dim3(kBlock), 0, stream, a.q, a.k, a.v, a.rate, a.dt, a.N, a.H, a.D, cl2,
                         a.scale, a.state, (T*)a.y, first);
    else
      hipLaunchKernelGGL((k_decay_step<T, 1>), dim3(count), dim3(kBlock), 0, stream, a.q, a.k, a.v, a.rate, a.dt, a.N, a.H, a.D, cl2,
                         a.scale, a.state, (T*)a.y, first);
  });
}

}  // namespace
}  // namespace atlhip
