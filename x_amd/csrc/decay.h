// Linear attention with a decay for each head: what its entry points hand to the kernels of a type (decay_kernels.h).
#pragma once
#include "typed.h"

namespace atlhip {

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

struct DecayFwd {
  Rows q, k, v;
  const float* h0;
  float scale;
  void* y;
  float* last;
  void* states;                            // spans of the stretches, and from span_bytes on their sums or states
  int64_t span_bytes;
};
struct DecayBwd {
  Rows q, k, v, gy;
  const float *h0, *glast;
  float scale;
  void *gq, *gk, *gv;
  float* gh0;
  const void* states;                      // the forward's
  void* ws;                                // the same from the end
  int64_t span_bytes;
};
struct DecayStep {
  Rows q, k, v;
  const float *rate, *dt;
  int64_t N;
  int H, D;
  float scale;
  float* state;
  void* y;
};

// T: float, bf16_t, f16_t, each in a file of its own (a minute of compiling each).
template <typename T>
void decay_fwd(const DecayGeo& d, const DecayFwd& a, hipStream_t stream);
template <typename T>
void decay_bwd(const DecayGeo& d, const DecayBwd& a, hipStream_t stream);
template <typename T>
void decay_step(const DecayStep& a, hipStream_t stream);

}  // namespace atlhip
