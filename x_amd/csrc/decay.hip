// Linear attention with a decay for each head: sizes, checks and entry points (the kernels: decay_kernels.h).
#include "decay.h"
#include "../../include/atl_hip.h"

#include <algorithm>

namespace atlhip {
namespace {

constexpr int kMaxHead = 128;
constexpr int64_t kMaxStride = (int64_t)1 << 22;

// Tokens of a stretch: the stretches of all heads, and half a stretch for every window's last, are 1536 workgroups, six a
// compute unit (half and twice as many were up to 20% slower, by the width), whole pairs of chunks, four pairs at least.
int64_t stretch_len(int64_t N, int64_t B, int64_t H) {
  constexpr int64_t kGroups = 1536, kPair = 64;
  const int64_t left = std::max(kGroups - B * H / 2, kGroups / 2);
  const int64_t pairs = (N * H / left + kPair - 1) / kPair;
  return kPair * std::min<int64_t>(std::max<int64_t>(pairs, 4), 512);
}

bool decay_ok(int dtype, int64_t N, int64_t B, int64_t H, int64_t D) {
  return dtype_ok(dtype) && N >= 0 && B >= 0 && H >= 1 && D >= 1 && D <= kMaxHead && N < ((int64_t)1 << 40) &&
         B < ((int64_t)1 << 31) && H * D < kMaxStride;
}
// Rows within reach of a chunk's 32-bit offsets, none on another (a single row's stride says nothing).
bool strides_ok(Rows& r, int64_t N, int64_t D) {
  if (N < 2) r.sn = D;
  return r.sh >= 0 && r.sn >= D && r.sn < kMaxStride;
}

int64_t decay_entries(int64_t N, int64_t B, int64_t H) { return N / stretch_len(N, B, H) + 1; }
int64_t decay_span_bytes(int64_t N, int64_t B, int64_t H) { return (decay_entries(N, B, H) * H * 16 + 255) / 256 * 256; }

template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == kF32) f(float{});
  else if (dtype == kBF16) f(bf16_t{});
  else f(f16_t{});
}

DecayGeo decay_geo(int64_t N, int64_t B, int64_t H, int64_t D, const int64_t* start, const float* dt, const float* rate) {
  DecayGeo d{};
  d.start = start; d.dt = dt; d.rate = rate;
  d.N = N; d.B = B; d.L = stretch_len(N, B, H);
  d.slots = N / d.L + B + 2;
  d.H = (int)H; d.D = (int)D;
  return d;
}

}  // namespace
}  // namespace atlhip

using namespace atlhip;

extern "C" {

int64_t atl_decay_attn_states_bytes(int64_t N, int64_t B, int64_t H, int64_t D) {
  if (!decay_ok(kF32, N, B, H, D)) return -1;
  return N <= stretch_len(N, B, H) ? 0 : decay_span_bytes(N, B, H) + decay_entries(N, B, H) * H * D * D * 4;
}

int atl_decay_attn_fwd(const void* q, int64_t sqn, int64_t sqh, const void* k, int64_t skn, int64_t skh, const void* v,
                       int64_t svn, int64_t svh, int dtype, int64_t N, int64_t H, int64_t D, const float* rate,
                       const int64_t* start, int64_t B, const float* dt, const float* h0, double scale, void* y, float* last,
                       void* states, int64_t states_bytes, hipStream_t stream) {
  Rows rq{q, sqn, sqh}, rk{k, skn, skh}, rv{v, svn, svh};
  if (!decay_ok(dtype, N, B, H, D) || (N > 0 && !(strides_ok(rq, N, D) && strides_ok(rk, N, D) && strides_ok(rv, N, D)))) { set_error("decay_attn_fwd: bad sizes N=%lld B=%lld H=%lld D=%lld type %d", (long long)N, (long long)B, (long long)H, (long long)D, dtype); return 1; }
  const int64_t need = atl_decay_attn_states_bytes(N, B, H, D);
  if (!start || !rate || (N > 0 && (!q || !k || !v || !y)) || (need && !states)) { set_error("decay_attn_fwd: null argument"); return 1; }
  if (states_bytes < need) { set_error("decay_attn_fwd: states of %lld bytes, need %lld", (long long)states_bytes, (long long)need); return 1; }
  const DecayGeo d = decay_geo(N, B, H, D, start, dt, rate);
  const DecayFwd a{rq, rk, rv, h0, (float)scale, y, last, states, decay_span_bytes(N, B, H)};
  by_type(dtype, [&](auto t) { decay_fwd<decltype(t)>(d, a, stream); });
  return check_launch("decay_attn_fwd");
}

int atl_decay_attn_bwd(const void* q, int64_t sqn, int64_t sqh, const void* k, int64_t skn, int64_t skh, const void* v,
                       int64_t svn, int64_t svh, const void* gy, int64_t sgn, int64_t sgh, int dtype, int64_t N, int64_t H,
                       int64_t D, const float* rate, const int64_t* start, int64_t B, const float* dt, const float* h0,
                       const float* glast, double scale, const void* states, void* gq, void* gk, void* gv, float* gh0, void* ws,
                       int64_t ws_bytes, hipStream_t stream) {
  Rows rq{q, sqn, sqh}, rk{k, skn, skh}, rv{v, svn, svh}, rg{gy, sgn, sgh};
  if (!decay_ok(dtype, N, B, H, D) || (N > 0 && !(strides_ok(rq, N, D) && strides_ok(rk, N, D) && strides_ok(rv, N, D) && strides_ok(rg, N, D)))) { set_error("decay_attn_bwd: bad sizes N=%lld B=%lld H=%lld D=%lld type %d", (long long)N, (long long)B, (long long)H, (long long)D, dtype); return 1; }
  const int64_t need = atl_decay_attn_states_bytes(N, B, H, D);
  if (!start || !rate || (N > 0 && (!q || !k || !v || !gy || !gq || !gk || !gv)) || (need && (!states || !ws))) { set_error("decay_attn_bwd: null argument"); return 1; }
  if (ws_bytes < need) { set_error("decay_attn_bwd: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)need); return 1; }
  const DecayGeo d = decay_geo(N, B, H, D, start, dt, rate);
  const DecayBwd a{rq, rk, rv, rg, h0, glast, (float)scale, gq, gk, gv, gh0, states, ws, decay_span_bytes(N, B, H)};
  by_type(dtype, [&](auto t) { decay_bwd<decltype(t)>(d, a, stream); });
  return check_launch("decay_attn_bwd");
}

int atl_decay_attn_step(const void* q, int64_t sqn, int64_t sqh, const void* k, int64_t skn, int64_t skh, const void* v,
                        int64_t svn, int64_t svh, int dtype, int64_t N, int64_t H, int64_t D, const float* rate, const float* dt,
                        double scale, float* state, void* y, hipStream_t stream) {
  if (!decay_ok(dtype, N, 0, H, D) || (N > 0 && (sqn < 0 || sqh < 0 || skn < 0 || skh < 0 || svn < 0 || svh < 0))) { set_error("decay_attn_step: bad sizes N=%lld H=%lld D=%lld type %d", (long long)N, (long long)H, (long long)D, dtype); return 1; }
  if (N == 0) return 0;
  if (!q || !k || !v || !rate || !state || !y) { set_error("decay_attn_step: null argument"); return 1; }
  const DecayStep a{{q, sqn, sqh}, {k, skn, skh}, {v, svn, svh}, rate, dt, N, (int)H, (int)D, (float)scale, state, y};
  by_type(dtype, [&](auto t) { decay_step<decltype(t)>(a, stream); });
  return check_launch("decay_attn_step");
}

}  // extern "C"
