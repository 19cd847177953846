// Linear attention with a decay for each head: sizes, checks and entry points (the kernels: decay_kernels.h).
#include "decay.h"
#include "../../include/atl_hip.h"

#include <algorithm>

namespace atlhip {
namespace {

constexpr int kMaxHead = 128;
constexpr int64_t kMaxStride = (int64_t)1 << 22;

// Tokens of a stretch: whole pairs of chunks, four pairs at least.  The stretches of all heads, and half a stretch for every
// window's last, are whole rounds of workgroups: past 64 channels two rounds of two a compute unit (four waves each, two a
// SIMD), past 32 two rounds of four, up to 32 one and a half a SIMD, all at once.  Chosen by bfloat16 cases; microseconds,
// forward + backward, by their number:
//   65k x 8 x 128   512: 1195   768: 942   1024: 951                 180k x 6 x 64   1024: 813   2048: 711   2900: 787
//   30k x 16 x 128  512: 1059   768: 978   1024: 902                 102k x 4 x 64   1024: 422   2048: 361   2900: 364
//   1M x 2 x 32     768: 657   1536: 572   2048: 648                 400k x 4 x 32    768: 640   1536: 509   2048: 554
// The rule counts workgroups, not the states that stretches write, join and read, and so is off where there are few windows
// of wide heads, and in other types:
//   100k x 4 x 128, 3 windows           512: 695   1024: 826         250k x 4 x 64, 1 window        1024: 672   2048: 706
//   40k x 6 x 100, float32              512: 1158  1024: 1238        251k x 3 x 45, float32         1024: 1100  2048: 1131
//   90k x 8 x 96, float16               512: 1634  1024: 1687        100k x 8 x 32, float32         1536: 539   2048: 498
int64_t stretch_len(int64_t N, int64_t B, int64_t H, int64_t D) {
  constexpr int64_t kPair = 64;
  const int64_t groups = D <= 32 ? 1536 : D <= 64 ? 2048 : 1024;
  const int64_t left = std::max(groups - B * H / 2, groups / 2);
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

int64_t decay_entries(int64_t N, int64_t B, int64_t H, int64_t D) { return N / stretch_len(N, B, H, D) + 1; }
int64_t decay_span_bytes(int64_t N, int64_t B, int64_t H, int64_t D) { return (decay_entries(N, B, H, D) * H * 16 + 255) / 256 * 256; }

template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == kF32) f(float{});
  else if (dtype == kBF16) f(bf16_t{});
  else f(f16_t{});
}

DecayGeo decay_geo(int64_t N, int64_t B, int64_t H, int64_t D, const int64_t* start, const float* dt, const float* rate) {
  DecayGeo d{};
  d.start = start; d.dt = dt; d.rate = rate;
  d.N = N; d.B = B; d.L = stretch_len(N, B, H, D);
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
  return N <= stretch_len(N, B, H, D) ? 0 : decay_span_bytes(N, B, H, D) + decay_entries(N, B, H, D) * H * D * D * 4;
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
  const DecayFwd a{rq, rk, rv, h0, (float)scale, y, last, states, decay_span_bytes(N, B, H, D)};
  by_type(dtype, [&](auto t) { decay_fwd<decltype(t)>(d, a, stream); });
  return check_launch("decay_attn_fwd");
}

int atl_decay_attn_bwd(const void* q, int64_t sqn, int64_t sqh, const void* k, int64_t skn, int64_t skh, const void* v,
                       int64_t svn, int64_t svh, const void* gy, int64_t sgn, int64_t sgh, int dtype, int64_t N, int64_t H,
                       int64_t D, const float* rate, const int64_t* start, int64_t B, const float* dt, const float* h0,
                       const float* glast, double scale, const void* states, void* gq, void* gk, void* gv, float* gh0, void* ws,
                       int64_t ws_bytes, hipStream_t stream) {
  Rows rq{q, sqn, sqh}, rk{k, skn, skh}, rv{v, svn, svh}, rg{gy, sgn, sgh};
  if (!decay_ok(dtype, N, B, H, D) || (N > 0 && !(strides_ok(rq, N, D) && strides_ok(rk, N, D) && strides_ok(rv, N, D) && (!gy || strides_ok(rg, N, D))))) { set_error("decay_attn_bwd: bad sizes N=%lld B=%lld H=%lld D=%lld type %d", (long long)N, (long long)B, (long long)H, (long long)D, dtype); return 1; }
  const int64_t need = atl_decay_attn_states_bytes(N, B, H, D);
  if (!start || !rate || (N > 0 && (!q || !k || !v || !gq || !gk || !gv)) || (need && (!states || !ws))) { set_error("decay_attn_bwd: null argument"); return 1; }
  if (ws_bytes < need) { set_error("decay_attn_bwd: workspace of %lld bytes, need %lld", (long long)ws_bytes, (long long)need); return 1; }
  const DecayGeo d = decay_geo(N, B, H, D, start, dt, rate);
  const DecayBwd a{rq, rk, rv, rg, h0, glast, (float)scale, gq, gk, gv, gh0, states, ws, decay_span_bytes(N, B, H, D)};
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
