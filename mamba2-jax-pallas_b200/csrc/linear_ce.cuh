// What the two forms of the linear cross entropy (linear_ce.cu, linear_ce_small.cu) share: a
// row's results from the statistics of its logits.
#pragma once
#include "common.cuh"

namespace ssd {
namespace ce {

constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.6931471805599453;

__device__ __forceinline__ int64_t target_at(const void* y, int is64, int64_t t) {
  return is64 ? __ldg(static_cast<const long long*>(y) + t) : (int64_t)__ldg(static_cast<const int*>(y) + t);
}

// A row's results from its statistics (float2: maximum times log2(e), sum of 2^(s log2(e) - that),
// the target left out), by one warp; the few values behind the sum in f64.
struct RowResult {
  float loss, lse;
  float pm1;               // p - 1 of the target
  float top, inv;          // p of another column: inv * 2^(s log2(e) - top)
};

__device__ __forceinline__ RowResult warp_row(const float2* stats, int ns, const float* picked, int target) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY;
  for (int i = lane; i < ns; i += 32) top = fmaxf(top, stats[i].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (top == -INFINITY) top = 0.f;
  double others = 0;
  for (int i = lane; i < ns; i += 32) {
    const float2 s = stats[i];
    others += (double)(s.y * exp2f(s.x - top));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) others += __shfl_xor_sync(0xffffffffu, others, o);
  const double anchor = LN2 * (double)top;
  RowResult r;
  r.top = top;
  if (target < 0) {        // an invalid target: its loss is NaN, and so is its gradient
    r.loss = r.pm1 = r.inv = NAN;
    r.lse = (float)(anchor + log(others));
    return r;
  }
  const double s = (double)*picked, d = anchor - s;
  if (others == 0.0) {     // nothing but the target has mass: p is 1 whatever its logit
    const bool ok = s > -INFINITY && s < INFINITY;
    r.loss = r.pm1 = r.inv = ok ? 0.f : NAN;
    r.lse = ok ? (float)s : NAN;
    return r;
  }
  // others / e^s: the odds against the target; past e^600 they are infinite as far as f32 goes (s may
  // be -inf, which leaves the others' sum alone)
  const double odds = others * exp(d);
  const bool far = d > 600.0;
  double loss = far ? log(others) + d : log1p(odds);
  if (!(s < INFINITY)) loss = NAN;   // an infinite or NaN logit, as the formula has it
  r.loss = (float)loss;
  r.lse = (float)(far ? anchor + log(others) : loss + s);
  r.pm1 = (float)(!(s < INFINITY) ? NAN : far ? -1.0 : -odds / (1.0 + odds));
  r.inv = (float)(1.0 / (others + exp(-d)));
  return r;
}

// What the gradients need of a row: p of a column other than the target's is f 2^(s log2(e) - top).
struct RowFactors {
  float top, f, at_y;
};

}  // namespace ce
}  // namespace ssd
