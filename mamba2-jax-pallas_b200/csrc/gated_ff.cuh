// What the forms of the gated feed-forward block (gated_ff.cu, gated_ff_few.cu) share: the activations.
#pragma once
#include "common.cuh"

namespace ssd {
namespace ff {

__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.f, 1.f + exp2f(v * -1.4426950408889634f)); }

// act(g), and with `slope` act'(g); one of ssd_activation_t.
template <int ACT>
__device__ __forceinline__ float activate(float g, float* slope) {
  if constexpr (ACT == SSD_ACT_RELU) {
    if (slope) *slope = g > 0.f ? 1.f : 0.f;
    return g < 0.f ? 0.f : g;
  } else if constexpr (ACT == SSD_ACT_GELU) {   // g Phi(g); Phi' is the normal density
    const float p = 0.5f * erfcf(g * -0.70710678118654752f);
    if (slope) *slope = fmaf(g * exp2f(g * g * -0.72134752044448170f), 0.39894228040143268f, p);
    return g * p;
  } else if constexpr (ACT == SSD_ACT_GELU_TANH) {   // (1 + tanh z) / 2 = sigmoid(2 z)
    const float k = 1.5957691216057308f, q = fminf(g * g, 1e30f);   // 2 sqrt(2 / pi); beyond 1e15 p is 0 or 1, and 0 times q has to be 0
    const float p = sigmoid(k * g * fmaf(0.044715f, q, 1.f));
    if (slope) *slope = fmaf(g * p * (1.f - p), k * fmaf(3.f * 0.044715f, q, 1.f), p);
    return g * p;
  } else {
    const float p = sigmoid(g);
    if (slope) *slope = p * fmaf(g, 1.f - p, 1.f);
    return g * p;
  }
}

// The same with the activation known at run time.
__device__ __forceinline__ float activate(int act, float g, float* slope) {
  switch (act) {
    case SSD_ACT_RELU: return activate<SSD_ACT_RELU>(g, slope);
    case SSD_ACT_GELU: return activate<SSD_ACT_GELU>(g, slope);
    case SSD_ACT_GELU_TANH: return activate<SSD_ACT_GELU_TANH>(g, slope);
    default: return activate<SSD_ACT_SILU>(g, slope);
  }
}

}  // namespace ff
}  // namespace ssd
