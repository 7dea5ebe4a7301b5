// The gate activations of the gated feed-forward product and their derivatives
// (gated.cu), in float32.
//
//   silu       a(g) = g s(g),              a' = s + g s (1 - s),  s(g) = 1 / (1 + e^-g)
//   gelu       a(g) = g Phi(g),            a' = Phi + g phi
//   gelu_tanh  a(g) = g (1 + tanh y) / 2 = g s(2 y),  a' = s + g s (1 - s) 2 y',
//              y = sqrt(2 / pi) (g + 0.044715 g^3)
// All three are g times a distribution-like factor that is computed without
// cancellation on either side, so far negative gates keep their relative
// precision. The fast exponential and division are off by some 1e-6, three
// orders below the rounding of a 16-bit result.
#pragma once

#include "common.cuh"

namespace gfx {
namespace gated {

enum : int { kSilu = 0, kGelu = 1, kGeluTanh = 2 };

__device__ __forceinline__ float sigmoid(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

constexpr float kRoot2OverPi = 0.7978845608028654f, kCubic = 0.044715f, kInvRoot2Pi = 0.3989422804014327f;

template <int kAct>
__device__ __forceinline__ float activation(float g) {
  if constexpr (kAct == kSilu) return g * sigmoid(g);
  if constexpr (kAct == kGelu) return g * normcdff(g);
  return g * sigmoid(2.0f * kRoot2OverPi * g * (1.0f + kCubic * g * g));
}

// a(g) and a'(g)
template <int kAct>
__device__ __forceinline__ void activation_grad(float g, float& a, float& da) {
  if constexpr (kAct == kSilu) {
    const float s = sigmoid(g);
    a = g * s;
    da = s + a * (1.0f - s);
  } else if constexpr (kAct == kGelu) {
    const float c = normcdff(g);
    a = g * c;
    da = c + g * kInvRoot2Pi * __expf(-0.5f * g * g);
  } else {
    const float s = sigmoid(2.0f * kRoot2OverPi * g * (1.0f + kCubic * g * g));
    a = g * s;
    const float t = a * (1.0f - s);
    // far out s (1 - s) is 0 and the cubic's slope may be infinite
    da = s + (t == 0.0f ? 0.0f : t * 2.0f * kRoot2OverPi * (1.0f + 3.0f * kCubic * g * g));
  }
}

}  // namespace gated
}  // namespace gfx
