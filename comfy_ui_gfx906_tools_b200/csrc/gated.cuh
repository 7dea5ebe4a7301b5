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
//
// Phi(-x) = e^(-x^2 / 2) P(t) / 2 for x >= 0 with t = 1 / (1 + 0.35 x / sqrt 2),
// the form of Abramowitz and Stegun 7.1.26; P's eight coefficients are fitted
// here to erfcx by reweighted least squares to 8.3e-7 of its value for every x
// (2e-6 with float32's own rounding above g = -5). It takes 18 instructions
// and its exponential is phi's, where normcdff took the epilogue past the
// matrix product.
#pragma once

#include "common.cuh"

namespace gfx {
namespace gated {

enum : int { kSilu = 0, kGelu = 1, kGeluTanh = 2 };

__device__ __forceinline__ float sigmoid(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

constexpr float kRoot2OverPi = 0.7978845608028654f, kCubic = 0.044715f, kInvRoot2Pi = 0.3989422804014327f;

// Phi(g), and e^(-g^2 / 2) in `e`
__device__ __forceinline__ float normal_cdf(float g, float& e) {
  constexpr float kC[8] = {0.19746628403663635f, 0.197453111410141f,     0.18590933084487915f, 0.154672309756279f,
                           0.1629437953233719f,  -0.014549784362316132f, 0.20120933651924133f, -0.08510520309209824f};
  const float t = __fdividef(1.0f, 1.0f + (0.35f * 0.7071067811865476f) * fabsf(g));
  float p = kC[7];
#pragma unroll
  for (int i = 6; i >= 0; --i) p = p * t + kC[i];
  e = __expf(-0.5f * g * g);
  const float q = 0.5f * p * t * e;
  return g < 0.0f ? q : 1.0f - q;
}

template <int kAct>
__device__ __forceinline__ float activation(float g) {
  if constexpr (kAct == kSilu) return g * sigmoid(g);
  if constexpr (kAct == kGelu) {
    float e;
    return g * normal_cdf(g, e);
  }
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
    float e;
    const float c = normal_cdf(g, e);
    a = g * c;
    da = c + g * kInvRoot2Pi * e;
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
