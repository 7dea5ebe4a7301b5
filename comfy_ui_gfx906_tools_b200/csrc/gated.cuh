// The gate activations of the gated feed-forward product and their derivatives
// (gated.cu), in float32.
//
//   silu       a(g) = g s(g),              a' = s + g s (1 - s),  s(g) = 1 / (1 + e^-g)
//   gelu       a(g) = g Phi(g),            a' = Phi + g phi
//   gelu_tanh  a(g) = g (1 + tanh y) / 2 = g s(2 y),  a' = s + g s (1 - s) 2 y',
//              y = sqrt(2 / pi) (g + 0.044715 g^3)
// All three are g times a distribution-like factor that is computed without
// cancellation on either side, so far negative gates keep their relative
// precision. Nothing overflows on the way: the logistic function of -x is taken
// as e^-x / (1 + e^-x), where 1 / (1 + e^x) would be 0 from x = 87 on, while
// g times it is still far above bfloat16's smallest steps.
//
// The exponential's instruction and the reciprocal's are documented to 2^-22 and
// 2^-23, CUDA's fast exponential (in Phi) to 2 + 1.17 |x| steps for e^x; rounding
// the argument moves e^x by some |x| half steps more. By these bounds a value is
// within 1e-6 of itself near g = 0 (gelu 3e-6), 1e-5 at silu's g = -20 or gelu's
// -6, and 4e-5 at the far end, where the exponential's argument is -90: a tenth of
// half a float16 step.
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

constexpr float kRoot2OverPi = 0.7978845608028654f, kCubic = 0.044715f, kInvRoot2Pi = 0.3989422804014327f;
constexpr float kHalfLog2E = 0.72134752044448170368f;

// 1 / (1 + e^-x) from z = -|x| log2(e) / 2 and x's sign. e^-|x| is the square of 2^z, whose instruction flushes results
// below 2^-126 to 0 and does not come near them before |x| = 174.
__device__ __forceinline__ float logistic(float z, bool negative) {
  float h, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(z));
  const float e = h * h;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return (negative ? e : 1.0f) * r;
}

// silu's factor s(g), and gelu_tanh's s(2 y)
__device__ __forceinline__ float sigmoid(float g) { return logistic(-kHalfLog2E * fabsf(g), g < 0.0f); }
__device__ __forceinline__ float tanh_factor(float g) {
  constexpr float kA = -2.0f * kHalfLog2E * kRoot2OverPi;
  return logistic(fabsf(g) * (kA + kA * kCubic * (g * g)), g < 0.0f);
}

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
  return g * tanh_factor(g);
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
    const float s = tanh_factor(g);
    a = g * s;
    const float t = a * (1.0f - s);
    // far out s (1 - s) is 0 and the cubic's slope may be infinite
    da = s + (t == 0.0f ? 0.0f : t * 2.0f * kRoot2OverPi * (1.0f + 3.0f * kCubic * g * g));
  }
}

}  // namespace gated
}  // namespace gfx
