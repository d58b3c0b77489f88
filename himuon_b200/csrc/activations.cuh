// Activations of the gated feed-forward block and their derivatives, in fp32.
#pragma once

#include <cuda_runtime.h>

#include "gated_mlp.h"

namespace himuon {

// silu(g) = g / (1 + e^-g), and the tanh form of gelu by 0.5 (1 + tanh z) = 1 / (1 + e^-2z): no difference of near values.
// Far below 0 the exponential runs over to infinity, and the quotient is 0 as it has to be (__fdividef gives 0 from divisors of 2^126 on): an exponent that
// stops somewhere leaves a sigmoid above 0, which a gate of -1e36 turns into -18.  A gate of -inf gives NaN, as -inf times 0 does.
constexpr float kGeluC = 0.7978845608028654f, kGeluA = 0.044715f;      // sqrt(2 / pi)
constexpr float kLargest = 3e38f;

template <int ACT>
__device__ __forceinline__ float activate(float g) {
  if constexpr (ACT == kSilu) return __fdividef(g, 1.f + __expf(-g));
  if constexpr (ACT == kGelu) return 0.5f * g * erfcf(g * -0.70710678f);
  if constexpr (ACT == kGeluTanh) return __fdividef(g, 1.f + __expf(-2.f * kGeluC * g * (1.f + kGeluA * g * g)));
  return g < 0.f ? 0.f : g;                       // (NaN stays)
}
// The activation and its derivative.  (e * s, which is 1 - s, has to stay a number where e is infinite and s is 0: e stops at the largest of them there.)
template <int ACT>
__device__ __forceinline__ void activate_grad(float g, float& a, float& d) {
  if constexpr (ACT == kSilu) {
    const float e = __expf(-g), s = __fdividef(1.f, 1.f + e);
    a = g * s;
    d = s * (1.f + g * (fminf(e, kLargest) * s));
  } else if constexpr (ACT == kGelu) {
    const float phi = 0.5f * erfcf(g * -0.70710678f);
    a = g * phi;
    d = phi + g * 0.3989422804f * __expf(-0.5f * g * g);
  } else if constexpr (ACT == kGeluTanh) {
    // (beyond 30 the sigmoid is what it is there, while the polynomial would run over; NaN stays)
    const float z = fminf(fmaxf(g, -30.f), 30.f), e = __expf(-2.f * kGeluC * z * (1.f + kGeluA * z * z)), s = __fdividef(1.f, 1.f + e);
    a = g * s;
    d = s + z * (fminf(e, kLargest) * s) * s * (2.f * kGeluC * (1.f + 3.f * kGeluA * z * z));
    if (g != g) d = g;
  } else {
    a = g < 0.f ? 0.f : g;
    d = g <= 0.f ? 0.f : 1.f;
  }
}

}  // namespace himuon
