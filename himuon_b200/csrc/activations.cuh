// Activations of the gated feed-forward block and their derivatives, in fp32.
#pragma once

#include <cuda_runtime.h>

#include "gated_mlp.h"

namespace himuon {

// silu(g) = g / (1 + e^-g), and the tanh form of gelu by 0.5 (1 + tanh z) = 1 / (1 + e^-2z): no difference of near values.
constexpr float kGeluC = 0.7978845608028654f, kGeluA = 0.044715f;      // sqrt(2 / pi)

template <int ACT>
__device__ __forceinline__ float activate(float g) {
  if constexpr (ACT == kSilu) return __fdividef(g, 1.f + __expf(fminf(-g, 80.f)));
  if constexpr (ACT == kGelu) return 0.5f * g * erfcf(g * -0.70710678f);
  if constexpr (ACT == kGeluTanh) return __fdividef(g, 1.f + __expf(fminf(-2.f * kGeluC * g * (1.f + kGeluA * g * g), 80.f)));
  return g < 0.f ? 0.f : g;                       // (NaN stays)
}
// The activation and its derivative.  (The exponent stops at 80, where the sigmoid is 2e-35: e * s stays a number.)
template <int ACT>
__device__ __forceinline__ void activate_grad(float g, float& a, float& d) {
  if constexpr (ACT == kSilu) {
    const float e = __expf(fminf(-g, 80.f)), s = __fdividef(1.f, 1.f + e);
    a = g * s;
    d = s * (1.f + g * (e * s));
  } else if constexpr (ACT == kGelu) {
    const float phi = 0.5f * erfcf(g * -0.70710678f);
    a = g * phi;
    d = phi + g * 0.3989422804f * __expf(-0.5f * g * g);
  } else if constexpr (ACT == kGeluTanh) {
    // (beyond 30 the sigmoid is what it is there, while the polynomial would run over; NaN stays)
    const float z = fminf(fmaxf(g, -30.f), 30.f), e = __expf(fminf(-2.f * kGeluC * z * (1.f + kGeluA * z * z), 80.f)), s = __fdividef(1.f, 1.f + e);
    a = g * s;
    d = s + z * (e * s) * s * (2.f * kGeluC * (1.f + 3.f * kGeluA * z * z));
    if (g != g) d = g;
  } else {
    a = g < 0.f ? 0.f : g;
    d = g <= 0.f ? 0.f : 1.f;
  }
}

}  // namespace himuon
