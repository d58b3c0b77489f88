// The running sums behind log probabilities and entropy, shared by the kernels on logits and on hidden states.
#pragma once

#include "sm100_common.cuh"

namespace himuon {

constexpr float kLog2eS = 1.4426950408889634f;
constexpr float kFar = -1.0e4f;                   // d below this: e^d is 0 in fp32, and d * e^d has to be as well


// Sums over some logits of a row, relative to the largest of them: s = sum e^(x-m), t = sum (x-m) e^(x-m).
struct Sums { float m, s, t; };
__device__ __forceinline__ Sums moved(const Sums& a, float m) {     // a's sums relative to m >= a.m
  if (a.m == -INFINITY) return Sums{m, a.s, a.t};                   // 0, or NaN
  const float d = fmaxf(a.m - m, kFar), f = exp2f(d * kLog2eS);
  return Sums{m, a.s * f, f * (a.t + d * a.s)};
}
__device__ __forceinline__ Sums merged(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m);
  const Sums x = moved(a, m), y = moved(b, m);
  return Sums{m, x.s + y.s, x.t + y.t};
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <int N>
__device__ __forceinline__ float largest(const float (&x)[N]) {
  float mx = x[0];
#pragma unroll
  for (int i = 1; i + 1 < N; i += 2) mx = max3(mx, x[i], x[i + 1]);
  return N % 2 ? mx : fmaxf(mx, x[N - 1]);
}
// Adds N logits, the largest of which is mx, to the sums.
template <int N>
__device__ __forceinline__ void take(Sums& a, const float (&x)[N], float mx) {
  if (mx > a.m) a = moved(a, mx);
  const float base = a.m == -INFINITY ? 0.f : a.m;    // nothing but -inf so far: d = -inf, e^d = 0
  const f32x2 nbase = pack2(-base, -base), l2e = pack2(kLog2eS, kLog2eS);
  f32x2 s[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)}, t[2] = {s[0], s[0]};
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const f32x2 d = add2(pack2(x[2 * i], x[2 * i + 1]), nbase);
    float y0, y1;
    unpack2(mul2(d, l2e), y0, y1);
    const f32x2 e = pack2(exp2f(y0), exp2f(y1));
    s[i & 1] = add2(s[i & 1], e);
    t[i & 1] = fma2(d, e, t[i & 1]);
  }
  float s0, s1, t0, t1;
  unpack2(add2(s[0], s[1]), s0, s1);
  unpack2(add2(t[0], t[1]), t0, t1);
  t0 += t1;
  if (t0 != t0) {                                     // -inf among them: 0 times -inf.  (A maximum for each logit costs a tenth of the pass.)
    t0 = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = x[i] - base;
      t0 = fmaf(fmaxf(d, kFar), exp2f(d * kLog2eS), t0);
    }
  }
  a.s += s0 + s1;
  a.t += t0;
}
__device__ __forceinline__ Sums lanes_merged(Sums a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = merged(a, Sums{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.t, o)});
  return a;
}

// What a row's sums say: m and log s (0 and INFINITY for a row of nothing but -inf), and the entropy.
struct RowScore { float m, log_s, entropy; };
__device__ __forceinline__ RowScore row_score(const Sums& a) {
  if (a.s == 0.f) return RowScore{0.f, INFINITY, 0.f};
  const float log_s = static_cast<float>(log(static_cast<double>(a.s)));      // (logf is the approximate one in this build)
  return RowScore{a.m, log_s, log_s - a.t / a.s};
}
__device__ __forceinline__ float nan_f() { return __uint_as_float(0x7FFFFFFFu); }

// What the gradient of a row is made of:  dx_j = g [j = y] - p_j (c0 + h log p_j),  c0 = g + h H.
struct RowGrad { float m, log_s, c0, h, g; int y; };
__device__ __forceinline__ RowGrad row_grad(const float2* stats, const float* entropy, const long long* ids, const float* g_log_probs,
                                            const float* g_entropy, long long ignore, int vocab, long long row) {
  RowGrad r;
  const float2 st = stats[row];
  const long long id = ids[row];
  const bool counted = id != ignore && id >= 0 && id < vocab;
  r.m = st.x;
  r.log_s = st.y;
  r.y = counted && st.y != INFINITY ? static_cast<int>(id) : -1;              // (INFINITY: a row of nothing but -inf)
  r.g = counted && g_log_probs ? g_log_probs[row] : 0.f;
  r.h = g_entropy ? g_entropy[row] : 0.f;
  r.c0 = fmaf(r.h, entropy[row], r.g);
  return r;
}
__device__ __forceinline__ float grad_of(const RowGrad& r, float x, int column) {
  const float lp = (x - r.m) - r.log_s, d = -exp2f(lp * kLog2eS) * fmaf(r.h, fmaxf(lp, kFar), r.c0);
  return column == r.y ? d + r.g : d;
}

}  // namespace himuon
