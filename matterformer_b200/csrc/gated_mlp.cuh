// What the kernels of the gated feed-forward block share: its activations, and the entry of the kernels for few tokens.
#pragma once

#include "common.cuh"

namespace mf {

// act(z) = z s(w(z)) with the logistic function s: w = z is SiLU; w = 2 sqrt(2/pi) (z + 0.044715 z^3) is GELU in its tanh form, since
// (1 + tanh(a)) / 2 = s(2 a), and nothing cancels for large negative z.  The derivative is s + z s (1 - s) w'.
// Beyond |z| = 64 GELU is 0 or z in fp32: the clamp keeps the cube and w' finite.
template <int kAct>
__device__ __forceinline__ float2 logistic2(float2 z, float2& slope) {  // slope: w'
  constexpr float kLog2e = 1.4426950408889634f;
  float2 w = mul2(z, make_float2(-kLog2e, -kLog2e));
  if constexpr (kAct == MF_ACT_GELU_TANH) {
    constexpr float kBeta = 1.5957691216057308f, kKappa = 0.044715f;
    const float2 c = make_float2(fminf(fmaxf(z.x, -64.f), 64.f), fminf(fmaxf(z.y, -64.f), 64.f)), c2 = mul2(c, c);
    const float a = -kLog2e * kBeta;
    w = mul2(c, fma2(c2, make_float2(a * kKappa, a * kKappa), make_float2(a, a)));
    slope = fma2(c2, make_float2(3.f * kBeta * kKappa, 3.f * kBeta * kKappa), make_float2(kBeta, kBeta));
  }
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(w.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(w.y));
  e = add2(e, make_float2(1.f, 1.f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(e.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(e.y));
  return e;
}
template <int kAct>
__device__ __forceinline__ float2 activation2(float2 z) {
  float2 unused;
  return mul2(z, logistic2<kAct>(z, unused));
}
// act(z) and act'(z)
template <int kAct>
__device__ __forceinline__ void activation2(float2 z, float2& value, float2& slope) {
  float2 dw;
  const float2 s = logistic2<kAct>(z, dw);
  value = mul2(z, s);
  float2 t = mul2(value, fma2(s, make_float2(-1.f, -1.f), make_float2(1.f, 1.f)));
  if constexpr (kAct == MF_ACT_GELU_TANH) t = mul2(t, dw);
  slope = add2(s, t);
}

// The forward pass of at most kSmallRows tokens (gated_mlp_small.cu).
constexpr int kSmallRows = 32;
int gated_mlp_small_forward(const MfGatedMlpArgs* a, cudaStream_t stream);

}  // namespace mf
