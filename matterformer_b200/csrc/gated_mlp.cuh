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

// ---- pre-activations between the passes ------------------------------------------------------------------------------
// Kept in 16 bits, 16 neighbouring channels of a token scaled by a power of two that goes by the largest, with its exponent in a byte (the
// bytes of 64 channels, four for gate, four for up, lie together, token by token).  Rounded to the block's type like everything else
// that goes through memory, they alone put the gradients 1.75 times as far from 64 bits as the rounding of the gradients does;
// with a bit more it is 1.5 times, with three 1.4.  With P the power of two in the largest of a group:
//   bf16: fp16 with the largest below 2^15: 11 bits down to 2^-28 P.
//   fp16: sign, 4 bits of exponent, 11 of fraction: 12 bits down to 2^-13 P, from there steps of 2^-24 P.  What an fp32 value below
//   2^-112 has in its bits 12-26 is that form, subnormals included: a multiplication and a shift round to it.  (3 bits of exponent and 12 of
//   fraction keep a bit more of most values, but less than fp16 itself from 2^-7 P on and nothing below 2^-18 P: channels beside an
//   outlier would lose their gradients.)
// A group with an infinity or NaN: bf16 passes it on beside the values that fp16 can hold; fp16 is NaN in all 16.
// The larger of two magnitudes: in fp16 a NaN wins, so that its group is known; in bf16 the others decide, a NaN needs no exponent.
template <typename T>
__device__ __forceinline__ float group_max(float a, float b) {
  if constexpr (!std::is_same<T, __half>::value) return fmaxf(a, b);
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t group_exponent(float largest) {  // of the largest magnitude
  const uint32_t e = __float_as_uint(largest) >> 23;
  return e == 255u ? (std::is_same<T, __half>::value ? 255u : 141u) : e < 15u ? 15u : e;
}
__device__ __forceinline__ float2 twice(float x) { return make_float2(x, x); }
template <typename T>
__device__ __forceinline__ float2 group_scale(uint32_t exponent) {
  return twice(__uint_as_float((268u - exponent) << 23));  // the largest comes below 2^15
}
template <typename T>
__device__ __forceinline__ float2 group_unscale(uint32_t exponent) {
  if (std::is_same<T, __half>::value && exponent == 255u) return twice(__uint_as_float(0x7fffffffu));
  return twice(__uint_as_float((exponent - 14u) << 23));
}
template <typename T>
__device__ __forceinline__ uint32_t pack_pre(float2 v, float2 scale) {
  v = mul2(v, scale);
  if constexpr (std::is_same<T, __half>::value) {
    v = mul2(v, twice(__uint_as_float(1u << 22)));  // 2^-127
    const uint32_t a = __float_as_uint(v.x) + 0x800u, b = __float_as_uint(v.y) + 0x800u;
    return (a >> 12 & 0x7fffu) | (a >> 16 & 0x8000u) | (b << 4 & 0x7fff0000u) | (b & 0x80000000u);
  } else {
    return pack2<__half>(v.x, v.y);
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack_pre(uint32_t w, float2 unscale) {
  float2 v;
  if constexpr (std::is_same<T, __half>::value) {
    v = make_float2(__uint_as_float((w << 12 & 0x07fff000u) | (w << 16 & 0x80000000u)), __uint_as_float((w >> 4 & 0x07fff000u) | (w & 0x80000000u)));
    v = mul2(v, twice(__uint_as_float(254u << 23)));  // 2^127
  } else {
    v = unpack2<__half>(w);
  }
  return mul2(v, unscale);
}
inline size_t gated_mlp_pre_values(int64_t rows, int64_t hidden) { return align_up((size_t)rows * 2 * (size_t)hidden * 2, 256); }  // bytes before the exponents

// The kernels for few tokens (gated_mlp_small.cu) take up to 16, up to 32 where there are few weights: they read the tokens again for
// every 16 channels.  us, 16 | 17 | 32 tokens there, 33 on tcgen05 tiles: 512 x 2048 7.7 | 9.9 | 11.1, 12.8; 1024 x 4096 14 | 23 | 27, 20;
// 2048 x 8192 28 | 40 | 43, 32; 4096 x 10 928 73 | 93 | 103, 68.
inline bool gated_mlp_small(const MfGatedMlpArgs* a) { return a->rows <= 16 || (a->rows <= 32 && (int64_t)a->dim * a->hidden <= 1 << 21); }
int gated_mlp_small_forward(const MfGatedMlpArgs* a, cudaStream_t stream);

}  // namespace mf
