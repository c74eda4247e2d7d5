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
// with two more bits it is 1.45 times, with three 1.42.  With P the power of two in the largest of a group:
//   bf16: fp16 with the largest below 2^15: 11 bits down to 2^-28 P.
//   fp16: sign, 3 bits of exponent, 12 of fraction: 13 bits down to 2^-5 P, from there steps of 2^-17 P.  That is less than fp16 itself has
//   from 2^-7 P on, and channels beside an outlier would lose their gradients: a group with such a value takes a bit of the fraction for the
//   exponent, 12 bits down to 2^-13 P and steps of 2^-24 P below, and the byte's top bit.  (That form for all groups: 1.52 times.)  What
//   an fp32 value below 2^-120 (2^-112) has in its bits 11-25 (12-26) is that form, subnormals included: a multiplication and a shift round
//   to it.  The exponent, from 2^-62 to 2^62, takes 7 bits: sums of products of fp16 values are multiples of 2^-48, at most 2^60.
// A group with an infinity or NaN: bf16 passes it on beside the values that fp16 can hold; fp16 is NaN in all 16.
template <typename T>
struct PreGroup {  // magnitudes of a group
  float most = 0.f, least = INFINITY;
  // in fp16 a NaN wins, so that its group is known; in bf16 the others decide, a NaN needs no exponent
  __device__ __forceinline__ static float larger(float a, float b) {
    if constexpr (!std::is_same<T, __half>::value) return fmaxf(a, b);
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
  }
  __device__ __forceinline__ void add(float a, float b) {
    most = larger(most, larger(fabsf(a), fabsf(b)));
    least = fminf(least, fminf(fabsf(a), fabsf(b)));
  }
  __device__ __forceinline__ void exchange(uint32_t lanes, int with) {
    most = larger(most, __shfl_xor_sync(lanes, most, with));
    least = fminf(least, __shfl_xor_sync(lanes, least, with));
  }
  __device__ __forceinline__ uint32_t code() const {
    uint32_t e = __float_as_uint(most) >> 23;
    if constexpr (!std::is_same<T, __half>::value) return e == 255u ? 141u : e < 15u ? 15u : e;
    if (e > 189u) return 127u;
    if (e < 65u) e = 65u;
    return (e - 64u) | (least < __uint_as_float((e - 7u) << 23) ? 128u : 0u);
  }
};
__device__ __forceinline__ float2 twice(float x) { return make_float2(x, x); }
// What a group's code says: the factor that brings the largest to [2^14, 2^15) or back from there; in fp16 how the bits are cut.
template <typename T>
struct PreForm {
  float2 factor, tiny;
  uint32_t narrow = 0u;  // fp16: a bit less of the fraction
  __device__ __forceinline__ PreForm(uint32_t code, bool back) {
    uint32_t e = code;
    if constexpr (std::is_same<T, __half>::value) {
      narrow = code >> 7, e = (code & 127u) + 64u;
      tiny = twice(__uint_as_float(narrow ? 1u << 22 : 1u << 14));  // 2^-127 : 2^-135
      factor = twice(__uint_as_float(!back ? (268u - e) << 23 : e == 191u ? 0x7fffffffu : (e - (narrow ? 14u : 6u)) << 23));
    } else {
      factor = twice(__uint_as_float((back ? e - 14u : 268u - e) << 23));
    }
  }
  __device__ __forceinline__ uint32_t pack(float2 v) const {
    v = mul2(v, factor);
    if constexpr (std::is_same<T, __half>::value) {
      v = mul2(v, tiny);
      const uint32_t half = 0x400u << narrow, a = __float_as_uint(v.x) + half, b = __float_as_uint(v.y) + half;
      return (a >> (11u + narrow) & 0x7fffu) | (a >> 16 & 0x8000u) | (b << (5u - narrow) & 0x7fff0000u) | (b & 0x80000000u);
    } else {
      return pack2<__half>(v.x, v.y);
    }
  }
  __device__ __forceinline__ float2 unpack(uint32_t w) const {
    float2 v;
    if constexpr (std::is_same<T, __half>::value) {
      const uint32_t a = (w & 0x7fffu) << (11u + narrow), b = (w & 0x7fff0000u) >> (5u - narrow);
      v = make_float2(__uint_as_float(a | (w << 16 & 0x80000000u)), __uint_as_float(b | (w & 0x80000000u)));
      v = mul2(v, twice(__uint_as_float(254u << 23)));  // 2^127
    } else {
      v = unpack2<__half>(w);
    }
    return mul2(v, factor);
  }
};
inline size_t gated_mlp_pre_values(int64_t rows, int64_t hidden) { return align_up((size_t)rows * 2 * (size_t)hidden * 2, 256); }  // bytes before the exponents

// The kernels for few tokens (gated_mlp_small.cu) take up to 16, up to 32 where there are few weights: they read the tokens again for
// every 16 channels.  us, 16 | 17 | 32 tokens there, 33 on tcgen05 tiles: 512 x 2048 7.7 | 9.9 | 11.1, 12.8; 1024 x 4096 14 | 23 | 27, 20;
// 2048 x 8192 28 | 40 | 43, 32; 4096 x 10 928 73 | 93 | 103, 68.  (The line goes by the number of tokens: between 9 and 16 of them the widest
// weights lose some 5 us to it.)
inline bool gated_mlp_small(const MfGatedMlpArgs* a) { return a->rows <= 16 || (a->rows <= 32 && (int64_t)a->dim * a->hidden <= 1 << 21); }
int gated_mlp_small_forward(const MfGatedMlpArgs* a, cudaStream_t stream);

}  // namespace mf
