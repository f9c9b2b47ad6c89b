// Activations with their first two derivatives, in fp32.
//
//   silu       a = z s, s = 1 / (1 + e^-z)                        a' = s (1 + z (1 - s))       a'' = s (1 - s) (2 + z (1 - 2 s))
//   gelu       a = z F, F the normal distribution, f its density  a' = F + z f                 a'' = f (2 - z^2)
//   gelu_tanh  a = z s(u), u = sqrt(8 / pi) (z + 0.044715 z^3): (1 + tanh(u / 2)) / 2 is s(u), which keeps its relative precision for z < 0
//
// Two forms.  Precise: the CUDA library's functions, for float32.  Fast, for results that are rounded to 11 bits or fewer: ex2 and rcp
// (2^-22 each), and F(-a) = e^(-a^2 / 2) P(1 / (1 + 0.31 a)) for a >= 0: the form of Hastings' approximations of the error function, P of
// degree 6 fitted to the relative error (4.7e-6 over 0 <= a <= 16), since a is used where F is 1e-5 as well.
#pragma once

#include "attn_b200.h"
#include "tc_common.cuh"

namespace attn {

enum Activation { ACT_NONE = ATTN_ACT_NONE, ACT_SILU = ATTN_ACT_SILU, ACT_GELU = ATTN_ACT_GELU, ACT_GELU_TANH = ATTN_ACT_GELU_TANH };

__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// s(u), s(-u) = 1 - s(u) and s(-u) - s(u), none of them a difference of larger numbers
struct Logistic { float s, rest, turn; };
template <bool PRECISE>
__device__ __forceinline__ Logistic logistic(float u) {
  const float e = PRECISE ? expf(-fabsf(u)) : tc::ex2(-kLog2e * fabsf(u));      // at most 1
  const float large = PRECISE ? 1.f / (1.f + e) : fast_rcp(1.f + e), small = e * large, turn = (1.f - e) * large;
  return u < 0.f ? Logistic{small, large, turn} : Logistic{large, small, -turn};
}

// F(z) and f(z)
template <bool PRECISE>
__device__ __forceinline__ void normal(float z, float& F, float& f) {
  constexpr float kDensity = 0.3989422804014327f;      // 1 / sqrt(2 pi)
  if constexpr (PRECISE) {
    F = normcdff(z);
    f = kDensity * expf(-0.5f * z * z);
  } else {
    const float a = fabsf(z), t = fast_rcp(fmaf(0.31f, a, 1.f)), e = tc::ex2(-0.5f * kLog2e * z * z);
    float p = -0.07392913f;
    p = fmaf(p, t, 0.18045032f);
    p = fmaf(p, t, 0.01574473f);
    p = fmaf(p, t, 0.13342978f);
    p = fmaf(p, t, 0.12044128f);
    p = fmaf(p, t, 0.1238607f);
    const float below = e * p * t;
    F = z < 0.f ? below : 1.f - below;
    f = kDensity * e;
  }
}

// a(z); with ORDER 1 and 2 its derivatives too.  Beyond the bound (what lies there is 0 or z in fp32) z is replaced by it wherever another
// factor is 0, so that no product of 0 and infinity is formed.
template <int ACT, bool PRECISE, int ORDER>
__device__ __forceinline__ void activate(float z, float& a, float& d1, float& d2) {
  constexpr float kBound = ACT == ACT_SILU ? 200.f : 30.f;
  const float c = fminf(fmaxf(z, -kBound), kBound);
  d1 = d2 = 0.f;
  if constexpr (ACT == ACT_NONE) {
    a = z;
    d1 = 1.f;
  } else if constexpr (ACT == ACT_SILU) {
    const Logistic l = logistic<PRECISE>(z);
    a = z * l.s;
    if constexpr (ORDER >= 1) d1 = l.s * fmaf(l.rest, c, 1.f);
    if constexpr (ORDER >= 2) d2 = l.s * l.rest * fmaf(c, l.turn, 2.f);
  } else if constexpr (ACT == ACT_GELU) {
    float F, f;
    normal<PRECISE>(c, F, f);
    a = z * F;
    if constexpr (ORDER >= 1) d1 = fmaf(c, f, F);
    if constexpr (ORDER >= 2) d2 = f * fmaf(-c, c, 2.f);
  } else {
    constexpr float kRoot = 1.5957691216057308f, kCube = 0.044715f;      // sqrt(8 / pi)
    const Logistic l = logistic<PRECISE>(kRoot * c * fmaf(kCube * c, c, 1.f));
    a = z * l.s;
    if constexpr (ORDER >= 1) {
      const float u1 = kRoot * fmaf(3.f * kCube * c, c, 1.f);
      d1 = l.s * fmaf(c * u1, l.rest, 1.f);
      if constexpr (ORDER >= 2) d2 = l.s * l.rest * fmaf(c, fmaf(l.turn * u1, u1, 6.f * kRoot * kCube * c), 2.f * u1);
    }
  }
  if (z != z) a = d1 = d2 = z;      // the bound drops it
}

// f(tc::Int<activation>): the switch lies outside of the loops over elements
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  if (act == ACT_SILU) f(tc::Int<ACT_SILU>{});
  else if (act == ACT_GELU) f(tc::Int<ACT_GELU>{});
  else if (act == ACT_GELU_TANH) f(tc::Int<ACT_GELU_TANH>{});
  else f(tc::Int<ACT_NONE>{});
}

// A value that is kept for the backward in T: within its finite range, so that the derivatives there are those of a very large z.
template <typename T> __device__ __forceinline__ float within(float v) { return v; }
template <> __device__ __forceinline__ float within<__half>(float v) { return v > 65504.f ? 65504.f : v < -65504.f ? -65504.f : v; }
template <> __device__ __forceinline__ float within<__nv_bfloat16>(float v) {
  constexpr float kMost = 3.3895313892515355e38f;
  return v > kMost ? kMost : v < -kMost ? -kMost : v;
}

}  // namespace attn
