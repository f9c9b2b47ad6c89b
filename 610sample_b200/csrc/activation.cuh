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

// The fast form of two elements at a time, in packed arithmetic: the products' epilogues compute it for every element of a tile, in the time that the
// tensor cores take for the next one.  a(z), for any z; with GRAD its derivative too, for finite z and NaN.
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float bounded(float v, float most) {      // NaN stays
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(most));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(-most));
  return v;
}
template <int ACT, bool GRAD>
__device__ __forceinline__ void activate2(float2 z, float2& a, float2& d) {
  if constexpr (ACT == ACT_NONE) {
    a = z;
    d = both(1.f);
  } else if constexpr (ACT == ACT_GELU) {
    const float2 m = make_float2(fminf(fabsf(z.x), 40.f), fminf(fabsf(z.y), 40.f));      // what lies below 40 is 0; NaN comes back with z itself
    const float2 t1 = __ffma2_rn(both(0.31f), m, both(1.f)), t = make_float2(fast_rcp(t1.x), fast_rcp(t1.y));
    const float2 q = __fmul2_rn(__fmul2_rn(m, m), both(-0.5f * kLog2e)), e = make_float2(tc::ex2(q.x), tc::ex2(q.y));
    float2 p = __ffma2_rn(both(-0.07392913f), t, both(0.18045032f));
    p = __ffma2_rn(p, t, both(0.01574473f));
    p = __ffma2_rn(p, t, both(0.13342978f));
    p = __ffma2_rn(p, t, both(0.12044128f));
    p = __ffma2_rn(p, t, both(0.1238607f));
    const float2 below = __fmul2_rn(__fmul2_rn(e, t), p), half = __fmul2_rn(z, both(0.5f));
    // max(z, 0) - |z| F(-|z|)
    a = __ffma2_rn(make_float2(-m.x, -m.y), below, make_float2(fmaf(0.5f, fabsf(z.x), half.x), fmaf(0.5f, fabsf(z.y), half.y)));
    if constexpr (GRAD) {
      const float2 F = make_float2(z.x < 0.f ? below.x : 1.f - below.x, z.y < 0.f ? below.y : 1.f - below.y);
      d = __ffma2_rn(__fmul2_rn(z, both(0.3989422804014327f)), e, F);
    }
  } else {
    constexpr float kRoot = 1.5957691216057308f, kCube = 0.044715f;      // sqrt(8 / pi)
    float2 c = z, u = z;
    if constexpr (ACT == ACT_GELU_TANH) {
      if constexpr (GRAD) c = make_float2(bounded(z.x, 30.f), bounded(z.y, 30.f));
      u = __fmul2_rn(c, __ffma2_rn(__fmul2_rn(c, c), both(kRoot * kCube), both(kRoot)));
    }
    const float2 q = __fmul2_rn(u, both(-kLog2e)), e = __fadd2_rn(make_float2(tc::ex2(q.x), tc::ex2(q.y)), both(1.f));
    const float2 s = make_float2(fast_rcp(e.x), fast_rcp(e.y));
    a = __fmul2_rn(z, s);
    if constexpr (GRAD) {      // a' = s + c u' s (1 - s)
      float2 w = __fmul2_rn(c, s);
      if constexpr (ACT == ACT_GELU_TANH) w = __fmul2_rn(w, __ffma2_rn(__fmul2_rn(c, c), both(3.f * kRoot * kCube), both(kRoot)));
      d = __ffma2_rn(w, __fadd2_rn(both(1.f), make_float2(-s.x, -s.y)), s);
    }
  }
}

// What a gated product keeps of a half-precision call, 20 bits a value: 16 in a plane of the type's size, and 4 of either value in a plane of bytes.  A
// product of two values that were rounded to the type, rounded again, would have gradients 3.0e-3 (bf16) from 64 bits in the 2-norm, where rounding the
// gradients' own factors and results makes 2.4e-3; 4 more bits cost 1 byte beside 4.  bf16: sign, 8 bits of exponent, 11 of mantissa; f16: 6 and
// 13, since a(z) u may be in its range where z or u is not.  Codes are the nearest ones and are read as they stand, so that 0 stays 0: what gradients have
// as a factor vanishes with it.
template <typename T> struct Kept;
template <> struct Kept<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t code(float v) {      // in the upper 20 bits
    const uint32_t b = __float_as_uint(v);
    return (b & 0x80000000u) | min((b & 0x7fffffffu) + 0x800u, 0x7fc00000u);      // NaN would carry into the sign
  }
  static __device__ __forceinline__ float value(uint32_t code) { return __uint_as_float(code & 0xfffff000u); }
};
template <> struct Kept<__half> {
  // the exponent moved to where 6 bits hold it: normal numbers from 2^-15, below them 2^-28 apart; from 2^46 on NaN
  static __device__ __forceinline__ uint32_t code(float v) {
    const uint32_t b = __float_as_uint(v * 0x1p-111f);
    return (b & 0x80000000u) | min((b & 0x7fffffffu) + 0x200u, 0x1f800000u) << 2;
  }
  static __device__ __forceinline__ float value(uint32_t code) {
    const float v = __uint_as_float((code & 0x80000000u) | (code & 0x7ffff000u) >> 2) * 0x1p111f;
    return fabsf(v) >= 0x1p46f ? NAN : v;      // the codes that are f16's NaN and infinities
  }
};
// The planes' words of four values of either: the upper halves in pairs, and a word of bytes, bits of z low and of u high
__device__ __forceinline__ uint32_t kept_high(uint32_t c0, uint32_t c1) { return __byte_perm(c0, c1, 0x7632); }
__device__ __forceinline__ uint32_t kept_nibbles(const uint32_t (&c)[4]) {      // bits 12 to 15 of each, in the upper halves of bytes
  return __byte_perm(__byte_perm(c[0], c[1], 0x0051), __byte_perm(c[2], c[3], 0x0051), 0x5410);
}
__device__ __forceinline__ uint32_t kept_low(const uint32_t (&z)[4], const uint32_t (&u)[4]) {
  return (kept_nibbles(z) >> 4 & 0x0f0f0f0fu) | (kept_nibbles(u) & 0xf0f0f0f0u);
}
// the codes of value E of four from the halves' pair that holds it and the nibbles' word, 0xf0 or 0x0f of `low` in its place
__device__ __forceinline__ uint32_t kept_z(uint32_t low) { return low << 4 & 0xf0f0f0f0u; }
__device__ __forceinline__ uint32_t kept_u(uint32_t low) { return low & 0xf0f0f0f0u; }
template <int E> __device__ __forceinline__ uint32_t kept_code(uint32_t high, uint32_t nibbles) {
  constexpr uint32_t kHalf = (E & 1) ? 0x3200u : 0x1000u;      // the half's two bytes on top, the nibble's byte below; what is below that is not read
  return __byte_perm(high, nibbles, kHalf | (4u + E) << 4 | (4u + E));
}

// f(tc::Int<activation>): the switch lies outside of the loops over elements
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  if (act == ACT_SILU) f(tc::Int<ACT_SILU>{});
  else if (act == ACT_GELU) f(tc::Int<ACT_GELU>{});
  else if (act == ACT_GELU_TANH) f(tc::Int<ACT_GELU_TANH>{});
  else f(tc::Int<ACT_NONE>{});
}

// Two arguments of an activation that are kept for the backward, of half types in f16 within its finite range: three more bits than bf16 has, and beyond 65504
// every derivative is what it is there.  (Kept in bf16, the gradients of
// 300 x 768 -> 520 were 2.4e-3 from 64 bits in the 2-norm; 2.3e-3 now.)
__device__ __forceinline__ uint32_t pack_argument(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T> struct ArgumentOf { typedef __half type; };
template <> struct ArgumentOf<float> { typedef float type; };

}  // namespace attn
