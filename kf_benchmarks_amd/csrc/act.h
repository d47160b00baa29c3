// Activations fused into group norm, the causal convolution and the selective
// scan, as functions of the value u before the activation.
#pragma once
#include "common.h"

namespace kfb {

// codes of ops/nn.py _FUSED_ACTS
enum FusedAct : int { ACT_LINEAR = 0, ACT_RELU = 1, ACT_RELU6 = 2, ACT_TANH = 3, ACT_SILU = 4 };

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// v_exp_f32 / v_rcp_f32 are good to about 1 ulp; log2(e) u is rounded once, a
// relative error of |u| 2^-24 in the exponential and less in the sigmoid.
__device__ __forceinline__ float sigmoidf(float u) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * u));
}

// u * sigmoid(u): below about -88 the exponential is infinite and u * 0 = -0,
// but -inf * 0 would be NaN: the limit is 0.  (NaN comes through the sigmoid.)
__device__ __forceinline__ float siluf(float u) { return fmaxf(u, -3.4e38f) * sigmoidf(u); }

__device__ __forceinline__ float dsiluf(float u) {
  const float s = sigmoidf(u);
  if (s == 0.f) return 0.f;  // u (1 - s) s with u = -inf
  if (u == INFINITY) return 1.f;
  return s * (1.f + u * (1.f - s));
}

__device__ __forceinline__ float tanh_f(float u) {
  // 1 - 2 / (1 + e^{2|u|}); near 0 the odd series, where the difference cancels
  const float a = fabsf(u);
  const float e = __builtin_amdgcn_exp2f(2.f * LOG2E * a);
  const float big = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + e);
  const float q = a * a;
  const float small =
      a * (1.f + q * (-1.f / 3 + q * (2.f / 15 + q * (-17.f / 315 + q * (62.f / 2835)))));
  return copysignf(a < 0.25f ? small : big, u);
}

// The piecewise linear ones are y = clamp(u, lo, hi), with comparisons that are
// false for NaN: NaN stays NaN, and NaN bounds clamp nothing.
enum ActClass : int { CLAMP = 0, TANH = 1, SILU = 2 };

struct Act {
  int kind;  // ActClass: a template parameter of the kernels
  float lo, hi;
};

inline Act act_of(int code) {
  const float none = __builtin_nanf("");
  switch (code) {
    case ACT_RELU: return Act{CLAMP, 0.f, none};
    case ACT_RELU6: return Act{CLAMP, 0.f, 6.f};
    case ACT_TANH: return Act{TANH, none, none};
    case ACT_SILU: return Act{SILU, none, none};
    default: return Act{CLAMP, none, none};
  }
}

template <int KIND> __device__ __forceinline__ float act_fwd(float u, const Act& a) {
  if constexpr (KIND == TANH) return tanh_f(u);
  else if constexpr (KIND == SILU) return siluf(u);
  else return u < a.lo ? a.lo : u > a.hi ? a.hi : u;
}

// dact/du at u; the gradient at the kinks 0 and 6 is 0.
template <int KIND> __device__ __forceinline__ float act_grad(float u, const Act& a) {
  if constexpr (KIND == TANH) {
    const float t = tanh_f(u);
    return 1.f - t * t;
  } else if constexpr (KIND == SILU) {
    return dsiluf(u);
  } else {
    return u <= a.lo || u >= a.hi ? 0.f : 1.f;
  }
}

#define KFB_DISPATCH_ACT(kind, KIND, ...)                             \
  switch (kind) {                                                     \
    case kfb::TANH: { constexpr int KIND = kfb::TANH; __VA_ARGS__; break; } \
    case kfb::SILU: { constexpr int KIND = kfb::SILU; __VA_ARGS__; break; } \
    default: { constexpr int KIND = kfb::CLAMP; __VA_ARGS__; break; }  \
  }

// log(1 + e^v) = max(v, 0) + log1p(e), e = e^-|v|, to a few ulp for any v.
// The rounding error of log2(e) |v|, kept from the fused multiply-add, comes back
// as a first-order factor of e.  With w = 1 + e rounded and c = e - (w - 1), both
// exact, log1p(e) = log(w) + c / w, and c alone is as good: it counts where w is
// near 1 (for small e log(w) loses what the rounding of w drops).
__device__ __forceinline__ float softplusf(float v) {
  const float m = fmaxf(-fabsf(v), -200.f);  // e^-200 is 0 either way
  const float p = LOG2E * m, lo = fmaf(LOG2E, m, -p);
  float e = __builtin_amdgcn_exp2f(p);
  e = fmaf(e, LN2 * lo, e);
  const float w = 1.f + e;
  return fmaf(LN2, __builtin_amdgcn_logf(w), e - (w - 1.f)) + (v < 0.f ? 0.f : v);  // NaN stays
}

}  // namespace kfb
