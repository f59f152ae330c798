// A gate's arithmetic: h = act(g) u and its gradients.
#pragma once
#include "common.h"

namespace sd {

// act(g).  SILU: g / (1 + exp(-g)), one exponential and one reciprocal, 4 roundings and g's of the exponent: within 2^-21 of itself where |g| < 16.
// An exponential that overflows gives the zero that the quotient rounds to.
__device__ inline float gate_value(int act, float g) {
  if (act == SD_ACT_SILU) return g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f));
  return act_apply(act, g);
}
// act(g) and act'(g) together: they share what is dear.  GELU: Phi(g) from the root of its tail, phi(g) one exponential more.
__device__ inline void gate_slope(int act, float g, float& value, float& slope) {
  if (act == SD_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f));
    value = g * s;
    slope = __builtin_fmaf(value, 1.f - s, s);
  } else if (act == SD_ACT_GELU) {
    const float root = normal_tail_root(fabsf(g)), below = g >= 0.f ? __builtin_fmaf(-root, root, 1.f) : root * root;
    value = g * below;
    slope = __builtin_fmaf(g * 0.39894228040143268f, __builtin_amdgcn_exp2f((g * -0.72134752044448170f) * g), below);
  } else {
    value = act_apply(act, g);
    slope = act_derivative(act, g);
  }
}

}  // namespace sd
