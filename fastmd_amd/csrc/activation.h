// Activations of the feed-forward block and the group norm, and their derivatives, in float32.
#pragma once

#include "common.h"

constexpr int kActNone = 0, kActSilu = 1, kActGelu = 2, kActRelu = 3;

struct ActValue {
  float value, slope;
};

// exp(x) to 2 ulp: 2^t by the instruction, t = x log2(e), and what the rounding of t left. |x| is cut at 104, where exp is 0 or infinite.
__device__ __forceinline__ float exp_near(float x) {
  x = __builtin_amdgcn_fmed3f(x, -104.f, 104.f);
  const float t = x * 1.44269502162933f, rest = fmaf(x, 1.92596303e-8f, fmaf(x, 1.44269502162933f, -t));
  return __builtin_amdgcn_exp2f(t) * fmaf(rest, 0.69314718f, 1.f);
}

// silu: z s, s (1 + z (1 - s)) with s = 1 / (1 + exp(-z)) (reciprocal to 1 ulp; 1 - s = exp(-z) s where s is near 1); gelu: z P,
// P + z p with the normal distribution P(z) = (1 + erf(z / sqrt 2)) / 2 and its density p. FAST, for results that are rounded
// to bf16 at once: silu's exponential by the instruction alone, off by |z| 2^-24 of itself, and 1 - s as it is.
template <bool FAST = false>
__device__ __forceinline__ ActValue activation(float z, int act) {
  if (act == kActSilu) {
    if (FAST) {
      const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
      return {z * s, s * fmaf(z, 1.f - s, 1.f)};
    }
    const float e = exp_near(-z), s = __builtin_amdgcn_rcpf(1.f + e);
    return {z * s, s * (1.f + z * (z < 0.f ? 1.f - s : e * s))};
  }
  if (act == kActGelu) {
    // 0.5 erfc(-z / sqrt 2): no cancellation where z is far below 0
    const float p = 0.5f * erfcf(-z * 0.70710678118654752f);
    return {z * p, p + z * exp_near(-0.5f * z * z) * 0.39894228040143268f};
  }
  if (act == kActRelu) return {z > 0.f || z != z ? z : 0.f, z > 0.f ? 1.f : 0.f};
  return {z, 1.f};
}
