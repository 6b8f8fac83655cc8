// Activations of the feed-forward block and the group norm, and their derivatives, in float32.
#pragma once

#include "common.h"

constexpr int kActNone = 0, kActSilu = 1, kActGelu = 2, kActRelu = 3;

struct ActValue {
  float value, slope;
};

// silu: z s, s (1 + z (1 - s)) with s = 1 / (1 + exp(-z)) (reciprocal to 1 ulp; 1 - s = exp(-z) s where s is near 1); gelu: z P, P + z p with the normal
// distribution P(z) = (1 + erf(z / sqrt 2)) / 2 and its density p
__device__ __forceinline__ ActValue activation(float z, int act) {
  if (act == kActSilu) {
    const float e = expf(-z), s = __builtin_amdgcn_rcpf(1.f + e);
    return {z * s, s * (1.f + z * (z < 0.f ? 1.f - s : e * s))};
  }
  if (act == kActGelu) {
    // 0.5 erfc(-z / sqrt 2): no cancellation where z is far below 0
    const float p = 0.5f * erfcf(-z * 0.70710678118654752f);
    return {z * p, p + z * expf(-0.5f * z * z) * 0.39894228040143268f};
  }
  if (act == kActRelu) return {z > 0.f || z != z ? z : 0.f, z > 0.f ? 1.f : 0.f};
  return {z, 1.f};
}
