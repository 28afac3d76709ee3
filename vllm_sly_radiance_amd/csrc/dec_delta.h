// What the forms of the gated delta rule share: the gates of a token and value head.
#pragma once
#include <hip/hip_runtime.h>

namespace dec {

__device__ __forceinline__ float decay_rate(float a_log) { return -expf(a_log); }

// g = -exp(a_log) softplus(a + dt_bias), rate = decay_rate(a_log).
__device__ __forceinline__ float log_decay(float a, float rate, float dt_bias) {
  const float x = a + dt_bias;
  return rate * (fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))));
}

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

}  // namespace dec
