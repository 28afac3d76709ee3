// What the forms of the gated delta rule share: the gates of a token and value head, and the lengths of keys and
// queries.
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

// A row's squares are added in fp32. Where they or the products with a state could leave its range, the row is
// scaled by a power of two first, which changes nothing else: p = unit_power(its largest magnitude) brings that to
// [1, 2) (what is below 2^-126 to less, what is above 2^127 to less than 4; what is not finite stays so).
__device__ __forceinline__ float unit_power(float top) {
  const int e = (int)(__float_as_uint(top) >> 23);
  return __uint_as_float((uint32_t)(254 - min(max(e, 1), 253)) << 23);
}
// Squares that need none of that: lengths of 2^-6 to 2^6, and so states up to 2^120.
__device__ __forceinline__ bool plain_squares(float x) { return x >= 0x1p-12f && x <= 0x1p12f; }
// x / sqrt(squares + eps p^2), the squares those of a row times p. (Where eps p^2 leaves the range, it is so much
// more than the squares, 2^36 at most, that they do not count.)
__device__ __forceinline__ float over_length(float x, float squares, float eps, float p) {
  const float least = eps * p;
  return least * p < __builtin_inff() ? x / sqrtf(fmaf(least, p, squares)) : x / (sqrtf(eps) * p);
}

}  // namespace dec
