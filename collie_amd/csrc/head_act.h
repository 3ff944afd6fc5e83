// Activations of the linear and gated layers, in float32: f(z) and f'(z).
#pragma once

#include "head_types.h"

namespace collie {

constexpr float kLeakySlope = 0.01f;  // F.leaky_relu's default, as in the hybrid head

// f(z) over N values; `act` is the same for the whole launch, so the branch is taken once
template <int N>
__device__ __forceinline__ void act_values(int act, float (&v)[N]) {
  switch (act) {
    case COLLIE_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] > 0.0f || v[i] != v[i] ? v[i] : 0.0f;
      break;
    case COLLIE_ACT_LEAKY_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] > 0.0f ? v[i] : v[i] * kLeakySlope;
      break;
    case COLLIE_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = sigmoidf_(v[i]);
      break;
    case COLLIE_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] * sigmoidf_(v[i]);
      break;
    case COLLIE_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] * (0.5f * (1.0f + erff(v[i] * 0.70710678118654752f)));
      break;
    default: break;
  }
}

// v = f(z) and d = f'(z); the slope of relu and leaky_relu at 0 is that of the negative side
template <int N>
__device__ __forceinline__ void act_slopes(int act, float (&v)[N], float (&d)[N]) {
  switch (act) {
    case COLLIE_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        d[i] = v[i] > 0.0f ? 1.0f : 0.0f;
        v[i] = v[i] > 0.0f || v[i] != v[i] ? v[i] : 0.0f;
      }
      break;
    case COLLIE_ACT_LEAKY_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        d[i] = v[i] > 0.0f ? 1.0f : kLeakySlope;
        v[i] *= d[i];
      }
      break;
    case COLLIE_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] = sigmoidf_(v[i]);
        d[i] = v[i] * (1.0f - v[i]);
      }
      break;
    case COLLIE_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float s = sigmoidf_(v[i]);
        d[i] = s * (1.0f + v[i] * (1.0f - s));
        v[i] *= s;
      }
      break;
    case COLLIE_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float cdf = 0.5f * (1.0f + erff(v[i] * 0.70710678118654752f));
        d[i] = cdf + v[i] * (0.39894228040143268f * expf(-0.5f * v[i] * v[i]));
        v[i] *= cdf;
      }
      break;
    default:
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = 1.0f;
      break;
  }
}

// A pre-activation kept for the backward pass.  It is kept in the layer's own type: f' and f of it
// are off by half a step of that type times a slope of about one, which is what the gradient is
// rounded by anyway, and float32 would double what the forward pass writes.  float16 ends at 65504,
// where every activation here has reached its end: a larger value is kept as that one, because an
// infinity would turn z (1 - sigmoid(z)) into inf * 0.
template <typename T>
__device__ __forceinline__ float kept(float z) {
  return z;
}
template <>
__device__ __forceinline__ float kept<f16_t>(float z) {
  return fabsf(z) < INFINITY ? fminf(fmaxf(z, -65504.0f), 65504.0f) : z;
}

}  // namespace collie
