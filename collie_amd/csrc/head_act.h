// Activations of the linear and gated layers, in float32: f(z) and f'(z).
#pragma once

#include "head_types.h"

namespace collie {

constexpr float kLeakySlope = 0.01f;  // F.leaky_relu's default, as in the hybrid head

// exp(x + low), x of magnitude below 100 and low a part below its last bit: 2^t with t = x log2(e) in two
// parts (the product and what it was rounded by).  The library's expf and division took a third of the
// gated layer's forward pass (16,384 x 2,048 x 5,504: 988 us with them).
__device__ __forceinline__ float fast_exp(float x, float low = 0.0f) {
  const float t = x * 1.44269504f;
  const float rest = fmaf(x, 1.44269504f, -t) + fmaf(x, 1.92596299e-8f, low * 1.44269504f);
  const float e = __builtin_amdgcn_exp2f(t);
  // beyond, e is at an end of the range (infinite times a correction would be NaN)
  return fabsf(t) < 126.0f ? fmaf(e, rest * 0.693147181f, e) : e;
}
// 1 / (1 + exp(-z)) to about two steps of float32
__device__ __forceinline__ float fast_sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + fast_exp(-z));
}

// Phi(z), the normal distribution function, to eight half steps of float32 of its value on either side,
// and exp(-z^2 / 2) with it, without a branch: Phi(-|z|) = t P(t) exp(-z^2 / 2), t = 1 / (1 + 0.35 |z|).
// P is the polynomial of degree 8 with the least relative error (3.2e-8) against
// erfc(x) exp(x^2) / (2 t), x = |z| / sqrt(2), over |z| <= 14, found by Remez's exchange from erfc in
// 40 digits.  What z^2 is rounded by would be 50 half steps of the exponential at |z| = 10, so it goes in
// as the low part.  The library's erff cost the forward pass of 720,896 x 256 x 128 (float32) 100 us of
// 580.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, fabsf(z), 1.0f));
  float p = fmaf(t, -0.0291459142f, 0.143971623f);
  p = fmaf(t, p, -0.255714108f);
  p = fmaf(t, p, 0.159174003f);
  p = fmaf(t, p, -0.0231097335f);
  p = fmaf(t, p, 0.105507964f);
  p = fmaf(t, p, 0.119832877f);
  p = fmaf(t, p, 0.139861868f);
  p = fmaf(t, p, 0.139621404f);
  const float h = z * z;
  e = fast_exp(-0.5f * h, -0.5f * fmaf(z, z, -h));
  const float tail = p * t * e;
  return z < 0.0f ? tail : 1.0f - tail;
}

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
      for (int i = 0; i < N; ++i) v[i] = fast_sigmoid(v[i]);
      break;
    case COLLIE_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] * fast_sigmoid(v[i]);
      break;
    case COLLIE_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float e;
        v[i] *= normal_cdf(v[i], e);
      }
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
        v[i] = fast_sigmoid(v[i]);
        d[i] = v[i] * (1.0f - v[i]);
      }
      break;
    case COLLIE_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float s = fast_sigmoid(v[i]);
        d[i] = s * (1.0f + v[i] * (1.0f - s));
        v[i] *= s;
      }
      break;
    case COLLIE_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float e;
        const float cdf = normal_cdf(v[i], e);
        d[i] = fmaf(v[i] * 0.39894228f, e, cdf);
        v[i] *= cdf;
      }
      break;
    default:
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = 1.0f;
      break;
  }
}

// Pre-activations kept for the backward pass are float32, in the linear layer (where f' is smooth) and in
// the gated one (whose gradients contain f, f' and u).  16 bits of z are not enough for f'(z): a relative
// change d of z is one of d z f''(z) / f'(z), |z| times as much in a sigmoid's tail and without bound next
// to the zero of silu's or gelu's slope.  Of relu and leaky_relu only the sign counts, so the linear layer
// keeps their z in its own type, and what is positive as something positive.
__host__ __device__ constexpr bool kept_in_float(int act) { return act >= COLLIE_ACT_SIGMOID; }

template <typename T>
__device__ __forceinline__ float kept_sign(float z) {
  constexpr float least = std::is_same<T, f16_t>::value ? 6.10351562e-5f : 1.17549435e-38f;
  return z > 0.0f && z < least ? least : z;
}

}  // namespace collie
