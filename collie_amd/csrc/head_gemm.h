// The product that the linear and gated layers are made of (head_gemm.hip), and what is done to its
// results.
#pragma once

#include "head_act.h"

namespace collie {

// element (i, k) of an operand: p[i * rs + k * ks]
struct Mat {
  const void* p;
  int64_t rs, ks;
};

enum Epilogue { kEpiLinear, kEpiGated, kEpiStore };

struct Gemm {
  Mat a, b;
  const void* b2;        // second matrix of b's shape, or NULL
  int64_t k_split;       // without kEpiGated: k >= k_split reads b2 at k - k_split, and of either
  int64_t k_valid;       // matrix only the first k_valid are there (the rest is padding: zero)
  int64_t m, n, k;
  // the first `full` tiles are computed whole; the depth of the others is cut into `splits` parts of
  // k_chunk, whose sums go to partial [splits, tiles - full, accumulators, tile rows, tile columns]
  int64_t full;
  int splits;
  int64_t k_chunk;
  float* partial;
  // epilogue
  int act;
  const void *bias, *bias2;
  const void* residual;
  int64_t res_ld;
  void *keep, *keep2;    // pre-activations for the backward pass [m, n], or NULL (see head_act.h)
  void *c, *c2;          // output [m, n]; with kEpiStore rows >= row_split are c2's, and of either
  int64_t row_split;     // only the first row_valid are wanted
  int64_t row_valid;
  bool stream;           // the results are stored past the caches
  const uint32_t* over;  // float16, kEpiStore: where not 0, a is kDzScale times what it stands for
};

// float16 ends at 65504, and an activation gradient (dy u f'(g) in the gated layer) may go past that
// although its products with the weights do not.  Where any finite one of a call does, all are stored
// times this power of two, and the products are divided by it again in float32.  Values below 2^-17 are
// then rounded to multiples of it, so it is no smaller: what lies past 1.6e7 stays infinite.
constexpr float kDzScale = 1.0f / 256.0f;
constexpr float kHalfMax = 65504.0f;

// what to multiply a result of this launch by
template <typename T, int EPI>
__device__ __forceinline__ float result_scale(const Gemm& g) {
  if constexpr (EPI == kEpiStore && std::is_same<T, f16_t>::value)
    if (g.over && *g.over) return 1.0f / kDzScale;
  return 1.0f;
}

// biases of the columns col .. col + W
template <typename T, int EPI, int W>
__device__ __forceinline__ void load_biases(const Gemm& g, int64_t col, float (&b)[W], float (&b2)[W]) {
#pragma unroll
  for (int j = 0; j < W; ++j) b[j] = b2[j] = 0.0f;
  if (EPI == kEpiStore || g.bias == nullptr || col >= g.n) return;
  const int left = g.n - col < W ? static_cast<int>(g.n - col) : W;
  load_pack<T, W>(static_cast<const T*>(g.bias) + col, left, b);
  if constexpr (EPI == kEpiGated) load_pack<T, W>(static_cast<const T*>(g.bias2) + col, left, b2);
}

// results at (row, col .. col + W): columns of one row that one thread holds
template <typename T, int EPI, int W>
__device__ __forceinline__ void finish_row(const Gemm& g, int64_t row, int64_t col, float (&v)[W],
                                           float (&u)[W], const float (&b)[W], const float (&b2)[W],
                                           float scale) {
  if (row >= g.m || col >= g.n) return;
  const int left = g.n - col < W ? static_cast<int>(g.n - col) : W;
  const int64_t at = row * g.n + col;
  if constexpr (EPI == kEpiStore) {
    if constexpr (std::is_same<T, f16_t>::value) {
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] *= scale;
    }
    T* c = static_cast<T*>(row < g.row_split ? g.c : g.c2);
    const int64_t r = row < g.row_split ? row : row - g.row_split;
    if (c && r < g.row_valid) store_pack<T, W>(c + r * g.n + col, left, v, g.stream);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      v[j] += b[j];
      if (EPI == kEpiGated) u[j] += b2[j];
    }
    float t[W];
    if (g.keep) {
      if constexpr (EPI == kEpiGated) {
        store_pack<float, W>(static_cast<float*>(g.keep) + at, left, v, g.stream);
        store_pack<float, W>(static_cast<float*>(g.keep2) + at, left, u, g.stream);
      } else if (kept_in_float(g.act)) {
        store_pack<float, W>(static_cast<float*>(g.keep) + at, left, v, g.stream);
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j) t[j] = kept_sign<T>(v[j]);
        store_pack<T, W>(static_cast<T*>(g.keep) + at, left, t, g.stream);
      }
    }
    act_values(g.act, v);
    if constexpr (EPI == kEpiGated) {
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] *= u[j];
    } else if (g.residual) {
      load_pack<T, W>(static_cast<const T*>(g.residual) + row * g.res_ld + col, left, t);
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] += t[j];
    }
    store_pack<T, W>(static_cast<T*>(g.c) + at, left, v, g.stream);
  }
}

}  // namespace collie
