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
  int64_t b2_offset;     // b2 - b, in elements
  int64_t m, n, k;
  int64_t k_chunk;       // depth of one of the `splits` parts
  int splits;
  // epilogue
  int act;
  const void *bias, *bias2;
  const void* residual;
  int64_t res_ld;
  void *keep, *keep2;    // pre-activations for the backward pass [m, n], or NULL
  void *c, *c2;          // output [m, n]; with kEpiStore rows >= row_split are c2's, and of either
  int64_t row_split;     // only the first row_valid are wanted
  int64_t row_valid;
  float* partial;        // splits > 1: [splits, accumulators, m, n] sums of the parts of the depth
};

// the sums of one part of the depth
template <int EPI, int W>
__device__ __forceinline__ void store_part(const Gemm& g, int64_t row, int64_t col, int64_t part,
                                           const float (&v)[W], const float (&u)[W]) {
  if (row >= g.m || col >= g.n) return;
  const int left = g.n - col < W ? static_cast<int>(g.n - col) : W;
  constexpr int NB = EPI == kEpiGated ? 2 : 1;
  float* p = g.partial + part * NB * g.m * g.n + row * g.n + col;
  store_pack<float, W>(p, left, v);
  if constexpr (NB == 2) store_pack<float, W>(p + g.m * g.n, left, u);
}

// results at (row, col .. col + W): columns of one row that one thread holds
template <typename T, int EPI, int W>
__device__ __forceinline__ void finish_row(const Gemm& g, int64_t row, int64_t col, float (&v)[W],
                                           float (&u)[W]) {
  if (row >= g.m || col >= g.n) return;
  const int left = g.n - col < W ? static_cast<int>(g.n - col) : W;
  const int64_t at = row * g.n + col;
  if constexpr (EPI == kEpiStore) {
    T* c = static_cast<T*>(row < g.row_split ? g.c : g.c2);
    const int64_t r = row < g.row_split ? row : row - g.row_split;
    if (c && r < g.row_valid) store_pack<T, W>(c + r * g.n + col, left, v);
  } else {
    float add[W];
    if (g.bias) {
      load_pack<T, W>(static_cast<const T*>(g.bias) + col, left, add);
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] += add[j];
      if constexpr (EPI == kEpiGated) {
        load_pack<T, W>(static_cast<const T*>(g.bias2) + col, left, add);
#pragma unroll
        for (int j = 0; j < W; ++j) u[j] += add[j];
      }
    }
    if (g.keep) {
#pragma unroll
      for (int j = 0; j < W; ++j) add[j] = kept<T>(v[j]);
      store_pack<T, W>(static_cast<T*>(g.keep) + at, left, add);
      if constexpr (EPI == kEpiGated) {
#pragma unroll
        for (int j = 0; j < W; ++j) add[j] = kept<T>(u[j]);
        store_pack<T, W>(static_cast<T*>(g.keep2) + at, left, add);
      }
    }
    act_values(g.act, v);
    if constexpr (EPI == kEpiGated) {
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] *= u[j];
    } else if (g.residual) {
      load_pack<T, W>(static_cast<const T*>(g.residual) + row * g.res_ld + col, left, add);
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] += add[j];
    }
    store_pack<T, W>(static_cast<T*>(g.c) + at, left, v);
  }
}

}  // namespace collie
