// Element types of the ranking-head operators (embed_rows.hip, layer_norm.hip, head_gemm.hip):
// float32, bfloat16 and float16 storage, float32 arithmetic.
#pragma once

#include "common.h"

namespace collie {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// V consecutive elements at any element address.  The hardware takes 16-byte global accesses at any
// byte address, so rows of odd widths and views with odd offsets need no kernels of their own.
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[V];
};

template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));  // elements of one 16-byte access

// v[j] = p[j] for j < n, 0 elsewhere
template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* __restrict__ p, int n, float (&v)[V]) {
  if (n >= V) {
    const Pack<T, V> a = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = static_cast<float>(a.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = j < n ? static_cast<float>(p[j]) : 0.0f;
  }
}

// The same where the caller knows that a row holds whole packs only and `p` can always be read: one
// unconditional load, so that several stay in flight; zeros where !ok.
template <bool WHOLE, typename T, int V>
__device__ __forceinline__ void load_row(const T* __restrict__ p, int n, bool ok, float (&v)[V]) {
  if constexpr (WHOLE) {
    const Pack<T, V> a = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = ok ? static_cast<float>(a.v[j]) : 0.0f;
  } else {
    load_pack<T, V>(p, ok ? n : 0, v);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* __restrict__ p, int n, const float (&v)[V]) {
  if (n >= V) {
    Pack<T, V> a;
#pragma unroll
    for (int j = 0; j < V; ++j) a.v[j] = static_cast<T>(v[j]);
    *reinterpret_cast<Pack<T, V>*>(p) = a;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < n) p[j] = static_cast<T>(v[j]);
  }
}

// calls f.template operator()<T>() with the element type of a COLLIE_F32 / BF16 / F16 tag
template <typename F>
int with_type(int32_t dtype, const char* who, F&& f) {
  switch (dtype) {
    case COLLIE_F32: return f(static_cast<float*>(nullptr));
    case COLLIE_BF16: return f(static_cast<bf16_t*>(nullptr));
    case COLLIE_F16: return f(static_cast<f16_t*>(nullptr));
    default: set_error("%s: unknown element type %d", who, dtype); return -1;
  }
}

inline size_t type_size(int32_t dtype) { return dtype == COLLIE_F32 ? 4 : 2; }

}  // namespace collie
