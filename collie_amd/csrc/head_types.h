// Element types of the ranking-head operators (embed_rows.hip, layer_norm.hip, head_gemm.hip):
// float32, bfloat16 and float16 storage, float32 arithmetic.
#pragma once

#include "common.h"

#include <type_traits>

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

// The 16 bytes of a row of `dim` values from column c on, zeros past its end (and all zeros where !ok).
// `row` must be readable; WHOLE: dim is a whole number of packs and c is below it, one unconditional
// load, so that several stay in flight.  (Where a row ends inside a pack: loading its last whole pack
// and shifting it, without a branch, was slower than the branch: 24,001 x 1,023 bf16, layer norm
// forward 41 against 36 us.)
template <bool WHOLE, typename T, int V>
__device__ __forceinline__ Pack<T, V> row_pack(const T* __restrict__ row, int c, int dim, bool ok) {
  static_assert(V * sizeof(T) == 16, "a pack is 16 bytes");
  Pack<T, V> a;
  if constexpr (WHOLE) {
    a = *reinterpret_cast<const Pack<T, V>*>(row + c);
    if (!ok) a = Pack<T, V>{};
  } else if (ok && c + V <= dim) {
    a = *reinterpret_cast<const Pack<T, V>*>(row + c);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) a.v[j] = ok && c + j < dim ? row[c + j] : static_cast<T>(0.0f);
  }
  return a;
}

template <bool WHOLE, typename T, int V>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int c, int dim, bool ok,
                                         float (&v)[V]) {
  const Pack<T, V> a = row_pack<WHOLE, T, V>(row, c, dim, ok);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = static_cast<float>(a.v[j]);
}

// the first n of V values: at most one store of each power of two
template <typename T, int V, int AT, int PART>
__device__ __forceinline__ void store_parts(T* __restrict__ p, int n, const Pack<T, V>& a) {
  if constexpr (PART >= 1) {
    if (n & PART) {
      Pack<T, PART> b;
#pragma unroll
      for (int j = 0; j < PART; ++j) b.v[j] = a.v[AT + j];
      *reinterpret_cast<Pack<T, PART>*>(p + AT) = b;
      store_parts<T, V, AT + PART, PART / 2>(p, n, a);
    } else {
      store_parts<T, V, AT, PART / 2>(p, n, a);
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* __restrict__ p, int n, const float (&v)[V]) {
  if (n >= V) {
    Pack<T, V> a;
#pragma unroll
    for (int j = 0; j < V; ++j) a.v[j] = static_cast<T>(v[j]);
    *reinterpret_cast<Pack<T, V>*>(p) = a;
  } else if (n > 0) {
    Pack<T, V> a;
#pragma unroll
    for (int j = 0; j < V; ++j) a.v[j] = static_cast<T>(v[j]);
    store_parts<T, V, 0, V / 2>(p, n, a);
  }
}

// Results of this many bytes and more are stored past the caches: whoever reads them finds little of
// them there anyway, and the tables and operands that are read meanwhile stay.
constexpr int64_t kStreamBytes = int64_t{64} << 20;

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* __restrict__ p, int n, const float (&v)[V], bool stream) {
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  constexpr int N = kVec<T>;
  if constexpr (V % N == 0) {
    if (stream && n >= V && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
#pragma unroll
      for (int i = 0; i < V; i += N) {
        Pack<T, N> a;
#pragma unroll
        for (int j = 0; j < N; ++j) a.v[j] = static_cast<T>(v[i + j]);
        __builtin_nontemporal_store(__builtin_bit_cast(words, a), reinterpret_cast<words*>(p + i));
      }
      return;
    }
  }
  store_pack<T, V>(p, n, v);
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

}  // namespace collie
