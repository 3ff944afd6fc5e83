// K11: embedding lookup with scaling, and its gradient by sorted ids.
//   y[i] = s W[id_i]                     (an id outside the table gives a zero row and sets *status)
//   dW[r] = s sum_{i : id_i = r} dy[i]   (rows without an entry are 0)
// Both are bound by memory.  The gradient is a sum over entries in a fixed order, without
// floating-point atomics: the ids are sorted (stable), then summed by chunks of kChunk sorted
// entries, whatever rows they belong to, so that one row with a tenth of all entries costs as much
// as as many rows with one entry.  A run of equal ids inside a chunk is a finished row; a run that
// goes on past a chunk's border becomes one of the chunk's (at most two) entries of the next, kChunk
// / 2 times shorter, list, which the same kernel sums until one chunk is left.
#include "head_types.h"
#include "rowsort.h"

namespace collie {
namespace {

constexpr int kBlock = 256;
constexpr int kChunk = 64;                     // entries per chunk
constexpr int kUnroll = 8;                     // rows in flight per lane
constexpr uint32_t kNoKey = 0xffffffffu;       // no entry (keys are rows, below 2^31)

// `lpr` lanes per row, a power of two: at most a wave, and no more than the row has 16-byte chunks
inline int lanes_per_row(int64_t dim, int v) {
  int l = 1;
  while (l < kWave && static_cast<int64_t>(l) * v < dim) l <<= 1;
  return l;
}

// WHOLE: a row is a whole number of 16-byte packs
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kBlock) void embed_rows_kernel(
    const T* __restrict__ table, int64_t num_rows, int dim, const void* __restrict__ ids,
    int ids_dtype, int64_t n, float scale, T* __restrict__ out, int32_t* __restrict__ status,
    int lpr) {
  constexpr int V = kVec<T>;
  constexpr int R = 4;  // rows in flight per lane group
  const int sub = threadIdx.x & (lpr - 1);
  const int groups = kBlock / lpr;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * groups * R + threadIdx.x / lpr;
  int64_t id[R];
  bool ok[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = first + r * groups;
    id[r] = i < n ? load_idx(ids, ids_dtype, i) : 0;
    ok[r] = id[r] >= 0 && id[r] < num_rows;
    if (!ok[r] && status && sub == 0) atomicOr(status, 1);
  }
  for (int c = sub * V; c < dim; c += lpr * V) {
    float v[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r)
      load_row<WHOLE, T, V>(table + (ok[r] ? id[r] : 0) * dim + c, dim - c, ok[r], v[r]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t i = first + r * groups;
#pragma unroll
      for (int j = 0; j < V; ++j) v[r][j] *= scale;
      if (i < n) store_pack<T, V>(out + i * dim + c, dim - c, v[r]);
    }
  }
}

// sort keys (the row; `num_rows`, which sorts last, for ids that take no gradient) and entry
// numbers, and zeros into the whole gradient: rows without an entry keep them
__global__ __launch_bounds__(kBlock) void grad_entries_kernel(
    const void* __restrict__ ids, int ids_dtype, int64_t n, int64_t num_rows, int64_t padding_idx,
    uint32_t* __restrict__ keys, uint32_t* __restrict__ codes, char* __restrict__ grad,
    int64_t grad_bytes, int32_t* __restrict__ status) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kBlock;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
  for (int64_t i = t0; i < n; i += stride) {
    const int64_t id = load_idx(ids, ids_dtype, i);
    const bool ok = id >= 0 && id < num_rows;
    if (!ok && status) atomicOr(status, 1);
    keys[i] = static_cast<uint32_t>(ok && id != padding_idx ? id : num_rows);
    codes[i] = static_cast<uint32_t>(i);
  }
  const int64_t n16 = grad_bytes / 16;
  for (int64_t i = t0; i < n16; i += stride)
    reinterpret_cast<uint4*>(grad)[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = 8 * n16 + t0; i < grad_bytes / 2; i += stride)
    reinterpret_cast<uint16_t*>(grad)[i] = 0;
}

// Sums the runs of equal keys of `m` sorted entries.  Entry e is row codes[e] of `src` (row e where
// codes is NULL).  Finished rows go to `grad` (times scale, rounded once); the runs that cross a
// chunk's borders go to next_keys / next_sums [2 * chunks].
template <typename S, typename T, bool WHOLE>
__global__ __launch_bounds__(kBlock) void sum_runs_kernel(
    const uint32_t* __restrict__ keys, const uint32_t* __restrict__ codes, int64_t m,
    const S* __restrict__ src, int64_t src_ld, int64_t num_rows, int dim, float scale,
    T* __restrict__ grad, uint32_t* __restrict__ next_keys, float* __restrict__ next_sums, int lpr) {
  constexpr int V = kVec<S>;
  const int sub = threadIdx.x & (lpr - 1);
  const int64_t chunk = static_cast<int64_t>(blockIdx.x) * (kBlock / lpr) + threadIdx.x / lpr;
  const int64_t lo = chunk * kChunk;
  if (lo >= m) return;
  const int64_t hi = lo + kChunk < m ? lo + kChunk : m;
  const uint32_t first_key = keys[lo], last_key = keys[hi - 1];
  const uint32_t rows = static_cast<uint32_t>(num_rows);
  const bool from_before = lo > 0 && keys[lo - 1] == first_key && first_key < rows;
  const bool goes_on = hi < m && keys[hi] == last_key && last_key < rows;
  const bool one_run = first_key == last_key;
  if (sub == 0 && blockIdx.y == 0 && next_keys) {
    // a chunk inside one long run has one sum: its second slot has the same key and adds zero
    next_keys[2 * chunk] = from_before || (one_run && goes_on) ? first_key : kNoKey;
    next_keys[2 * chunk + 1] = goes_on || (one_run && from_before) ? last_key : kNoKey;
  }
  const int c = (blockIdx.y * lpr + sub) * V;
  if (c >= dim) return;
  const int left = dim - c;
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0.0f;
  uint32_t key = first_key;
  bool first_run = true;
  auto finish = [&](bool is_last) {
    const bool open_left = first_run && from_before;
    const bool open_right = is_last && goes_on;
    if (open_left || open_right) {
      // the sum of a run that fills the chunk goes to the first slot
      const int slot = first_run ? 0 : 1;
      store_pack<float, V>(next_sums + (2 * chunk + slot) * dim + c, left, sum);
      if (first_run && is_last) {
        float zero[V];
#pragma unroll
        for (int j = 0; j < V; ++j) zero[j] = 0.0f;
        store_pack<float, V>(next_sums + (2 * chunk + 1) * dim + c, left, zero);
      }
    } else if (key < rows) {
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] *= scale;
      store_pack<T, V>(grad + static_cast<int64_t>(key) * dim + c, left, sum);
    }
    first_run = false;
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
  };
  for (int64_t e0 = lo; e0 < hi; e0 += kUnroll) {
    uint32_t k[kUnroll];
    float v[kUnroll][V];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t e = e0 + u < hi ? e0 + u : lo;
      k[u] = keys[e];
      const int64_t row = codes ? static_cast<int64_t>(codes[e]) : e;
      load_row<WHOLE, S, V>(src + row * src_ld + c, left, k[u] < rows, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (e0 + u >= hi) break;
      if (k[u] != key) {
        finish(false);
        key = k[u];
      }
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += v[u][j];
    }
  }
  finish(true);
}

struct GradWs {
  SortWs sort;
  uint32_t* keys[2];  // the two lists of open runs that take turns
  float* sums[2];
  size_t bytes;
};

inline int64_t chunks_of(int64_t m) { return (m + kChunk - 1) / kChunk; }

GradWs carve_grad_ws(void* base, int64_t n, int dim) {
  Carver c(base);
  GradWs w;
  carve_pair_sort_ws(c, w.sort, n);
  int64_t m = n;
  for (int i = 0; i < 2; ++i) {
    m = 2 * chunks_of(m);
    w.keys[i] = c.take<uint32_t>(m);
    w.sums[i] = c.take<float>(static_cast<size_t>(m) * dim);
  }
  w.bytes = align_up(c.off, 256);
  return w;
}

template <typename S, typename T>
int launch_sum_runs(const uint32_t* keys, const uint32_t* codes, int64_t m, const S* src,
                    int64_t src_ld, int64_t num_rows, int dim, float scale, T* grad,
                    uint32_t* next_keys, float* next_sums, hipStream_t stream) {
  constexpr int V = kVec<S>;
  const int lpr = lanes_per_row(dim, V);
  const int64_t groups = kBlock / lpr;
  const dim3 grid(static_cast<unsigned>((chunks_of(m) + groups - 1) / groups),
                  static_cast<unsigned>((dim + lpr * V - 1) / (lpr * V)));
  auto* kernel = dim % V == 0 ? sum_runs_kernel<S, T, true> : sum_runs_kernel<S, T, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kBlock), 0, stream, keys, codes, m, src, src_ld, num_rows,
                     dim, scale, grad, next_keys, next_sums, lpr);
  return check_launch("sum_runs_kernel");
}

int check_table(const char* who, int64_t num_rows, int32_t dim, int64_t n) {
  COLLIE_REQUIRE(num_rows >= 1 && num_rows < (int64_t{1} << 31) - 1, "%s: bad number of rows", who);
  COLLIE_REQUIRE(dim >= 1 && dim <= (1 << 20), "%s: dim must be in [1, 2^20]", who);
  COLLIE_REQUIRE(n >= 0 && n < (int64_t{1} << 31), "%s: bad number of ids", who);
  return 0;
}

}  // namespace
}  // namespace collie

using namespace collie;

extern "C" int collie_embedding_rows(const void* table, int32_t dtype, int64_t num_rows, int32_t dim,
                                     const void* ids, int32_t ids_dtype, int64_t n, float scale,
                                     void* out, int32_t* status, collie_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (check_table("embedding_rows", num_rows, dim, n)) return -1;
  COLLIE_REQUIRE(ids_dtype == COLLIE_I32 || ids_dtype == COLLIE_I64, "embedding_rows: bad id type");
  if (n == 0) return 0;
  COLLIE_REQUIRE(table && ids && out, "embedding_rows: NULL pointer");
  return with_type(dtype, "embedding_rows", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const int lpr = lanes_per_row(dim, kVec<T>);
    const int64_t per_block = static_cast<int64_t>(kBlock / lpr) * 4;
    auto* kernel = dim % kVec<T> == 0 ? embed_rows_kernel<T, true> : embed_rows_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((n + per_block - 1) / per_block)),
                       dim3(kBlock), 0, stream, static_cast<const T*>(table), num_rows, dim, ids,
                       ids_dtype, n, scale, static_cast<T*>(out), status, lpr);
    return check_launch("embed_rows_kernel");
  });
}

extern "C" size_t collie_embedding_rows_grad_workspace_bytes(int64_t n, int32_t dim) {
  if (n < 1 || dim < 1) return 256;
  return carve_grad_ws(nullptr, n, dim).bytes;
}

extern "C" int collie_embedding_rows_grad(const void* ids, int32_t ids_dtype, int64_t n,
                                          const void* dy, int64_t dy_ld, int32_t dtype,
                                          int64_t num_rows, int32_t dim, float scale,
                                          int64_t padding_idx, void* grad, void* workspace,
                                          size_t workspace_bytes, int32_t* status,
                                          collie_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (check_table("embedding_rows_grad", num_rows, dim, n)) return -1;
  COLLIE_REQUIRE(n < (int64_t{1} << 30), "embedding_rows_grad: at most 2^30 - 1 ids");
  COLLIE_REQUIRE(ids_dtype == COLLIE_I32 || ids_dtype == COLLIE_I64,
                 "embedding_rows_grad: bad id type");
  COLLIE_REQUIRE(grad && (n == 0 || (ids && dy)), "embedding_rows_grad: NULL pointer");
  COLLIE_REQUIRE(n <= 1 || dy_ld >= dim, "embedding_rows_grad: rows of dy overlap");
  COLLIE_REQUIRE(reinterpret_cast<uintptr_t>(grad) % 16 == 0,
                 "embedding_rows_grad: grad must be aligned to 16 bytes");
  const GradWs w = carve_grad_ws(workspace, n < 1 ? 1 : n, dim);
  COLLIE_REQUIRE(n == 0 || (workspace && workspace_bytes >= w.bytes),
                 "workspace too small: need %zu bytes, got %zu", w.bytes, workspace_bytes);
  return with_type(dtype, "embedding_rows_grad", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const int64_t grad_bytes = num_rows * dim * static_cast<int64_t>(sizeof(T));
    int64_t blocks = (n > grad_bytes / 16 ? n : grad_bytes / 16) / (4 * kBlock) + 1;
    if (blocks > 4096) blocks = 4096;
    hipLaunchKernelGGL(grad_entries_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kBlock), 0,
                       stream, ids, ids_dtype, n, num_rows, padding_idx, w.sort.ekeys,
                       w.sort.ecodes, static_cast<char*>(grad), grad_bytes, status);
    if (check_launch("grad_entries_kernel")) return -2;
    if (n == 0) return 0;
    const int64_t nkeys = num_rows + 1;
    if (sort_pairs(w.sort, nkeys, stream)) return -1;
    T* out = static_cast<T*>(grad);
    int64_t m = n;
    int rc = launch_sum_runs<T, T>(sorted_keys(w.sort, nkeys), sorted_vals(w.sort, nkeys), m,
                                   static_cast<const T*>(dy), dy_ld, num_rows, dim, scale, out,
                                   w.keys[0], w.sums[0], stream);
    for (int turn = 0; !rc && chunks_of(m) > 1; turn ^= 1) {
      m = 2 * chunks_of(m);
      rc = launch_sum_runs<float, T>(w.keys[turn], nullptr, m, w.sums[turn], dim, num_rows, dim,
                                     scale, out, w.keys[turn ^ 1], w.sums[turn ^ 1], stream);
    }
    return rc;
  });
}
