// K11: embedding lookup with scaling, and its gradient by sorted ids.
//   y[i] = s W[id_i]                     (an id outside the table gives a zero row and sets *status)
//   dW[r] = s sum_{i : id_i = r} dy[i]   (rows without an entry are 0)
// Both are bound by memory.  The gradient is a sum over entries in a fixed order, without
// floating-point atomics: the ids are sorted (stable), then summed by chunks of sorted entries,
// whatever rows they belong to, so that one row with a tenth of all entries costs as much as as many
// rows with one entry.  A run of equal ids inside a chunk is a finished row; runs that cross chunks
// are put together in LDS, and what crosses the workgroup's borders becomes its (at most two) entries
// of the next list, hundreds of times shorter, which the same kernel sums until one workgroup is left.
#include "head_types.h"
#include "rowsort.h"

namespace collie {
namespace {

constexpr int kBlock = 256;
constexpr int kMaxChunk = 64;                  // entries per lane group
constexpr int kMaxEntries = 1024;              // entries per workgroup
constexpr int kLookupRows = 4;                 // rows in flight per lane group of the lookup
constexpr int kAhead = 8;                      // rows on their way while as many are summed
constexpr uint32_t kNoKey = 0xffffffffu;       // no entry (keys are rows, below 2^31)

// `lpr` lanes per row, a power of two: at most a wave, and no more than the row has 16-byte packs, but
// at least `least`
inline int lanes_per_row(int64_t dim, int v, int least) {
  int l = least;
  while (l < kWave && static_cast<int64_t>(l) * v < dim) l <<= 1;
  return l;
}

// WHOLE: a row is a whole number of 16-byte packs
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kBlock) void embed_rows_kernel(
    const T* __restrict__ table, int64_t num_rows, int dim, const void* __restrict__ ids,
    int ids_dtype, int64_t n, float scale, T* __restrict__ out, int32_t* __restrict__ status, int lpr,
    bool stream_out) {
  constexpr int V = kVec<T>;
  constexpr int R = kLookupRows;
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
      load_row<WHOLE, T, V>(table + (ok[r] ? id[r] : 0) * dim, c, dim, ok[r], v[r]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t i = first + r * groups;
#pragma unroll
      for (int j = 0; j < V; ++j) v[r][j] *= scale;
      if (i < n) store_pack<T, V>(out + i * dim + c, dim - c, v[r], stream_out);
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
  // a workgroup fills one contiguous piece (512 MB: 6 TB/s; round-robin 16-byte stores 3.7)
  const int64_t n16 = grad_bytes / 16;
  const int64_t piece = (n16 + gridDim.x - 1) / gridDim.x;
  const int64_t end = (blockIdx.x + 1) * piece < n16 ? (blockIdx.x + 1) * piece : n16;
  for (int64_t i = blockIdx.x * piece + threadIdx.x; i < end; i += kBlock)
    reinterpret_cast<uint4*>(grad)[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = 8 * n16 + t0; i < grad_bytes / 2; i += stride)
    reinterpret_cast<uint16_t*>(grad)[i] = 0;
}

// Sums the runs of equal keys of `m` sorted entries.  Entry e is row codes[e] of `src` (row e where
// codes is NULL).  Finished rows go to `grad` (times scale, rounded once); the runs that cross the
// borders of a workgroup go to next_keys / next_sums [2 * workgroups].  A lane group of `lpr` lanes
// sums `chunk` entries.
template <typename S, typename T, bool WHOLE>
__global__ __launch_bounds__(kBlock) void sum_runs_kernel(
    const uint32_t* __restrict__ keys, const uint32_t* __restrict__ codes, int64_t m,
    const S* __restrict__ src, int64_t src_ld, int64_t num_rows, int dim, float scale,
    T* __restrict__ grad, uint32_t* __restrict__ next_keys, float* __restrict__ next_sums, int lpr,
    int chunk) {
  constexpr int V = kVec<S>;
  __shared__ uint32_t skey[kMaxEntries + 2], scode[kMaxEntries];  // skey[0]: the entry before
  __shared__ uint32_t open_key[kBlock][2];
  __shared__ float open_sum[2][kBlock * V];  // of a group's first run, and of its last
  const int groups = kBlock / lpr, sub = threadIdx.x & (lpr - 1), group = threadIdx.x / lpr;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * groups * chunk;
  const int entries = static_cast<int>(m - base < groups * chunk ? m - base : groups * chunk);
  const uint32_t rows = static_cast<uint32_t>(num_rows);
  for (int e = threadIdx.x; e < entries + 2; e += kBlock) {
    const int64_t at = base + e - 1;
    skey[e] = at >= 0 && at < m ? keys[at] : kNoKey;
  }
  for (int e = threadIdx.x; e < entries; e += kBlock)
    scode[e] = codes ? codes[base + e] : static_cast<uint32_t>(base + e);
  open_key[group][0] = open_key[group][1] = kNoKey;
  __syncthreads();
  const uint32_t* key_of = skey + 1;
  const int c = (blockIdx.y * lpr + sub) * V;
  const int left = dim - c;
  const int lo = group * chunk, hi = lo + chunk < entries ? lo + chunk : entries;
  // sums of a run that is not closed: with the row's columns of this lane
  float* open0 = open_sum[0] + threadIdx.x * V;
  float* open1 = open_sum[1] + threadIdx.x * V;
  if (lo < hi) {
    const uint32_t first_key = key_of[lo], last_key = key_of[hi - 1];
    const bool from_before = key_of[lo - 1] == first_key && first_key < rows;
    const bool goes_on = key_of[hi] == last_key && last_key < rows;
    const bool one_run = first_key == last_key;
    if (sub == 0) {
      // a chunk inside one long run has one sum: its second slot has the same key and adds zero
      open_key[group][0] = from_before || (one_run && goes_on) ? first_key : kNoKey;
      open_key[group][1] = goes_on || (one_run && from_before) ? last_key : kNoKey;
    }
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = open0[j] = open1[j] = 0.0f;
    uint32_t key = first_key;
    bool first_run = true;
    auto finish = [&](bool is_last) {
      if ((first_run && from_before) || (is_last && goes_on)) {
        float* to = first_run ? open0 : open1;
#pragma unroll
        for (int j = 0; j < V; ++j) to[j] = sum[j];
      } else if (key < rows && left > 0) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] *= scale;
        store_pack<T, V>(grad + static_cast<int64_t>(key) * dim + c, left, sum);
      }
      first_run = false;
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] = 0.0f;
    };
    Pack<S, V> v[2][kAhead];
    auto fetch = [&](Pack<S, V> (&to)[kAhead], int e0) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int e = e0 + u < hi ? e0 + u : lo;
        to[u] = row_pack<WHOLE, S, V>(src + static_cast<int64_t>(scode[e]) * src_ld,
                                      left > 0 ? c : 0, dim, true);
      }
    };
    auto add = [&](const Pack<S, V> (&from)[kAhead], int e0) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (e0 + u < hi) {
          const uint32_t k = key_of[e0 + u];
          if (k != key) {
            finish(false);
            key = k;
          }
          if (k < rows) {
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += static_cast<float>(from[u].v[j]);
          }
        }
      }
    };
    fetch(v[0], lo);
    for (int e0 = lo; e0 < hi; e0 += 2 * kAhead) {
      if (e0 + kAhead < hi) fetch(v[1], e0 + kAhead);
      add(v[0], e0);
      if (e0 + 2 * kAhead < hi) fetch(v[0], e0 + 2 * kAhead);
      add(v[1], e0 + kAhead);
    }
    finish(true);
  }
  __syncthreads();
  // The open sums in order, two per group: a run of them is added up by the group that holds its
  // start.  What is open at the workgroup's left border is its first entry of the next list, at its
  // right border its second one.
  const uint32_t first_key = key_of[0], last_key = key_of[entries - 1];
  const bool from_before = key_of[-1] == first_key && first_key < rows;
  const bool goes_on = key_of[entries] == last_key && last_key < rows;
  const bool one_run = first_key == last_key;
  if (threadIdx.x == 0 && blockIdx.y == 0) {
    next_keys[2 * blockIdx.x] = from_before || (one_run && goes_on) ? first_key : kNoKey;
    next_keys[2 * blockIdx.x + 1] = goes_on || (one_run && from_before) ? last_key : kNoKey;
  }
  const uint32_t* list = &open_key[0][0];
  for (int s = 2 * group; s < 2 * group + 2; ++s) {
    const uint32_t key = list[s];
    if (key == kNoKey || (s > 0 && list[s - 1] == key)) continue;
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.0f;
    for (int e = s; e < 2 * groups && list[e] == key; ++e) {
      const float* from = open_sum[e & 1] + ((e >> 1) * lpr + sub) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += from[j];
    }
    if (left <= 0) continue;
    const bool open_left = from_before && key == first_key;
    const bool open_right = goes_on && key == last_key;
    if (open_left || open_right) {
      const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (key == first_key ? 0 : 1);
      store_pack<float, V>(next_sums + slot * dim + c, left, sum);
      if (one_run) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] = 0.0f;
        store_pack<float, V>(next_sums + (slot + 1) * dim + c, left, sum);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] *= scale;
      store_pack<T, V>(grad + static_cast<int64_t>(key) * dim + c, left, sum);
    }
  }
}

// lanes per row and entries per lane group, at most kMaxEntries per workgroup.  Fewer where there are
// not enough of them for eight workgroups on every CU; the later lists are short, and one more launch costs
// more than 32 entries one after another.
struct RunShape {
  int lpr, chunk;
  int64_t blocks;
};
RunShape run_shape(int64_t m, int dim, int v, bool later) {
  RunShape r;
  // eight lanes also where fewer would do: of a run that fills the workgroup one lane group adds up the
  // open sums of all, and there are 32 of them then, not 256 (1 column, 65,536 skewed ids: 105 -> 55 us)
  r.lpr = lanes_per_row(dim, v, 8);
  const int groups = kBlock / r.lpr;
  const int most = kMaxEntries / groups < kMaxChunk ? kMaxEntries / groups : kMaxChunk;
  r.chunk = most;
  if (later)
    r.chunk = most < 32 ? most : 32;
  else
    while (r.chunk > 8 && m < static_cast<int64_t>(2048) * groups * r.chunk) r.chunk /= 2;
  r.blocks = (m + groups * r.chunk - 1) / (groups * r.chunk);
  return r;
}

struct GradWs {
  SortWs sort;
  uint32_t* keys[2];  // the two lists of open runs that take turns
  float* sums[2];
  size_t bytes;
};

GradWs carve_grad_ws(void* base, int64_t n, int dim) {
  Carver c(base);
  GradWs w;
  carve_pair_sort_ws(c, w.sort, n);
  // the first list has two entries per workgroup; lanes per row are fewest for 16-bit values
  int64_t m = 0;
  for (int v : {4, 8}) {
    const int64_t blocks = run_shape(n, dim, v, false).blocks;
    m = m > 2 * blocks ? m : 2 * blocks;
  }
  for (int i = 0; i < 2; ++i) {
    w.keys[i] = c.take<uint32_t>(m);
    w.sums[i] = c.take<float>(static_cast<size_t>(m) * dim);
  }
  w.bytes = align_up(c.off, 256);
  return w;
}

// returns the number of workgroups
template <typename S, typename T>
int64_t launch_sum_runs(const uint32_t* keys, const uint32_t* codes, int64_t m, const S* src,
                        int64_t src_ld, int64_t num_rows, int dim, float scale, T* grad,
                        uint32_t* next_keys, float* next_sums, hipStream_t stream) {
  constexpr int V = kVec<S>;
  const RunShape r = run_shape(m, dim, V, codes == nullptr);
  const dim3 grid(static_cast<unsigned>(r.blocks),
                  static_cast<unsigned>((dim + r.lpr * V - 1) / (r.lpr * V)));
  auto* kernel = dim % V == 0 ? sum_runs_kernel<S, T, true> : sum_runs_kernel<S, T, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kBlock), 0, stream, keys, codes, m, src, src_ld, num_rows,
                     dim, scale, grad, next_keys, next_sums, r.lpr, r.chunk);
  return check_launch("sum_runs_kernel") ? -1 : r.blocks;
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
    const int lpr = lanes_per_row(dim, kVec<T>, 1);
    const int64_t per_block = static_cast<int64_t>(kBlock / lpr) * kLookupRows;
    auto* kernel = dim % kVec<T> == 0 ? embed_rows_kernel<T, true> : embed_rows_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((n + per_block - 1) / per_block)),
                       dim3(kBlock), 0, stream, static_cast<const T*>(table), num_rows, dim, ids,
                       ids_dtype, n, scale, static_cast<T*>(out), status, lpr,
                       n * dim * static_cast<int64_t>(sizeof(T)) >= kStreamBytes);
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
    int64_t fill = (n > grad_bytes / 16 ? n : grad_bytes / 16) / (4 * kBlock) + 1;
    if (fill > 4096) fill = 4096;
    hipLaunchKernelGGL(grad_entries_kernel, dim3(static_cast<unsigned>(fill)), dim3(kBlock), 0,
                       stream, ids, ids_dtype, n, num_rows, padding_idx, w.sort.ekeys,
                       w.sort.ecodes, static_cast<char*>(grad), grad_bytes, status);
    if (check_launch("grad_entries_kernel")) return -2;
    if (n == 0) return 0;
    const int64_t nkeys = num_rows + 1;
    if (sort_pairs(w.sort, nkeys, stream)) return -1;
    T* out = static_cast<T*>(grad);
    int64_t blocks = launch_sum_runs<T, T>(sorted_keys(w.sort, nkeys), sorted_vals(w.sort, nkeys), n,
                                           static_cast<const T*>(dy), dy_ld, num_rows, dim, scale,
                                           out, w.keys[0], w.sums[0], stream);
    for (int turn = 0; blocks > 1; turn ^= 1)
      blocks = launch_sum_runs<float, T>(w.keys[turn], nullptr, 2 * blocks, w.sums[turn], dim,
                                         num_rows, dim, scale, out, w.keys[turn ^ 1],
                                         w.sums[turn ^ 1], stream);
    return blocks < 0 ? -2 : 0;
  });
}
