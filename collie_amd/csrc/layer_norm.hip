// K12: layer normalisation over the last dimension and its gradient.
//   m = mean(x), v = mean((x - m)^2), r = 1 / sqrt(v + eps), h = (x - m) r, y = h w + b
//   g = dy w, dx = r (g - mean(g) - h mean(g h)), dw = sum over rows of dy h, db = sum of dy
// Bound by memory: the forward pass reads x and writes y, the backward pass reads x and dy and
// writes dx.  A row stays in the registers of the TPR lanes that own it (NV packs of 16 bytes each),
// so the variance is the centred one and costs no second read.  In the backward pass a lane keeps
// the sums of its own columns over all rows of its workgroup; one workgroup writes one partial, and
// a second launch adds the partials in fixed order (no floating-point atomics).
// Rows too wide for the registers of a workgroup (over kMaxPacks packs per lane) are read again
// from the caches instead (the *_wide kernels).
#include "head_types.h"

namespace collie {
namespace {

constexpr int kBlock = 256;
constexpr int kMaxPartials = 1024;  // workgroups of the backward pass: four on every CU
constexpr int kRedCols = 64, kRedRows = 16;

struct NormParams {
  const void* x;
  const void* dy;
  const void* w;     // NULL: ones
  const void* b;     // NULL: zeros
  void* y;           // backward: dx (NULL: not wanted)
  float* mean;       // [2, rows]: the mean, and what is left of it after rounding
  float* rstd;
  float* partial;    // backward: [workgroups, 2, dim] (NULL: not wanted)
  void *dw, *db;     // backward with one workgroup: the sums themselves, of the parameters' type
  int64_t rows, x_ld, dy_ld;
  int dim;
  int w_f32;         // w and b are float32 (else: the rows' type)
  float eps;
  bool stream;       // the result is stored past the caches
};

template <typename T, int V>
__device__ __forceinline__ void load_param(const void* p, int f32, int c, int n, float other,
                                           float (&v)[V]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = other;
  } else if (f32) {
    load_pack<float, V>(static_cast<const float*>(p) + c, n, v);
  } else {
    load_pack<T, V>(static_cast<const T*>(p) + c, n, v);
  }
}

// sums over the TPR lanes of a row (TPR = 256: the workgroup)
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&s)[N]) {
  constexpr int W = TPR < kWave ? TPR : kWave;
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = group_sum<W>(s[i]);
  if constexpr (TPR > kWave) {
    __shared__ float sh[N][TPR / kWave];
    __syncthreads();  // the sums of the previous call have been read
    if (lane_id() == 0)
      for (int i = 0; i < N; ++i) sh[i][threadIdx.x / kWave] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s[i] = 0.0f;
#pragma unroll
      for (int w = 0; w < TPR / kWave; ++w) s[i] += sh[i][w];
    }
  }
}

// mean of squares about a point that is `off` from the mean -> variance
__device__ __forceinline__ float variance(float squares, float off) {
  const float v = fmaf(-off, off, squares);
  return v < 0.0f ? 0.0f : v;  // (NaN stays)
}

__device__ __forceinline__ void keep_stats(const NormParams& p, int64_t row, float first, float off,
                                           float rstd) {
  const float mean = first + off;
  p.mean[row] = mean;
  p.mean[p.rows + row] = off - (mean - first);
  p.rstd[row] = rstd;
}

// lane `sub` of a row owns the packs sub, sub + TPR, ...; WHOLE: dim is a whole number of packs
template <typename T, int TPR, int NV, bool WHOLE>
__global__ __launch_bounds__(kBlock) void norm_fwd_kernel(const NormParams p) {
  constexpr int V = kVec<T>;
  constexpr int G = kBlock / TPR;
  const int sub = threadIdx.x % TPR;
  const float inv = 1.0f / static_cast<float>(p.dim);
  float w[NV][V], b[NV][V];
  int col[NV], left[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + sub) * V;
    left[i] = c < p.dim ? p.dim - c : 0;
    col[i] = left[i] ? c : 0;
    load_param<T, V>(p.w, p.w_f32, col[i], left[i], 1.0f, w[i]);
    load_param<T, V>(p.b, p.w_f32, col[i], left[i], 0.0f, b[i]);
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * G;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * G; r0 < p.rows; r0 += step) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool live = row < p.rows;  // TPR = 256: always, so every thread meets the barriers
    const T* x = static_cast<const T*>(p.x) + (live ? row : 0) * p.x_ld;
    float v[NV][V], s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) load_row<WHOLE, T, V>(x, col[i], p.dim, left[i] > 0, v[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += v[i][j];
    row_sums<TPR>(s);
    const float first = s[0] * inv;
    // what the mean was rounded by is the mean of what is left: a constant row has no variance then,
    // however large its value (1e6 over 49 columns: the sum times 1 / 49 is 0.06 off)
    float c[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = j < left[i] ? v[i][j] - first : 0.0f;
        c[0] += v[i][j];
        c[1] = fmaf(v[i][j], v[i][j], c[1]);
      }
    row_sums<TPR>(c);
    const float off = c[0] * inv;
    const float rstd = 1.0f / sqrtf(variance(c[1] * inv, off) + p.eps);
    if (!live) continue;
    T* y = static_cast<T*>(p.y) + row * p.dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = fmaf((v[i][j] - off) * rstd, w[i][j], b[i][j]);
      if (left[i] > 0) store_pack<T, V>(y + col[i], left[i], v[i], p.stream);
    }
    if (sub == 0 && p.mean) keep_stats(p, row, first, off, rstd);
  }
}

template <typename T, int TPR, int NV, bool WHOLE>
__global__ __launch_bounds__(kBlock) void norm_bwd_kernel(const NormParams p) {
  constexpr int V = kVec<T>;
  constexpr int G = kBlock / TPR;
  const int sub = threadIdx.x % TPR;
  const float inv = 1.0f / static_cast<float>(p.dim);
  float w[NV][V], dw[NV][V], db[NV][V];
  int col[NV], left[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + sub) * V;
    left[i] = c < p.dim ? p.dim - c : 0;
    col[i] = left[i] ? c : 0;
    load_param<T, V>(p.w, p.w_f32, col[i], left[i], 1.0f, w[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.0f;
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * G;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * G; r0 < p.rows; r0 += step) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool live = row < p.rows;
    const int64_t at = live ? row : 0;
    const T* x = static_cast<const T*>(p.x) + at * p.x_ld;
    const T* dy = static_cast<const T*>(p.dy) + at * p.dy_ld;
    const float mean = p.mean[at], low = p.mean[p.rows + at], rstd = p.rstd[at];
    float h[NV][V], g[NV][V], s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      load_row<WHOLE, T, V>(x, col[i], p.dim, left[i] > 0, h[i]);
      load_row<WHOLE, T, V>(dy, col[i], p.dim, left[i] > 0 && live, g[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[i][j] = j < left[i] ? (h[i][j] - mean - low) * rstd : 0.0f;
        if (live) {
          dw[i][j] = fmaf(g[i][j], h[i][j], dw[i][j]);
          db[i][j] += g[i][j];
        }
        g[i][j] *= w[i][j];
        s[0] += g[i][j];
        s[1] = fmaf(g[i][j], h[i][j], s[1]);
      }
    if (p.y == nullptr) continue;
    row_sums<TPR>(s);
    if (!live) continue;
    const float mg = s[0] * inv, mgh = s[1] * inv;
    T* dx = static_cast<T*>(p.y) + row * p.dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) g[i][j] = rstd * (g[i][j] - fmaf(h[i][j], mgh, mg));
      if (left[i] > 0) store_pack<T, V>(dx + col[i], left[i], g[i], p.stream);
    }
  }
  if (p.partial == nullptr) return;
  float* out = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * p.dim;
  const bool last = gridDim.x == 1;
  // the G rows that were worked on side by side, added in order
  __shared__ float sh[G][TPR * NV * V];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    void* final_out = which ? p.db : p.dw;
    if (G == 1 && !last) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (left[i] > 0)
          store_pack<float, V>(out + which * p.dim + col[i], left[i], which ? db[i] : dw[i]);
      continue;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j)
        sh[threadIdx.x / TPR][(i * TPR + sub) * V + j] = which ? db[i][j] : dw[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < p.dim; c += kBlock) {
      float t = 0.0f;
#pragma unroll
      for (int k = 0; k < G; ++k) t += sh[k][c];
      if (!last)
        out[which * p.dim + c] = t;
      else if (final_out && p.w_f32)
        static_cast<float*>(final_out)[c] = t;
      else if (final_out)
        static_cast<T*>(final_out)[c] = static_cast<T>(t);
    }
  }
}

// ---- rows too wide for the registers: one workgroup per row, every pass reads it again ------------
template <typename T>
__global__ __launch_bounds__(kBlock) void norm_fwd_wide_kernel(const NormParams p) {
  constexpr int V = kVec<T>;
  const float inv = 1.0f / static_cast<float>(p.dim);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
    float v[V], s[1] = {0.0f};
    for (int c = threadIdx.x * V; c < p.dim; c += kBlock * V) {
      load_pack<T, V>(x + c, p.dim - c, v);
#pragma unroll
      for (int j = 0; j < V; ++j) s[0] += v[j];
    }
    row_sums<kBlock>(s);
    const float first = s[0] * inv;
    float t[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x * V; c < p.dim; c += kBlock * V) {
      load_pack<T, V>(x + c, p.dim - c, v);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = c + j < p.dim ? v[j] - first : 0.0f;
        t[0] += d;
        t[1] = fmaf(d, d, t[1]);
      }
    }
    row_sums<kBlock>(t);
    const float off = t[0] * inv;
    const float rstd = 1.0f / sqrtf(variance(t[1] * inv, off) + p.eps);
    T* y = static_cast<T*>(p.y) + row * p.dim;
    for (int c = threadIdx.x * V; c < p.dim; c += kBlock * V) {
      float w[V], b[V];
      load_pack<T, V>(x + c, p.dim - c, v);
      load_param<T, V>(p.w, p.w_f32, c, p.dim - c, 1.0f, w);
      load_param<T, V>(p.b, p.w_f32, c, p.dim - c, 0.0f, b);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = fmaf((v[j] - first - off) * rstd, w[j], b[j]);
      store_pack<T, V>(y + c, p.dim - c, v);
    }
    if (threadIdx.x == 0 && p.mean) keep_stats(p, row, first, off, rstd);
  }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void norm_dx_wide_kernel(const NormParams p) {
  constexpr int V = kVec<T>;
  const float inv = 1.0f / static_cast<float>(p.dim);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
    const T* dy = static_cast<const T*>(p.dy) + row * p.dy_ld;
    const float mean = p.mean[row], low = p.mean[p.rows + row], rstd = p.rstd[row];
    float h[V], g[V], w[V], s[2] = {0.0f, 0.0f};
    auto load = [&](int c) {
      load_pack<T, V>(x + c, p.dim - c, h);
      load_pack<T, V>(dy + c, p.dim - c, g);
      load_param<T, V>(p.w, p.w_f32, c, p.dim - c, 1.0f, w);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[j] = c + j < p.dim ? (h[j] - mean - low) * rstd : 0.0f;
        g[j] *= w[j];
      }
    };
    for (int c = threadIdx.x * V; c < p.dim; c += kBlock * V) {
      load(c);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[0] += g[j];
        s[1] = fmaf(g[j], h[j], s[1]);
      }
    }
    row_sums<kBlock>(s);
    const float mg = s[0] * inv, mgh = s[1] * inv;
    T* dx = static_cast<T*>(p.y) + row * p.dim;
    for (int c = threadIdx.x * V; c < p.dim; c += kBlock * V) {
      load(c);
#pragma unroll
      for (int j = 0; j < V; ++j) g[j] = rstd * (g[j] - fmaf(h[j], mgh, mg));
      store_pack<T, V>(dx + c, p.dim - c, g);
    }
  }
}

// workgroup (i, k): columns [256 i, ...) over every gridDim.y-th row from k on
template <typename T>
__global__ __launch_bounds__(kBlock) void norm_dw_wide_kernel(const NormParams p) {
  const int c = blockIdx.x * kBlock + threadIdx.x;
  if (c >= p.dim) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float g = static_cast<float>(static_cast<const T*>(p.dy)[row * p.dy_ld + c]);
    const float x = static_cast<float>(static_cast<const T*>(p.x)[row * p.x_ld + c]);
    dw = fmaf(g, (x - p.mean[row] - p.mean[p.rows + row]) * p.rstd[row], dw);
    db += g;
  }
  float* out = p.partial + static_cast<int64_t>(blockIdx.y) * 2 * p.dim;
  out[c] = dw;
  out[p.dim + c] = db;
}

// dw, db from the partials: a workgroup adds 64 columns, 16 slices of the partials side by side
template <typename T>
__global__ __launch_bounds__(kRedCols* kRedRows) void norm_reduce_kernel(
    const float* __restrict__ partial, int count, int dim, int out_f32, void* __restrict__ dw,
    void* __restrict__ db) {
  __shared__ float sh[kRedRows][kRedCols];
  const int cx = threadIdx.x % kRedCols, ry = threadIdx.x / kRedCols;
  const int c = blockIdx.x * kRedCols + cx;
  float t = 0.0f;
  if (c < 2 * dim) {
#pragma unroll 8
    for (int k = ry; k < count; k += kRedRows) t += partial[static_cast<int64_t>(k) * 2 * dim + c];
  }
  sh[ry][cx] = t;
  __syncthreads();
  if (ry != 0 || c >= 2 * dim) return;
  t = 0.0f;
#pragma unroll
  for (int k = 0; k < kRedRows; ++k) t += sh[k][cx];
  void* out = c < dim ? dw : db;
  if (out == nullptr) return;
  const int at = c < dim ? c : c - dim;
  if (out_f32)
    static_cast<float*>(out)[at] = t;
  else
    static_cast<T*>(out)[at] = static_cast<T>(t);
}

// lanes per row and packs per lane, from the packs of a row; tpr = 0: the wide kernels
constexpr int kMaxPacks = 8;
struct NormShape {
  int tpr, nv;
};
template <typename T>
NormShape norm_shape(int dim) {
  const int packs = (dim + kVec<T> - 1) / kVec<T>;
  if (packs <= 16) return {16, 1};
  if (packs <= 32) return {32, 1};
  if (packs <= 64) return {64, 1};
  if (packs <= 128) return {64, 2};
  if (packs <= 256) return {64, 4};
  if (packs <= 512) return {256, 2};
  if (packs <= 1024) return {256, 4};
  // 8 packs of 8 values would be 64 registers per array: only float32 rows get that many
  if (packs <= 2048 && kVec<T> == 4) return {256, kMaxPacks};
  return {0, 0};
}

// workgroups of the backward pass; the partials of at least four rows per lane group are added in
// registers before anything is written
template <typename T>
int norm_partials(int64_t rows, int dim) {
  const NormShape s = norm_shape<T>(dim);
  const int64_t per = s.tpr ? 4 * (kBlock / s.tpr) : 64;
  const int64_t want = (rows + per - 1) / per;
  const int64_t most = s.tpr ? kMaxPartials : 64;
  return static_cast<int>(want < 1 ? 1 : want < most ? want : most);
}

template <typename T, bool BWD>
int launch_norm(const NormParams& p, unsigned grid, hipStream_t stream) {
  const NormShape s = norm_shape<T>(p.dim);
  const bool whole = p.dim % kVec<T> == 0;
#define COLLIE_NORM(TPR, NV)                                                                        \
  if (s.tpr == TPR && s.nv == NV) {                                                                 \
    auto* kernel = BWD ? (whole ? norm_bwd_kernel<T, TPR, NV, true> : norm_bwd_kernel<T, TPR, NV, false>)  \
                       : (whole ? norm_fwd_kernel<T, TPR, NV, true> : norm_fwd_kernel<T, TPR, NV, false>); \
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kBlock), 0, stream, p);                             \
    return check_launch("layer norm kernel");                                                       \
  }
  COLLIE_NORM(16, 1)
  COLLIE_NORM(32, 1)
  COLLIE_NORM(64, 1)
  COLLIE_NORM(64, 2)
  COLLIE_NORM(64, 4)
  COLLIE_NORM(256, 2)
  COLLIE_NORM(256, 4)
  if constexpr (kVec<T> == 4) {
    COLLIE_NORM(256, 8)
  }
#undef COLLIE_NORM
  set_error("layer_norm: no kernel for %d columns", p.dim);
  return -1;
}

int check_norm(const char* who, int64_t rows, int32_t dim, int64_t x_ld, int32_t w_dtype,
               int32_t dtype) {
  COLLIE_REQUIRE(rows >= 0 && rows < (int64_t{1} << 40), "%s: bad number of rows", who);
  COLLIE_REQUIRE(dim >= 1 && dim <= (1 << 20), "%s: dim must be in [1, 2^20]", who);
  COLLIE_REQUIRE(rows <= 1 || x_ld >= dim, "%s: rows overlap", who);
  COLLIE_REQUIRE(w_dtype == dtype || w_dtype == COLLIE_F32,
                 "%s: weight and bias are float32 or of the rows' type", who);
  return 0;
}

}  // namespace
}  // namespace collie

using namespace collie;

extern "C" int collie_layer_norm_forward(const void* x, int64_t x_ld, int32_t dtype, int64_t rows,
                                         int32_t dim, const void* weight, const void* bias,
                                         int32_t w_dtype, float eps, void* y, float* mean,
                                         float* rstd, collie_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (check_norm("layer_norm_forward", rows, dim, x_ld, w_dtype, dtype)) return -1;
  COLLIE_REQUIRE(eps >= 0.0f, "layer_norm_forward: eps must not be negative");
  if (rows == 0) return 0;
  COLLIE_REQUIRE(x && y, "layer_norm_forward: NULL pointer");
  COLLIE_REQUIRE((mean == nullptr) == (rstd == nullptr),
                 "layer_norm_forward: mean and rstd belong together");
  return with_type(dtype, "layer_norm_forward", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    NormParams p;
    memset(&p, 0, sizeof(p));
    p.x = x;
    p.w = weight;
    p.b = bias;
    p.y = y;
    p.mean = mean;
    p.rstd = rstd;
    p.rows = rows;
    p.x_ld = x_ld;
    p.dim = dim;
    p.w_f32 = w_dtype == COLLIE_F32;
    p.eps = eps;
    p.stream = rows * dim * static_cast<int64_t>(sizeof(T)) >= kStreamBytes;
    const NormShape s = norm_shape<T>(dim);
    const int64_t groups = s.tpr ? kBlock / s.tpr : 1;
    int64_t grid = (rows + groups - 1) / groups;
    if (grid > 8192) grid = 8192;
    if (s.tpr) return launch_norm<T, false>(p, static_cast<unsigned>(grid), stream);
    hipLaunchKernelGGL(norm_fwd_wide_kernel<T>, dim3(static_cast<unsigned>(grid)), dim3(kBlock), 0,
                       stream, p);
    return check_launch("norm_fwd_wide_kernel");
  });
}

extern "C" size_t collie_layer_norm_backward_workspace_bytes(int64_t rows, int32_t dim) {
  if (rows < 1 || dim < 1) return 256;
  const int a = norm_partials<float>(rows, dim), b = norm_partials<bf16_t>(rows, dim);
  return align_up(static_cast<size_t>(a > b ? a : b) * 2 * dim * sizeof(float), 256);
}

extern "C" int collie_layer_norm_backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld,
                                          int32_t dtype, int64_t rows, int32_t dim,
                                          const void* weight, int32_t w_dtype, const float* mean,
                                          const float* rstd, void* dx, void* dweight, void* dbias,
                                          void* workspace, size_t workspace_bytes,
                                          collie_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (check_norm("layer_norm_backward", rows, dim, x_ld, w_dtype, dtype)) return -1;
  COLLIE_REQUIRE(rows <= 1 || dy_ld >= dim, "layer_norm_backward: rows of dy overlap");
  COLLIE_REQUIRE(rows == 0 || (dy && x && mean && rstd), "layer_norm_backward: NULL pointer");
  const bool sums = dweight || dbias;
  COLLIE_REQUIRE(!sums || rows == 0 ||
                     (workspace && workspace_bytes >=
                                       collie_layer_norm_backward_workspace_bytes(rows, dim)),
                 "workspace too small: need %zu bytes, got %zu",
                 collie_layer_norm_backward_workspace_bytes(rows, dim), workspace_bytes);
  return with_type(dtype, "layer_norm_backward", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    NormParams p;
    memset(&p, 0, sizeof(p));
    p.x = x;
    p.dy = dy;
    p.w = weight;
    p.y = dx;
    p.mean = const_cast<float*>(mean);
    p.rstd = const_cast<float*>(rstd);
    p.partial = sums ? static_cast<float*>(workspace) : nullptr;
    p.rows = rows;
    p.x_ld = x_ld;
    p.dy_ld = dy_ld;
    p.dim = dim;
    p.w_f32 = w_dtype == COLLIE_F32;
    p.stream = rows * dim * static_cast<int64_t>(sizeof(T)) >= kStreamBytes;
    const int count = rows ? norm_partials<T>(rows, dim) : 0;
    p.dw = dweight;
    p.db = dbias;
    const NormShape s = norm_shape<T>(dim);
    if (rows && s.tpr && (dx || sums)) {
      if (const int rc = launch_norm<T, true>(p, static_cast<unsigned>(count), stream)) return rc;
      if (count == 1) return 0;  // the workgroup has written the sums
    } else if (rows) {
      if (dx) {
        hipLaunchKernelGGL(norm_dx_wide_kernel<T>, dim3(static_cast<unsigned>(rows < 8192 ? rows : 8192)),
                           dim3(kBlock), 0, stream, p);
        if (check_launch("norm_dx_wide_kernel")) return -2;
      }
      if (sums) {
        hipLaunchKernelGGL(norm_dw_wide_kernel<T>, dim3((dim + kBlock - 1) / kBlock, count),
                           dim3(kBlock), 0, stream, p);
        if (check_launch("norm_dw_wide_kernel")) return -2;
      }
    }
    if (!sums) return 0;
    hipLaunchKernelGGL(norm_reduce_kernel<T>, dim3((2 * dim + kRedCols - 1) / kRedCols),
                       dim3(kRedCols * kRedRows), 0, stream, p.partial, count, dim, p.w_f32, dweight,
                       dbias);
    return check_launch("norm_reduce_kernel");
  });
}
