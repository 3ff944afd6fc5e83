// K13: the linear layer with bias, activation and residual, and the gated layer, with their
// gradients.
//   linear   z = x W^T + b                      y = f(z) + residual
//            dz = dy f'(z)                      dx = dz W, dW = dz^T x, db = column sums of dz
//   gated    g = x Wg^T + bg, u = x Wu^T + bu   y = f(g) u
//            dg = dy u f'(g), du = dy f(g)      dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
// Everything is a matrix product with something done to its result, so there is one product kernel:
// the gated forward pass has two accumulators per output, the gated dx runs over [dg | du] and
// [Wg ; Wu] as one product of twice the depth, and both weight gradients are one product whose rows
// are the columns of [dg | du].  Products are summed in float32.
#include "head_act.h"

namespace collie {
namespace {

constexpr int kBlock = 256;

// element (i, k) of an operand: p[i * rs + k * ks]
struct Mat {
  const void* p;
  int64_t rs, ks;
};

enum Epilogue { kEpiLinear, kEpiGated, kEpiStore, kEpiPartial };

struct Gemm {
  Mat a, b;
  const void* b2;        // second matrix of b's shape, or NULL
  int64_t k_split;       // without kEpiGated: k >= k_split reads b2 at k - k_split, and of either
  int64_t k_valid;       // matrix only the first k_valid are there (the rest is padding: zero)
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
  float* partial;        // kEpiPartial: [splits, m, n]
};

// results at (row, col .. col + W): columns of one row that one thread holds
template <typename T, int EPI, int W>
__device__ __forceinline__ void finish_row(const Gemm& g, int64_t row, int64_t col, float (&v)[W],
                                           float (&u)[W]) {
  if (row >= g.m || col >= g.n) return;
  const int left = g.n - col < W ? static_cast<int>(g.n - col) : W;
  const int64_t at = row * g.n + col;
  if constexpr (EPI == kEpiPartial) {
    store_pack<float, W>(g.partial + static_cast<int64_t>(blockIdx.z) * g.m * g.n + at, left, v);
  } else if constexpr (EPI == kEpiStore) {
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

// ---- any sizes, any strides: 64 x 64 results per workgroup, 4 x 4 per thread ----------------------
constexpr int kTile = 64, kDepth = 16;

template <typename T, int EPI>
__global__ __launch_bounds__(kBlock) void gemm_any_kernel(const Gemm g) {
  constexpr bool PAIR = EPI == kEpiGated;
  __shared__ float as[kDepth][kTile + 4], bs[kDepth][kTile + 4], us[PAIR ? kDepth : 1][kTile + 4];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kTile;
  const int64_t col0 = static_cast<int64_t>(blockIdx.y) * kTile;
  const int64_t k0 = static_cast<int64_t>(blockIdx.z) * g.k_chunk;
  const int64_t k1 = k0 + g.k_chunk < g.k ? k0 + g.k_chunk : g.k;
  float acc[4][4], acc2[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = acc2[i][j] = 0.0f;
  for (int64_t kk = k0; kk < k1; kk += kDepth) {
    for (int e = threadIdx.x; e < kTile * kDepth; e += kBlock) {
      // neighbouring threads walk the direction that is contiguous in memory
      const int ak = g.a.ks == 1 ? e % kDepth : e / kTile, ai = g.a.ks == 1 ? e / kDepth : e % kTile;
      const int64_t r = row0 + ai, k = kk + ak;
      as[ak][ai] = r < g.m && k < k1 ? static_cast<float>(static_cast<const T*>(
                                           g.a.p)[r * g.a.rs + k * g.a.ks]) : 0.0f;
      const int bk = g.b.ks == 1 ? e % kDepth : e / kTile, bi = g.b.ks == 1 ? e / kDepth : e % kTile;
      const int64_t c = col0 + bi;
      int64_t kb = kk + bk;
      bool in = c < g.n && kb < k1;
      const T* b = static_cast<const T*>(g.b.p);
      if (PAIR) {
        us[PAIR ? bk : 0][bi] = in ? static_cast<float>(static_cast<const T*>(
                                         g.b2)[c * g.b.rs + kb * g.b.ks]) : 0.0f;
      } else if (g.b2) {
        if (kb >= g.k_split) {
          b = static_cast<const T*>(g.b2);
          kb -= g.k_split;
        }
        in = in && kb < g.k_valid;
      }
      bs[bk][bi] = in ? static_cast<float>(b[c * g.b.rs + kb * g.b.ks]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      float a[4], b[4], u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = as[k][ty * 4 + i];
        b[i] = bs[k][tx * 4 + i];
        if (PAIR) u[i] = us[PAIR ? k : 0][tx * 4 + i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
          if (PAIR) acc2[i][j] = fmaf(a[i], u[j], acc2[i][j]);
        }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    finish_row<T, EPI, 4>(g, row0 + ty * 4 + i, col0 + tx * 4, acc[i], acc2[i]);
}

// ---- dz = dy f'(z) (linear), [dg | du] (gated), and the column sums for the bias gradients --------
struct ActBwd {
  const void *dy, *z, *u;  // z: kept pre-activation (NULL: identity); u: the gated layer's second one
  void* dz;                // [m, dz_ld]; NULL: only the column sums are wanted
  float* partial;          // [gridDim.y, pair * n] or NULL
  int64_t m, n, dy_ld, dz_ld;
  int64_t rows_per_part;
  int act;
};
constexpr int kActLanes = 32;
constexpr int kActRows = kBlock / kActLanes;

template <typename T, bool PAIR>
__global__ __launch_bounds__(kBlock) void act_bwd_kernel(const ActBwd p) {
  constexpr int V = kVec<T>;
  const int lane = threadIdx.x % kActLanes, ry = threadIdx.x / kActLanes;
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * kActLanes + lane) * V;
  const int left = col < p.n ? (p.n - col < V ? static_cast<int>(p.n - col) : V) : 0;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * p.rows_per_part;
  const int64_t r1 = r0 + p.rows_per_part < p.m ? r0 + p.rows_per_part : p.m;
  float sum[V], sum2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = sum2[j] = 0.0f;
  if (left > 0) {
    for (int64_t row = r0 + ry; row < r1; row += kActRows) {
      float dy[V], z[V], d[V], u[V];
      load_pack<T, V>(static_cast<const T*>(p.dy) + row * p.dy_ld + col, left, dy);
      if (p.z) {
        load_pack<T, V>(static_cast<const T*>(p.z) + row * p.n + col, left, z);
        if (PAIR) load_pack<T, V>(static_cast<const T*>(p.u) + row * p.n + col, left, u);
        act_slopes(p.act, z, d);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (PAIR) {
          const float t = dy[j];
          dy[j] = t * u[j] * d[j];
          u[j] = t * z[j];
          sum2[j] += u[j];
        } else if (p.z) {
          dy[j] *= d[j];
        }
        sum[j] += dy[j];
      }
      if (p.dz) {
        // up to the padded width: what lies past n_out is 0
        T* dz = static_cast<T*>(p.dz) + row * p.dz_ld + col;
        const int64_t half = p.dz_ld / (PAIR ? 2 : 1);
        const int room = half - col < V ? static_cast<int>(half - col) : V;
        store_pack<T, V>(dz, room, dy);
        if (PAIR) store_pack<T, V>(dz + half, room, u);
      }
    }
  }
  if (p.partial == nullptr) return;
  __shared__ float sh[kActRows][kActLanes * V];
#pragma unroll
  for (int which = 0; which < (PAIR ? 2 : 1); ++which) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) sh[ry][lane * V + j] = which ? sum2[j] : sum[j];
    __syncthreads();
    for (int c = threadIdx.x; c < kActLanes * V; c += kBlock) {
      const int64_t at = static_cast<int64_t>(blockIdx.x) * kActLanes * V + c;
      if (at >= p.n) continue;
      float t = 0.0f;
#pragma unroll
      for (int k = 0; k < kActRows; ++k) t += sh[k][c];
      p.partial[(static_cast<int64_t>(blockIdx.y) * (PAIR ? 2 : 1) + which) * p.n + at] = t;
    }
  }
}

// out[c] = sum over `count` partials of partial[k][c], c < width, in fixed order; columns from
// `split` on belong to out2, and of either only the first `valid` are wanted.  64 columns x 16 slices of the partials per workgroup.
constexpr int kRedCols = 64, kRedRows = 16;
template <typename T>
__global__ __launch_bounds__(kRedCols* kRedRows) void sum_partials_kernel(
    const float* __restrict__ partial, int64_t count, int64_t width, int64_t split, int64_t valid,
    T* __restrict__ out, T* __restrict__ out2) {
  __shared__ float sh[kRedRows][kRedCols];
  const int cx = threadIdx.x % kRedCols, ry = threadIdx.x / kRedCols;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kRedCols + cx;
  float t = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (int64_t k = ry; k < count; k += kRedRows) t += partial[k * width + c];
  }
  sh[ry][cx] = t;
  __syncthreads();
  if (ry != 0 || c >= width) return;
  t = 0.0f;
#pragma unroll
  for (int k = 0; k < kRedRows; ++k) t += sh[k][cx];
  T* o = c < split ? out : out2;
  const int64_t at = c < split ? c : c - split;
  if (o && at < valid) o[at] = static_cast<T>(t);
}

template <typename T>
int sum_partials(const float* partial, int64_t count, int64_t width, int64_t split, int64_t valid,
                 void* out, void* out2, hipStream_t stream) {
  hipLaunchKernelGGL(sum_partials_kernel<T>, dim3(static_cast<unsigned>((width + kRedCols - 1) / kRedCols)),
                     dim3(kRedCols * kRedRows), 0, stream, partial, count, width, split,
                     valid, static_cast<T*>(out), static_cast<T*>(out2));
  return check_launch("sum_partials_kernel");
}

template <typename T, int EPI>
int launch_gemm(const Gemm& g, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((g.m + kTile - 1) / kTile),
                  static_cast<unsigned>((g.n + kTile - 1) / kTile), static_cast<unsigned>(g.splits));
  hipLaunchKernelGGL((gemm_any_kernel<T, EPI>), grid, dim3(kBlock), 0, stream, g);
  return check_launch("gemm_any_kernel");
}

// parts of the depth of a weight gradient: enough workgroups for every CU, each at least 256 deep
int weight_splits(int64_t rows, int64_t n, int64_t m) {
  const int64_t tiles = ((n + kTile - 1) / kTile) * ((m + kTile - 1) / kTile);
  int64_t s = (1024 + tiles - 1) / tiles;
  if (s > rows / 256) s = rows / 256;
  return static_cast<int>(s < 1 ? 1 : s);
}

// rows per slice of the column sums, and slices
constexpr int64_t kActParts = 512;
int64_t act_parts(int64_t m) {
  const int64_t parts = (m + 4 * kActRows - 1) / (4 * kActRows);
  return parts < kActParts ? parts : kActParts;
}

// columns of one half of dz: whole 16-byte packs
int64_t padded(int64_t n, int32_t dtype) {
  const int64_t v = 16 / static_cast<int64_t>(type_size(dtype));
  return (n + v - 1) / v * v;
}

struct BwdWs {
  void* dz;
  float* act_partial;
  float* w_partial;
  int splits;
  size_t bytes;
};

BwdWs carve_bwd(void* base, int32_t dtype, int64_t m, int64_t n_in, int64_t n_out, bool pair) {
  Carver c(base);
  BwdWs w;
  const int64_t wide = pair ? 2 : 1;
  w.dz = c.take<char>(static_cast<size_t>(m) * wide * padded(n_out, dtype) * type_size(dtype));
  w.act_partial = c.take<float>(static_cast<size_t>(act_parts(m)) * wide * n_out);
  w.splits = weight_splits(m, wide * n_out, n_in);
  w.w_partial = c.take<float>(w.splits > 1 ? static_cast<size_t>(w.splits) * wide * padded(n_out, dtype) * n_in : 1);
  w.bytes = align_up(c.off, 256);
  return w;
}

int check_layer(const char* who, int64_t m, int32_t n_in, int32_t n_out, int64_t x_ld, int32_t act) {
  COLLIE_REQUIRE(m >= 0 && m < (int64_t{1} << 31), "%s: bad number of rows", who);
  COLLIE_REQUIRE(n_in >= 1 && n_out >= 1 && n_in <= (1 << 20) && n_out <= (1 << 20),
                 "%s: widths must be in [1, 2^20]", who);
  COLLIE_REQUIRE(m <= 1 || x_ld >= n_in, "%s: rows of x overlap", who);
  COLLIE_REQUIRE(act >= COLLIE_ACT_IDENTITY && act <= COLLIE_ACT_GELU, "%s: unknown activation %d",
                 who, act);
  return 0;
}

template <typename T>
int layer_forward(const void* x, int64_t x_ld, const void* w, const void* w2, const void* bias,
                  const void* bias2, const void* residual, int64_t res_ld, int64_t m, int64_t n_in,
                  int64_t n_out, int act, void* keep, void* keep2, void* y, hipStream_t stream) {
  Gemm g;
  memset(&g, 0, sizeof(g));
  g.a = {x, x_ld, 1};
  g.b = {w, n_in, 1};
  g.b2 = w2;
  g.m = m;
  g.n = n_out;
  g.k = g.k_chunk = n_in;
  g.splits = 1;
  g.act = act;
  g.bias = bias;
  g.bias2 = bias2;
  g.residual = residual;
  g.res_ld = res_ld;
  g.keep = keep;
  g.keep2 = keep2;
  g.c = y;
  return w2 ? launch_gemm<T, kEpiGated>(g, stream) : launch_gemm<T, kEpiLinear>(g, stream);
}

template <typename T>
int layer_backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, const void* w,
                   const void* w2, const void* z, const void* u, int32_t dtype, int64_t m,
                   int64_t n_in, int64_t n_out, int act, void* dx, void* dw, void* dw2, void* db,
                   void* db2, void* workspace, hipStream_t stream) {
  const bool pair = w2 != nullptr;
  const BwdWs ws = carve_bwd(workspace, dtype, m, n_in, n_out, pair);
  const int64_t wide = pair ? 2 : 1;
  const void* dz = dy;
  int64_t dz_ld = dy_ld, half = n_out;
  const bool sums = db || db2;
  if (z || sums) {
    ActBwd p;
    memset(&p, 0, sizeof(p));
    p.dy = dy;
    p.z = z;
    p.u = u;
    p.m = m;
    p.n = n_out;
    p.dy_ld = dy_ld;
    p.act = act;
    if (z) {
      half = padded(n_out, dtype);
      dz_ld = wide * half;
      dz = p.dz = ws.dz;
      p.dz_ld = dz_ld;
    }
    p.partial = sums ? ws.act_partial : nullptr;
    const int64_t parts = act_parts(m);
    p.rows_per_part = (m + parts - 1) / parts;
    const int64_t cols = kActLanes * kVec<T>;
    const dim3 grid(static_cast<unsigned>((n_out + cols - 1) / cols), static_cast<unsigned>(parts));
    if (pair)
      hipLaunchKernelGGL((act_bwd_kernel<T, true>), grid, dim3(kBlock), 0, stream, p);
    else
      hipLaunchKernelGGL((act_bwd_kernel<T, false>), grid, dim3(kBlock), 0, stream, p);
    if (check_launch("act_bwd_kernel")) return -2;
    if (sums) {
      if (const int rc = sum_partials<T>(ws.act_partial, parts, wide * n_out, n_out, n_out, db, db2,
                                           stream))
        return rc;
    }
  }
  Gemm g;
  if (dx) {
    memset(&g, 0, sizeof(g));
    g.a = {dz, dz_ld, 1};
    g.b = {w, 1, n_in};
    g.b2 = w2;
    g.k_split = half;
    g.k_valid = n_out;
    g.m = m;
    g.n = n_in;
    g.k = g.k_chunk = pair ? half + n_out : n_out;
    g.splits = 1;
    g.c = dx;
    g.row_split = g.row_valid = m;
    if (const int rc = launch_gemm<T, kEpiStore>(g, stream)) return rc;
  }
  if (dw || dw2) {
    memset(&g, 0, sizeof(g));
    g.a = {dz, 1, dz_ld};
    g.b = {x, 1, x_ld};
    g.m = pair ? half + n_out : n_out;
    g.n = n_in;
    g.k = m;
    g.splits = ws.splits;
    g.k_chunk = (m + g.splits - 1) / g.splits;
    g.row_split = half;
    g.row_valid = n_out;
    g.c = dw;
    g.c2 = dw2;
    g.partial = ws.w_partial;
    if (g.splits == 1) return launch_gemm<T, kEpiStore>(g, stream);
    if (const int rc = launch_gemm<T, kEpiPartial>(g, stream)) return rc;
    return sum_partials<T>(ws.w_partial, g.splits, g.m * g.n, half * g.n, n_out * g.n, dw, dw2,
                           stream);
  }
  return 0;
}

}  // namespace
}  // namespace collie

using namespace collie;

extern "C" size_t collie_layer_backward_workspace_bytes(int32_t dtype, int64_t m, int32_t n_in,
                                                        int32_t n_out, int32_t pair) {
  if (m < 1 || n_in < 1 || n_out < 1) return 256;
  return carve_bwd(nullptr, dtype, m, n_in, n_out, pair != 0).bytes;
}

extern "C" int collie_linear_forward(const void* x, int64_t x_ld, int32_t dtype, int64_t m,
                                     int32_t n_in, const void* weight, const void* bias,
                                     int32_t n_out, int32_t act, const void* residual,
                                     int64_t res_ld, void* keep, void* y, collie_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (check_layer("linear_forward", m, n_in, n_out, x_ld, act)) return -1;
  COLLIE_REQUIRE(!residual || m <= 1 || res_ld >= n_out, "linear_forward: rows of residual overlap");
  if (m == 0) return 0;
  COLLIE_REQUIRE(x && weight && y, "linear_forward: NULL pointer");
  return with_type(dtype, "linear_forward", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    return layer_forward<T>(x, x_ld, weight, nullptr, bias, nullptr, residual, res_ld, m, n_in,
                            n_out, act, keep, nullptr, y, stream);
  });
}

extern "C" int collie_gated_forward(const void* x, int64_t x_ld, int32_t dtype, int64_t m,
                                    int32_t n_in, const void* gate_weight, const void* up_weight,
                                    const void* gate_bias, const void* up_bias, int32_t n_out,
                                    int32_t act, void* keep_gate, void* keep_up, void* y,
                                    collie_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (check_layer("gated_forward", m, n_in, n_out, x_ld, act)) return -1;
  COLLIE_REQUIRE((gate_bias == nullptr) == (up_bias == nullptr),
                 "gated_forward: both biases or none");
  COLLIE_REQUIRE((keep_gate == nullptr) == (keep_up == nullptr),
                 "gated_forward: keep_gate and keep_up belong together");
  if (m == 0) return 0;
  COLLIE_REQUIRE(x && gate_weight && up_weight && y, "gated_forward: NULL pointer");
  return with_type(dtype, "gated_forward", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    return layer_forward<T>(x, x_ld, gate_weight, up_weight, gate_bias, up_bias, nullptr, 0, m, n_in,
                            n_out, act, keep_gate, keep_up, y, stream);
  });
}

extern "C" int collie_linear_backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld,
                                      int32_t dtype, int64_t m, int32_t n_in, const void* weight,
                                      int32_t n_out, int32_t act, const void* kept_z, void* dx,
                                      void* dweight, void* dbias, void* workspace,
                                      size_t workspace_bytes, collie_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (check_layer("linear_backward", m, n_in, n_out, x_ld, act)) return -1;
  COLLIE_REQUIRE(m <= 1 || dy_ld >= n_out, "linear_backward: rows of dy overlap");
  COLLIE_REQUIRE(m >= 1, "linear_backward: no rows");
  COLLIE_REQUIRE(dy && x && weight, "linear_backward: NULL pointer");
  COLLIE_REQUIRE((act == COLLIE_ACT_IDENTITY) == (kept_z == nullptr),
                 "linear_backward: kept_z is what the forward pass kept (NULL for the identity)");
  const size_t need = collie_layer_backward_workspace_bytes(dtype, m, n_in, n_out, 0);
  COLLIE_REQUIRE(workspace && workspace_bytes >= need, "workspace too small: need %zu bytes, got %zu",
                 need, workspace_bytes);
  return with_type(dtype, "linear_backward", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    return layer_backward<T>(dy, dy_ld, x, x_ld, weight, nullptr, kept_z, nullptr, dtype, m, n_in,
                             n_out, act, dx, dweight, nullptr, dbias, nullptr, workspace, stream);
  });
}

extern "C" int collie_gated_backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld,
                                     int32_t dtype, int64_t m, int32_t n_in, const void* gate_weight,
                                     const void* up_weight, int32_t n_out, int32_t act,
                                     const void* kept_gate, const void* kept_up, void* dx,
                                     void* dgate_weight, void* dup_weight, void* dgate_bias,
                                     void* dup_bias, void* workspace, size_t workspace_bytes,
                                     collie_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (check_layer("gated_backward", m, n_in, n_out, x_ld, act)) return -1;
  COLLIE_REQUIRE(m <= 1 || dy_ld >= n_out, "gated_backward: rows of dy overlap");
  COLLIE_REQUIRE(m >= 1, "gated_backward: no rows");
  COLLIE_REQUIRE(dy && x && gate_weight && up_weight && kept_gate && kept_up,
                 "gated_backward: NULL pointer");
  const size_t need = collie_layer_backward_workspace_bytes(dtype, m, n_in, n_out, 1);
  COLLIE_REQUIRE(workspace && workspace_bytes >= need, "workspace too small: need %zu bytes, got %zu",
                 need, workspace_bytes);
  return with_type(dtype, "gated_backward", [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    return layer_backward<T>(dy, dy_ld, x, x_ld, gate_weight, up_weight, kept_gate, kept_up, dtype, m,
                             n_in, n_out, act, dx, dgate_weight, dup_weight, dgate_bias, dup_bias,
                             workspace, stream);
  });
}
