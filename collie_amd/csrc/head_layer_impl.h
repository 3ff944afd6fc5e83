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
#pragma once

#include "head_layer.h"
#include "head_tile.h"

namespace collie {
namespace {

constexpr int kBlock = 256;

// ---- dz = dy f'(z) (linear), [dg | du] (gated), and the column sums for the bias gradients --------
// dz goes to the products in the element type, because that is what the matrix instructions multiply:
// one more rounding in dx and dW of 16-bit layers (1.41 times the error of one, in the mean; more bits
// would take two products instead of one).  The bias gradients are summed before it.
struct ActBwd {
  const void *dy;
  const void *z, *u;       // kept pre-activations (head_act.h; NULL: identity)
  void* dz;                // [m, dz_ld]; NULL: only the column sums are wanted
  float* partial;          // [gridDim.y, pair * n]: column sums, or NULL
  void *db, *db2;          // gridDim.y = 1: the sums themselves (either may be NULL) instead
  int64_t m, n, dy_ld, dz_ld;
  int64_t rows_per_part;
  int act;
  bool stream;             // dz is stored past the caches
  uint32_t* over;          // float16 (or NULL): set where a finite value of dz is past the type's range,
  bool again;              // and the second launch, which stores dz times kDzScale if it is set
};
constexpr int kActLanes = 32;
constexpr int kActRows = kBlock / kActLanes;

__device__ __forceinline__ bool past_half(float v) {
  return fabsf(v) > kHalfMax && fabsf(v) < INFINITY;
}

template <typename T, bool PAIR>
__global__ __launch_bounds__(kBlock) void act_bwd_kernel(const ActBwd p) {
  constexpr int V = kVec<T>;
  constexpr bool HALF = std::is_same<T, f16_t>::value;
  if (HALF && p.again && *p.over == 0) return;
  const int lane = threadIdx.x % kActLanes, ry = threadIdx.x / kActLanes;
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * kActLanes + lane) * V;
  const int left = col < p.n ? (p.n - col < V ? static_cast<int>(p.n - col) : V) : 0;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * p.rows_per_part;
  const int64_t r1 = r0 + p.rows_per_part < p.m ? r0 + p.rows_per_part : p.m;
  float sum[V], sum2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = sum2[j] = 0.0f;
  bool over = false;
  if (left > 0) {
    for (int64_t row = r0 + ry; row < r1; row += kActRows) {
      float dy[V], z[V], d[V], u[V];
      load_pack<T, V>(static_cast<const T*>(p.dy) + row * p.dy_ld + col, left, dy);
      if (p.z) {
        if (PAIR || kept_in_float(p.act))
          load_pack<float, V>(static_cast<const float*>(p.z) + row * p.n + col, left, z);
        else
          load_pack<T, V>(static_cast<const T*>(p.z) + row * p.n + col, left, z);
        if (PAIR) load_pack<float, V>(static_cast<const float*>(p.u) + row * p.n + col, left, u);
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
        if (HALF) {
          over = over || past_half(dy[j]) || (PAIR && past_half(u[j]));
          if (p.again) {
            dy[j] *= kDzScale;
            if (PAIR) u[j] *= kDzScale;
          }
        }
      }
      if (p.dz) {
        // up to the padded width: what lies past n_out is 0
        T* dz = static_cast<T*>(p.dz) + row * p.dz_ld + col;
        const int64_t half = p.dz_ld / (PAIR ? 2 : 1);
        const int room = half - col < V ? static_cast<int>(half - col) : V;
        store_pack<T, V>(dz, room, dy, p.stream);
        if (PAIR) store_pack<T, V>(dz + half, room, u, p.stream);
      }
    }
  }
  if (HALF && p.over && !p.again && __any(over) && (threadIdx.x & (kWave - 1)) == 0) atomicOr(p.over, 1u);
  if (p.partial == nullptr && p.db == nullptr && p.db2 == nullptr) return;
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
      if (p.partial) {
        p.partial[(static_cast<int64_t>(blockIdx.y) * (PAIR ? 2 : 1) + which) * p.n + at] = t;
      } else {
        T* db = static_cast<T*>(which ? p.db2 : p.db);
        if (db) db[at] = static_cast<T>(t);
      }
    }
  }
}

__global__ void clear_word_kernel(uint32_t* word) { *word = 0; }

// out[c] = sum over `count` partials of partial[k][c], c < width, in fixed order; columns from
// `split` on belong to out2.  64 columns x 16 slices of the partials per workgroup.
constexpr int kRedCols = 64, kRedRows = 16;
template <typename T>
__global__ __launch_bounds__(kRedCols* kRedRows) void sum_partials_kernel(
    const float* __restrict__ partial, int64_t count, int64_t width, int64_t split,
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
  if (o) o[c < split ? c : c - split] = static_cast<T>(t);
}

template <typename T>
int sum_partials(const float* partial, int64_t count, int64_t width, int64_t split, void* out,
                 void* out2, hipStream_t stream) {
  hipLaunchKernelGGL(sum_partials_kernel<T>, dim3(static_cast<unsigned>((width + kRedCols - 1) / kRedCols)),
                     dim3(kRedCols * kRedRows), 0, stream, partial, count, width, split,
                     static_cast<T*>(out), static_cast<T*>(out2));
  return check_launch("sum_partials_kernel");
}

// ---- laying an operand out for the tiles -----------------------------------------------------------
// The tiles load whole aligned 16-byte packs.  Rows of another width or alignment are copied once
// into rows of whole packs, zeros behind them: one more pass over that operand, for odd widths only.
// All operands of a call go in one launch.
struct PackJobs {
  static constexpr int kMax = 4;
  int n;
  const void* src[kMax];
  void* dst[kMax];
  int64_t ld[kMax], cols[kMax], packs[kMax], total[kMax];  // packs per row, and in all
};

template <typename T>
__global__ __launch_bounds__(kBlock) void pack_rows_kernel(const PackJobs jobs) {
  constexpr int V = kVec<T>;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kBlock;
  for (int k = 0; k < jobs.n; ++k) {
    const T* src = static_cast<const T*>(jobs.src[k]);
    T* dst = static_cast<T*>(jobs.dst[k]);
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < jobs.total[k];
         i += stride) {
      const int64_t row = i / jobs.packs[k], c = (i - row * jobs.packs[k]) * V;
      const int64_t left = jobs.cols[k] - c;
      float v[V];
      load_pack<T, V>(src + row * jobs.ld[k] + c, left < V ? static_cast<int>(left) : V, v);
      store_pack<T, V>(dst + i * V, V, v);
    }
  }
}

template <typename T>
bool whole_packs(const void* p, int64_t ld, int64_t cols) {
  // (a stage's loads have 32-bit offsets from its first row)
  return ld * static_cast<int64_t>(sizeof(T)) < (int64_t{1} << 23) && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % kVec<T> == 0 && cols % kVec<T> == 0;
}

// columns of a row of whole packs
template <typename T>
int64_t padded(int64_t n) {
  return (n + kVec<T> - 1) / kVec<T> * kVec<T>;
}

// `p` in rows of whole packs: itself, or its copy at `room`, which launch_packs() makes
template <typename T>
void lay_out(PackJobs& jobs, const void*& p, int64_t& ld, int64_t rows, int64_t cols, void* room) {
  if (whole_packs<T>(p, ld, cols)) return;
  const int k = jobs.n++;
  jobs.src[k] = p;
  jobs.dst[k] = room;
  jobs.ld[k] = ld;
  jobs.cols[k] = cols;
  jobs.packs[k] = padded<T>(cols) / kVec<T>;
  jobs.total[k] = rows * jobs.packs[k];
  p = room;
  ld = padded<T>(cols);
}

template <typename T>
int launch_packs(const PackJobs& jobs, hipStream_t stream) {
  if (jobs.n == 0) return 0;
  int64_t grid = 1;
  for (int k = 0; k < jobs.n; ++k) {
    const int64_t blocks = (jobs.total[k] + kBlock - 1) / kBlock;
    grid = grid > blocks ? grid : blocks;
  }
  hipLaunchKernelGGL(pack_rows_kernel<T>, dim3(static_cast<unsigned>(grid < 8192 ? grid : 8192)),
                     dim3(kBlock), 0, stream, jobs);
  return check_launch("pack_rows_kernel");
}

// ---- which kernel, and how many parts of the depth -------------------------------------------------
constexpr int64_t kSkinnyRows = 64;  // rows of the kernel that streams the weights
constexpr int64_t kCus = 256;

// A CU holds one workgroup of the 256 x 256 kernel, two of the 128 x 128 one or three of the 128 x 64
// one (LDS), which is there for narrow results: 48 columns fill a third of a 128-wide tile.  The tiles that
// fill whole rounds of the chip are computed as they are; those left over may be cut along the depth,
// so that they fill a round too: 344 tiles of 256 (a weight gradient of 11,008 x 2,048 over 16,384
// rows) took two rounds, 947 us, and take 745 cut.  Tile and parts are the ones with the least time by:
// the products at the rate that all workgroups together reach on large matrices; the stores of a tile
// at a CU's share of a copy's bandwidth (of the workgroups that share a CU one stores while the others
// multiply, so that only its own stores count); a start and an end of a few microseconds.  Against what
// was measured, 128 x 64 / 128 x 128 / 256 x 256 (us): float32 720,896 x 128 -> 256 528 / 463 / 517,
// 200,000 x 256 -> 512 445 / 378 / 431, 65,536 x 1,024 -> 512 492 / 398 / 402, 16,384 x 2,048 -> 5,504
// 2,535 / 2,052 / 1,825; bfloat16 20,000 x 256 -> 256 with kept values 17 / 21 / 34, 720,896 x 64 -> 128
// 56 / 61 / 92, 8,192 x 1,024 -> 4,096 103 / 79 / 84, gated 16,384 x 2,048 -> 5,504 970 / 810 / 757.
struct Plan {
  int bm, bn;
  int64_t slots;  // workgroups that the chip holds
  int64_t tiles, full, splits, k_chunk;
};

// out_bytes: what is stored per accumulator
template <typename T>
Plan plan_gemm(int64_t m, int64_t n, int64_t k, bool pair, double out_bytes) {
  const int64_t depth = 128 / static_cast<int64_t>(sizeof(T));
  const int64_t stages = (k + depth - 1) / depth;
  struct Shape {
    int bm, bn, per_cu;
    double rate16, rate32, ends;
  };
  static const Shape shapes[] = {{128, 64, 3, 0.72e15, 1.48e14, 1.2e-6},
                                 {128, 128, 2, 0.95e15, 1.95e14, 1.5e-6},
                                 {256, 256, 1, 1.12e15, 2.24e14, 3e-6}};
  const double cu_bandwidth = 4.7e12 / kCus;
  Plan best;
  memset(&best, 0, sizeof(best));
  double best_time = 0.0;
  for (const Shape& c : shapes) {
    const int64_t slots = kCus * c.per_cu;
    const int64_t tiles = ((m + c.bm - 1) / c.bm) * ((n * (pair ? 2 : 1) + c.bn - 1) / c.bn);
    const int64_t full = tiles / slots * slots, rest = tiles - full;
    const double area = static_cast<double>(c.bm) * c.bn;
    const double stage = 2.0 * area * depth * slots / (sizeof(T) == 2 ? c.rate16 : c.rate32);
    auto tile_time = [&](int64_t n_stages, double bytes) {
      return n_stages * stage + area * bytes / cu_bandwidth + c.ends;
    };
    for (int64_t q = 0; q <= 4; ++q) {
      int64_t s = q == 0 || rest == 0 ? 1 : q * slots / rest;
      if (s > stages / 4) s = stages / 4;
      if (s < 1) s = 1;
      const int64_t part = (stages + s - 1) / s;
      s = (stages + part - 1) / part;
      const int64_t rounds = (rest * s + slots - 1) / slots;
      double time = tile_time(stages, out_bytes) * (full / slots);
      time += rounds * tile_time(part, s > 1 ? 4.0 : out_bytes);
      // the parts' sums are read again, by a launch of its own
      if (s > 1) time += 4e-6 + (4.0 * s + out_bytes) * rest * area / 4e12;
      if (best.bm == 0 || time < best_time) {
        best_time = time;
        best = {c.bm, c.bn, slots, tiles, s > 1 ? full : tiles, s, part * depth};
      }
    }
  }
  return best;
}

// what the forward pass stores per accumulator when the backward pass is to follow (the linear layer's
// kept values in its own type: the workspace is asked for before the activation is known)
template <typename T>
double stored_bytes(bool pair) {
  return pair ? (sizeof(T) + 8.0) / 2 : 2.0 * sizeof(T);
}

// the products of a layer: x W^T, dz W (gated: over [dg | du] in one) and dz^T x (the columns of [dg | du])
template <typename T>
Plan plan_of(Product product, int64_t m, int64_t n_in, int64_t n_out, bool pair) {
  const int64_t both = pair ? padded<T>(n_out) + n_out : n_out;
  switch (product) {
    case kForward: return plan_gemm<T>(m, n_out, n_in, pair, stored_bytes<T>(pair));
    case kDx: return plan_gemm<T>(m, n_in, both, false, sizeof(T));
    default: return plan_gemm<T>(both, n_in, m, false, sizeof(T));
  }
}

size_t partial_floats(const Plan& p) {
  return static_cast<size_t>(p.splits > 1 ? p.splits * (p.tiles - p.full) * p.bm * p.bn : 0);
}

template <typename T, int BM, int BN, int WM, int WN, bool AKC, bool BKC, int EPI, bool CAT>
int launch_tile(const Gemm& g, const Plan& p, hipStream_t stream) {
  const int64_t rest = p.tiles - p.full;
  const int64_t total = p.full + rest * p.splits;
  hipLaunchKernelGGL((gemm_tile_kernel<T, BM, BN, WM, WN, AKC, BKC, EPI, CAT>),
                     dim3(static_cast<unsigned>(total < p.slots ? total : p.slots)),
                     dim3(kWave * WM * WN), 0, stream, g);
  if (check_launch("gemm_tile_kernel")) return -2;
  if (rest == 0) return 0;
  constexpr int64_t per_tile = BM * BN / (EPI == kEpiGated ? 2 : 1) / 4 / kWave;
  const dim3 grid(static_cast<unsigned>(rest * per_tile));
  if (p.splits <= 8)
    hipLaunchKernelGGL((gemm_finish_kernel<T, BM, BN, EPI, 1>), grid, dim3(kWave), 0, stream, g);
  else
    hipLaunchKernelGGL((gemm_finish_kernel<T, BM, BN, EPI, 8>), grid, dim3(kWave * 8), 0, stream, g);
  return check_launch("gemm_finish_kernel");
}

template <typename T, bool AKC, bool BKC, int EPI, bool CAT>
int launch_tiles(Gemm& g, const Plan& p, hipStream_t stream) {
  g.stream = g.m * g.n * static_cast<int64_t>(sizeof(T)) >= kStreamBytes;
  g.full = p.full;
  g.splits = static_cast<int>(p.splits);
  g.k_chunk = p.k_chunk;
  if (p.bn == 64) return launch_tile<T, 128, 64, 4, 1, AKC, BKC, EPI, CAT>(g, p, stream);
  if (p.bn == 128) return launch_tile<T, 128, 128, 2, 2, AKC, BKC, EPI, CAT>(g, p, stream);
  return launch_tile<T, 256, 256, 2, 4, AKC, BKC, EPI, CAT>(g, p, stream);
}

template <typename T, int EPI>
int launch_skinny(const Gemm& g, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((g.n + 15) / 16)), block(kWave * kSkinnyWaves);
  const bool whole = g.k % kVec<T> == 0;
#define COLLIE_SKINNY(MT)                                                                        \
  if (g.m <= 16 * MT) {                                                                          \
    auto* kernel = whole ? gemm_skinny_kernel<T, MT, EPI, true> : gemm_skinny_kernel<T, MT, EPI, false>; \
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, g);                                       \
    return check_launch("gemm_skinny_kernel");                                                   \
  }
  COLLIE_SKINNY(1)
  COLLIE_SKINNY(2)
  COLLIE_SKINNY(4)
#undef COLLIE_SKINNY
  set_error("matrix product: too many rows for the streaming kernel");
  return -1;
}

// slices of the rows for the column sums: together with the column blocks about eight workgroups per
// CU (with two, 720,896 x 128 float32 ran at 2.8 of the 4.7 TB/s a copy reaches), each of at least
// four rows per lane group
int64_t act_parts(int64_t m, int64_t n, int64_t v) {
  const int64_t columns = (n + kActLanes * v - 1) / (kActLanes * v);
  int64_t parts = (2048 + columns - 1) / columns;
  if (parts < 64) parts = 64;
  if (m <= 16 * kActRows) return 1;  // the sums at once: one launch less
  const int64_t most = (m + 4 * kActRows - 1) / (4 * kActRows);
  return parts < most ? parts : most;
}

// Workspaces.  An operand's room is there only if the operand is not in whole packs already.
struct FwdWs {
  void *x, *w, *w2;
  float* partial;
  size_t bytes;
};

template <typename T>
FwdWs carve_fwd(void* base, const void* x, int64_t x_ld, int64_t m, int64_t n_in, const void* w,
                const void* w2, int64_t n_out) {
  Carver c(base);
  FwdWs ws;
  memset(&ws, 0, sizeof(ws));
  if (m > kSkinnyRows) {
    const size_t wide = static_cast<size_t>(padded<T>(n_in));
    if (!whole_packs<T>(x, x_ld, n_in)) ws.x = c.take<T>(m * wide);
    if (!whole_packs<T>(w, n_in, n_in)) ws.w = c.take<T>(n_out * wide);
    if (w2 && !whole_packs<T>(w2, n_in, n_in)) ws.w2 = c.take<T>(n_out * wide);
    ws.partial = c.take<float>(partial_floats(plan_of<T>(kForward, m, n_in, n_out, w2 != nullptr)));
  }
  ws.bytes = align_up(c.off, 256) + 256;
  return ws;
}

struct BwdWs {
  void *dz, *x, *w, *w2;
  float* act_partial;
  float* partial;
  uint32_t* over;
  size_t bytes;
};

template <typename T>
BwdWs carve_bwd(void* base, const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, int64_t m,
                int64_t n_in, const void* w, const void* w2, int64_t n_out, int act) {
  Carver c(base);
  BwdWs ws;
  memset(&ws, 0, sizeof(ws));
  const int64_t pair = w2 ? 2 : 1;
  const int64_t half = padded<T>(n_out);
  const size_t wide = static_cast<size_t>(padded<T>(n_in));
  if (w2 || act != COLLIE_ACT_IDENTITY || !whole_packs<T>(dy, dy_ld, n_out))
    ws.dz = c.take<T>(static_cast<size_t>(m) * pair * half);
  if (!whole_packs<T>(x, x_ld, n_in)) ws.x = c.take<T>(m * wide);
  if (!whole_packs<T>(w, n_in, n_in)) ws.w = c.take<T>(n_out * wide);
  if (w2 && !whole_packs<T>(w2, n_in, n_in)) ws.w2 = c.take<T>(n_out * wide);
  ws.act_partial = c.take<float>(static_cast<size_t>(act_parts(m, n_out, kVec<T>)) * pair * n_out);
  const size_t a = partial_floats(plan_of<T>(kDx, m, n_in, n_out, w2 != nullptr));
  const size_t b = partial_floats(plan_of<T>(kDw, m, n_in, n_out, w2 != nullptr));
  ws.partial = c.take<float>(a > b ? a : b);
  ws.over = c.take<uint32_t>(1);
  ws.bytes = align_up(c.off, 256) + 256;
  return ws;
}

template <typename T>
int layer_forward(const void* x, int64_t x_ld, const void* w, const void* w2, const void* bias,
                  const void* bias2, const void* residual, int64_t res_ld, int64_t m, int64_t n_in,
                  int64_t n_out, int act, void* keep, void* keep2, void* y, void* workspace,
                  hipStream_t stream) {
  Gemm g;
  memset(&g, 0, sizeof(g));
  g.m = m;
  g.n = n_out;
  g.k = n_in;
  g.act = act;
  g.bias = bias;
  g.bias2 = bias2;
  g.residual = residual;
  g.res_ld = res_ld;
  g.keep = keep;
  g.keep2 = keep2;
  g.c = y;
  int64_t ld = n_in, ld2 = n_in;
  if (m > kSkinnyRows) {
    const FwdWs ws = carve_fwd<T>(workspace, x, x_ld, m, n_in, w, w2, n_out);
    g.partial = ws.partial;
    PackJobs jobs;
    jobs.n = 0;
    lay_out<T>(jobs, x, x_ld, m, n_in, ws.x);
    lay_out<T>(jobs, w, ld, n_out, n_in, ws.w);
    if (w2) lay_out<T>(jobs, w2, ld2, n_out, n_in, ws.w2);
    if (launch_packs<T>(jobs, stream)) return -2;
  }
  g.a = {x, x_ld, 1};
  g.b = {w, ld, 1};
  g.b2 = w2;
  if (m <= kSkinnyRows)
    return w2 ? launch_skinny<T, kEpiGated>(g, stream) : launch_skinny<T, kEpiLinear>(g, stream);
  const Plan p = plan_of<T>(kForward, m, n_in, n_out, w2 != nullptr);
  return w2 ? launch_tiles<T, true, true, kEpiGated, false>(g, p, stream)
            : launch_tiles<T, true, true, kEpiLinear, false>(g, p, stream);
}

template <typename T>
int layer_backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, const void* w,
                   const void* w2, const void* z, const void* u, int64_t m, int64_t n_in,
                   int64_t n_out, int act, void* dx, void* dw, void* dw2, void* db, void* db2,
                   void* workspace, hipStream_t stream) {
  const bool pair = w2 != nullptr;
  const BwdWs ws = carve_bwd<T>(workspace, dy, dy_ld, x, x_ld, m, n_in, w, w2, n_out, act);
  const int64_t wide = pair ? 2 : 1;
  const int64_t half = padded<T>(n_out);
  const void* dz = dy;
  int64_t dz_ld = dy_ld;
  const uint32_t* over = nullptr;
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
      dz = p.dz = ws.dz;
      dz_ld = p.dz_ld = wide * half;
      p.stream = m * dz_ld * static_cast<int64_t>(sizeof(T)) >= kStreamBytes;
    }
    const int64_t parts = act_parts(m, n_out, kVec<T>);
    if (sums && parts > 1) {
      p.partial = ws.act_partial;
    } else {
      p.db = db;
      p.db2 = db2;
    }
    p.rows_per_part = (m + parts - 1) / parts;
    // (|f'| is at most 1 but for silu and gelu)
    if (std::is_same<T, f16_t>::value && z && (dx || dw || dw2) &&
        (pair || act == COLLIE_ACT_SILU || act == COLLIE_ACT_GELU)) {
      p.over = ws.over;
      hipLaunchKernelGGL(clear_word_kernel, dim3(1), dim3(1), 0, stream, p.over);
      if (check_launch("clear_word_kernel")) return -2;
    }
    const int64_t cols = kActLanes * kVec<T>;
    const dim3 grid(static_cast<unsigned>((n_out + cols - 1) / cols), static_cast<unsigned>(parts));
    auto* kernel = pair ? act_bwd_kernel<T, true> : act_bwd_kernel<T, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(kBlock), 0, stream, p);
    if (check_launch("act_bwd_kernel")) return -2;
    over = p.over;
    if (p.over) {
      ActBwd again = p;
      again.again = true;
      again.partial = nullptr;
      again.db = again.db2 = nullptr;
      hipLaunchKernelGGL(kernel, grid, dim3(kBlock), 0, stream, again);
      if (check_launch("act_bwd_kernel")) return -2;
    }
    if (p.partial) {
      if (const int rc = sum_partials<T>(ws.act_partial, parts, wide * n_out, n_out, db, db2, stream))
        return rc;
    }
  }
  if (!dx && !dw && !dw2) return 0;
  PackJobs jobs;
  jobs.n = 0;
  int64_t ld = n_in, ld2 = n_in;
  if (!z) lay_out<T>(jobs, dz, dz_ld, m, n_out, ws.dz);
  if (dx) {
    lay_out<T>(jobs, w, ld, n_out, n_in, ws.w);
    if (pair) lay_out<T>(jobs, w2, ld2, n_out, n_in, ws.w2);
  }
  if (dw || dw2) lay_out<T>(jobs, x, x_ld, m, n_in, ws.x);
  if (launch_packs<T>(jobs, stream)) return -2;
  Gemm g;
  if (dx) {
    memset(&g, 0, sizeof(g));
    g.a = {dz, dz_ld, 1};
    g.b = {w, 1, ld};
    g.b2 = w2;
    g.k_split = half;
    g.k_valid = n_out;
    g.m = m;
    g.n = n_in;
    g.k = pair ? half + n_out : n_out;
    g.c = dx;
    g.over = over;
    g.row_split = g.row_valid = m;
    g.partial = ws.partial;
    const Plan p = plan_of<T>(kDx, m, n_in, n_out, pair);
    const int rc = pair ? launch_tiles<T, true, false, kEpiStore, true>(g, p, stream)
                        : launch_tiles<T, true, false, kEpiStore, false>(g, p, stream);
    if (rc) return rc;
  }
  if (dw || dw2) {
    memset(&g, 0, sizeof(g));
    g.a = {dz, 1, dz_ld};
    g.b = {x, 1, x_ld};
    g.m = pair ? half + n_out : n_out;
    g.n = n_in;
    g.k = m;
    g.row_split = half;
    g.row_valid = n_out;
    g.c = dw;
    g.c2 = dw2;
    g.over = over;
    g.partial = ws.partial;
    return launch_tiles<T, false, false, kEpiStore, false>(
        g, plan_of<T>(kDw, m, n_in, n_out, pair), stream);
  }
  return 0;
}

}  // namespace

template <typename T>
size_t HeadLayer<T>::forward_bytes(const void* x, int64_t x_ld, int64_t m, int64_t n_in,
                                   const void* w, const void* w2, int64_t n_out) {
  return carve_fwd<T>(nullptr, x, x_ld, m, n_in, w, w2, n_out).bytes;
}

template <typename T>
size_t HeadLayer<T>::backward_bytes(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld,
                                    int64_t m, int64_t n_in, const void* w, const void* w2,
                                    int64_t n_out, int act) {
  return carve_bwd<T>(nullptr, dy, dy_ld, x, x_ld, m, n_in, w, w2, n_out, act).bytes;
}

template <typename T>
void HeadLayer<T>::plan(Product product, int64_t m, int64_t n_in, int64_t n_out, bool pair,
                        int64_t (&out)[5]) {
  if (product == kForward && m <= kSkinnyRows) {
    memset(out, 0, sizeof(out));
    return;
  }
  const Plan p = plan_of<T>(product, m, n_in, n_out, pair);
  const int64_t values[5] = {p.bm, p.bn, p.tiles, p.full, p.splits};
  memcpy(out, values, sizeof(out));
}

template <typename T>
int HeadLayer<T>::forward(const void* x, int64_t x_ld, const void* w, const void* w2,
                          const void* bias, const void* bias2, const void* residual, int64_t res_ld,
                          int64_t m, int64_t n_in, int64_t n_out, int act, void* keep, void* keep2,
                          void* y, void* workspace, hipStream_t stream) {
  return layer_forward<T>(x, x_ld, w, w2, bias, bias2, residual, res_ld, m, n_in, n_out, act, keep,
                          keep2, y, workspace, stream);
}

template <typename T>
int HeadLayer<T>::backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, const void* w,
                           const void* w2, const void* z, const void* u, int64_t m, int64_t n_in,
                           int64_t n_out, int act, void* dx, void* dw, void* dw2, void* db, void* db2,
                           void* workspace, hipStream_t stream) {
  return layer_backward<T>(dy, dy_ld, x, x_ld, w, w2, z, u, m, n_in, n_out, act, dx, dw, dw2, db, db2,
                           workspace, stream);
}

}  // namespace collie
