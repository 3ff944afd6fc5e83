// The tiled matrix product of the linear and gated layers (head_gemm.hip): C = A B^T over tiles of
// BM x BN results, both operands through LDS, products on the matrix cores.
//
// An operand is "along k" (KC: element (i, k) at p[i ld + k], as a layer's input and weight are in
// the forward pass) or "across k" (RC: at p[k ld + i], as the weight is in dx = dz W and both
// operands are in dW = dz^T x).  Either way a stage holds 128 bytes per operand row: 64 values of 16
// bits or 32 of float32, brought in by 16-byte LDS-DMA loads (no registers in between), one stage
// ahead of the products.
//   KC image: [row][8 chunks of 16 bytes], chunk c of row r at slot c ^ (r / 2 & 7): the 16 rows a
//     fragment read touches then lie in 16 different 16-byte columns of the 256 bytes of all banks.
//   RC image: [k][row chunks]; 16-bit fragments are read by the transposing LDS load (four k of one
//     row per lane, 16 lanes sharing 4 k x 16 rows), float32 ones element by element; the chunk
//     index is XORed with k so that the rows of one read do not meet in the same banks.
// The DMA destination is linear in the lane, so the XOR is applied to the lane's source address.
// Matrix instruction: 16 x 16 results, its rows are the product's columns: a lane ends up with four
// neighbouring columns of one row of C, which it stores together.
#pragma once

#include "head_gemm.h"

namespace collie {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

__device__ uint4 g_zero_chunk;  // what a load past the depth reads

// 16 bytes per lane from `g` to LDS at `lds` (wave-uniform) + 16 * lane.  In asm, because after the
// builtin every later LDS read waits for all outstanding loads; the waits here are explicit.
__device__ __forceinline__ void dma16(const void* g, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(lds)
               : "memory", "m0");
}
__device__ __forceinline__ void wait_dma() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// A fragment: 16 rows by 32 k (16-bit) or 16 k (float32); lane l holds row l % 16 and
// k = 8 (l / 16) + j, or 4 (l / 16) + j.
template <typename T>
struct Frag {
  s16x8 v;
};
template <>
struct Frag<float> {
  f32x4 v;
};

template <typename T>
__device__ __forceinline__ void multiply(const Frag<T>& a, const Frag<T>& b, f32x4& c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[t], b.v[t], c, 0, 0, 0);
  } else if constexpr (std::is_same<T, bf16_t>::value) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.v),
                                                __builtin_bit_cast(bf16x8, b.v), c, 0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.v),
                                               __builtin_bit_cast(f16x8, b.v), c, 0, 0, 0);
  }
}

// One operand's image of a stage: R rows x 128 bytes.
template <typename T, int R, bool KC>
struct Image {
  static constexpr int kBytes = R * 128;
  static constexpr int kDepth = 128 / static_cast<int>(sizeof(T));
  static constexpr int kRowChunks = KC ? 8 : R * static_cast<int>(sizeof(T)) / 16;  // image row

  static __device__ __forceinline__ int swizzle(int row) {
    if (KC) return (row >> 1) & 7;
    if (sizeof(T) == 2) return ((row & 3) | ((row >> 1) & 4)) << 1;
    return ((row >> 2) & 3) << 2;
  }
  // image row and source chunk of the 16 bytes at linear position `at`
  static __device__ __forceinline__ void source(int at, int& row, int& chunk) {
    row = at / kRowChunks;
    chunk = (at % kRowChunks) ^ swizzle(row);
  }
  // fragment `step` (of 2) of the 16 rows from row0 on
  static __device__ __forceinline__ Frag<T> read(const char* img, int row0, int step, int lane) {
    const int r = lane & 15, g = lane >> 4;
    Frag<T> f;
    if constexpr (KC) {
      const int row = row0 + r;
      const char* p = img + row * 128 + ((4 * step + g) ^ swizzle(row)) * 16;
      f.v = *reinterpret_cast<const decltype(f.v)*>(p);
    } else if constexpr (sizeof(T) == 2) {
      s16x4 part[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = 32 * step + 8 * g + 4 * h + (r >> 2);
        const int chunk = (row0 >> 3) + ((r & 3) >> 1);
        const char* p = img + k * (R * 2) + (chunk ^ swizzle(k)) * 16 + (r & 1) * 8;
        part[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(p));
      }
      f.v = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int k = 16 * step + 4 * g + t;
        const int chunk = (row0 >> 2) + (r >> 2);
        f.v[t] = *reinterpret_cast<const float*>(img + k * (R * 4) + (chunk ^ swizzle(k)) * 16 +
                                                 (r & 3) * 4);
      }
    }
    return f;
  }
};

// The loads of one operand: every thread brings N x 16 bytes of a stage.
//   rows0: first row of the tile; `rows` of the operand (further ones are clamped: their products go
//   nowhere).  With SECOND, image rows from R / 2 on are rows of `p2` (the gated forward pass); with
//   CAT, k from k_split on is k - k_split of `p2`, and of either only k < k_valid is there.
template <typename T, int R, bool KC, int THREADS, bool SECOND, bool CAT>
struct Feed {
  using Img = Image<T, R, KC>;
  static constexpr int N = Img::kBytes / 16 / THREADS;
  static constexpr int V = kVec<T>;
  const T* p[N];
  int kk[N];  // k within the stage
  int64_t ld;

  __device__ __forceinline__ void init(const void* base, const void* base2, int64_t ld_, int64_t row0,
                                       int64_t rows, int64_t k0, int tid) {
    ld = ld_;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      int r, c;
      Img::source(j * THREADS + tid, r, c);
      if (KC) {
        const bool second = SECOND && r >= R / 2;
        int64_t row = row0 + (second ? r - R / 2 : r);
        row = row < rows ? row : rows - 1;
        kk[j] = c * V;
        p[j] = static_cast<const T*>(second ? base2 : base) + row * ld + k0 + kk[j];
      } else {
        // an operand whose rows are no whole number of packs is one that was laid out with padding
        const int64_t end = (rows + V - 1) / V * V;
        int64_t col = row0 + c * V;
        col = col < end ? col : end - V;
        kk[j] = r;
        p[j] = static_cast<const T*>(base) + col + (CAT ? 0 : (k0 + r) * ld);
      }
    }
  }

  // issues the loads of the stage at depth k (up to k1) into the image at LDS address `lds`
  __device__ __forceinline__ void issue(uint32_t lds, int64_t k, int64_t k1, const Gemm& g) {
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds + (threadIdx.x / kWave) * kWave * 16);
    const bool whole = k + Img::kDepth <= k1;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const void* q = p[j];
      if constexpr (CAT) {
        int64_t at = k + kk[j];
        const bool second = at >= g.k_split;
        const bool in = at < k1;
        if (second) at -= g.k_split;
        q = p[j] + (second ? g.b2_offset : 0) + at * ld;
        if (!in || at >= g.k_valid) q = &g_zero_chunk;
      } else {
        if (!whole && k + kk[j] >= k1) q = &g_zero_chunk;
        p[j] += KC ? static_cast<int64_t>(Img::kDepth) : Img::kDepth * ld;
      }
      dma16(q, to + j * THREADS * 16);
    }
  }
};

// Tiles in an order that keeps the operands in the caches: workgroups go round the 8 XCDs, so XCD x
// gets the x-th run of tiles; inside a run, kBand row tiles by all column tiles.
__device__ __forceinline__ void tile_of(int64_t id, int64_t total, int64_t tiles_m, int64_t tiles_n,
                                        int64_t& tm, int64_t& tn, int64_t& part) {
  constexpr int64_t kBand = 8;
  const int64_t q = total / 8, r = total % 8, x = id % 8;
  id = x * q + (x < r ? x : r) + id / 8;
  part = id / (tiles_m * tiles_n);
  id -= part * tiles_m * tiles_n;
  const int64_t band = id / (kBand * tiles_n);
  const int64_t high = tiles_m - band * kBand < kBand ? tiles_m - band * kBand : kBand;
  id -= band * kBand * tiles_n;
  tm = band * kBand + id % high;
  tn = id / high;
}

template <typename T, int BM, int BN, int WM, int WN, bool AKC, bool BKC, int EPI, bool CAT>
__global__ __launch_bounds__(kWave* WM* WN, 2) void gemm_tile_kernel(const Gemm g) {
  constexpr bool PAIR = EPI == kEpiGated;
  constexpr int THREADS = kWave * WM * WN;
  constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
  constexpr int TN = PAIR ? BN / 2 : BN;  // columns of C per tile
  constexpr int HALF = PAIR ? NT / 2 : NT;
  using ImgA = Image<T, BM, AKC>;
  using ImgB = Image<T, BN, BKC>;
  constexpr int kStage = ImgA::kBytes + ImgB::kBytes;
  constexpr int kDepth = ImgA::kDepth;
  __shared__ __attribute__((aligned(16))) char lds[2 * kStage];
  const uint32_t lds0 =
      static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wm = wave / WN, wn = wave % WN;

  const int64_t tiles_m = (g.m + BM - 1) / BM, tiles_n = (g.n + TN - 1) / TN;
  int64_t tm, tn, part;
  tile_of(blockIdx.x, gridDim.x, tiles_m, tiles_n, tm, tn, part);
  const int64_t row0 = tm * BM, col0 = tn * TN;
  const int64_t k0 = part * g.k_chunk;
  const int64_t k1 = k0 + g.k_chunk < g.k ? k0 + g.k_chunk : g.k;

  Feed<T, BM, AKC, THREADS, false, false> fa;
  Feed<T, BN, BKC, THREADS, PAIR, CAT> fb;
  fa.init(g.a.p, nullptr, AKC ? g.a.rs : g.a.ks, row0, g.m, k0, tid);
  fb.init(g.b.p, g.b2, BKC ? g.b.rs : g.b.ks, col0, g.n, k0, tid);

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  fa.issue(lds0, k0, k1, g);
  fb.issue(lds0 + ImgA::kBytes, k0, k1, g);
  int cur = 0;
  for (int64_t k = k0; k < k1; k += kDepth) {
    wait_dma();      // this wave's loads of the stage have landed
    tile_barrier();  // everyone's have, and the other stage has been read
    if (k + kDepth < k1) {
      const uint32_t to = lds0 + (cur ^ 1) * kStage;
      fa.issue(to, k + kDepth, k1, g);
      fb.issue(to + ImgA::kBytes, k + kDepth, k1, g);
    }
    const char* ia = lds + cur * kStage;
    const char* ib = ia + ImgA::kBytes;
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      Frag<T> b[NT], a[MT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int row = PAIR ? (j / HALF) * (BN / 2) + wn * (TN / WN) + (j % HALF) * 16
                             : wn * (BN / WN) + j * 16;
        b[j] = ImgB::read(ib, row, step, lane);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) a[i] = ImgA::read(ia, wm * (BM / WM) + i * 16, step, lane);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) multiply<T>(b[j], a[i], acc[i][j]);
    }
    cur ^= 1;
  }

  const int r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < HALF; ++j) {
      float v[4], u[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        v[t] = acc[i][j][t];
        u[t] = PAIR ? acc[i][PAIR ? j + HALF : j][t] : 0.0f;
      }
      const int64_t row = row0 + wm * (BM / WM) + i * 16 + r;
      const int64_t col = col0 + wn * (TN / WN) + j * 16 + 4 * q;
      if (g.splits > 1)
        store_part<EPI, 4>(g, row, col, part, v, u);
      else
        finish_row<T, EPI, 4>(g, row, col, v, u);
    }
}

// The product of at most 16 MT rows, where reading the weights is all there is to it: a workgroup of
// eight waves owns 16 columns of C, the waves share out the depth (64 values at a time, so that
// every row of a weight is read in whole cache lines) and add their sums in order through LDS.  Loads
// go straight to registers; any alignment and any depth.
constexpr int kSkinnyWaves = 8;
template <typename T, int MT, int EPI, bool WHOLE>
__global__ __launch_bounds__(kWave* kSkinnyWaves) void gemm_skinny_kernel(const Gemm g) {
  constexpr bool PAIR = EPI == kEpiGated;
  constexpr int NB = PAIR ? 2 : 1;
  constexpr int V = kVec<T>;
  constexpr int kStep = 4 * V;   // k per fragment
  constexpr int kRun = 2;        // fragments a wave takes in a row
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int r = lane & 15, q = lane >> 4;
  const int64_t col0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int64_t col = col0 + r < g.n ? col0 + r : g.n - 1;
  const T* w[2] = {static_cast<const T*>(g.b.p) + col * g.b.rs,
                   static_cast<const T*>(g.b2) + col * g.b.rs};
  const T* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t row = i * 16 + r < g.m ? i * 16 + r : g.m - 1;
    x[i] = static_cast<const T*>(g.a.p) + row * g.a.rs;
  }
  f32x4 acc[MT][NB];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto load = [&](const T* p, int64_t k) {
    Frag<T> f;
    if constexpr (WHOLE) {
      const Pack<T, V> v = *reinterpret_cast<const Pack<T, V>*>(p + (k < g.k ? k : 0));
      f.v = __builtin_bit_cast(decltype(f.v), v);
      if (k >= g.k) f.v = decltype(f.v){};
    } else {
      Pack<T, V> v;
      if (k + V <= g.k) {
        v = *reinterpret_cast<const Pack<T, V>*>(p + k);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v.v[j] = k + j < g.k ? p[k + j] : static_cast<T>(0.0f);
      }
      f.v = __builtin_bit_cast(decltype(f.v), v);
    }
    return f;
  };
#pragma unroll 2
  for (int64_t k = wave * (kRun * kStep); k < g.k; k += kSkinnyWaves * kRun * kStep) {
    Frag<T> b[kRun][NB], a[kRun][MT];
#pragma unroll
    for (int s = 0; s < kRun; ++s) {
      const int64_t at = k + s * kStep + q * V;
#pragma unroll
      for (int j = 0; j < NB; ++j) b[s][j] = load(w[j], at);
#pragma unroll
      for (int i = 0; i < MT; ++i) a[s][i] = load(x[i], at);
    }
#pragma unroll
    for (int s = 0; s < kRun; ++s)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) multiply<T>(b[s][j], a[s][i], acc[i][j]);
  }
  __shared__ f32x4 sums[kSkinnyWaves][MT][NB][kWave];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) sums[wave][i][j][lane] = acc[i][j];
  __syncthreads();
  for (int i = wave; i < MT; i += kSkinnyWaves) {
    float v[4], u[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      v[t] = u[t] = 0.0f;
#pragma unroll
      for (int s = 0; s < kSkinnyWaves; ++s) {
        v[t] += sums[s][i][0][lane][t];
        if (PAIR) u[t] += sums[s][i][PAIR ? 1 : 0][lane][t];
      }
    }
    finish_row<T, EPI, 4>(g, i * 16 + r, col0 + 4 * q, v, u);
  }
}

// The parts of the depth added in order, then the epilogue.  64 x 4 results per workgroup; with
// SLICES > 1 the parts are shared out over the waves, whose sums are added in order through LDS.
template <typename T, int EPI, int SLICES>
__global__ __launch_bounds__(kWave* SLICES) void gemm_finish_kernel(const Gemm g) {
  constexpr int NB = EPI == kEpiGated ? 2 : 1;
  const int lane = threadIdx.x & (kWave - 1), slice = threadIdx.x / kWave;
  const int64_t packs = (g.n + 3) / 4;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kWave + lane;
  const int64_t row = at / packs, col = (at - row * packs) * 4;
  const bool in = row < g.m;
  const int left = in ? static_cast<int>(g.n - col < 4 ? g.n - col : 4) : 0;
  float v[2][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[0][j] = v[1][j] = 0.0f;
  if (in) {
    const float* p = g.partial + row * g.n + col;
#pragma unroll 4
    for (int s = slice; s < g.splits; s += SLICES) {
      float t[4];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        load_pack<float, 4>(p + (static_cast<int64_t>(s) * NB + b) * g.m * g.n, left, t);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[b][j] += t[j];
      }
    }
  }
  if constexpr (SLICES > 1) {
    __shared__ float sh[SLICES][NB][kWave][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) sh[slice][b][lane][j] = v[b][j];
    __syncthreads();
    if (slice != 0) return;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int s = 1; s < SLICES; ++s) v[b][j] += sh[s][b][lane][j];
  }
  if (in) finish_row<T, EPI, 4>(g, row, col, v[0], v[1]);
}

}  // namespace collie
