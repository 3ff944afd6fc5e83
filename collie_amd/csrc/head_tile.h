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

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

static __device__ uint4 g_zero_chunk;  // what a load past the depth reads

// 16 bytes per lane from `g` to LDS at `lds` (wave-uniform) + 16 * lane.  In asm, because after the
// builtin every later LDS read waits for all outstanding loads; the waits here are explicit.
__device__ __forceinline__ void dma16(const void* g, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(lds)
               : "memory", "m0");
}
// the same from a base that is the same for the wave and a lane's byte offset
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2" ::"v"(off), "s"(lds),
               "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void wait_dma() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

constexpr int kMfma = 0x008, kDsRead = 0x100;  // groups of __builtin_amdgcn_sched_group_barrier

// A fragment: 16 rows by 32 k; lane l holds row l % 16 and k = 8 (l / 16) + j.
template <typename T>
struct Frag {
  s16x8 v;
};
template <>
struct Frag<float> {
  float v[8];
};

// A float32 fragment as three bfloat16 ones, x = hi + mid + lo exactly: 8 significant bits each, what
// is left after rounding to the nearest.  Of the nine products of two such numbers the six of
// weight 2^-16 and more are summed; the others are below 2^-23 of the product, which is what float32
// rounds it by.  Six bfloat16 instructions do 32 k in 96 cycles; the float32 ones need 256.  Values
// without a finite bfloat16 (infinities, NaN, the top of the range) make sums that are not finite:
// the tile is then computed again with the float32 instructions (gemm_tile_kernel).  Parts end at
// bfloat16's smallest number: at most 2^-134 times the other factor is lost, which is float32's own
// rounding down to 2^-110.
struct Split {
  bf16x8 hi, mid, lo;
};
__device__ __forceinline__ uint32_t round_pair(const f32x2& x) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
}
__device__ __forceinline__ float low_value(uint32_t pair) {
  return __builtin_bit_cast(float, pair << 16);
}
__device__ __forceinline__ float high_value(uint32_t pair) {
  return __builtin_bit_cast(float, pair & 0xffff0000u);
}
template <typename T>
__device__ __forceinline__ Split split(const Frag<T>& f) {
  Split s;
  if constexpr (sizeof(T) == 4) {
    // two values per conversion: 44 instructions
    u32x4 hi, mid, lo;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 x = {f.v[2 * j], f.v[2 * j + 1]};
      hi[j] = round_pair(x);
      const f32x2 r = {x[0] - low_value(hi[j]), x[1] - high_value(hi[j])};
      mid[j] = round_pair(r);
      lo[j] = round_pair(f32x2{r[0] - low_value(mid[j]), r[1] - high_value(mid[j])});
    }
    s.hi = __builtin_bit_cast(bf16x8, hi);
    s.mid = __builtin_bit_cast(bf16x8, mid);
    s.lo = __builtin_bit_cast(bf16x8, lo);
  }
  return s;
}

__device__ __forceinline__ f32x4 mfma_bf16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ void multiply(const Split& a, const Split& b, f32x4& c) {
  c = mfma_bf16(a.lo, b.hi, c);   // the smallest first
  c = mfma_bf16(a.hi, b.lo, c);
  c = mfma_bf16(a.mid, b.mid, c);
  c = mfma_bf16(a.mid, b.hi, c);
  c = mfma_bf16(a.hi, b.mid, c);
  c = mfma_bf16(a.hi, b.hi, c);
}

template <typename T>
__device__ __forceinline__ void multiply(const Frag<T>& a, const Frag<T>& b, f32x4& c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int t = 0; t < 8; ++t) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[t], b.v[t], c, 0, 0, 0);
  } else if constexpr (std::is_same<T, bf16_t>::value) {
    c = mfma_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v), c);
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
    if (sizeof(T) == 2 && R == 64) return (((row >> 1) & 1) | ((row >> 2) & 2)) << 1;
    if (sizeof(T) == 2) return ((row & 3) | ((row >> 1) & 4)) << 1;
    return ((row >> 3) & 3) << 2;
  }
  // image row and source chunk of the 16 bytes at linear position `at`
  static __device__ __forceinline__ void source(int at, int& row, int& chunk) {
    row = at / kRowChunks;
    chunk = (at % kRowChunks) ^ swizzle(row);
  }
  static constexpr int kSteps = kDepth / 32;  // fragments along the depth
  // fragment `step` of the 16 rows from row0 on
  static __device__ __forceinline__ Frag<T> read(const char* img, int row0, int step, int lane) {
    const int r = lane & 15, g = lane >> 4;
    Frag<T> f;
    if constexpr (KC && sizeof(T) == 2) {
      const int row = row0 + r;
      f.v = *reinterpret_cast<const s16x8*>(img + row * 128 + ((4 * step + g) ^ swizzle(row)) * 16);
    } else if constexpr (KC) {
      const int row = row0 + r;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 v =
            *reinterpret_cast<const f32x4*>(img + row * 128 + ((2 * g + h) ^ swizzle(row)) * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) f.v[4 * h + j] = v[j];
      }
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
      for (int j = 0; j < 8; ++j) {
        const int k = 8 * g + j;
        const int chunk = (row0 >> 2) + (r >> 2);
        f.v[j] = *reinterpret_cast<const float*>(img + k * (R * 4) + (chunk ^ swizzle(k)) * 16 +
                                                 (r & 3) * 4);
      }
    }
    return f;
  }
};

// The loads of one operand: every thread brings N x 16 bytes of a stage, from a base that is the same
// for the workgroup and moves by one stage, and offsets that stay.
//   row0: first row of the tile; `rows` of the operand (further ones are clamped: their products go
//   nowhere).  With SECOND, image rows from R / 2 on are rows of a second matrix (the gated forward
//   pass); with CAT, k from k_split on is k - k_split of a second matrix, and of either only
//   k < k_valid is there.
template <typename T, int R, bool KC, int THREADS, bool SECOND, bool CAT>
struct Feed {
  using Img = Image<T, R, KC>;
  static constexpr int N = Img::kBytes / 16 / THREADS;
  static constexpr int V = kVec<T>;
  static constexpr int kSize = static_cast<int>(sizeof(T));
  static_assert(!SECOND || (KC && N % 2 == 0), "the halves of an image are whole loads");
  uint32_t off[N];            // bytes from the base: the host keeps 256 rows below 2^31
  const char *base, *base2;   // of the next stage (base2 with CAT: at k - k_split)
  int64_t step;

  __device__ __forceinline__ void init(const void* p, const void* p2, int64_t ld, int64_t row0,
                                       int64_t rows, int64_t k0, int64_t k_split, int tid) {
    const int64_t at = KC ? row0 * ld + k0 : k0 * ld + row0;
    base = static_cast<const char*>(p) + at * kSize;
    if (SECOND || CAT) base2 = static_cast<const char*>(p2) + (at - (CAT ? k_split * ld : 0)) * kSize;
    step = KC ? 128 : Img::kDepth * ld * kSize;
    const int last = static_cast<int>(rows - row0 < (SECOND ? R / 2 : R) ? rows - row0 : (SECOND ? R / 2 : R)) - 1;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      int r, c;
      Img::source(j * THREADS + tid, r, c);
      if (KC) {
        if (SECOND && j >= N / 2) r -= R / 2;
        off[j] = static_cast<uint32_t>((r < last ? r : last) * static_cast<int>(ld * kSize) + c * 16);
      } else {
        // an operand whose rows are no whole number of packs is one that was laid out with padding
        off[j] = static_cast<uint32_t>(r * static_cast<int>(ld * kSize) +
                                       (c < last / V ? c : last / V) * 16);
      }
    }
  }

  // issues the loads of the stage at depth k (up to k1) into the image at LDS address `lds`
  __device__ __forceinline__ void issue(uint32_t lds, int64_t k, int64_t k1, const Gemm& g) {
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds + (threadIdx.x / kWave) * kWave * 16);
    const bool second = CAT && k >= g.k_split;
    const int64_t end = !CAT ? k1 : second ? g.k_split + g.k_valid : g.k_valid;
    if (k + Img::kDepth <= (end < k1 ? end : k1)) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        dma16(second || (SECOND && j >= N / 2) ? base2 : base, off[j], to + j * THREADS * 16);
    } else {
      // the end of the depth, or of the first matrix: lane by lane, zeros past it
#pragma unroll
      for (int j = 0; j < N; ++j) {
        int r, c;
        Img::source(j * THREADS + threadIdx.x, r, c);
        const int64_t at = k + (KC ? c * V : r);
        const bool two = CAT ? at >= g.k_split : SECOND && j >= N / 2;
        bool in = at < k1;
        if (CAT) in = in && at - (two ? g.k_split : 0) < g.k_valid;
        const char* q = (two ? base2 : base) + off[j];
        dma16(in ? q : reinterpret_cast<const char*>(&g_zero_chunk), to + j * THREADS * 16);
      }
    }
    base += step;
    if (SECOND || CAT) base2 += step;
  }
};

// Lanes l, l + 16, l + 32, l + 48 hold columns 4 q .. 4 q + 3 (q = l / 16) of one row of two 16-column
// tiles; afterwards lane row q holds half q / 2 of tile q % 2.
__device__ __forceinline__ void spread2(const f32x4& t0, const f32x4& t1, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(t0[j]), __float_as_uint(t1[j]),
                                                    false, false);
    const uint32_t a = s[0], b = s[1];  // (a bit_cast of a vector's element would take element 0)
    v[j] = __uint_as_float(a);
    v[4 + j] = __uint_as_float(b);
  }
}

// Workgroups go round the 8 XCDs: XCD x gets the x-th run of the numbers below `total`.
__device__ __forceinline__ int64_t xcd_order(int64_t id, int64_t total) {
  const int64_t q = total / 8, r = total % 8, x = id % 8;
  return x * q + (x < r ? x : r) + id / 8;
}

// Tile number -> row and column tile: kBand row tiles by all column tiles, then the next band, so
// that the tiles of a run share operands in their XCD's cache.
__device__ __forceinline__ void tile_at(int64_t id, int64_t tiles_m, int64_t tiles_n, int64_t& tm,
                                        int64_t& tn) {
  constexpr int64_t kBand = 8;
  const int64_t band = id / (kBand * tiles_n);
  const int64_t high = tiles_m - band * kBand < kBand ? tiles_m - band * kBand : kBand;
  id -= band * kBand * tiles_n;
  tm = band * kBand + id % high;
  tn = id / high;
}

// The grid is at most what the chip holds: a workgroup works on one tile (or one part of the depth of
// a tile) after another, and the first stage of the next one is loaded under the last products and
// the epilogue of the one before.
template <typename T, int BM, int BN, int WM, int WN, bool AKC, bool BKC, int EPI, bool CAT>
__global__ __launch_bounds__(kWave* WM* WN, BN == 64 ? 3 : 2) void gemm_tile_kernel(const Gemm g) {
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
  const int64_t rest = tiles_m * tiles_n - g.full;
  const int64_t total = g.full + rest * g.splits;
  struct Work {
    int64_t slot, row0, col0, k0, k1;  // slot: of the partial sums, -1 for a whole tile
  };
  auto work_at = [&](int64_t n) {
    Work w;
    int64_t id, tm, tn;
    if (n >= g.full) {
      id = xcd_order(n - g.full, rest * g.splits);
      w.slot = id;
      w.k0 = id / rest * g.k_chunk;
      w.k1 = w.k0 + g.k_chunk < g.k ? w.k0 + g.k_chunk : g.k;
      id = g.full + id % rest;
    } else {
      id = xcd_order(n, g.full);
      w.slot = -1;
      w.k0 = 0;
      w.k1 = g.k;
    }
    tile_at(id, tiles_m, tiles_n, tm, tn);
    w.row0 = tm * BM;
    w.col0 = tn * TN;
    return w;
  };

  Feed<T, BM, AKC, THREADS, false, false> fa;
  Feed<T, BN, BKC, THREADS, PAIR, CAT> fb;
  auto start = [&](const Work& w, uint32_t to) {
    fa.init(g.a.p, nullptr, AKC ? g.a.rs : g.a.ks, w.row0, g.m, w.k0, 0, tid);
    fb.init(g.b.p, g.b2, BKC ? g.b.rs : g.b.ks, w.col0, g.n, w.k0, g.k_split, tid);
    fa.issue(to, w.k0, w.k1, g);
    fb.issue(to + ImgA::kBytes, w.k0, w.k1, g);
  };
  f32x4 acc[MT][NT];
  auto b_row = [&](int j) {
    return PAIR ? (j / HALF) * (BN / 2) + wn * (TN / WN) + (j % HALF) * 16 : wn * (BN / WN) + j * 16;
  };
  // float32: EXACT takes the float32 instructions
  auto products = [&](const char* ia, auto exact) {
    constexpr bool EXACT = decltype(exact)::value;
    const char* ib = ia + ImgA::kBytes;
    if constexpr (sizeof(T) == 4 && !EXACT) {
      Split b[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) b[j] = split(ImgB::read(ib, b_row(j), 0, lane));
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const Split a = split(ImgA::read(ia, wm * (BM / WM) + i * 16, 0, lane));
#pragma unroll
        for (int j = 0; j < NT; ++j) multiply(b[j], a, acc[i][j]);
      }
    } else {
#pragma unroll
      for (int step = 0; step < ImgA::kSteps; ++step) {
        Frag<T> b[NT], a[MT];
#pragma unroll
        for (int j = 0; j < NT; ++j) b[j] = ImgB::read(ib, b_row(j), step, lane);
#pragma unroll
        for (int i = 0; i < MT; ++i) a[i] = ImgA::read(ia, wm * (BM / WM) + i * 16, step, lane);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) multiply<T>(b[j], a[i], acc[i][j]);
      }
      if constexpr (sizeof(T) == 2) {
        // the order of the above: the fragments of the next row tiles are on their way while those at
        // hand are multiplied (8,192^3: 1,025 -> 990 us)
        constexpr int RA = AKC ? 1 : 2, RB = BKC ? 1 : 2;  // LDS reads per fragment
        __builtin_amdgcn_sched_group_barrier(kDsRead, NT * RB + 2 * RA, 0);
#pragma unroll
        for (int step = 0; step < 2; ++step) {
#pragma unroll
          for (int i = 0; i < MT - 2; ++i) {
            __builtin_amdgcn_sched_group_barrier(kMfma, NT, 0);
            __builtin_amdgcn_sched_group_barrier(kDsRead, RA, 0);
          }
          if (step == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              __builtin_amdgcn_sched_group_barrier(kMfma, NT, 0);
              __builtin_amdgcn_sched_group_barrier(kDsRead, NT * RB / 2 + RA, 0);
            }
          } else {
            __builtin_amdgcn_sched_group_barrier(kMfma, 2 * NT, 0);
          }
        }
      }
    }
  };
  auto clear = [&] {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  };

  static_assert(NT == 4, "four column tiles per wave");
  constexpr int W = sizeof(T) == 4 ? 4 : 8;  // columns that a lane stores together
  constexpr int G = 4 * HALF / W;

  const float scale = result_scale<T, EPI>(g);
  int64_t n = blockIdx.x;
  Work now = work_at(n);
  int cur = 0;
  start(now, lds0);
  while (true) {
    const bool more = n + gridDim.x < total;
    const Work next = more ? work_at(n + gridDim.x) : now;
    clear();
    wait_dma();  // this wave's loads of the first stage have landed (so they have further down)
    for (int64_t k = now.k0; k < now.k1; k += kDepth) {
      tile_barrier();  // every wave's loads have landed, and the other stage has been read
      const uint32_t to = lds0 + (cur ^ 1) * kStage;
      if (k + kDepth < now.k1) {
        fa.issue(to, k + kDepth, now.k1, g);
        fb.issue(to + ImgA::kBytes, k + kDepth, now.k1, g);
      } else if (more) {
        start(next, to);
      }
      products(lds + cur * kStage, std::false_type{});
      cur ^= 1;
      if (k + kDepth < now.k1) wait_dma();
    }
    if constexpr (sizeof(T) == 4) {
      bool finite = true;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int t = 0; t < 4; ++t) finite = finite && fabsf(acc[i][j][t]) < INFINITY;
      if (__syncthreads_or(!finite)) {
        // once more, one stage at a time in the stage that holds nothing, then the next tile's first
        // stage again (the loads above went on from there)
        clear();
        const uint32_t to = lds0 + (cur ^ 1) * kStage;
        for (int64_t k = now.k0; k < now.k1; k += kDepth) {
          wait_dma();
          tile_barrier();
          if (k == now.k0) {
            start(now, to);
          } else {
            fa.issue(to, k, now.k1, g);
            fb.issue(to + ImgA::kBytes, k, now.k1, g);
          }
          wait_dma();
          tile_barrier();
          products(lds + (cur ^ 1) * kStage, std::true_type{});
        }
        tile_barrier();
        if (more) start(next, lds0 + cur * kStage);
      }
    }

    // A lane has four neighbouring columns of each column tile.  Of float32, four lanes then store a
    // 64-byte piece of a row; of 16 bits, lanes exchange halves of two tiles to the same end.
    const int r = lane & 15, q = lane >> 4;
    const int lc0 = wn * (TN / WN) + (W == 4 ? 4 * q : 16 * (q & 1) + 8 * (q >> 1));
    float b[G][W], b2[G][W];
#pragma unroll
    for (int k = 0; k < G; ++k)
      if (now.slot < 0) load_biases<T, EPI, W>(g, now.col0 + lc0 + k * 4 * W, b[k], b2[k]);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int lr = wm * (BM / WM) + i * 16 + r;
#pragma unroll
      for (int k = 0; k < G; ++k) {
        const int lc = lc0 + k * 4 * W;
        float v[W], u[W];
        if constexpr (W == 4) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            v[t] = acc[i][k][t];
            u[t] = acc[i][PAIR ? k + HALF : k][t];
          }
        } else {
          spread2(acc[i][2 * k], acc[i][2 * k + 1], v);
          if constexpr (PAIR) spread2(acc[i][2], acc[i][3], u);
        }
        if (now.slot >= 0) {
          float* p = g.partial + (now.slot * (PAIR ? 2 : 1) * BM + lr) * TN + lc;
          store_pack<float, W>(p, W, v);
          if (PAIR) store_pack<float, W>(p + BM * TN, W, u);
        } else {
          finish_row<T, EPI, W>(g, now.row0 + lr, now.col0 + lc, v, u, b[k], b2[k], scale);
        }
      }
    }
    if (!more) break;
    n += gridDim.x;
    now = next;
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
  constexpr int kStep = 32;      // k per fragment
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
    T v[8];
#pragma unroll
    for (int h = 0; h < 8; h += V) {
      Pack<T, V> pack;
      if constexpr (WHOLE) {
        pack = *reinterpret_cast<const Pack<T, V>*>(p + (k + h < g.k ? k + h : 0));
#pragma unroll
        for (int j = 0; j < V; ++j) v[h + j] = k + h < g.k ? pack.v[j] : static_cast<T>(0.0f);
      } else if (k + h + V <= g.k) {
        pack = *reinterpret_cast<const Pack<T, V>*>(p + k + h);
#pragma unroll
        for (int j = 0; j < V; ++j) v[h + j] = pack.v[j];
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[h + j] = k + h + j < g.k ? p[k + h + j] : static_cast<T>(0.0f);
      }
    }
    __builtin_memcpy(&f.v, v, sizeof(v));
    return f;
  };
#pragma unroll 2
  for (int64_t k = wave * (kRun * kStep); k < g.k; k += kSkinnyWaves * kRun * kStep) {
    Frag<T> b[kRun][NB], a[kRun][MT];
#pragma unroll
    for (int s = 0; s < kRun; ++s) {
      const int64_t at = k + s * kStep + q * 8;
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
  float bias[4], bias2[4];
  load_biases<T, EPI, 4>(g, col0 + 4 * q, bias, bias2);
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
    finish_row<T, EPI, 4>(g, i * 16 + r, col0 + 4 * q, v, u, bias, bias2, 1.0f);
  }
}

// The parts of the depth of the cut tiles added in order, then the epilogue: 64 x 4 results of one
// tile per workgroup; with SLICES > 1 the parts are shared out over the waves, whose sums are added
// in order through LDS.
template <typename T, int BM, int BN, int EPI, int SLICES>
__global__ __launch_bounds__(kWave* SLICES) void gemm_finish_kernel(const Gemm g) {
  constexpr int NB = EPI == kEpiGated ? 2 : 1;
  constexpr int TN = BN / NB;
  constexpr int kPacks = BM * TN / 4;
  const int lane = threadIdx.x & (kWave - 1), slice = threadIdx.x / kWave;
  const int64_t tiles_m = (g.m + BM - 1) / BM, tiles_n = (g.n + TN - 1) / TN;
  const int64_t rest = tiles_m * tiles_n - g.full;
  const int64_t tile = blockIdx.x / (kPacks / kWave);
  const int pack = blockIdx.x % (kPacks / kWave) * kWave + lane;
  const int lr = pack / (TN / 4), lc = pack % (TN / 4) * 4;
  int64_t tm, tn;
  tile_at(g.full + tile, tiles_m, tiles_n, tm, tn);
  const int64_t row = tm * BM + lr, col = tn * TN + lc;
  const float* p = g.partial + (tile * NB * BM + lr) * TN + lc;
  f32x4 sum[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) sum[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (row < g.m && col < g.n) {
#pragma unroll 4
    for (int s = slice; s < g.splits; s += SLICES)
#pragma unroll
      for (int b = 0; b < NB; ++b)
        sum[b] += *reinterpret_cast<const f32x4*>(p + (s * rest * NB + b) * BM * TN);
  }
  if constexpr (SLICES > 1) {
    __shared__ f32x4 sh[SLICES][NB][kWave];
#pragma unroll
    for (int b = 0; b < NB; ++b) sh[slice][b][lane] = sum[b];
    __syncthreads();
    if (slice != 0) return;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int s = 1; s < SLICES; ++s) sum[b] += sh[s][b][lane];
  }
  float v[4], u[4], bias[4], bias2[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = sum[0][j];
    u[j] = sum[NB - 1][j];
  }
  load_biases<T, EPI, 4>(g, col, bias, bias2);
  finish_row<T, EPI, 4>(g, row, col, v, u, bias, bias2, result_scale<T, EPI>(g));
}

}  // namespace collie
