// 8-bit integer dense operators: quantisation of rows, and the product of a
// matrix quantised by row (token) with one quantised by row (output channel):
//
//   y[n, m] = (sum_k qx[n, k] qw[m, k]) sx[n] sw[m],
//
// sums exact in 32-bit integers (K < 2^17), on tcgen05 kind::i8.
//
// Up to four rows: CUDA cores (rows_kernel).  Tile kernel (few rows, or a long
// contraction and few tiles): one CTA computes 128 features (lanes of the
// accumulator) x NT rows of x over a slice of the contraction; the slices of a
// tile are the CTAs of a cluster and are added through distributed shared
// memory.  64 rows of 4096 to 4096: 8.0 us (16.8 MB of weights, 2.6 us of memory
// time), bounded by its start, the stages' latency and the join.  More rows:
// int8_pair.cuh.
#include <algorithm>
#include <cooperative_groups.h>

#include "int8_pair.cuh"

namespace ds {
namespace int8 {
namespace {

namespace cg = cooperative_groups;
using namespace ds::rows;

__device__ int g_err;   // bit 1: a bounded wait gave up

// ---------------------------------------------------------------- quantisation

__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  const int lane = threadIdx.x & 31;
  if (lane == 0) red[threadIdx.x >> 5] = v;
  row_barrier();
  return __reduce_max_sync(0xffffffffu, lane < warps ? red[lane] : 0u);
}

// Bits of the largest magnitude of a vector as f32 (bits of non-negative values
// order as the values, infinities and NaN above).
template <typename T, int VEC>
__device__ __forceinline__ uint32_t top_of(const Pack<T, VEC>& k) {
  if constexpr (VEC == 8) {
    uint32_t t = __vmaxu2(__vmaxu2(k.raw.x & 0x7FFF7FFFu, k.raw.y & 0x7FFF7FFFu),
                          __vmaxu2(k.raw.z & 0x7FFF7FFFu, k.raw.w & 0x7FFF7FFFu));
    t = max(t & 0xFFFFu, t >> 16);
    return std::is_same<T, __half>::value ? __float_as_uint(__half2float(__ushort_as_half((uint16_t)t))) : t << 16;
  } else {
    float v[VEC];
    k.get(v);
    uint32_t t = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) t = max(t, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    return t;
  }
}

// A block takes rows blockIdx.x, + gridDim.x ..., blockDim.y at a time, V times
// VEC values a thread; THREADS: of a row, which they fill, or 0, or -1: rows of
// any columns and strides, through lines.  The next row is loaded while this one
// is coded.  16384 x 4096 bf16: 35 us, 5.8 TB/s; with 16 values a thread instead
// of 32 37 us, without the row ahead 65.  Through lines 75 us (single values, in
// registers or through lines, 93 to 112).
template <typename T, int V, int THREADS>
__global__ void __maxnreg__(V <= 2 * (int)sizeof(T) ? 80 : 128) quantize_kernel(const T* __restrict__ x, int64_t rows,
                                                                                int cols, int64_t ld,
                                                                                uint8_t* __restrict__ codes,
                                                                                int64_t pitch,
                                                                                float* __restrict__ scales) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr bool kLines = THREADS < 0;
  extern __shared__ uint4 smem[];
  __shared__ uint32_t red[kMostRows][2][32];
  launch_dependents();
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  auto column = [&](int i) { return (i * (THREADS > 0 ? THREADS : (int)blockDim.x) + (int)threadIdx.x) * VEC; };
  auto inside = [&](int i) { return THREADS > 0 || column(i) < cols; };
  Lines<T> lines;
  lines.template place<kStages>(smem, x, cols);
  Pack<T, VEC> k[V];
  auto fetch = [&](int stage, int64_t row) {
    if constexpr (kLines) {
      if (row < rows) lines.copy(stage, x + row * ld);
      Slots::commit();
    } else {
      if (row >= rows) return;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (inside(i)) k[i].load(x + row * ld + column(i));
    }
  };
  int turn = 0, stage = 0;
  int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
#pragma unroll
  for (int i = 0; i < (kLines ? kStages - 1 : 1); ++i) fetch(i, row + i * step);
  for (; row < rows; row += step, turn ^= 1) {
    if constexpr (kLines) {
      Slots::wait<kStages - 2>();
      line_barrier();   // the row is here, and the one before it read
      fetch(stage ? stage - 1 : kStages - 1, row + (kStages - 1) * step);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!inside(i)) continue;
        k[i].raw = lines.vector(stage, x + row * ld, column(i));
        if (column(i) + VEC > cols) k[i].cut(cols - column(i));
      }
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    float v[V][VEC];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (!inside(i)) continue;
      top = max(top, top_of(k[i]));
      k[i].get(v[i]);
    }
    if constexpr (!kLines) fetch(0, row + step);   // on its way during the rest
    const float s = scale_of(row_max(top, red[threadIdx.y][turn]));
    if (threadIdx.x == 0) scales[row] = s;
    const Coder coder(s);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (!inside(i)) continue;
      uint32_t q[VEC];
      coder.codes(v[i], q);
      uint8_t* at = codes + row * pitch + column(i);
      if (kLines && column(i) + VEC > cols) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (column(i) + j < cols) at[j] = (uint8_t)q[j];
        continue;
      }
      uint32_t w[VEC / 4];
#pragma unroll
      for (int j = 0; j < VEC / 4; ++j) w[j] = pack_codes(q[4 * j], q[4 * j + 1], q[4 * j + 2], q[4 * j + 3]);
      if constexpr (VEC == 8) *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(at) = w[0];
    }
  }
}

// Rows that no block's registers hold: read twice, one value a thread.
template <typename T>
__global__ void __launch_bounds__(1024) quantize_long_kernel(const T* __restrict__ x, int cols, int64_t ld,
                                                             uint8_t* __restrict__ codes, int64_t pitch,
                                                             float* __restrict__ scales) {
  __shared__ uint32_t red[32];
  launch_dependents();
  const int64_t row = blockIdx.x;
  const T* src = x + row * ld;
  uint32_t top = 0;
  for (int c = threadIdx.x; c < cols; c += blockDim.x) top = max(top, __float_as_uint((float)src[c]) & 0x7FFFFFFFu);
  const float s = scale_of(row_max(top, red));
  if (threadIdx.x == 0) scales[row] = s;
  const Coder coder(s);
  for (int c = threadIdx.x; c < cols; c += blockDim.x) {
    float v[2] = {(float)src[c], 0.0f};
    uint32_t q[2];
    coder.codes(v, q);
    codes[row * pitch + c] = (uint8_t)q[0];
  }
}

// Values of codes, VEC a thread: eight where the result's rows lie on 16 bytes,
// otherwise (ANY) the 16 bytes of a granule of the result, whose codes are a
// window of two.  STREAM: the result leaves L2 first, so that the codes, which
// their quantisation may just have left there, do not; for results that do not fit
// into L2, whose next reader has to fetch most of them either way.  To bf16 in rows
// of 4096, with quantisation before it: 16384 of them 65.6 us instead of 71.7,
// 18432 77.8 (81.9), from 20480 on none is gained (24576: 107.6, 106.8).  Of codes
// from memory, alone or with a layer norm or a product reading the result: 40.9
// (40.1), 94.2 (93.6) and 71.7 us (70.9).  With the result inside L2 that reader
// would pay: 8192 rows and a product 42.5 us instead of 36.9.
template <typename T, bool ANY, bool STREAM>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ codes, int64_t pitch,
                                                         const float* __restrict__ scales, int64_t rows, int cols,
                                                         T* __restrict__ out) {
  constexpr int PER = 16 / sizeof(T), VEC = ANY ? PER : 8;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= rows) return;
  const float s = scales[row];
  const uint8_t* from = codes + row * pitch;
  T* dst = out + row * cols;
  // columns of the row in its first granule that are another's
  const int skip = ANY ? (int)(reinterpret_cast<uintptr_t>(dst) & 15) / (int)sizeof(T) : 0;
  for (int c = (int)threadIdx.x * VEC - skip; c < cols; c += blockDim.x * VEC) {
    if (ANY && (c < 0 || c + VEC > cols)) {
      for (int j = max(c, 0); j < min(c + VEC, cols); ++j) dst[j] = narrow<T>((float)(int8_t)from[j] * s);
      continue;
    }
    // c + skip is a multiple of VEC
    uint32_t w[VEC / 4];
    if constexpr (VEC == 8) {
      uint2 q = *reinterpret_cast<const uint2*>(from + c + skip);
      if (ANY && skip) {
        const uint2 before = *reinterpret_cast<const uint2*>(from + c + skip - 8);
        const uint32_t a = skip < 4 ? before.y : before.x, b = skip < 4 ? q.x : before.y, e = skip < 4 ? q.y : q.x;
        const int bits = 8 * (4 - (skip & 3));
        q = make_uint2(__funnelshift_rc(a, b, bits), __funnelshift_rc(b, e, bits));
      }
      w[0] = q.x, w[1] = q.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(from + c + skip);
      if (skip) w[0] = __funnelshift_r(*reinterpret_cast<const uint32_t*>(from + c + skip - 4), w[0], 8 * (4 - skip));
    }
    float v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (float)(int8_t)(w[j / 4] >> (8 * (j & 3))) * s;
#pragma unroll
    for (int h = 0; h < VEC / PER; ++h) {
      float part[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) part[j] = v[h * PER + j];
      put<T, PER, STREAM>(dst + c + h * PER, part);
    }
  }
}

// ---------------------------------------------------------------- product of few rows

struct TileParams {
  CUtensorMap a, b;            // codes of the weights, of x
  const float *sw, *sx;
  int M, N;                    // features, rows of x
  int ksteps;                  // stages of 128 codes
  void* out;                   // out[n * ldo + m]
  int64_t ldo;
  int out_dtype;
  int* err;
};

template <int NT>
struct TileShape {
  static constexpr int kStage = 16384 + NT * 128;
  // less than half of an SM, so that the next launch's CTAs join this one's and
  // their weights are on their way while it finishes
  static constexpr int kStages = std::min(6, 110 * 1024 / kStage);
  static constexpr int kSmem = 1024 + kStages * kStage;
  static constexpr int kCols = NT < 32 ? 32 : NT;
  static_assert(kStages * kStage >= NT * 128 * 4, "stages hold the partial tile");
};

constexpr int kTileThreads = 320;   // warp 0 copies, warp 1 MMA, warps 2-9 epilogue (two a lane quarter)

// Elements (m, n0 .. n0 + J - 1) of the result, nv of them inside; sx: the
// scales of row n0 and on.
template <int J>
__device__ __forceinline__ void tile_store(const TileParams& p, int m, float sw, int n0, int nv, const float* sx,
                                           const int (&v)[J]) {
  if (m >= p.M) return;
  const int64_t at = (int64_t)n0 * p.ldo + m;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (j >= nv) continue;
    const float y = scaled(v[j], sx[j], sw);
    if (p.out_dtype == DS_F32) static_cast<float*>(p.out)[at + j * p.ldo] = y;
    else if (p.out_dtype == DS_F16) static_cast<__half*>(p.out)[at + j * p.ldo] = __float2half_rn(y);
    else static_cast<__nv_bfloat16*>(p.out)[at + j * p.ldo] = __float2bfloat16_rn(y);
  }
}

// Sums this CTA's share of the tile's `rows` rows over the partial tiles
// [NT][128] of the cluster.  The reads of four rows from all slices are in
// flight together.
template <int NT, int SLICES>
__device__ __forceinline__ void tile_join(const TileParams& p, int* part, int slice, int turn, int m, int mi, float sw,
                                          int n0, int rows, const float* sx) {
  cg::cluster_group cluster = cg::this_cluster();
  const int* src[SLICES];
#pragma unroll
  for (int r = 0; r < SLICES; ++r) src[r] = cluster.map_shared_rank(part, r) + mi;
  const int share = (rows + SLICES - 1) / SLICES, end = min(rows, (slice + 1) * share);
  for (int n = slice * share + 4 * turn; n < end; n += 8) {
    int w[SLICES][4];
#pragma unroll
    for (int r = 0; r < SLICES; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) w[r][j] = src[r][min(n + j, end - 1) * 128];
    int v[4] = {};
#pragma unroll
    for (int r = 0; r < SLICES; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += w[r][j];
    tile_store(p, m, sw, n0 + n, end - n, sx + n, v);
  }
}

// Eight values of a row from p on, the first n of them (0 behind).
template <typename X>
__device__ __forceinline__ void load8(const X* p, int n, bool vec, float (&v)[8]) {
  if (vec && n >= 8) {
    constexpr int kPer = 16 / sizeof(X);
#pragma unroll
    for (int h = 0; h < 8 / kPer; ++h) {
      Pack<X, kPer> k;
      k.load_kept(p + h * kPer);
      float f[kPer];
      k.get(f);
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[h * kPer + j] = f[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? (float)p[j] : 0.0f;
  }
}

template <int NT>
__global__ void __launch_bounds__(kTileThreads, 2) tile_kernel(const __grid_constant__ TileParams p) {
  using C = TileShape<NT>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ __align__(8) uint64_t full[S], empty[S], accfull;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  cg::cluster_group cluster = cg::this_cluster();
  const int slices = cluster.dim_blocks().x, slice = cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mts = (p.M + 127) / 128, tile = blockIdx.x / slices;
  const int m0 = tile % mts * 128, n0 = tile / mts * NT, rows = min(NT, p.N - n0);
  const int it0 = (int)((int64_t)p.ksteps * slice / slices), its = (int)((int64_t)p.ksteps * (slice + 1) / slices) - it0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&accfull, 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tc5::alloc(&tmem_base, C::kCols);
  tc5::fence_before();
  __syncthreads();
  tc5::fence_after();
  const uint32_t tb = tmem_base;
  volatile int* abort = &abort_flag;
  launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      auto weights = [&](int g) {
        mbar_arrive_expect_tx(&full[g % S], C::kStage);
        tma_load_2d(smem + g % S * C::kStage, &p.a, (it0 + g) * 128, m0, &full[g % S]);
      };
      auto codes = [&](int g) {
        tma_load_2d(smem + g % S * C::kStage + 16384, &p.b, (it0 + g) * 128, n0, &full[g % S]);
      };
      // The weights of the first stages need nothing of the launch before this
      // one in the stream: that is one of the same call, and the call's first
      // launch began after all earlier work had ended.
      const int early = min(S, its);
      for (int g = 0; g < early; ++g) weights(g);
      wait_prior_grid();
      for (int g = 0; g < early; ++g) codes(g);
      int g = early;
      for (; g < its; ++g) {
        if (!ds::pair::wait(&empty[g % S], ((g / S) - 1) & 1, abort, p.err)) break;
        weights(g);
        codes(g);
      }
      // never leave with copies in flight into this CTA's shared memory
      for (int j = g - S < 0 ? 0 : g - S; j < g; ++j) mbar_wait_bounded(&full[j % S], (j / S) & 1, 200000000ull);
    }
  } else if (warp == 1) {
    const uint64_t ops = tc5::sdesc_sw128(smem_u32(smem));
    constexpr uint32_t id = idesc(128, NT);
    for (int g = 0; g < its; ++g) {
      const int s = g % S;
      if (!ds::pair::wait_all(&full[s], (g / S) & 1, abort, p.err)) break;
      tc5::fence_after();
      if (elect_one()) {
        const uint64_t ad = ops + (uint64_t)((s * C::kStage) >> 4), bd = ad + (16384 >> 4);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) mma(tb, ad + 2 * kk, bd + 2 * kk, id, (g | kk) != 0);
        tc5::commit(&empty[s]);
      }
      __syncwarp();
    }
    // all issued MMAs complete before the accumulators are read or released
    if (elect_one()) tc5::commit(&accfull);
    __syncwarp();
    ds::pair::wait_all(&accfull, 0, abort, p.err);
  } else {
    ds::pair::wait_all(&accfull, 0, abort, p.err);
  }
  tc5::fence_after();

  // ---- epilogue: thread = one feature (lane of tensor memory)
  wait_prior_grid();
  const int q = warp & 3, turn = (warp - 2) >> 2, mi = q * 32 + lane, m = m0 + mi;
  int* part = reinterpret_cast<int*>(smem);   // [NT][128]
  const float* sx = p.sx + n0;
  const float sw = warp >= 2 && m < p.M ? p.sw[m] : 0.0f;
  if (warp >= 2) {
    for (int c0 = 16 * turn; c0 < rows; c0 += 32) {
      float f[16];
      int v[16];
      tc5::ld_x16_nowait(tc5::lane_quarter(tb + c0, q), f);
      tc5::wait_ld();
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = __float_as_int(f[j]);
      if (slices > 1) {
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c0 + j) * 128 + mi] = v[j];
      } else {
        tile_store(p, m, sw, n0 + c0, rows - c0, sx + c0, v);
      }
    }
  }
  if (slices > 1) {
    cluster.sync();
    if (warp >= 2) {
      if (slices == 8) tile_join<NT, 8>(p, part, slice, turn, m, mi, sw, n0, rows, sx);
      else if (slices == 4) tile_join<NT, 4>(p, part, slice, turn, m, mi, sw, n0, rows, sx);
      else tile_join<NT, 2>(p, part, slice, turn, m, mi, sw, n0, rows, sx);
    }
    cluster.sync();   // partial tiles stay until every CTA has read them
  }
  tc5::fence_before();
  __syncthreads();
  if (warp == 1) {
    tc5::fence_after();
    tc5::dealloc(tb, C::kCols);
  }
}

// ---------------------------------------------------------------- product of single rows

struct VecParams {
  const uint8_t* w;            // codes of the weights
  int64_t pitch;
  const float *sw, *sx;        // sx: scales of x where it comes as codes
  const void* x;
  int64_t ldx;                 // of codes
  int vec;                     // every 8 values of x start on 16 bytes
  int cols, M, N;              // K, features, rows of x (up to T)
  void* out;
  int64_t ldo;
  int out_dtype;
};

// 16 codes of a row from `at` on, of which n (1 or more) are left; what lies
// behind the row's end is not touched.
__device__ __forceinline__ uint4 codes_at(const uint8_t* at, int n) {
  if (n >= 16) return __ldcs(reinterpret_cast<const uint4*>(at));
  uint32_t q[4] = {};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < n) q[j >> 2] |= (uint32_t)at[j] << (8 * (j & 3));
  return make_uint4(q[0], q[1], q[2], q[3]);
}

// Up to T rows of x by F features a block, on CUDA cores: a thread keeps 16
// columns (of every blockDim.x * 16), so it quantises just what it multiplies,
// and all F rows of weights are on their way before x has been looked at.  X:
// type of x, one row of values, or int8_t where a launch before this one has
// quantised it (every block that quantises does all of it: two rows took 12.8 us
// that way).
// No cluster, no tensor memory: bounded by the stream of weights and the start
// of a launch.  The grid is one wave of blocks where it
// can be (by_features).  One row of 4096 to 4096: 8.4 us with its launch, 2.6 of
// them the weights at memory speed.
template <typename X, int T, int F>
__global__ void __launch_bounds__(256) rows_kernel(const VecParams p) {
  constexpr bool kCoded = std::is_same<X, int8_t>::value;
  static_assert(kCoded || T == 1, "only a single row comes as values");
  __shared__ uint32_t tops[8];
  __shared__ int part[8][F * T];
  __shared__ float sx[T];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int f0 = blockIdx.x * F, wide = blockDim.x * 16;
  const X* x = static_cast<const X*>(p.x);
  uint4 w[F];
  auto weights = [&](int c) {
#pragma unroll
    for (int f = 0; f < F; ++f) {
      w[f] = make_uint4(0u, 0u, 0u, 0u);
      if (f0 + f < p.M && c < p.cols) w[f] = codes_at(p.w + (f0 + f) * p.pitch + c, p.cols - c);
    }
  };
  weights(threadIdx.x * 16);
  [[maybe_unused]] float scale;
  if constexpr (kCoded) {
    launch_dependents();
    wait_prior_grid();
    if (threadIdx.x < T) sx[threadIdx.x] = threadIdx.x < p.N ? p.sx[threadIdx.x] : 0.0f;
  } else {
    uint32_t top = 0;
    for (int c = threadIdx.x * 16; c < p.cols; c += wide) {
#pragma unroll
      for (int h = 0; h < 16; h += 8) {
        float v[8];
        load8(x + c + h, p.cols - c - h, p.vec, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    for (int i = 0; i < warps; ++i) top = max(top, tops[i]);
    scale = scale_of(top);
    if (threadIdx.x == 0) sx[0] = scale;
  }
  int acc[F][T] = {};
  for (int c = threadIdx.x * 16;; c += wide) {
    uint32_t q[T][4];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      if constexpr (kCoded) {
        uint4 k = make_uint4(0u, 0u, 0u, 0u);
        if (t < p.N && c < p.cols) k = codes_at(reinterpret_cast<const uint8_t*>(x) + t * p.ldx + c, p.cols - c);
        q[t][0] = k.x, q[t][1] = k.y, q[t][2] = k.z, q[t][3] = k.w;
      } else {
        const Coder coder(scale);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[8];
          uint32_t k[8];
          load8(x + c + 8 * h, p.cols - c - 8 * h, p.vec, v);
          coder.codes(v, k);
          q[t][2 * h] = pack_codes(k[0], k[1], k[2], k[3]), q[t][2 * h + 1] = pack_codes(k[4], k[5], k[6], k[7]);
        }
      }
    }
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const uint32_t k[4] = {w[f].x, w[f].y, w[f].z, w[f].w};
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[f][t] = __dp4a((int)k[j], (int)q[t][j], acc[f][t]);
    }
    if (c + wide >= p.cols) break;
    weights(c + wide);
  }
#pragma unroll
  for (int f = 0; f < F; ++f)
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int v = __reduce_add_sync(0xffffffffu, acc[f][t]);
      if (lane == 0) part[warp][f * T + t] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < F * T; i += blockDim.x) {
    const int f = i / T, t = i % T;
    if (f0 + f >= p.M || t >= p.N) continue;
    int v = 0;
    for (int k = 0; k < warps; ++k) v += part[k][i];
    const float y = scaled(v, sx[t], p.sw[f0 + f]);
    const int64_t at = t * p.ldo + f0 + f;
    if (p.out_dtype == DS_F32) static_cast<float*>(p.out)[at] = y;
    else if (p.out_dtype == DS_F16) static_cast<__half*>(p.out)[at] = __float2half_rn(y);
    else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
  }
}

// ---------------------------------------------------------------- host side

constexpr int kMostCols = (1 << 17) - 1;   // 2^14 K stays inside an s32 sum

int64_t pitch_of(int64_t cols) { return (cols + kPitch - 1) / kPitch * kPitch; }

// Codes of a matrix [rows, cols], rows pitch bytes apart, in boxes of 128 codes
// x box_rows (zeros outside).
bool map_codes(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t pitch, int box_rows) {
  return grouped::encode_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, rows, cols, pitch, 128, box_rows,
                            CU_TENSOR_MAP_SWIZZLE_128B);
}

int* err_word() {
  static SymbolOnce known;
  return ds::symbol_address(&known, &g_err);
}

int launch_quantize(const void* x, int dtype, int64_t rows, int cols, int64_t ld, uint8_t* codes, int64_t pitch,
                    float* scales, cudaStream_t s) {
  const int es = elements(dtype);
  const bool vec = vectors(x, rows, cols, ld, es);
  int st = DS_OK;
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    const T* src = static_cast<const T*>(x);
    if (cols > 64 * 1024 / es || (!vec && kStages * Lines<T>::pitch_of(cols) > kMostSmem)) {
      quantize_long_kernel<T><<<(unsigned)rows, 1024, 0, s>>>(src, cols, ld, codes, pitch, scales);
      return;
    }
    // 16 values a thread; many rows are shared out in 32, as the maximum over a
    // row's threads takes much of the work otherwise (but not f32 through lines:
    // too few registers, 8192 x 4096 with its dequantisation 110 us instead of 88)
    const bool many = rows >= 4 * (int64_t)ds::sm_count() && (vec || es == 2);
    const Shape sh = shape_of(cols, 16 / es, many ? 32 : 16, 512, 256);
    by_shape<T, 2 * sizeof(T), 8, true>(sh, cols, vec, [&](auto, auto v, auto threads) {
      st = launch_rows<quantize_kernel<T, decltype(v)::value, decltype(threads)::value>>(
          sh, rows, vec ? 0 : kStages * Lines<T>::pitch_of(cols), s, src, rows, cols, ld, codes, pitch, scales);
    });
  });
  if (st != DS_OK) return st;
  DS_CHECK_LAUNCH("int8 quantize_kernel");
  return DS_OK;
}

// Rows of x as a call gives them: values, or codes (DS_I8) with their scales.
struct Input {
  const void* p;
  const float* scales;
  int dtype;
  int64_t rows, ld;
  int cols;
};

template <int NT>
int launch_tiles(TileParams& p, const Input& x, const DsInt8& w, int slices, cudaStream_t s, bool chained) {
  using C = TileShape<NT>;
  const bool ok = map_codes(&p.a, w.codes, w.rows, w.cols, w.pitch, 128) &&
                  map_codes(&p.b, x.p, x.rows, x.cols, x.ld, NT);
  DS_REQUIRE(ok, DS_ECUDA, "int8: tensor map encoding failed");
  static SmemOnce once;
  const int st = ds::allow_smem(&once, reinterpret_cast<const void*>(&tile_kernel<NT>), C::kSmem);
  if (st != DS_OK) return st;
  const int64_t tiles = (p.M + 127) / 128 * (int64_t)((p.N + NT - 1) / NT);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * slices));
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)slices;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = chained ? 2 : 1;
  DS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, tile_kernel<NT>, p));
  return DS_OK;
}

// Result [rows, cols], whose rows start on 16 bytes, in boxes of 128 bytes x 32 rows.
bool map_result(CUtensorMap* m, void* y, int64_t rows, int64_t cols, int dtype) {
  const int es = elements(dtype);
  return grouped::encode_2d(m, dtype == DS_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, y,
                            rows, cols, cols * es, 128 / es, 32, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int NT>
int launch_pairs(PairParams& p, const Input& x, const DsInt8& w, cudaStream_t s, bool chained) {
  using C = pairs::Shape<NT>;
  const bool ok = map_codes(&p.a, x.p, x.rows, x.cols, x.ld, 128) &&
                  map_codes(&p.b, w.codes, w.rows, w.cols, w.pitch, NT / 2);
  DS_REQUIRE(ok, DS_ECUDA, "int8: tensor map encoding failed");
  const int64_t tiles = (p.M + 255) / 256 * (int64_t)((p.N + NT - 1) / NT);
  DS_REQUIRE(tiles < ((int64_t)1 << 31), DS_ERANGE, "int8: too many tiles");
  static SmemOnce once;
  const int st = ds::allow_smem(&once, reinterpret_cast<const void*>(&pairs::pair_kernel<NT>), C::kSmem);
  if (st != DS_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, ds::sm_count() / 2)));
  cfg.blockDim = dim3(pairs::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = chained ? 1 : 0;
  DS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, pairs::pair_kernel<NT>, p));
  return DS_OK;
}

// Rows up to which the product runs on CUDA cores: four of 4096 to 4096 take
// 10.4 us with their quantisation (the tile kernel 10.8), of 1024 to 1024 6.3
// (8.4); eight 14.5 (10.8).
constexpr int kVecRows = 4;

template <typename X, int T, int F>
int launch_vec(const VecParams& p, cudaStream_t s, bool chained) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.M + F - 1) / F));
  cfg.blockDim = dim3((unsigned)std::min(256, (p.cols + 511) / 512 * 32));
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = chained ? 1 : 0;
  DS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, rows_kernel<X, T, F>, p));
  return DS_OK;
}

// Features a block: the fewest that leave one wave of two blocks an SM.
template <typename X, int T>
int by_features(const VecParams& p, cudaStream_t s, bool chained) {
  const int64_t wave = 2 * (int64_t)ds::sm_count();
  if (p.M <= 4 * wave) return launch_vec<X, T, 4>(p, s, chained);
  if constexpr (T < 4) {
    if (p.M > 8 * wave) return launch_vec<X, T, 16>(p, s, chained);
  }
  return launch_vec<X, T, 8>(p, s, chained);
}

int launch_rows_kernel(const Input& x, const DsInt8& w, void* y, int out_dtype, cudaStream_t s, bool chained) {
  VecParams p = {reinterpret_cast<const uint8_t*>(w.codes), w.pitch, w.scales, x.scales, x.p, x.ld, 0, x.cols,
                 (int)w.rows, (int)x.rows, y, w.rows, out_dtype};
  int st = DS_OK;
  if (x.dtype == DS_I8) {
    if (x.rows == 1) return by_features<int8_t, 1>(p, s, chained);
    if (x.rows == 2) return by_features<int8_t, 2>(p, s, chained);
    return by_features<int8_t, 4>(p, s, chained);
  }
  p.vec = ds::aligned(x.p, 16);
  by_type(x.dtype, [&](auto t) {
    using X = decltype(t);
    st = by_features<X, 1>(p, s, false);
  });
  return st;
}

// Estimated times in ns of both tensor core kernels, fitted to the figures of
// K x N = 1024 x 1024 to 8192 x 8192 with 64 to 2048 rows of codes (within 15 %
// there).  The pair kernel takes a launch and, for each wave of tiles, its
// stages, 360, 270 or 234 ns each at 256, 128 or 64 columns; it wins where one
// wave has work for most pairs (4096 x 4096, 512 rows: 13.6 us, the tile kernel
// 17.5).  The tile kernel shares a contraction out among up to eight CTAs; it
// wins where it is long and the result small (8192 x 512, 512 rows: 12 us, the
// pair kernel 20).
// Results whose rows do not start on 16 bytes (boxed false) leave it row by row:
// 20 ns a column and wave more.
int64_t pair_ns(int64_t rows, int64_t cols, int ksteps, int nt, bool boxed) {
  const int64_t tiles = (rows + 255) / 256 * ((cols + nt - 1) / nt), pairs = ds::sm_count() / 2;
  return 4800 + (tiles + pairs - 1) / pairs * (ksteps * (nt == 256 ? 360 : nt == 128 ? 270 : 234) + (boxed ? 0 : 20 * nt));
}

// `slices`: of the contraction, enough to give every SM a CTA, at least two stages each.
int64_t tile_ns(int64_t rows, int64_t cols, int ksteps, int nt, int* slices) {
  const int64_t tiles = (cols + 127) / 128 * ((rows + nt - 1) / nt), sms = ds::sm_count();
  int s = 1;
  while (s < 8 && tiles * s * 2 <= sms && ksteps / (s * 2) >= 2) s *= 2;
  *slices = s;
  return 5000 + 8 * nt + 310 * ((ksteps + s - 1) / s) * std::max(tiles * s, sms) / sms + (s > 1 ? 4 * nt * s : 0);
}

// y = x W^T.
int product(const Input& x, const DsInt8& w, void* y, int out_dtype, int* err, cudaStream_t s, bool chained) {
  if (x.rows <= kVecRows) return launch_rows_kernel(x, w, y, out_dtype, s, chained);
  const int ksteps = (int)((w.cols + 127) / 128), nt = x.rows <= 16 ? 16 : x.rows <= 32 ? 32 : x.rows <= 64 ? 64 : 128;
  int slices, wide = 256;
  const int64_t by_tiles = tile_ns(x.rows, w.rows, ksteps, nt, &slices);
  const bool boxed = ds::aligned(y, 16) && w.rows * elements(out_dtype) % 16 == 0;
  int64_t by_pairs = pair_ns(x.rows, w.rows, ksteps, 256, boxed);
  for (int n : {128, 64}) {
    const int64_t t = pair_ns(x.rows, w.rows, ksteps, n, boxed);
    if (t < by_pairs) by_pairs = t, wide = n;
  }
  if (x.rows > 64 && by_pairs < by_tiles) {
    PairParams p = {};
    p.sx = x.scales, p.sw = w.scales, p.y = y, p.ldy = w.rows, p.out_dtype = out_dtype;
    p.boxed = boxed && map_result(&p.out, y, x.rows, w.rows, out_dtype);
    p.M = (int)x.rows, p.N = (int)w.rows, p.ksteps = ksteps, p.err = err;
    if (wide == 256) return launch_pairs<256>(p, x, w, s, chained);
    if (wide == 128) return launch_pairs<128>(p, x, w, s, chained);
    return launch_pairs<64>(p, x, w, s, chained);
  }
  TileParams p = {};
  p.sw = w.scales, p.sx = x.scales, p.M = (int)w.rows, p.N = (int)x.rows, p.ksteps = ksteps, p.err = err;
  p.out = y, p.ldo = w.rows, p.out_dtype = out_dtype;
  if (nt == 16) return launch_tiles<16>(p, x, w, slices, s, chained);
  if (nt == 32) return launch_tiles<32>(p, x, w, slices, s, chained);
  if (nt == 64) return launch_tiles<64>(p, x, w, slices, s, chained);
  return launch_tiles<128>(p, x, w, slices, s, chained);
}

// Workspace for x given as values; a single row is quantised by the product's
// own kernel (a launch and its workspace less: 8.4 us for 4096 to 4096 instead
// of 9.8, and 42 of host time instead of 50).
size_t x_bytes(int64_t rows, int64_t cols) {
  if (rows <= 1) return 0;
  return grouped::up((size_t)rows * pitch_of(cols), 256) + grouped::up((size_t)rows * 4, 256);
}

}  // namespace
}  // namespace int8
}  // namespace ds

using namespace ds::int8;

extern "C" int ds_int8_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ld, int8_t* codes,
                                int64_t pitch, float* scales, void* stream) {
  DS_REQUIRE(x_dtype == DS_F32 || x_dtype == DS_BF16 || x_dtype == DS_F16, DS_EINVAL,
             "int8_quantize: x must be f32, bf16 or f16");
  DS_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && cols >= 1 && cols <= kMostCols, DS_ERANGE,
             "int8_quantize: rows must be in [0, 2^31), cols in [1, 2^17)");
  DS_REQUIRE(rows <= 1 || ld >= cols, DS_EINVAL, "int8_quantize: row stride below cols");
  DS_REQUIRE(pitch >= cols && pitch % kPitch == 0, DS_EINVAL,
             "int8_quantize: the codes' rows must be a multiple of 16 bytes apart, and hold cols");
  if (rows == 0) return DS_OK;
  DS_REQUIRE(x && codes && scales, DS_EINVAL, "int8_quantize: null pointer");
  DS_REQUIRE(ds::aligned(x, ds::rows::elements(x_dtype)) && ds::aligned(codes, 16) && ds::aligned(scales, 4), DS_EALIGN,
             "int8_quantize: x and scales must be aligned to their elements, codes to 16 bytes");
  return launch_quantize(x, x_dtype, rows, (int)cols, ld, reinterpret_cast<uint8_t*>(codes), pitch, scales,
                         static_cast<cudaStream_t>(stream));
}

extern "C" int ds_int8_dequantize(const int8_t* codes, int64_t pitch, const float* scales, int64_t rows, int64_t cols,
                                  void* out, int out_dtype, void* stream) {
  DS_REQUIRE(out_dtype == DS_F32 || out_dtype == DS_BF16 || out_dtype == DS_F16, DS_EINVAL,
             "int8_dequantize: out must be f32, bf16 or f16");
  DS_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && cols >= 1 && cols <= kMostCols, DS_ERANGE,
             "int8_dequantize: rows must be in [0, 2^31), cols in [1, 2^17)");
  DS_REQUIRE(pitch >= cols && pitch % kPitch == 0, DS_EINVAL,
             "int8_dequantize: the codes' rows must be a multiple of 16 bytes apart, and hold cols");
  if (rows == 0) return DS_OK;
  const int es = ds::rows::elements(out_dtype);
  DS_REQUIRE(codes && scales && out, DS_EINVAL, "int8_dequantize: null pointer");
  DS_REQUIRE(ds::aligned(codes, 16) && ds::aligned(scales, 4) && ds::aligned(out, es), DS_EALIGN,
             "int8_dequantize: codes must be 16-byte aligned, scales and out to their elements");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint8_t* src = reinterpret_cast<const uint8_t*>(codes);
  const bool vec = ds::aligned(out, 16) && cols % 8 == 0;
  const int n = (int)(vec ? cols / 8 : (cols * es + 14) / 16 + 1), threads = std::min(256, (n + 31) / 32 * 32);
  const dim3 block(threads, 256 / threads);
  const unsigned grid = (unsigned)((rows + block.y - 1) / block.y);
  ds::rows::by_type(out_dtype, [&](auto t) {
    using T = decltype(t);
    T* dst = static_cast<T*>(out);
    const bool stream = rows * cols * es >= (126 << 20);   // L2
    if (vec && stream) dequantize_kernel<T, false, true><<<grid, block, 0, s>>>(src, pitch, scales, rows, (int)cols, dst);
    else if (vec) dequantize_kernel<T, false, false><<<grid, block, 0, s>>>(src, pitch, scales, rows, (int)cols, dst);
    else if (stream) dequantize_kernel<T, true, true><<<grid, block, 0, s>>>(src, pitch, scales, rows, (int)cols, dst);
    else dequantize_kernel<T, true, false><<<grid, block, 0, s>>>(src, pitch, scales, rows, (int)cols, dst);
  });
  DS_CHECK_LAUNCH("int8 dequantize_kernel");
  return DS_OK;
}

extern "C" int ds_int8_linear_workspace_size(int64_t rows, int64_t cols, size_t* bytes) {
  DS_REQUIRE(bytes && rows >= 0 && cols >= 1, DS_EINVAL,
             "int8_linear_workspace_size: rows >= 0, cols >= 1 and an output expected");
  *bytes = x_bytes(rows, cols);
  return DS_OK;
}

extern "C" int ds_int8_linear(const void* x, const float* x_scales, int x_dtype, int64_t rows, int64_t ld,
                              const DsInt8* w, void* out, int out_dtype, void* workspace, size_t workspace_bytes,
                              void* stream) {
  DS_REQUIRE(w && w->codes && w->scales, DS_EINVAL, "int8_linear: null weight");
  DS_REQUIRE(w->rows >= 1 && w->rows <= (1 << 20) && w->cols >= 1 && w->cols <= kMostCols, DS_ERANGE,
             "int8_linear: weight rows must be in [1, 2^20], cols in [1, 2^17)");
  DS_REQUIRE(w->pitch >= w->cols && w->pitch % kPitch == 0, DS_EINVAL,
             "int8_linear: the weight's rows must be a multiple of 16 bytes apart, and hold its cols");
  DS_REQUIRE(ds::aligned(w->codes, 16) && ds::aligned(w->scales, 4), DS_EALIGN,
             "int8_linear: weight codes must be 16-byte aligned, scales to 4");
  DS_REQUIRE(x_dtype == DS_F32 || x_dtype == DS_BF16 || x_dtype == DS_F16 || x_dtype == DS_I8, DS_EINVAL,
             "int8_linear: x must be f32, bf16 or f16, or codes (i8) with scales");
  const bool coded = x_dtype == DS_I8;
  DS_REQUIRE(rows >= 0 && rows <= (1 << 22), DS_ERANGE, "int8_linear: rows must be in [0, 2^22]");
  DS_REQUIRE(out_dtype == DS_F32 || out_dtype == DS_BF16 || out_dtype == DS_F16, DS_EINVAL,
             "int8_linear: out must be f32, bf16 or f16");
  if (rows == 0) return DS_OK;
  DS_REQUIRE(x && (!coded || x_scales), DS_EINVAL, "int8_linear: null x");
  DS_REQUIRE(coded ? ld >= w->cols && ld % kPitch == 0 : rows <= 1 || ld >= w->cols, DS_EINVAL,
             "int8_linear: row stride of x below its columns, or that of its codes not a multiple of 16");
  DS_REQUIRE(coded ? ds::aligned(x, 16) && ds::aligned(x_scales, 4) : ds::aligned(x, ds::rows::elements(x_dtype)),
             DS_EALIGN, "int8_linear: x must be aligned to its elements, codes to 16 bytes");
  const size_t need = coded ? 0 : x_bytes(rows, w->cols);
  DS_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), DS_EINVAL,
             "int8_linear: workspace %zu bytes < required %zu", workspace_bytes, need);
  DS_REQUIRE(out && ds::aligned(out, ds::rows::elements(out_dtype)) && ds::aligned(workspace, 256), DS_EALIGN,
             "int8_linear: out must be aligned to its elements, the workspace to 256 bytes");
  DS_REQUIRE(ds::grouped::encode_fn() != nullptr, DS_ECUDA, "int8_linear: cuTensorMapEncodeTiled unavailable");
  int* err = err_word();
  DS_REQUIRE(err != nullptr, DS_ECUDA, "int8_linear: error word unavailable");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Input in = {x, x_scales, x_dtype, rows, ld, (int)w->cols};
  const bool first = !coded && rows > 1;
  if (first) {
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    float* scales = reinterpret_cast<float*>(codes + ds::grouped::up((size_t)rows * pitch_of(w->cols), 256));
    const int st = launch_quantize(x, x_dtype, rows, in.cols, ld, codes, pitch_of(w->cols), scales, s);
    if (st != DS_OK) return st;
    in = {codes, scales, DS_I8, rows, pitch_of(w->cols), in.cols};
  }
  return product(in, *w, out, out_dtype, err, s, first);
}

extern "C" int ds_int8_status(int32_t* err, void* stream) {
  DS_REQUIRE(err != nullptr, DS_EINVAL, "int8_status: null output");
  int* w = err_word();
  DS_REQUIRE(w != nullptr, DS_ECUDA, "int8_status: error word unavailable");
  return ds::take_error_word(w, err, static_cast<cudaStream_t>(stream));
}
