// Microscaled 4-bit dense operators: quantisation of activations, the product
// of two quantised matrices and the gated feed-forward block over quantised
// weights.
//
// Product y[n, m] = sum_k x[n, k] W[m, k] on tcgen05 kind::mxf4: packed codes
// straight from memory (two per byte, K-major, 128-byte swizzle), both scale
// sets in tensor memory, f32 accumulate.  Products of two codes and a power
// of two are exact, so the only error is that of the f32 sums.
//
// Tile kernel (up to 64 rows): one CTA computes 128 features (lanes) x NT rows
// of x over a slice of the contraction; the slices of a tile are the CTAs of a
// cluster and are added in slice order through distributed shared memory.  In
// the gated block 32 consecutive lanes are one block of h, so a warp quantises
// it with one maximum over its lanes.  Bounded by start-up: one row of 4096 to
// 4096 takes 5.7 us (8.9 MB, 1.4 us of memory time), the block of 4096 / 2048
// 10.7 us.  More rows: mx4_pair.cuh.
#include <algorithm>
#include <cooperative_groups.h>

#include "mx4_pair.cuh"

namespace ds {
namespace mx4 {
namespace {

namespace cg = cooperative_groups;

__device__ int g_err;   // bit 1: a bounded wait gave up

// ---------------------------------------------------------------- quantisation

// Sixteen values of a row, half a block, as they are stored: 16-bit types two
// a word.
template <typename T>
struct Half {
  static constexpr bool kF32 = sizeof(T) == 4, kF16 = std::is_same<T, __half>::value;
  static constexpr int kWords = kF32 ? 16 : 8;
  uint32_t w[kWords];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  // The first n, a multiple of 8, 16-byte aligned; STREAM: first to leave L2.
  template <bool STREAM = false>
  __device__ __forceinline__ void load(const T* p, int n) {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      if (i * 8 >= n * (kF32 ? 2 : 1)) continue;
      const uint4* at = reinterpret_cast<const uint4*>(p) + i;
      const uint4 a = STREAM ? __ldcs(at) : *at;
      w[4 * i] = a.x, w[4 * i + 1] = a.y, w[4 * i + 2] = a.z, w[4 * i + 3] = a.w;
    }
  }
  // The first n, one by one.
  __device__ __forceinline__ void load_some(const T* p, int n) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (j >= n) continue;
      if constexpr (kF32) w[j] = __float_as_uint(p[j]);
      else w[j >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[j] << (16 * (j & 1));
    }
  }
  // Bits of the block's largest magnitude as f32 (the bits of non-negative
  // values order as the values, infinities and NaN above); the other half is
  // the neighbouring lane's.
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (kF32) {
      uint32_t t = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) t = max(t, w[i] & 0x7FFFFFFFu);
      return max(t, __shfl_xor_sync(0xffffffffu, t, 1));
    } else {
      uint32_t t = w[0] & 0x7FFF7FFFu;
#pragma unroll
      for (int i = 1; i < 8; ++i) t = __vmaxu2(t, w[i] & 0x7FFF7FFFu);
      t = max(t & 0xFFFFu, t >> 16);
      t = max(t, __shfl_xor_sync(0xffffffffu, t, 1));
      return kF16 ? __float_as_uint(__half2float(__ushort_as_half((uint16_t)t))) : t << 16;
    }
  }
  // Codes of values 8 h .. 8 h + 7 times inv, a power of two.
  __device__ __forceinline__ uint32_t codes(int h, float inv) const {
    float v[8];
    if constexpr (kF32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[8 * h + i]) * inv;
    } else if constexpr (kF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[4 * h + i]));
        v[2 * i] = f.x * inv, v[2 * i + 1] = f.y * inv;
      }
    } else {
      // exact in bf16 too, which has f32's exponents; what leaves its normal
      // range rounds to code 0 either way
      const __nv_bfloat162 k = __float2bfloat162_rn(inv);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 m = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[4 * h + i]), k);
        const uint32_t u = *reinterpret_cast<const uint32_t*>(&m);
        v[2 * i] = __uint_as_float(u << 16), v[2 * i + 1] = __uint_as_float(u & 0xFFFF0000u);
      }
    }
    return e2m1x8(v);
  }
};

// How the rows of x lie: half blocks that follow one another through the whole
// matrix, 16-byte aligned ones in rows of any stride, or neither.
enum Rows { WHOLE, ALIGNED, ANY };

// A group is 16 values, two neighbours a block: 32 bytes loaded (64 in f32),
// one maximum over two lanes, 8 bytes stored, so a warp's code stores are
// whole lines.  A thread has its GROUPS loads in flight together.  Behind
// memory (27.5 us for 16384 x 4096 bf16, 6.2 TB/s) come the integer instructions of a
// block's scale and its places: with groups of 8, and a division per group,
// 47 us; with places by the group's number alone 41 us; hence half blocks.
template <typename T, int GROUPS, int ROWS>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, int64_t rows, int cols, int64_t ld,
                                                       uint2* __restrict__ packed, uint8_t* __restrict__ scales,
                                                       uint8_t* __restrict__ atoms) {
  // rows of many megabytes pass through, so that the codes stay in L2 for what
  // reads them next (quantising and dequantising 16384 x 4096: 64 -> 58 us)
  constexpr bool kStream = GROUPS > 1;
  launch_dependents();
  const uint32_t blocks = (cols + 31) / 32, per_row = blocks * 2;
  const int64_t first = (int64_t)blockIdx.x * (256 * GROUPS), row0 = first / per_row;
  const int tid = threadIdx.x, count = (int)min((int64_t)(256 * GROUPS), rows * per_row - first);
  const uint32_t t0 = (uint32_t)(first - row0 * per_row) + tid;
  const uint32_t rs = 256 / per_row, gs = 256 - rs * per_row;   // 256 groups on: rows, and groups of a row
  Half<T> v[GROUPS];
  if (ROWS == WHOLE) {
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
      v[k].clear();
      if (tid + 256 * k < count) v[k].template load<kStream>(x + (first + tid) * 16 + 4096 * k, 16);
    }
  } else {
    int64_t r = row0 + t0 / per_row;
    uint32_t g = t0 % per_row;
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
      v[k].clear();
      const int left = tid + 256 * k < count ? min(cols - (int)g * 16, 16) : 0;
      if (ROWS == ANY) v[k].load_some(x + r * ld + g * 16, left);
      else v[k].template load<kStream>(x + r * ld + g * 16, left);
      r += rs, g += gs;
      if (g >= per_row) g -= per_row, ++r;
    }
  }
  uint32_t s[GROUPS];
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) {
    s[k] = scale_byte(v[k].top());
    const float inv = inv_scale(s[k]);
    uint2 w = make_uint2(v[k].codes(0, inv), v[k].codes(1, inv));
    if (s[k] == 255u) w = make_uint2(0u, 0u);
    if (tid + 256 * k < count) packed[first + tid + 256 * k] = w;
  }
  if (tid & 1) return;
  if (scales) {
#pragma unroll
    for (int k = 0; k < GROUPS; ++k)
      if (tid + 256 * k < count) scales[(first + tid) / 2 + 128 * k] = (uint8_t)s[k];
  }
  if (atoms) {
    const uint32_t chunks = (blocks + 3) / 4;
    int64_t row = row0 + t0 / per_row;
    uint32_t g = t0 % per_row;
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
      if (tid + 256 * k < count) {
        uint8_t* at = atoms + atom_at(row, g >> 1, chunks);
        *at = (uint8_t)s[k];
        if (g == per_row - 2)   // blocks that fill up the last chunk: any scale but NaN
          for (uint32_t e = blocks; e < chunks * 4; ++e) at[e - blocks + 1] = 0;
      }
      row += rs, g += gs;
      if (g >= per_row) g -= per_row, ++row;
    }
  }
}

// The value of a code (its e2m1 pair already f16) times its scale: exact; the
// added 0 turns the second code of zero into +0.
__device__ __forceinline__ float2 values_of(uint32_t h2, float s) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
  return make_float2(fmaf(f.x, s, 0.0f), fmaf(f.y, s, 0.0f));
}

template <bool STREAM>
__device__ __forceinline__ void put(void* dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  if (STREAM) __stcs(static_cast<uint4*>(dst), make_uint4(a, b, c, d));
  else *static_cast<uint4*>(dst) = make_uint4(a, b, c, d);
}

// The values of 8 codes a thread: a 4-byte load, 16 or 32 bytes stored, whole
// lines a warp (rows of the result on 16 bytes, cols a multiple of 8).  Bounded
// by memory: 31 us for 16384 x 4096 bf16, 5.5 TB/s.
template <typename T, int GROUPS>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint32_t* __restrict__ packed,
                                                         const uint8_t* __restrict__ scales, int64_t rows, int cols,
                                                         T* __restrict__ out) {
  constexpr bool kStream = GROUPS > 1;   // many megabytes: first to leave L2
  const uint32_t blocks = (cols + 31) / 32, per_row = blocks * 4;
  const int64_t first = (int64_t)blockIdx.x * (256 * GROUPS), row0 = first / per_row;
  const uint32_t rem = (uint32_t)(first - row0 * per_row) + threadIdx.x;
  uint32_t w[GROUPS], sc[GROUPS];
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) {
    const uint32_t t = rem + 256 * k, r = t / per_row, g = t - r * per_row;
    const int64_t row = row0 + r;
    w[k] = row < rows ? packed[row * per_row + g] : 0u;
    sc[k] = row < rows ? scales[row * blocks + (g >> 2)] : 0u;
  }
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) {
    const uint32_t t = rem + 256 * k, r = t / per_row, g = t - r * per_row;
    const int64_t row = row0 + r;
    if (row >= rows || (int)g * 8 >= cols) continue;
    const float s = ds::u8m0_value(sc[k]);
    uint32_t h[4];
    e2m1x8_to_f16x2(w[k], h);
    float2 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = values_of(h[j], s);
    T* dst = out + row * cols + g * 8;
    if constexpr (sizeof(T) == 4) {
      put<kStream>(dst, __float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
      put<kStream>(dst + 4, __float_as_uint(v[2].x), __float_as_uint(v[2].y), __float_as_uint(v[3].x),
                   __float_as_uint(v[3].y));
    } else {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[j].x, v[j].y);
        o[j] = *reinterpret_cast<const uint32_t*>(&b);
      }
      put<kStream>(dst, o[0], o[1], o[2], o[3]);
    }
  }
}

// Any other result: a byte of codes a thread, so that a warp's single stores
// still fall on neighbouring addresses.
template <typename T>
__global__ void __launch_bounds__(256) dequantize_any_kernel(const uint8_t* __restrict__ packed,
                                                             const uint8_t* __restrict__ scales, int64_t rows, int cols,
                                                             T* __restrict__ out) {
  const uint32_t blocks = (cols + 31) / 32, pairs = (cols + 1) / 2;
  const int64_t first = (int64_t)blockIdx.x * 1024, row0 = first / pairs;
  const uint32_t rem = (uint32_t)(first - row0 * pairs) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t t = rem + 256 * k, r = t / pairs, g = t - r * pairs;
    const int64_t row = row0 + r;
    if (row >= rows) continue;
    const uint32_t code = packed[row * blocks * 16 + g];
    const float s = ds::u8m0_value(scales[row * blocks + (g >> 4)]);
    float lo, hi;
    tc5::e2m1x2_to_f32x2(code, lo, hi);
    T* dst = out + row * cols + g * 2;
    dst[0] = (T)fmaf(lo, s, 0.0f);
    if ((int)g * 2 + 1 < cols) dst[1] = (T)fmaf(hi, s, 0.0f);
  }
}

__global__ void __launch_bounds__(256) scale_atoms_kernel(const uint8_t* __restrict__ scales, int64_t rows, int blocks,
                                                          uint8_t* __restrict__ atoms) {
  const int chunks = (blocks + 3) / 4;
  const int64_t n = rows * chunks;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / chunks;
    const int c = (int)(i - row * chunks);
    uint32_t w = 0;
    for (int b = 0; b < 4; ++b)
      if (c * 4 + b < blocks) w |= (uint32_t)scales[row * blocks + c * 4 + b] << (8 * b);
    *reinterpret_cast<uint32_t*>(atoms + atom_at(row, c * 4, chunks)) = w;
  }
}

// ---------------------------------------------------------------- product

enum Mode { LINEAR, GATED };

struct TileParams {
  CUtensorMap a[2], b;         // weights (gated: W1, W3), rows of x
  const uint8_t* sa[2];        // their scale atoms
  const uint8_t* sb;
  const void* x;               // rows of x that the kernel quantises itself (b and sb unused then)
  int64_t ldx;
  int cols, vec;               // vec: every 16 values start on 16 bytes
  int M, N;                    // features, rows of x
  int blocks;                  // blocks of 32 along the contraction
  void* out;                   // LINEAR: out[n * ldo + m]
  int64_t ldo;
  int out_dtype;
  uint8_t* hq;                 // GATED: codes and atoms of h
  uint8_t* hs;
  float limit;
  int* err;
};

template <int MODE, int NT>
struct TileShape {
  static constexpr int kMats = MODE == GATED ? 2 : 1;
  static constexpr int kOps = kMats * 16384 + NT * 128;              // 256 codes of 128 features and NT rows
  static constexpr int kSf = (kMats + 1) * 2 * kAtom;
  static constexpr int kStage = kOps + (kSf + 1023) / 1024 * 1024;
  // less than half of an SM, so that the next launch's CTAs join this one's and
  // their weights are on their way while it finishes
  static constexpr int kStages = std::min(6, 111 * 1024 / kStage);
  static constexpr int kSmem = 1024 + kStages * kStage;
  static constexpr int kAcc = kMats * NT;
  static constexpr int kSfCols = (kMats + 1) * 8;
  static constexpr int kNeed = kAcc + 2 * kSfCols;
  static constexpr int kCols = kNeed <= 64 ? 64 : kNeed <= 128 ? 128 : kNeed <= 256 ? 256 : 512;
  static_assert(kOps % 1024 == 0 && kStages * kStage >= kMats * NT * 128 * 4, "stages hold the partial tile");
};

constexpr int kTileThreads = 320;   // warp 0 copies, warp 1 MMA, warps 2-9 epilogue (two a lane quarter)

// What becomes of the elements (m, n0 .. n0 + J - 1) of the tile, nv of them
// inside: rows of x n0.., feature m (lane of a full warp).  The columns go
// through each step together: a block's maximum, scale and codes are a chain
// of a few hundred cycles, and one column after the other made the epilogue of
// 64 rows 15 us long.
template <int MODE, int J>
__device__ __forceinline__ void tile_store(const TileParams& p, int m, int n0, int nv, const float (&v0)[J],
                                           const float (&v1)[J]) {
  if constexpr (MODE == LINEAR) {
    if (m >= p.M) return;
    const int64_t at = (int64_t)n0 * p.ldo + m;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (j >= nv) continue;
      if (p.out_dtype == DS_F32) static_cast<float*>(p.out)[at + j * p.ldo] = v0[j];
      else if (p.out_dtype == DS_F16) static_cast<__half*>(p.out)[at + j * p.ldo] = __float2half_rn(v0[j]);
      else static_cast<__nv_bfloat16*>(p.out)[at + j * p.ldo] = __float2bfloat16_rn(v0[j]);
    }
  } else {
    const int lane = threadIdx.x & 31, block = m >> 5, blocks = (p.M + 31) / 32, chunks = (blocks + 3) / 4;
    float h[J];
    int s[J];
    uint32_t w[J];
    // lanes past the features hold products with unset scales: no part of the block
#pragma unroll
    for (int j = 0; j < J; ++j) h[j] = m < p.M ? gate_unit(v0[j], v1[j], p.limit) : 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) s[j] = scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(h[j]) & 0x7FFFFFFFu));
#pragma unroll
    for (int j = 0; j < J; ++j) {
      w[j] = s[j] == 255 ? 0u : tc5::f32x2_to_e2m1x2(h[j] * inv_scale(s[j]), 0.0f) & 0xFu;
      if (w[j] == 8u) w[j] = 0u;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) w[j] |= __shfl_down_sync(0xffffffffu, w[j], 1) << 4;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (j >= nv) continue;
      if (block < blocks && (lane & 1) == 0)
        p.hq[((int64_t)(n0 + j) * blocks + block) * 16 + lane / 2] = (uint8_t)w[j];
      if (lane == 0) p.hs[atom_at(n0 + j, block, chunks)] = (uint8_t)s[j];
    }
  }
}

// Sums this CTA's share of the columns over the partial tiles [mats][NT][128]
// of the cluster, in slice order.  The reads of four columns from all slices
// are in flight together.
template <int MODE, int NT, int SLICES>
__device__ __forceinline__ void tile_join(const TileParams& p, float* part, int slice, int turn, int m, int mi) {
  constexpr int kMats = TileShape<MODE, NT>::kMats;
  cg::cluster_group cluster = cg::this_cluster();
  const float* src[SLICES];
#pragma unroll
  for (int r = 0; r < SLICES; ++r) src[r] = cluster.map_shared_rank(part, r) + mi;
  const int share = (p.N + SLICES - 1) / SLICES, end = min(p.N, (slice + 1) * share);
  for (int n = slice * share + 4 * turn; n < end; n += 8) {
    float w[SLICES][kMats][4];
#pragma unroll
    for (int r = 0; r < SLICES; ++r)
#pragma unroll
      for (int t = 0; t < kMats; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) w[r][t][j] = src[r][(t * NT + min(n + j, end - 1)) * 128];
    float v[2][4] = {};
#pragma unroll
    for (int r = 0; r < SLICES; ++r)
#pragma unroll
      for (int t = 0; t < kMats; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[t][j] += w[r][t][j];
    tile_store<MODE>(p, m, n, end - n, v[0], v[kMats - 1]);
  }
}

// One stage of x (256 columns from c0 on) quantised into the operand tile and
// its two atoms, by the eight warps of the later epilogue: half a block a
// thread, 16 rows.  Rows past x hold anything; their results are not stored.
template <typename X>
__device__ __forceinline__ void quantize_stage(const TileParams& p, uint8_t* tile, uint8_t* atoms, int c0) {
  const int t = threadIdx.x - 64, row = t >> 4, hb = t & 15;
  const int left = row < p.N ? p.cols - (c0 + hb * 16) : 0;
  const X* src = static_cast<const X*>(p.x) + row * p.ldx + c0 + hb * 16;
  Half<X> v;
  v.clear();
  if (p.vec) v.load(src, min(left, 16));
  else v.load_some(src, min(left, 16));
  const int s = scale_byte(v.top());
  const float inv = inv_scale(s);
  uint2 w = make_uint2(v.codes(0, inv), v.codes(1, inv));
  if (s == 255) w = make_uint2(0u, 0u);
  // 128-byte lines, 16-byte pieces swizzled by the line
  *reinterpret_cast<uint2*>(tile + row * 128 + (((hb >> 1) ^ (row & 7)) << 4) + (hb & 1) * 8) = w;
  if ((hb & 1) == 0) atoms[(hb >> 3) * kAtom + grouped::atom_off(row, (hb >> 1) & 3)] = (uint8_t)s;
}

// X: type of the rows of x that the kernel quantises itself (up to 16: every
// CTA its slice of the contraction, in place of a launch before this one), or
// void where x comes as codes.
template <int MODE, int NT, typename X>
__global__ void __launch_bounds__(kTileThreads, 2) tile_kernel(const __grid_constant__ TileParams p) {
  using C = TileShape<MODE, NT>;
  constexpr int S = C::kStages, kMats = C::kMats;
  constexpr bool kRaw = !std::is_void<X>::value;
  static_assert(!kRaw || NT == 16, "quantize_stage fills 16 rows");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ __align__(8) uint64_t full[S], empty[S], accfull;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  cg::cluster_group cluster = cg::this_cluster();
  const int slices = cluster.dim_blocks().x, slice = cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mt = blockIdx.x / slices, m0 = mt * 128;
  const int chunks = (p.blocks + 3) / 4, ksteps = (chunks + 1) / 2;   // a stage is two chunks of 128 codes
  const int it0 = (int)((int64_t)ksteps * slice / slices), it1 = (int)((int64_t)ksteps * (slice + 1) / slices);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], kRaw ? 9 : 1);   // the copies, and eight quantising warps
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
        const int it = it0 + g, na = min(2, chunks - 2 * it);   // atoms of this stage
        uint8_t* st = smem + g % S * C::kStage;
        uint64_t* bar = &full[g % S];
        mbar_arrive_expect_tx(bar, (kRaw ? kMats * 16384 : C::kOps) + (kRaw ? kMats : kMats + 1) * na * kAtom);
#pragma unroll
        for (int t = 0; t < kMats; ++t) {
          tma_load_2d(st + t * 16384, &p.a[t], it * 128, m0, bar);
          bulk_g2s(st + C::kOps + t * 2 * kAtom, p.sa[t] + ((int64_t)mt * chunks + 2 * it) * kAtom, na * kAtom, bar);
        }
      };
      auto rows = [&](int g) {
        if (kRaw) return;
        const int it = it0 + g, na = min(2, chunks - 2 * it);
        uint8_t* st = smem + g % S * C::kStage;
        tma_load_2d(st + kMats * 16384, &p.b, it * 128, 0, &full[g % S]);
        bulk_g2s(st + C::kOps + kMats * 2 * kAtom, p.sb + (int64_t)(2 * it) * kAtom, na * kAtom, &full[g % S]);
      };
      // The weights of the first stages need nothing of the launch before this
      // one in the stream: that is one of the same call, and the call's first
      // launch began after all earlier work had ended.
      const int n = it1 - it0, early = min(S, n);
      for (int g = 0; g < early; ++g) weights(g);
      wait_prior_grid();
      for (int g = 0; g < early; ++g) rows(g);
      int g = early;
      for (; g < n; ++g) {
        if (!ds::pair::wait(&empty[g % S], ((g / S) - 1) & 1, abort, p.err)) break;
        weights(g);
        rows(g);
      }
      // never leave with copies in flight into this CTA's shared memory
      for (int j = g - S < 0 ? 0 : g - S; j < g; ++j) mbar_wait_bounded(&full[j % S], (j / S) & 1, 200000000ull);
    }
  } else if (warp == 1) {
    const uint32_t idesc[2] = {tc5::idesc_mxf4(NT, 0), tc5::idesc_mxf4(NT, 2)};
    const uint64_t ops = tc5::sdesc_sw128(smem_u32(smem));
    for (int g = 0; g < it1 - it0; ++g) {
      const int s = g % S;
      if (!ds::pair::wait_all(&full[s], (g / S) & 1, abort, p.err)) break;
      tc5::fence_after();
      if (elect_one()) {
        const int left = p.blocks - 8 * (it0 + g);     // blocks from this stage on
        const int steps = min(4, (left + 1) / 2);      // MMAs of 64 codes (two blocks)
        const uint32_t sf = smem_u32(smem) + s * C::kStage + C::kOps;
        const uint32_t tsf = tb + C::kAcc + (g & 1) * C::kSfCols;   // [W (, W3), x][two atoms]
        for (int a = 0; a < (steps + 1) / 2; ++a)
#pragma unroll
          for (int t = 0; t <= kMats; ++t) copy_atom(tsf + 4 * (2 * t + a), sf + (2 * t + a) * kAtom);
        const uint64_t ad = ops + (uint64_t)((s * C::kStage) >> 4), bd = ad + ((kMats * 16384) >> 4);
        for (int kk = 0; kk < steps; ++kk)
#pragma unroll
          for (int t = 0; t < kMats; ++t)
            tc5::mma_mxf4(tb + t * NT, ad + t * (16384 >> 4) + 2 * kk, bd + 2 * kk, idesc[kk & 1],
                          tsf + 4 * (2 * t + (kk >> 1)), tsf + 4 * (2 * kMats + (kk >> 1)), (g | kk) != 0);
        tc5::commit(&empty[s]);
      }
      __syncwarp();
    }
    // all issued MMAs complete before the accumulators are read or released
    if (elect_one()) tc5::commit(&accfull);
    __syncwarp();
    ds::pair::wait_all(&accfull, 0, abort, p.err);
  } else {
    if constexpr (kRaw) {
      wait_prior_grid();
      for (int g = 0; g < it1 - it0; ++g) {
        if (g >= S && !ds::pair::wait_all(&empty[g % S], ((g / S) - 1) & 1, abort, p.err)) break;
        uint8_t* st = smem + g % S * C::kStage;
        quantize_stage<X>(p, st + kMats * 16384, st + C::kOps + kMats * 2 * kAtom, (it0 + g) * 256);
        fence_proxy_async_smem();   // the tensor core reads what this thread wrote
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[g % S]);
      }
    }
    ds::pair::wait_all(&accfull, 0, abort, p.err);
  }
  tc5::fence_after();

  // ---- epilogue: thread = one feature (lane of tensor memory)
  wait_prior_grid();
  const int q = warp & 3, turn = (warp - 2) >> 2, mi = q * 32 + lane, m = m0 + mi;
  float* part = reinterpret_cast<float*>(smem);   // [mats][NT][128]
  if (warp >= 2) {
    for (int c0 = 16 * turn; c0 < p.N; c0 += 32) {
      float v[kMats][16];
#pragma unroll
      for (int t = 0; t < kMats; ++t) tc5::ld_x16_nowait(tc5::lane_quarter(tb + t * NT + c0, q), v[t]);
      tc5::wait_ld();
      if (slices > 1) {
#pragma unroll
        for (int t = 0; t < kMats; ++t)
#pragma unroll
          for (int j = 0; j < 16; ++j) part[(t * NT + c0 + j) * 128 + mi] = v[t][j];
      } else {
        tile_store<MODE>(p, m, c0, p.N - c0, v[0], v[kMats - 1]);
      }
    }
  }
  if (slices > 1) {
    cluster.sync();
    if (warp >= 2) {
      if (slices == 8) tile_join<MODE, NT, 8>(p, part, slice, turn, m, mi);
      else if (slices == 4) tile_join<MODE, NT, 4>(p, part, slice, turn, m, mi);
      else tile_join<MODE, NT, 2>(p, part, slice, turn, m, mi);
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

// ---------------------------------------------------------------- host side

int64_t blocks_of(int64_t cols) { return (cols + 31) / 32; }
size_t atoms_bytes(int64_t rows, int64_t cols) {
  return (size_t)((rows + 127) / 128) * ((cols + 127) / 128) * kAtom;
}
size_t packed_bytes(int64_t rows, int64_t cols) { return (size_t)rows * blocks_of(cols) * 16; }

// Codes of a matrix as bytes [rows, 16 blocks]; a box is 128 bytes (256 codes) x box_rows.
bool map_codes(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int box_rows) {
  const int64_t bytes = blocks_of(cols) * 16;
  return grouped::encode_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, rows, bytes, bytes, 128, box_rows,
                            CU_TENSOR_MAP_SWIZZLE_128B);
}

int* err_word() {
  static SymbolOnce known;
  return ds::symbol_address(&known, &g_err);
}

// Groups of `size` values per thread: four, or one where that leaves SMs idle.
template <typename F>
int by_groups(int64_t rows, int64_t cols, int size, F launch) {
  const int64_t groups = rows * blocks_of(cols) * (32 / size);
  const int per = groups >= (int64_t)ds::sm_count() * 2 * 1024 ? 4 : 1;
  const int64_t grid = (groups + 256 * per - 1) / (256 * per);
  DS_REQUIRE(grid < ((int64_t)1 << 31), DS_ERANGE, "mx4: matrix too large");
  if (per == 4) launch(std::integral_constant<int, 4>(), (unsigned)grid);
  else launch(std::integral_constant<int, 1>(), (unsigned)grid);
  return DS_OK;
}

int launch_quantize(const void* x, int dtype, int64_t rows, int cols, int64_t ld, uint8_t* packed, uint8_t* scales,
                    uint8_t* atoms, cudaStream_t s) {
  const int es = dtype == DS_F32 ? 4 : 2;
  const bool vec = ds::aligned(x, 16) && cols % 8 == 0 && (rows == 1 || ld * es % 16 == 0);
  const bool whole = vec && cols % 32 == 0 && (rows == 1 || ld == cols);
  uint2* pk = reinterpret_cast<uint2*>(packed);
  const int st = by_groups(rows, cols, 16, [&](auto per, unsigned grid) {
    constexpr int G = decltype(per)::value;
    auto run = [&](auto* src) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(src)>>;
      if (whole) quantize_kernel<T, G, WHOLE><<<grid, 256, 0, s>>>(src, rows, cols, ld, pk, scales, atoms);
      else if (vec) quantize_kernel<T, G, ALIGNED><<<grid, 256, 0, s>>>(src, rows, cols, ld, pk, scales, atoms);
      else quantize_kernel<T, G, ANY><<<grid, 256, 0, s>>>(src, rows, cols, ld, pk, scales, atoms);
    };
    if (dtype == DS_F32) run(static_cast<const float*>(x));
    else if (dtype == DS_F16) run(static_cast<const __half*>(x));
    else run(static_cast<const __nv_bfloat16*>(x));
  });
  if (st != DS_OK) return st;
  DS_CHECK_LAUNCH("mx4 quantize_kernel");
  return DS_OK;
}

// The tile kernel quantises up to this many rows of x itself.
constexpr int kRawRows = 16;

// Rows of x as a call gives them: values, or codes (DS_U8) with their atoms.
struct Input {
  const void* p;
  const uint8_t* atoms;
  int dtype;
  int64_t rows, ld;
  int cols;
};

template <int MODE, int NT, typename X>
int launch_tiles(const TileParams& p, int slices, cudaStream_t s, bool chained) {
  using C = TileShape<MODE, NT>;
  static SmemOnce once;
  const int st = ds::allow_smem(&once, reinterpret_cast<const void*>(&tile_kernel<MODE, NT, X>), C::kSmem);
  if (st != DS_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.M + 127) / 128 * slices));
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
  DS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, tile_kernel<MODE, NT, X>, p));
  return DS_OK;
}

// The slices of the contraction: enough to give every SM a CTA, at least two
// stages each.
template <int MODE>
int run_tiles(TileParams& p, const Input& x, cudaStream_t s, bool chained) {
  const int64_t tiles = (p.M + 127) / 128;
  const int ksteps = (p.blocks + 7) / 8;
  int slices = 1;
  while (slices < 8 && tiles * slices * 2 <= ds::sm_count() && ksteps / (slices * 2) >= 2) slices *= 2;
  p.N = (int)x.rows;
  if (x.dtype != DS_U8) {
    p.x = x.p, p.ldx = x.ld, p.cols = x.cols;
    p.vec = ds::aligned(x.p, 16) && x.cols % 8 == 0 && (x.rows == 1 || x.ld * (x.dtype == DS_F32 ? 4 : 2) % 16 == 0);
    if (x.dtype == DS_F32) return launch_tiles<MODE, 16, float>(p, slices, s, chained);
    if (x.dtype == DS_F16) return launch_tiles<MODE, 16, __half>(p, slices, s, chained);
    return launch_tiles<MODE, 16, __nv_bfloat16>(p, slices, s, chained);
  }
  // one tile of all rows, so it starts at row 0 of a scale atom
  const int nt = x.rows <= 16 ? 16 : x.rows <= 32 ? 32 : 64;
  DS_REQUIRE(map_codes(&p.b, x.p, x.rows, x.cols, nt), DS_ECUDA, "mx4: tensor map encoding failed");
  p.sb = x.atoms;
  if (nt == 16) return launch_tiles<MODE, 16, void>(p, slices, s, chained);
  if (nt == 32) return launch_tiles<MODE, 32, void>(p, slices, s, chained);
  return launch_tiles<MODE, 64, void>(p, slices, s, chained);
}

// ---- pair kernel

// The pair kernel takes products of at least this many rows of x: at 64 the
// tile kernel is ahead (gated block of 4096 x 2048: 15.9 against 21.9 us, of
// 1024 x 1024 15.1 against 16.9), at 96 behind (25.5 against 22.1, 18.7 against
// 17.1).
constexpr int kPairRows = 65;

// Scale atoms as lines of 512 bytes (128 words); a box is two lines.
bool map_atoms(CUtensorMap* m, const void* base, int64_t rows, int64_t cols) {
  return grouped::encode_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, atoms_bytes(rows, cols) / kAtom, 128, kAtom, 128, 2,
                            CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Result [rows, cols] in boxes of 128 bytes x 32 rows; false where its rows do not start on 16 bytes.
bool map_result(CUtensorMap* m, void* y, int64_t rows, int64_t cols, int dtype) {
  const int es = dtype == DS_F32 ? 4 : 2;
  if (!ds::aligned(y, 16) || cols * es % 16 != 0) return false;
  return grouped::encode_2d(m, dtype == DS_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, y,
                            rows, cols, cols * es, 128 / es, 32, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <bool GATED>
int run_pairs(const PairParams& p, cudaStream_t s, bool chained) {
  constexpr int cols = GATED ? 128 : 256;
  const int64_t tiles = (p.M + 255) / 256 * (int64_t)((p.N + cols - 1) / cols);
  DS_REQUIRE(tiles < ((int64_t)1 << 31), DS_ERANGE, "mx4: too many tiles");
  static SmemOnce once;
  const int st = ds::allow_smem(&once, reinterpret_cast<const void*>(&pairs::pair_kernel<GATED>), pairs::Shape<GATED>::kSmem);
  if (st != DS_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, ds::sm_count() / 2)));
  cfg.blockDim = dim3(pairs::Shape<GATED>::kThreads);
  cfg.dynamicSmemBytes = pairs::Shape<GATED>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = chained ? 1 : 0;
  DS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, pairs::pair_kernel<GATED>, p));
  return DS_OK;
}

// y = x W^T.
int product(const Input& x, const DsMx4& w, void* y, int out_dtype, int* err, cudaStream_t s, bool chained) {
  if (x.rows >= kPairRows) {
    PairParams p = {};
    const bool ok = map_codes(&p.a, x.p, x.rows, w.cols, 128) && map_codes(&p.b[0], w.packed, w.rows, w.cols, 128) &&
                    map_atoms(&p.sa, x.atoms, x.rows, w.cols) && map_atoms(&p.sb[0], w.atoms, w.rows, w.cols);
    DS_REQUIRE(ok, DS_ECUDA, "mx4: tensor map encoding failed");
    p.boxed = map_result(&p.out, y, x.rows, w.rows, out_dtype);
    p.y = y, p.ldy = w.rows, p.out_dtype = out_dtype;
    p.M = (int)x.rows, p.N = (int)w.rows, p.blocks = (int)blocks_of(w.cols), p.err = err;
    return run_pairs<false>(p, s, chained);
  }
  TileParams p = {};
  DS_REQUIRE(map_codes(&p.a[0], w.packed, w.rows, w.cols, 128), DS_ECUDA, "mx4: tensor map encoding failed");
  p.sa[0] = w.atoms;
  p.M = (int)w.rows, p.blocks = (int)blocks_of(w.cols), p.err = err;
  p.out = y, p.ldo = w.rows, p.out_dtype = out_dtype;
  return run_tiles<LINEAR>(p, x, s, chained);
}

// Codes and atoms of h = the gated unit of x W1^T and x W3^T.
int gate_up(const Input& x, const DsMx4& w1, const DsMx4& w3, float limit, uint8_t* hq, uint8_t* hs, int* err,
            cudaStream_t s, bool chained) {
  if (x.rows >= kPairRows) {
    PairParams p = {};
    const bool ok = map_codes(&p.a, x.p, x.rows, w1.cols, 128) && map_codes(&p.b[0], w1.packed, w1.rows, w1.cols, 128) &&
                    map_codes(&p.b[1], w3.packed, w1.rows, w1.cols, 128) && map_atoms(&p.sa, x.atoms, x.rows, w1.cols) &&
                    map_atoms(&p.sb[0], w1.atoms, w1.rows, w1.cols) && map_atoms(&p.sb[1], w3.atoms, w1.rows, w1.cols);
    DS_REQUIRE(ok, DS_ECUDA, "mx4: tensor map encoding failed");
    p.hq = hq, p.hs = hs, p.limit = limit;
    p.M = (int)x.rows, p.N = (int)w1.rows, p.blocks = (int)blocks_of(w1.cols), p.err = err;
    return run_pairs<true>(p, s, chained);
  }
  TileParams p = {};
  const bool ok = map_codes(&p.a[0], w1.packed, w1.rows, w1.cols, 128) &&
                  map_codes(&p.a[1], w3.packed, w1.rows, w1.cols, 128);
  DS_REQUIRE(ok, DS_ECUDA, "mx4: tensor map encoding failed");
  p.sa[0] = w1.atoms, p.sa[1] = w3.atoms;
  p.M = (int)w1.rows, p.blocks = (int)blocks_of(w1.cols), p.err = err;
  p.hq = hq, p.hs = hs, p.limit = limit;
  return run_tiles<GATED>(p, x, s, chained);
}

int validate_weight(const DsMx4* w, const char* what) {
  DS_REQUIRE(w && w->packed && w->atoms, DS_EINVAL, "%s: null weight", what);
  DS_REQUIRE(w->rows >= 1 && w->rows <= (1 << 20) && w->cols >= 1 && w->cols <= (1 << 20), DS_ERANGE,
             "%s: weight rows and cols must be in [1, 2^20]", what);
  DS_REQUIRE(ds::aligned(w->packed, 16) && ds::aligned(w->atoms, 16), DS_EALIGN,
             "%s: weight codes and atoms must be 16-byte aligned", what);
  return DS_OK;
}

int validate_x(const void* x, const uint8_t* atoms, int dtype, int64_t rows, int cols, int64_t ld, const char* what) {
  DS_REQUIRE(dtype == DS_F32 || dtype == DS_BF16 || dtype == DS_F16 || (dtype == DS_U8 && (rows == 0 || atoms)), DS_EINVAL,
             "%s: x must be f32, bf16 or f16, or codes (u8) with atoms", what);
  DS_REQUIRE(rows >= 0 && rows <= (1 << 22), DS_ERANGE, "%s: rows must be in [0, 2^22]", what);
  DS_REQUIRE(rows == 0 || x, DS_EINVAL, "%s: null x", what);
  DS_REQUIRE(dtype == DS_U8 || rows <= 1 || ld >= cols, DS_EINVAL, "%s: row stride of x below its columns", what);
  DS_REQUIRE(ds::aligned(x, dtype == DS_U8 ? 16 : dtype == DS_F32 ? 4 : 2) && ds::aligned(atoms, 16), DS_EALIGN,
             "%s: x must be aligned to its elements, codes and atoms to 16 bytes", what);
  return DS_OK;
}

size_t quantized_bytes(int64_t rows, int64_t cols) {
  return grouped::up(packed_bytes(rows, cols), 256) + grouped::up(atoms_bytes(rows, cols), 256);
}

// Workspace for x given as values.
size_t x_bytes(int64_t rows, int64_t cols) { return rows <= kRawRows ? 0 : quantized_bytes(rows, cols); }

// Codes and atoms of x: as given, left to the tile kernel, or quantised into
// the workspace (then the next launch is chained to this one).
int quantized_x(Input& x, uint8_t*& ws, bool& chained, cudaStream_t s) {
  chained = false;
  if (x.dtype == DS_U8 || x.rows <= kRawRows) return DS_OK;
  uint8_t* sa = ws + grouped::up(packed_bytes(x.rows, x.cols), 256);
  const int st = launch_quantize(x.p, x.dtype, x.rows, x.cols, x.ld, ws, nullptr, sa, s);
  if (st != DS_OK) return st;
  x.p = ws, x.atoms = sa, x.dtype = DS_U8;
  ws += quantized_bytes(x.rows, x.cols);
  chained = true;
  return DS_OK;
}

}  // namespace
}  // namespace mx4
}  // namespace ds

using namespace ds::mx4;

extern "C" int ds_mx4_atoms_size(int64_t rows, int64_t cols, size_t* bytes) {
  DS_REQUIRE(bytes && rows >= 0 && cols >= 1, DS_EINVAL, "mx4_atoms_size: rows >= 0, cols >= 1 and an output expected");
  *bytes = atoms_bytes(rows, cols);
  return DS_OK;
}

extern "C" int ds_mx4_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ld, uint8_t* packed,
                               uint8_t* scales, uint8_t* atoms, void* stream) {
  DS_REQUIRE(x_dtype == DS_F32 || x_dtype == DS_BF16 || x_dtype == DS_F16, DS_EINVAL,
             "mx4_quantize: x must be f32, bf16 or f16");
  DS_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && cols >= 1 && cols <= (1 << 20), DS_ERANGE,
             "mx4_quantize: rows must be in [0, 2^31), cols in [1, 2^20]");
  DS_REQUIRE(rows <= 1 || ld >= cols, DS_EINVAL, "mx4_quantize: row stride below cols");
  if (rows == 0) return DS_OK;
  DS_REQUIRE(x && packed && scales, DS_EINVAL, "mx4_quantize: null pointer");
  DS_REQUIRE(ds::aligned(x, x_dtype == DS_F32 ? 4 : 2) && ds::aligned(packed, 16) && ds::aligned(atoms, 16), DS_EALIGN,
             "mx4_quantize: x must be aligned to its elements, codes and atoms to 16 bytes");
  return launch_quantize(x, x_dtype, rows, (int)cols, ld, packed, scales, atoms, static_cast<cudaStream_t>(stream));
}

extern "C" int ds_mx4_dequantize(const uint8_t* packed, const uint8_t* scales, int64_t rows, int64_t cols, void* out,
                                 int out_dtype, void* stream) {
  DS_REQUIRE(out_dtype == DS_F32 || out_dtype == DS_BF16, DS_EINVAL, "mx4_dequantize: out must be f32 or bf16");
  DS_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && cols >= 1 && cols <= (1 << 20), DS_ERANGE,
             "mx4_dequantize: rows must be in [0, 2^31), cols in [1, 2^20]");
  if (rows == 0) return DS_OK;
  DS_REQUIRE(packed && scales && out, DS_EINVAL, "mx4_dequantize: null pointer");
  DS_REQUIRE(ds::aligned(packed, 16) && ds::aligned(out, out_dtype == DS_F32 ? 4 : 2), DS_EALIGN,
             "mx4_dequantize: codes must be 16-byte aligned, out to its elements");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int C = (int)cols;
  if (ds::aligned(out, 16) && cols % 8 == 0) {
    const uint32_t* pk = reinterpret_cast<const uint32_t*>(packed);
    const int st = by_groups(rows, cols, 8, [&](auto per, unsigned grid) {
      constexpr int G = decltype(per)::value;
      if (out_dtype == DS_F32)
        dequantize_kernel<float, G><<<grid, 256, 0, s>>>(pk, scales, rows, C, static_cast<float*>(out));
      else
        dequantize_kernel<__nv_bfloat16, G><<<grid, 256, 0, s>>>(pk, scales, rows, C, static_cast<__nv_bfloat16*>(out));
    });
    if (st != DS_OK) return st;
  } else {
    const int64_t grid = (rows * ((cols + 1) / 2) + 1023) / 1024;
    DS_REQUIRE(grid < ((int64_t)1 << 31), DS_ERANGE, "mx4_dequantize: matrix too large");
    if (out_dtype == DS_F32)
      dequantize_any_kernel<<<(unsigned)grid, 256, 0, s>>>(packed, scales, rows, C, static_cast<float*>(out));
    else
      dequantize_any_kernel<<<(unsigned)grid, 256, 0, s>>>(packed, scales, rows, C, static_cast<__nv_bfloat16*>(out));
  }
  DS_CHECK_LAUNCH("mx4 dequantize_kernel");
  return DS_OK;
}

extern "C" int ds_mx4_scale_atoms(const uint8_t* scales, int64_t rows, int64_t cols, uint8_t* atoms, void* stream) {
  DS_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && cols >= 1 && cols <= (1 << 20), DS_ERANGE,
             "mx4_scale_atoms: rows must be in [0, 2^31), cols in [1, 2^20]");
  if (rows == 0) return DS_OK;
  DS_REQUIRE(scales && atoms, DS_EINVAL, "mx4_scale_atoms: null pointer");
  DS_REQUIRE(ds::aligned(atoms, 16), DS_EALIGN, "mx4_scale_atoms: atoms must be 16-byte aligned");
  const int64_t n = rows * ((cols + 127) / 128);
  const int grid = (int)std::min<int64_t>((n + 255) / 256, (int64_t)ds::sm_count() * 16);
  scale_atoms_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(scales, rows, (int)blocks_of(cols), atoms);
  DS_CHECK_LAUNCH("mx4 scale_atoms_kernel");
  return DS_OK;
}

extern "C" int ds_mx4_linear_workspace_size(int64_t rows, int64_t cols, size_t* bytes) {
  DS_REQUIRE(bytes && rows >= 0 && cols >= 1, DS_EINVAL,
             "mx4_linear_workspace_size: rows >= 0, cols >= 1 and an output expected");
  *bytes = x_bytes(rows, cols);
  return DS_OK;
}

extern "C" int ds_mx4_linear(const void* x, const uint8_t* x_atoms, int x_dtype, int64_t rows, int64_t ld,
                             const DsMx4* w, void* out, int out_dtype, void* workspace, size_t workspace_bytes,
                             void* stream) {
  int st = validate_weight(w, "mx4_linear");
  if (st != DS_OK) return st;
  if ((st = validate_x(x, x_atoms, x_dtype, rows, (int)w->cols, ld, "mx4_linear")) != DS_OK) return st;
  DS_REQUIRE(out_dtype == DS_F32 || out_dtype == DS_BF16 || out_dtype == DS_F16, DS_EINVAL,
             "mx4_linear: out must be f32, bf16 or f16");
  if (rows == 0) return DS_OK;
  const size_t need = x_dtype == DS_U8 ? 0 : x_bytes(rows, w->cols);
  DS_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), DS_EINVAL,
             "mx4_linear: workspace %zu bytes < required %zu", workspace_bytes, need);
  DS_REQUIRE(out && ds::aligned(out, out_dtype == DS_F32 ? 4 : 2) && ds::aligned(workspace, 256), DS_EALIGN,
             "mx4_linear: out must be aligned to its elements, the workspace to 256 bytes");
  DS_REQUIRE(ds::grouped::encode_fn() != nullptr, DS_ECUDA, "mx4_linear: cuTensorMapEncodeTiled unavailable");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  int* err = err_word();
  DS_REQUIRE(err != nullptr, DS_ECUDA, "mx4_linear: error word unavailable");
  Input in = {x, x_atoms, x_dtype, rows, ld, (int)w->cols};
  bool chained;
  if ((st = quantized_x(in, ws, chained, s)) != DS_OK) return st;
  return product(in, *w, out, out_dtype, err, s, chained);
}

extern "C" int ds_mx4_gated_ffn_workspace_size(int64_t rows, int64_t hidden, int64_t inter, size_t* bytes) {
  DS_REQUIRE(bytes && rows >= 0 && hidden >= 1 && inter >= 1, DS_EINVAL,
             "mx4_gated_ffn_workspace_size: rows >= 0, hidden >= 1, inter >= 1 and an output expected");
  *bytes = x_bytes(rows, hidden) + quantized_bytes(rows, inter);
  return DS_OK;
}

extern "C" int ds_mx4_gated_ffn(const void* x, const uint8_t* x_atoms, int x_dtype, int64_t rows, int64_t ld,
                                const DsMx4* w1, const DsMx4* w3, const DsMx4* w2, float limit, void* out,
                                int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int st;
  for (const DsMx4* w : {w1, w3, w2})
    if ((st = validate_weight(w, "mx4_gated_ffn")) != DS_OK) return st;
  const int64_t H = w1->cols, I = w1->rows;
  DS_REQUIRE(w3->rows == I && w3->cols == H && w2->rows == H && w2->cols == I, DS_EINVAL,
             "mx4_gated_ffn: w1 and w3 [I, H] and w2 [H, I] expected");
  if ((st = validate_x(x, x_atoms, x_dtype, rows, (int)H, ld, "mx4_gated_ffn")) != DS_OK) return st;
  DS_REQUIRE(out_dtype == DS_F32 || out_dtype == DS_BF16 || out_dtype == DS_F16, DS_EINVAL,
             "mx4_gated_ffn: out must be f32, bf16 or f16");
  DS_REQUIRE(limit >= 0.0f, DS_EINVAL, "mx4_gated_ffn: limit must be >= 0 (0: no clamps)");
  if (rows == 0) return DS_OK;
  const size_t need = (x_dtype == DS_U8 ? 0 : x_bytes(rows, H)) + quantized_bytes(rows, I);
  DS_REQUIRE(workspace && workspace_bytes >= need, DS_EINVAL, "mx4_gated_ffn: workspace %zu bytes < required %zu",
             workspace_bytes, need);
  DS_REQUIRE(out && ds::aligned(out, out_dtype == DS_F32 ? 4 : 2) && ds::aligned(workspace, 256), DS_EALIGN,
             "mx4_gated_ffn: out must be aligned to its elements, the workspace to 256 bytes");
  DS_REQUIRE(ds::grouped::encode_fn() != nullptr, DS_ECUDA, "mx4_gated_ffn: cuTensorMapEncodeTiled unavailable");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  int* err = err_word();
  DS_REQUIRE(err != nullptr, DS_ECUDA, "mx4_gated_ffn: error word unavailable");
  Input in = {x, x_atoms, x_dtype, rows, ld, (int)H};
  bool chained;
  if ((st = quantized_x(in, ws, chained, s)) != DS_OK) return st;
  uint8_t* hq = ws;
  uint8_t* hs = ws + ds::grouped::up(packed_bytes(rows, I), 256);
  if ((st = gate_up(in, *w1, *w3, limit, hq, hs, err, s, chained)) != DS_OK) return st;
  const Input h = {hq, hs, DS_U8, rows, 0, (int)I};
  return product(h, *w2, out, out_dtype, err, s, true);
}

extern "C" int ds_mx4_status(int32_t* err, void* stream) {
  DS_REQUIRE(err != nullptr, DS_EINVAL, "mx4_status: null output");
  int* w = err_word();
  DS_REQUIRE(w != nullptr, DS_ECUDA, "mx4_status: error word unavailable");
  return ds::take_error_word(w, err, static_cast<cudaStream_t>(stream));
}
