// Pieces of the dense 16-bit feed-forward kernels (gated_ffn.cu): operand
// tiles, tensor maps, descriptors and the gated unit with its derivative.
//
// Every product of the block and of its backward pass is one of
//   D[m, n] = sum_k A[m, k] B[n, k]
// over row-major 16-bit matrices.  An operand is "K-major" where the stored
// rows run along k (x, h, dy; weights in the forward pass) and "MN-major"
// where they run along m or n (weights in the backward pass, everything in a
// weight gradient); the tensor core reads both from 128-byte swizzled tiles,
// so nothing is transposed in memory.
#pragma once

#include "grouped.cuh"
#include "tc5.cuh"

namespace ds {
namespace dense {

using namespace ds::ptx;

constexpr int kBK = 64;                  // contraction per stage: 64 16-bit values = one 128-byte line
constexpr int kBoxBytes = 64 * 128;      // 64 lines of 128 bytes

// Shared-memory descriptor of an MN-major 16-bit tile: boxes of 64 k-lines x
// 64 values (128-byte swizzle); 8-line groups are 1024 bytes apart and the
// next 64 values of m or n follow kBoxBytes later.
__device__ __forceinline__ uint64_t sdesc_mn(uint32_t saddr) {
  uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)(kBoxBytes >> 4) << 16;   // leading offset: next 64 values of m / n
  d |= (uint64_t)64 << 32;                 // stride offset: next 8 k-lines
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// Descriptor of a tile and the 16-byte units that a step of 16 along k adds.
template <bool MN>
__device__ __forceinline__ uint64_t tile_desc(uint32_t saddr) {
  return MN ? sdesc_mn(saddr) : tc5::sdesc_sw128(saddr);
}
template <bool MN>
constexpr uint32_t kStep16 = MN ? (16 * 128) >> 4 : 32 >> 4;

// Instruction descriptor, kind::f16, f32 accumulate, A and B of one type.
__device__ __forceinline__ uint32_t idesc16(int f16, bool a_mn, bool b_mn, int m, int n) {
  const uint32_t ty = f16 ? 0u : 1u;
  return (1u << 4) | (ty << 7) | (ty << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Loads one operand tile of ROWS rows (m or n) x kBK into shared memory.
// k0 and r0 are multiples of 64, so the innermost coordinate stays 16-byte
// aligned whichever way the operand is stored; lines past the matrix read 0.
template <bool MN, int ROWS>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, int r0, int k0, uint64_t* bar) {
  if constexpr (MN) {
#pragma unroll
    for (int b = 0; b < ROWS / 64; ++b) tma_load_2d(dst + b * kBoxBytes, map, r0 + 64 * b, k0, bar);
  } else {
    tma_load_2d(dst, map, k0, r0, bar);
  }
}

// Tensor map of a row-major 16-bit matrix [rows, cols], boxes of 64 columns x
// box_rows rows.  ld (elements) and base must be 16-byte multiples.
inline bool map16(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  return grouped::encode_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, base, rows, cols, ld * 2, 64, box_rows,
                            CU_TENSOR_MAP_SWIZZLE_128B);
}

// The same of an f32 matrix, boxes of 32 x 32 (128-byte lines).
inline bool map32(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld) {
  return grouped::encode_2d(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, base, rows, cols, ld * 4, 32, 32,
                            CU_TENSOR_MAP_SWIZZLE_128B);
}

// A 16-bit matrix in boxes of 32 x 32 (64-byte lines).
inline bool map_slim(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld) {
  return grouped::encode_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, base, rows, cols, ld * 2, 32, 32,
                            CU_TENSOR_MAP_SWIZZLE_64B);
}

// ---------------------------------------------------------------- the gated unit

// h = silu(min(g, L)) * clip(u, -L, L); L = 0: no clamps.  The comparisons
// keep a NaN (fminf would drop it).  The fast exponential's relative error grows
// with |g|, 2^-22 near 0 and below 2^-16 at |g| = 88 (where h is 1e-36), the
// division's is 2^-22: well below the 16-bit rounding that follows.  Both have
// the right limits (0 for large negative g).
__device__ __forceinline__ void gate_clamp(float& g, float& u, float limit) {
  if (limit > 0.0f) {
    g = g > limit ? limit : g;
    u = u > limit ? limit : (u < -limit ? -limit : u);
  }
}

__device__ __forceinline__ float gate_unit(float g, float u, float limit) {
  gate_clamp(g, u, limit);
  return __fdividef(g, 1.0f + __expf(-g)) * u;
}

// Gradients of the unclamped g and u from dh.  With s = sigmoid(g'):
// d silu = s (1 + g' (1 - s)); a clamped value passes no gradient (one that
// equals the limit does, as the derivative from the inside).
__device__ __forceinline__ void gate_grad(float g, float u, float dh, float limit, float& dg, float& du) {
  float gc = g, uc = u;
  gate_clamp(gc, uc, limit);
  const float s = __fdividef(1.0f, 1.0f + __expf(-gc));
  dg = dh * uc * (s * (1.0f + gc * (1.0f - s)));
  du = dh * (gc * s);
  if (limit > 0.0f) {
    dg = g > limit ? 0.0f : dg;
    du = fabsf(u) <= limit ? du : 0.0f;
  }
}

// ---------------------------------------------------------------- values close to the limit
//
// The derivative of a clamp jumps at the limit, so which side of it an exact
// sum lies on decides over a whole gradient.  The tensor core's sum may lie on
// the other side: each step of 16 along the contraction cuts what its partial
// sum holds below f32's last place, and some of the products that it aligns.
// With S = |x_t|_2 |w_i|_2, which bounds the products' magnitudes together, a
// sum that ends near L has partial sums up to (S + L) / 2, and the errors of
// its n steps stay below (n + 1) 2^-23 (S + L): measured are 0.37 of that for
// products of one sign, 0.02 for normal data of 4096 terms.  Values no further
// than that from the limit are added up again in 64 bits by a warp (products
// of 16-bit values are exact in f32) and stored on the side where they belong.
// Only the stored g and u change: h is continuous at the limit.
//
// The tile kernel settles them itself.  The pair kernel lists them for a launch
// of their own: unit variance and a limit of 1.5 leave one value in 640 of 8192
// x 4096 x 2048 (a limit of 10 none), and its few epilogue warps would take 320
// us for what the whole GPU does in 55.  Where the list overflows, that launch
// looks through all stored values instead.

struct Near {
  const uint16_t* x;           // null: no clamps, or nothing is kept
  const uint16_t* w[2];        // W1, W3
  int64_t ldx, ldw[2];         // multiples of 8, bases on 16 bytes
  const float* nx;             // 2-norms of the rows of x, W1 and W3
  const float* nw[2];
  int K, f16;
  float limit, per;            // per: largest error of a sum, in units of S + L
  uint64_t* list;              // pair kernel: i | z << 31 | t << 32 of values to be settled
  unsigned long long* count;   // how many there are, those without room included
  uint32_t room;
};

__device__ __forceinline__ float from16(uint32_t bits, int f16) {
  return f16 ? __half2float(__ushort_as_half((uint16_t)bits)) : __uint_as_float(bits << 16);
}

// The exact sum for row t of x and row i of matrix z, by a warp, up to the
// rounding of 64-bit additions.
__device__ __forceinline__ double near_sum(const Near& p, int z, int64_t t, int64_t i) {
  const uint16_t *a = p.x + t * p.ldx, *b = z ? p.w[1] + i * p.ldw[1] : p.w[0] + i * p.ldw[0];
  const int lane = threadIdx.x & 31;
  double even = 0.0, odd = 0.0;
#pragma unroll 4
  for (int k = lane * 8; k + 8 <= p.K; k += 256) {
    const uint4 va = *reinterpret_cast<const uint4*>(a + k), vb = *reinterpret_cast<const uint4*>(b + k);
    const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      even += (double)(from16(wa[j] & 0xFFFFu, p.f16) * from16(wb[j] & 0xFFFFu, p.f16));
      odd += (double)(from16(wa[j] >> 16, p.f16) * from16(wb[j] >> 16, p.f16));
    }
  }
  const int k = p.K / 8 * 8 + lane;   // an uneven end
  if (k < p.K) even += (double)(from16(a[k], p.f16) * from16(b[k], p.f16));
  even += odd;
#pragma unroll
  for (int o = 16; o; o >>= 1) even += __shfl_xor_sync(0xffffffffu, even, o);
  return even;
}

// A settled value: rounded away from or towards zero, so that it does not
// cross the limit.
__device__ __forceinline__ float near_round(double v, float limit) {
  return fabs(v) <= (double)limit ? __double2float_rz(v) : v > 0 ? __double2float_ru(v) : __double2float_rd(v);
}

// How far from the limit a value is settled; a norm that is no number or
// passes f32 settles nothing (the sums are then no numbers either).
__device__ __forceinline__ float near_band(const Near& p, float nx, float nw) {
  const float b = p.per * (nx * nw + p.limit);
  return b <= 3.0e38f ? b : -1.0f;
}
__device__ __forceinline__ bool near_g(const Near& p, float g, float band) { return fabsf(g - p.limit) <= band; }
__device__ __forceinline__ bool near_u(const Near& p, float u, float band) { return fabsf(fabsf(u) - p.limit) <= band; }

// Settles the values of a warp whose bits are set in `near`, one after the
// other by all lanes.  at(lane, bit): row of x and row of the matrix;
// put(bit, v): the lane that the value belongs to keeps it.
template <typename At, typename Put>
__device__ __forceinline__ void near_settle(const Near& p, int z, uint32_t near, At at, Put put) {
  const int lane = threadIdx.x & 31;
  for (uint32_t any; (any = __ballot_sync(0xffffffffu, near != 0)) != 0;) {
    const int src = __ffs(any) - 1, bit = __ffs(__shfl_sync(0xffffffffu, near, src)) - 1;
    int64_t t, i;
    at(src, bit, t, i);
    const double v = near_sum(p, z, t, i);
    if (lane != src) continue;
    put(bit, near_round(v, p.limit));
    near &= near - 1;
  }
  __syncwarp();
}

// Lists the values of a warp whose bits are set in near[0] and near[1] (lane:
// row t of x, bit: row i0 + bit of the matrix), as far as there is room.
__device__ __forceinline__ void near_list(const Near& p, uint32_t (&near)[2], int64_t t, int i0) {
  const int lane = threadIdx.x & 31, mine = __popc(near[0]) + __popc(near[1]);
  if (!__any_sync(0xffffffffu, mine)) return;
  uint32_t at = mine;                    // this lane's values end at `at`
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, at, o);
    if (lane >= o) at += v;
  }
  unsigned long long to = lane == 31 ? atomicAdd(p.count, (unsigned long long)at) : 0ull;
  to = __shfl_sync(0xffffffffu, to, 31) + at - mine;
#pragma unroll
  for (int z = 0; z < 2; ++z)
    for (; near[z] && to < p.room; near[z] &= near[z] - 1)
      p.list[to++] = (uint64_t)t << 32 | (uint32_t)z << 31 | (uint32_t)(i0 + __ffs(near[z]) - 1);
}

// f32 -> 16-bit (round to nearest even), the low half of the result.
__device__ __forceinline__ uint16_t to16(float v, int f16) {
  return f16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, int f16) {
  if (f16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

}  // namespace dense
}  // namespace ds
