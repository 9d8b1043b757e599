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
// keep a NaN (fminf would drop it).  The fast exponential and division are
// good to about 2^-20, far below the 16-bit rounding that follows; both have
// the right limits (0 for g towards -infinity).
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
