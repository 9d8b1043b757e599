// Microscaled 4-bit format shared by the dense kernels in mx4.cu: scale rule,
// rounding, the tensor-core scale atoms and the copy of an atom into tensor
// memory.
//
// A row of K values is ceil(K / 32) blocks.  A block keeps 32 e2m1 codes (16
// bytes, low nibble first, zeros behind an uneven end) and one ue8m0 scale
// 2^(s - 127), s the smallest that brings the block's largest magnitude to 6
// or less (127 for a block of zeros).  A block that holds a NaN or an infinity
// gets s = 255, the format's NaN, so the value is not lost.
#pragma once

#include "grouped.cuh"
#include "tc5.cuh"

namespace ds {
namespace mx4 {

using namespace ds::ptx;

constexpr int kAtom = grouped::kSfAtom;   // scales of 128 rows x 4 blocks

// Scale byte from the bits of the block's largest magnitude.
__device__ __forceinline__ int scale_byte(uint32_t top) {
  // adding the mantissa bits above 1.5 carries into the exponent: ef - 2 or ef - 1
  const int s = max((int)((top + 0x3FFFFFu) >> 23) - 2, 0);
  return top >= 0x7F800000u ? 255 : top == 0u ? 127 : s;
}

// 2^(127 - s), s <= 253; 0 for the NaN scale (the codes are then all 0).
__device__ __forceinline__ float inv_scale(int s) { return s == 255 ? 0.0f : __uint_as_float((uint32_t)(254 - s) << 23); }

// Clears the sign of codes that rounded to 0: one code stands for 0.
__device__ __forceinline__ uint32_t no_negative_zero(uint32_t w) {
  const uint32_t nz = (w | (w >> 1) | (w >> 2)) & 0x11111111u;
  return w & (0x77777777u | (nz << 3));
}

// Eight scaled values to codes, the first in the lowest bits: to nearest, ties
// to the even code, at most 6 in magnitude.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t w;
  asm("{ .reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3}; }"
      : "=r"(w)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return no_negative_zero(w);
}

// Byte of (row, block) in a matrix's atoms [ceil(rows / 128)][chunks][512],
// chunks = ceil(blocks / 4).
__device__ __forceinline__ int64_t atom_at(int64_t row, int block, int chunks) {
  return ((row >> 7) * chunks + (block >> 2)) * kAtom + grouped::atom_off((int)(row & 127), block & 3);
}

// One atom from shared memory into four tensor-memory columns, replicated to
// the four lane quarters.  Ordered before the MMAs that this thread issues next.
__device__ __forceinline__ void copy_atom(uint32_t taddr, uint32_t saddr) {
  uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)8 << 32;   // 128 bytes between groups of 8 rows x 16 bytes
  d |= (uint64_t)1 << 46;   // no swizzle
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

// The gated unit (ds_gated_ffn's), from f32 sums: the clamps keep a NaN; the
// fast exponential's error grows with |g| (2^-22 near 0, below 2^-16 at 88), and
// what follows rounds to three bits.
__device__ __forceinline__ float gate_unit(float g, float u, float limit) {
  if (limit > 0.0f) {
    g = g > limit ? limit : g;
    u = u > limit ? limit : (u < -limit ? -limit : u);
  }
  return __fdividef(g, 1.0f + __expf(-g)) * u;
}

}  // namespace mx4
}  // namespace ds
