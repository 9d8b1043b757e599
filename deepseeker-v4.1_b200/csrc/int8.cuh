// Pieces of the 8-bit integer operators: the code of a value, the MMA and the
// scaled result.
//
// A row of K values is K codes q in -127 .. 127 (stored ones may be -128) and
// one f32 scale s = max |x| / 127, rounded to f32; q is the whole number
// nearest to the exact quotient x / s, the even one of two.
#pragma once

#include "grouped.cuh"
#include "pair.cuh"
#include "rows.cuh"
#include "tc5.cuh"

namespace ds {
namespace int8 {

using namespace ds::ptx;

// Codes are stored in rows whose distance is a multiple of this (and of no
// more: the tensor maps know where a row ends).
constexpr int kPitch = 16;

// The scale of a row whose largest magnitude has these bits: NaN for a NaN or
// an infinity, which stand above all numbers.
__device__ __forceinline__ float scale_of(uint32_t top) {
  return top >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float(top) / 127.0f;
}

// Code of x in the low byte of the result, by the scale s >= 2^-126 and inv =
// 1 / s.  x inv is off by a few parts in 2^24, so its rounding n (in the low
// bits of a sum with 1.5 * 2^23) is wrong by one at most, next to the middle
// of two codes; x - n s is exact (both are multiples of half the last place of
// s, and |x| <= 127.5 s), so comparing twice of it with s settles the code.
__device__ __forceinline__ uint32_t code_of(float x, float s, float inv) {
  constexpr float kMagic = 12582912.0f;
  const float r = fmaf(x, inv, kMagic);
  const float d = fmaf(-(r - kMagic), s, x), t = 2.0f * fabsf(d);
  uint32_t q = __float_as_uint(r);
  if (t > s || (t == s && (q & 1u))) q += d > 0.0f ? 1u : 0xFFFFFFFFu;
  return q & 0xFFu;
}

// The same for smaller scales, whose inverse may leave f32: the quotient in 64
// bits, which shows a tie only where there is one.  A scale of 0 has codes 0,
// and so has one that is no number.
__device__ __noinline__ uint32_t code_of_small(float x, float s) {
  if (!(s > 0.0f)) return 0u;
  const double q = rint((double)x / (double)s);
  return (uint32_t)(int)fmin(fmax(q, -127.0), 127.0) & 0xFFu;
}

// Instruction descriptor, kind::i8: s8 operands, s32 accumulators.
__device__ __forceinline__ constexpr uint32_t idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// D (+)= A * B, both s8 (K-major, 128-byte swizzle), K = 32.
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}
// The same by a pair of CTAs.
__device__ __forceinline__ void mma2(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(accumulate)
      : "memory");
}

// sum * a * b in f32: the smaller scale first, so that no step leaves f32
// where the result does not.  (Comparisons, as fminf would drop a NaN.)
__device__ __forceinline__ float scaled(int sum, float a, float b) {
  const bool less = a < b;
  return (float)sum * (less ? a : b) * (less ? b : a);
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool f16) {
  if (f16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

}  // namespace int8
}  // namespace ds
