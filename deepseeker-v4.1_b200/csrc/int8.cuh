// Pieces of the 8-bit integer operators: the code of a value, the MMA and the
// scaled result.
//
// A row of K values is K codes q in -127 .. 127 (stored ones may be -128) and
// one f32 scale s = max |x| * (1 / 127), both factors and the product in f32 (a
// unit of its last place from the quotient at most); q is the whole number
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
  return top >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float(top) * (1.0f / 127.0f);
}

// A row's scale as codes are formed with it.  Small ones (their inverse may
// leave f32) and the values go through a factor of 2^64, which is exact; a row
// whose scale is 0 or no number has codes 0.
struct Coder {
  float s, inv;
  bool small, none;

  __device__ __forceinline__ explicit Coder(float scale) : s(scale) {
    small = !(scale >= 7.8886091e-31f);   // 2^-100
    none = !(scale > 0.0f);
    if (small) s = none ? 1.0f : scale * 18446744073709551616.0f;
    inv = 1.0f / s;
  }
  // Codes of v, in the low bytes of q.  x inv is off by a few parts in 2^24, so
  // its rounding n (in the low bits of a sum with 1.5 * 2^23) is wrong by one at
  // most, next to the middle of two codes; x - n s is exact (both are multiples
  // of half the last place of s, and |x| <= 127.5 s), so comparing twice of it
  // with s settles the code, where any of them asks for it.
  template <int VEC>
  __device__ __forceinline__ void codes(float (&v)[VEC], uint32_t (&q)[VEC]) const {
    using rows::Values;
    constexpr float kMagic = 12582912.0f;
    if (small) {
      // a scale without its low bits may leave more than 127 of it
      const float most = 127.0f * s;
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = none ? 0.0f : fminf(fmaxf(v[j] * 18446744073709551616.0f, -most), most);
    }
    const Values<VEC> x(v), r = fma(x, Values<VEC>(inv), Values<VEC>(kMagic));
    float d[VEC], n[VEC], far = 0.0f;
    fma(r + Values<VEC>(-kMagic), Values<VEC>(-s), x).get(d);
    r.get(n);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      q[j] = __float_as_uint(n[j]);
      far = fmaxf(far, fabsf(d[j]));
    }
    if (2.0f * far < s) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float t = 2.0f * fabsf(d[j]);
      if (t > s || (t == s && (q[j] & 1u))) q[j] += d[j] > 0.0f ? 1u : 0xFFFFFFFFu;
    }
  }
};

// The low bytes of four codes as a word.
__device__ __forceinline__ uint32_t pack_codes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
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

// sum * a * b in f32: the scale nearer to 0 first (stored ones may be negative),
// so that no step leaves f32 where the result does not.  (Comparisons, as fminf
// would drop a NaN.)
__device__ __forceinline__ float scaled(int sum, float a, float b) {
  const bool less = fabsf(a) < fabsf(b);
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
