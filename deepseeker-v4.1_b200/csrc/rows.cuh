// Kernels over the rows of a matrix whose rows stay in registers: vectors as
// they are stored, sums over a row's threads, and how a row is shared out.
#pragma once

#include <algorithm>
#include <type_traits>

#include "ds_common.cuh"

namespace ds {
namespace rows {

// VEC neighbouring values as they are stored: 16 bytes, or one value.
template <typename T, int VEC>
struct Pack {
  static_assert(VEC == 1 || VEC * sizeof(T) == 16, "16 bytes or one value");
  using Raw = std::conditional_t<VEC == 1, T, uint4>;
  Raw raw;
  __device__ __forceinline__ void load(const T* p) { raw = __ldcs(reinterpret_cast<const Raw*>(p)); }
  __device__ __forceinline__ void load_kept(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
    if constexpr (VEC == 1) {
      v[0] = (float)raw;
    } else if constexpr (sizeof(T) == 4) {
      v[0] = __uint_as_float(raw.x), v[1] = __uint_as_float(raw.y);
      v[2] = __uint_as_float(raw.z), v[3] = __uint_as_float(raw.w);
    } else {
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 f;
        if constexpr (std::is_same<T, __half>::value) f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        else f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ T narrow(float v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

template <typename T, int VEC>
__device__ __forceinline__ void put(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *p = narrow<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the threads of a row: a warp (any number of them in a block), or
// the whole block, which then meets once.  The same value, bit for bit, in
// every thread.
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = warp_sum(v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  const int lane = threadIdx.x & 31;
  if (lane == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < warps ? red[lane] : 0.0f);
}

// ---------------------------------------------------------------- host side

// How a row is shared out: V vectors of VEC values for each of `threads`
// threads, `rows` rows a block.
struct Shape {
  int vec, v, threads, rows;
};

// Values per thread: up to `per`, so that 32 threads and more share a row;
// beyond 1024 (backward: 512) threads more.
inline Shape shape_of(int cols, int vec, int per, int most_threads) {
  Shape s;
  s.vec = vec;
  const int n = (cols + vec - 1) / vec;
  s.v = 1;
  while (s.v * vec < per && s.v * 32 < n) s.v *= 2;
  s.threads = 32;
  while (s.threads < most_threads && s.threads * s.v < n) s.threads *= 2;
  while (s.threads * s.v < n) s.v *= 2;
  // the last doubling may have left whole warps idle
  s.threads = ((n + s.v - 1) / s.v + 31) / 32 * 32;
  s.rows = s.threads == 32 ? 8 : 1;
  return s;
}

template <typename F>
void by_type(int dtype, F f) {
  if (dtype == DS_F32) f(float());
  else if (dtype == DS_F16) f(__half());
  else f(__nv_bfloat16());
}

// f(values per vector, vectors per thread)
template <typename T, int MOST, typename F>
void by_shape(const Shape& s, F f) {
  constexpr int kVec = 16 / sizeof(T);
  auto go = [&](auto vec) {
    constexpr int W = decltype(vec)::value;
    if (s.v == 1) f(vec, std::integral_constant<int, 1>());
    else if (s.v == 2) f(vec, std::integral_constant<int, 2>());
    else if (s.v == 4) f(vec, std::integral_constant<int, std::min(4, MOST / W)>());
    else if (s.v == 8) f(vec, std::integral_constant<int, std::min(8, MOST / W)>());
    else if (s.v == 16) f(vec, std::integral_constant<int, std::min(16, MOST / W)>());
    else f(vec, std::integral_constant<int, std::min(32, MOST / W)>());
  };
  if (s.vec == 1) go(std::integral_constant<int, 1>());
  else go(std::integral_constant<int, kVec>());
}

inline bool vectors(const void* p, int64_t rows, int64_t cols, int64_t ld, int es) {
  return ds::aligned(p, 16) && cols * es % 16 == 0 && (rows <= 1 || ld * es % 16 == 0);
}

inline int elements(int dtype) { return dtype == DS_F32 ? 4 : 2; }

}  // namespace rows
}  // namespace ds
