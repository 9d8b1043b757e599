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
  // Values from the n-th on become 0.
  __device__ __forceinline__ void cut(int n) {
    uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    constexpr int kPer = 4 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (n <= i * kPer) w[i] = 0;
      else if (kPer == 2 && n == i * kPer + 1) w[i] &= 0xFFFFu;
    }
    raw = make_uint4(w[0], w[1], w[2], w[3]);
  }
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

// STREAM: first to leave L2.
template <typename T, int VEC, bool STREAM = false>
__device__ __forceinline__ void put(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *p = narrow<T>(v[0]);
  } else {
    uint32_t w[4];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
    } else {
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
    }
    uint4* at = reinterpret_cast<uint4*>(p);
    const uint4 q = make_uint4(w[0], w[1], w[2], w[3]);
    if constexpr (STREAM) __stcs(at, q);
    else *at = q;
  }
}

// Arithmetic on VEC values, two an instruction where there are two.
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// VEC values, as pairs.
template <int VEC>
struct Values {
  static constexpr int kPairs = VEC / 2;
  uint64_t p[kPairs];
  __device__ __forceinline__ Values() {}
  __device__ __forceinline__ explicit Values(float all) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) p[i] = two(all, all);
  }
  __device__ __forceinline__ explicit Values(const float (&v)[VEC]) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) p[i] = two(v[2 * i], v[2 * i + 1]);
  }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) split(p[i], v[2 * i], v[2 * i + 1]);
  }
};
template <>
struct Values<1> {
  float p;
  __device__ __forceinline__ Values() {}
  __device__ __forceinline__ explicit Values(float v) : p(v) {}
  __device__ __forceinline__ explicit Values(const float (&v)[1]) : p(v[0]) {}
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = p; }
};
template <int VEC>
__device__ __forceinline__ Values<VEC> operator+(const Values<VEC>& a, const Values<VEC>& b) {
  Values<VEC> r;
  if constexpr (VEC == 1) {
    r.p = a.p + b.p;
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) r.p[i] = add2(a.p[i], b.p[i]);
  }
  return r;
}
template <int VEC>
__device__ __forceinline__ Values<VEC> operator*(const Values<VEC>& a, const Values<VEC>& b) {
  Values<VEC> r;
  if constexpr (VEC == 1) {
    r.p = a.p * b.p;
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) r.p[i] = mul2(a.p[i], b.p[i]);
  }
  return r;
}
template <int VEC>
__device__ __forceinline__ Values<VEC> fma(const Values<VEC>& a, const Values<VEC>& b, const Values<VEC>& c) {
  Values<VEC> r;
  if constexpr (VEC == 1) {
    r.p = fmaf(a.p, b.p, c.p);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) r.p[i] = fma2(a.p[i], b.p[i], c.p[i]);
  }
  return r;
}

template <int VEC>
__device__ __forceinline__ float total(const Values<VEC>& a) {
  if constexpr (VEC == 1) {
    return a.p;
  } else {
    uint64_t s = a.p[0];
#pragma unroll
    for (int i = 1; i < VEC / 2; ++i) s = add2(s, a.p[i]);
    float lo, hi;
    split(s, lo, hi);
    return lo + hi;
  }
}

// Slots of 16 bytes in shared memory, [slot][thread], that a thread fills with
// asynchronous copies and reads itself, so it waits for nothing but its own:
// rows on their way while others are in the registers, which alone do not hold
// the 50 KB that an SM needs in flight.
struct Slots {
  uint32_t mine, pitch;
  __device__ __forceinline__ explicit Slots(const void* smem)
      : mine(static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + (threadIdx.y * blockDim.x + threadIdx.x) * 16),
        pitch(blockDim.x * blockDim.y * 16) {}
  __device__ __forceinline__ void copy(int slot, const void* src) const {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mine + slot * pitch), "l"(src) : "memory");
  }
  static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  // All committed copies but those of the last N commits are here.
  template <int N>
  static __device__ __forceinline__ void wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
  }
  __device__ __forceinline__ uint4 read(int slot) const {
    uint4 q;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                 : "r"(mine + slot * pitch)
                 : "memory");
    return q;
  }
};

constexpr int kStages = 3;   // rows, or turns of rows, in a thread's slots

// Rows that begin or end anywhere, in lines of shared memory: byte for byte as
// they lie, wherever that is.  A row's threads copy the granules of 16 bytes that
// hold it, without what lies before the matrix or behind the row: a value on its
// way in a register would take four bytes whatever its size.
template <typename T>
struct Lines {
  // 16 beyond the granules: vector() reads two
  __host__ __device__ static constexpr int pitch_of(int cols) {
    return (cols * (int)sizeof(T) + 31 - (int)sizeof(T)) / 16 * 16 + 16;
  }
  const T* matrix;
  uint8_t* mine;
  int cols, pitch;
  // `which` of `of` matrices, STAGES lines of each for each of the block's rows
  template <int STAGES>
  __device__ __forceinline__ void place(void* smem, const void* matrix, int cols, int which = 0, int of = 1) {
    this->matrix = static_cast<const T*>(matrix), this->cols = cols, pitch = pitch_of(cols);
    mine = static_cast<uint8_t*>(smem) + (threadIdx.y * of + which) * STAGES * pitch;
  }
  static __device__ __forceinline__ int skip(const T* row) { return (int)(reinterpret_cast<uintptr_t>(row) & 15); }
  __device__ __forceinline__ void copy(int stage, const T* row) const {
    const int bytes = skip(row) + cols * (int)sizeof(T);
    const uint8_t* src = reinterpret_cast<const uint8_t*>(row) - skip(row);
    uint8_t* dst = mine + stage * pitch;
    for (int o = threadIdx.x * 16; o < bytes; o += blockDim.x * 16) {
      const int n = min(16, bytes - o);
      if (src + o < reinterpret_cast<const uint8_t*>(matrix)) {   // o = 0
        for (int b = skip(row); b < n; b += (int)sizeof(T))
          *reinterpret_cast<T*>(dst + b) = *reinterpret_cast<const T*>(src + b);
      } else {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         static_cast<uint32_t>(__cvta_generic_to_shared(dst + o))),
                     "l"(src + o), "r"(n)
                     : "memory");
      }
    }
  }
  // The row, value for value.
  __device__ __forceinline__ const T* at(int stage, const T* row) const {
    return reinterpret_cast<const T*>(mine + stage * pitch + skip(row));
  }
  // 16 bytes of it, whose first value is c, a multiple of a vector's: parts of two granules.
  __device__ __forceinline__ uint4 vector(int stage, const T* row, int c) const {
    const int off = skip(row), bits = (off & 3) * 8;
    const uint8_t* p = mine + stage * pitch + c * (int)sizeof(T);
    const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 16);
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint4 r;
    auto from = [&](auto words) {   // the same in all of a row's threads, so a branch
      constexpr int n = decltype(words)::value;
      r.x = __funnelshift_r(w[n], w[n + 1], bits);
      r.y = __funnelshift_r(w[n + 1], w[n + 2], bits);
      r.z = __funnelshift_r(w[n + 2], w[n + 3], bits);
      r.w = __funnelshift_r(w[n + 3], w[n + 4], bits);
    };
    if (off < 8) {
      if (off < 4) from(std::integral_constant<int, 0>());
      else from(std::integral_constant<int, 1>());
    } else if (off < 12) {
      from(std::integral_constant<int, 2>());
    } else {
      from(std::integral_constant<int, 3>());
    }
    return r;
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The warps of a row (threadIdx.y of several in a block) meet; a row of one
// warp needs none of this.
__device__ __forceinline__ void row_barrier() {
  asm volatile("bar.sync %0, %1;" ::"r"(threadIdx.y + 1), "r"(blockDim.x) : "memory");
}

// The same where a row may have one warp.
__device__ __forceinline__ void line_barrier() {
  if (blockDim.x == 32) __syncwarp();
  else row_barrier();
}

// Sum over the threads of a row, the same value, bit for bit, in every thread.
// red: 32 words of the row's.
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = warp_sum(v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  const int lane = threadIdx.x & 31;
  if (lane == 0) red[threadIdx.x >> 5] = v;
  row_barrier();
  return warp_sum(lane < warps ? red[lane] : 0.0f);
}

constexpr int kMostRows = 8;   // of a block

// First column of vector i of a thread's V.  Vectors: a row's threads side by
// side.  Single values: a warp's side by side, V times, so that their places are
// a constant apart.
template <int VEC, int V, int THREADS>
__device__ __forceinline__ int column_of(int i) {
  if constexpr (VEC == 1) return ((threadIdx.x >> 5) * V + i) * 32 + (threadIdx.x & 31);
  else return (i * (THREADS ? THREADS : blockDim.x) + threadIdx.x) * VEC;
}

// f(how many of a warp's V times 32 single values lie in the row: all of these,
// some of the next four, none of the rest), as a constant.  A warp that has the
// row's end would otherwise ask for each value and hold up the others (rows of
// 4064 values in place of 4096: a quarter of the time).
template <int V, int WHOLE = V, typename F>
__device__ __forceinline__ void by_end(int cols, F f) {
  if constexpr (WHOLE <= 0) f(std::integral_constant<int, 0>());
  else if (((int)(threadIdx.x >> 5) * V + WHOLE) * 32 <= cols) f(std::integral_constant<int, WHOLE>());
  else by_end<V, WHOLE - 4>(cols, f);
}

// ---------------------------------------------------------------- host side

// How a row is shared out: V vectors of VEC values for each of `threads`
// threads, `rows` rows a block.
struct Shape {
  int vec, v, threads, rows;
};

// A thread takes up to `per` values before a row gets more than a warp, and
// more only where `most_threads` threads do not hold the row; rows share a block
// of up to block_threads.
inline Shape shape_of(int cols, int vec, int per, int most_threads, int block_threads) {
  Shape s;
  s.vec = vec;
  const int n = (cols + vec - 1) / vec;
  s.v = 1;
  while (s.v * vec < per && s.v * 32 < n) s.v *= 2;
  while (s.v * most_threads < n) s.v *= 2;
  s.threads = ((n + s.v - 1) / s.v + 31) / 32 * 32;
  s.rows = std::max(1, std::min(kMostRows, block_threads / s.threads));
  return s;
}

template <typename F>
void by_type(int dtype, F f) {
  if (dtype == DS_F32) f(float());
  else if (dtype == DS_F16) f(__half());
  else f(__nv_bfloat16());
}

// f(values per vector, vectors per thread, threads of a row) with constants: up
// to MOST vectors of 16 bytes or 16 single values, or with LINES, -1 threads and
// vectors for rows that do not lie on 16 bytes.  Rows that FILLED vectors a
// thread fill get their number of threads as a constant, others 0: offsets that
// are constants and no checks of columns are worth a sixth of a pass over rows
// of 4096.
template <typename T, int FILLED, int MOST, bool LINES, typename F>
void by_shape(const Shape& s, int cols, bool vectors, F f) {
  using std::integral_constant;
  const integral_constant<int, 16 / (int)sizeof(T)> vec;
  const integral_constant<int, 1> one;
  const integral_constant<int, 0> any;
  auto by_v = [&](auto threads) {
    if (s.v == 1) f(vec, one, threads);
    else if (s.v == 2) f(vec, integral_constant<int, 2>(), threads);
    else if (s.v == 4) f(vec, integral_constant<int, std::min(4, MOST)>(), threads);
    else f(vec, integral_constant<int, std::min(8, MOST)>(), threads);
  };
  if constexpr (LINES) {
    if (!vectors) {
      by_v(integral_constant<int, -1>());
      return;
    }
  } else if (!vectors) {
    if (s.v == 1) f(one, one, any);
    else if (s.v == 2) f(one, integral_constant<int, 2>(), any);
    else if (s.v == 4) f(one, integral_constant<int, 4>(), any);
    else if (s.v == 8) f(one, integral_constant<int, 8>(), any);
    else f(one, integral_constant<int, 16>(), any);
    return;
  }
  if (s.v == FILLED && s.vec * s.v * s.threads == cols && s.threads <= 512) {
    const integral_constant<int, FILLED> v;
    if (s.threads == 32) f(vec, v, integral_constant<int, 32>());
    else if (s.threads == 64) f(vec, v, integral_constant<int, 64>());
    else if (s.threads == 128) f(vec, v, integral_constant<int, 128>());
    else if (s.threads == 160) f(vec, v, integral_constant<int, 160>());
    else if (s.threads == 256) f(vec, v, integral_constant<int, 256>());
    else if (s.threads == 320) f(vec, v, integral_constant<int, 320>());
    else if (s.threads == 512) f(vec, v, integral_constant<int, 512>());
    else f(vec, v, any);
  } else {
    by_v(any);
  }
}

constexpr int kMostSmem = 220 * 1024;   // dynamic, of a block

// Blocks of `kernel` that an SM holds, asked for once per size.
struct Residency {
  unsigned char known[33];   // by warps
};
inline int resident(Residency* r, const void* kernel, int threads, size_t smem) {
  unsigned char* at = &r->known[threads / 32];
  if (const int n = __atomic_load_n(at, __ATOMIC_RELAXED)) return n;
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    return 1;
  }
  __atomic_store_n(at, (unsigned char)n, __ATOMIC_RELAXED);
  return n;
}

// Launches KERNEL, which takes rows blockIdx.x, + gridDim.x ..., on as many
// blocks as are resident at a time; smem: bytes for each of a block's rows.
template <auto KERNEL, typename... A>
int launch_rows(const Shape& sh, int64_t rows, int smem, cudaStream_t s, const A&... args) {
  static Residency known;
  static SmemOnce once;
  const void* kernel = reinterpret_cast<const void*>(KERNEL);
  smem *= sh.rows;
  if (smem > 40 * 1024) {
    const int st = ds::allow_smem(&once, kernel, kMostSmem);
    if (st != DS_OK) return st;
  }
  const int most = std::min(resident(&known, kernel, sh.threads * sh.rows, 0), 227 * 1024 / (smem + 4 * 1024));
  const int64_t blocks = std::min<int64_t>((rows + sh.rows - 1) / sh.rows, (int64_t)ds::sm_count() * std::max(1, most));
  KERNEL<<<(unsigned)blocks, dim3(sh.threads, sh.rows), smem, s>>>(args...);
  return DS_OK;
}

inline bool vectors(const void* p, int64_t rows, int64_t cols, int64_t ld, int es) {
  return ds::aligned(p, 16) && cols * es % 16 == 0 && (rows <= 1 || ld * es % 16 == 0);
}

inline int elements(int dtype) { return dtype == DS_F32 ? 4 : 2; }

}  // namespace rows
}  // namespace ds
