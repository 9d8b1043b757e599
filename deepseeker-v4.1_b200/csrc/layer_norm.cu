// Layer norm over the features of a token, forward and backward.
//
//   mean = sum x / H, var = sum (x - mean)^2 / H, r = 1 / sqrt(var + eps)
//   xh = (x - mean) r,  y = xh w + b
//   g = dy w,  dx = r (g - sum g / H - xh sum(g xh) / H)
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Bounded by memory.  A row stays in the registers of the threads that loaded
// it, so x and dy are read once.  Sums, mean and r are f32.  The variance is
// summed from differences to the mean and xh is off by two roundings of its own
// in both passes, so a mean far from 0 costs no more than its own rounding.
#include <algorithm>
#include <type_traits>

#include "ptx.cuh"
#include "rows.cuh"

namespace ds {
namespace norm {
namespace {

using namespace ds::ptx;
using namespace ds::rows;

// VEC parameters (f32 or the type of x) from column c on as f32.
template <typename P, int VEC>
__device__ __forceinline__ void params(const P* p, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = (float)*p;
  } else {
    constexpr int kPer = 16 / sizeof(P);
#pragma unroll
    for (int h = 0; h < VEC / kPer; ++h) {
      Pack<P, kPer> k;
      k.load_kept(p + h * kPer);
      float f[kPer];
      k.get(f);
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[h * kPer + j] = f[j];
    }
  }
}

// f(vectors of a thread that are whole), see by_end.
template <int VEC, int V, int THREADS, typename F>
__device__ __forceinline__ void by_rows(int cols, F f) {
  if constexpr (THREADS > 0) f(std::integral_constant<int, V>());
  else if constexpr (VEC > 1) f(std::integral_constant<int, 0>());
  else by_end<V>(cols, f);
}

struct Forward {
  const void *x, *w, *b;
  void* y;
  float2* stats;              // mean and r of every row, or null
  int64_t rows, ld;
  int cols;
  float eps;
};

// 1 / sqrt(a), to the last bits by one step of Newton's method.
__device__ __forceinline__ float inverse_root(float a) {
  const float y = rsqrtf(a);
  return fmaf(0.5f * y, fmaf(-a * y, y, 1.0f), y);
}

// A block takes rows blockIdx.x, + gridDim.x ..., blockDim.y at a time, V times
// VEC values a thread; THREADS: of a row, which they fill, or 0.  Up to 16
// values, the parameters of a thread's columns stay in its registers.
//
// 16384 x 4096 bf16: 51 us, 5.2 TB/s (a plain copy of it: 43.5).  Behind memory
// come instructions: a row takes 250 in each warp beside its values (two sums,
// places, the root), so 16 values a thread, 80 registers (three blocks of 256
// threads an SM; with 64 or 96 59 us) and the next row loaded while this one is
// summed.  Measured beside it: no row ahead 72 us, eight values a thread 60, 32
// 54, 64 with the parameters in shared memory 60, rows through a ring in shared
// memory 64.
//
// Rows that do not lie on 16 bytes: single values through lines, 16384 x 4095
// bf16 90 us, 8192 x 4095 f32 51.  Measured beside it: single values in registers
// 119 and 65; vectors that are shifted out of the lines and into others 113 to
// 145 (bf16).
template <typename T, typename P, int VEC, int V, int THREADS>
__global__ void __maxnreg__(VEC == 1 && V <= 8 ? 64 : V * VEC <= 16 ? 80 : 128) forward_kernel(const Forward p) {
  __shared__ float red[kMostRows][2][32];
  const P* w = static_cast<const P*>(p.w);
  const P* b = static_cast<const P*>(p.b);
  // 1 / H in two parts: the mean is the rounded quotient.  With one part it can
  // miss the mean of equal values, and r takes that up to 1 / sqrt(eps) times.
  const float inv = 1.0f / p.cols, rest = fmaf(-inv, (float)p.cols, 1.0f) / p.cols;
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  auto column = [](int i) { return column_of<VEC, V, THREADS>(i); };
  by_rows<VEC, V, THREADS>(p.cols, [&](auto whole) {
    constexpr int kWhole = decltype(whole)::value;
    auto inside = [&](int i) { return i < kWhole || ((VEC > 1 || i < kWhole + 4) && column(i) < p.cols); };
    constexpr bool kKeep = V * VEC <= 16;
    Values<VEC> kw[kKeep ? V : 1], kb[kKeep ? V : 1];
    auto fetch_params = [&](int i, int to) {
      float f[VEC];
      kw[to] = Values<VEC>(1.0f), kb[to] = Values<VEC>(0.0f);
      if (w) params<P, VEC>(w + column(i), f), kw[to] = Values<VEC>(f);
      if (b) params<P, VEC>(b + column(i), f), kb[to] = Values<VEC>(f);
    };
    if constexpr (kKeep) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (inside(i)) fetch_params(i, i);
    }
    constexpr bool kLines = VEC == 1;
    extern __shared__ uint4 smem[];
    Lines<T> lines;
    lines.template place<kStages>(smem, p.x, p.cols);
    [[maybe_unused]] Pack<T, VEC> k[kLines ? 1 : V];
    auto fetch = [&](int stage, int64_t row) {
      const T* x = static_cast<const T*>(p.x) + row * p.ld;
      if constexpr (kLines) {
        if (row < p.rows) lines.copy(stage, x);
        Slots::commit();
      } else {
        if (row >= p.rows) return;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (inside(i)) k[i].load(x + column(i));
      }
    };
    int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    [[maybe_unused]] int stage = 0;
#pragma unroll
    for (int i = 0; i < (kLines ? kStages - 1 : 1); ++i) fetch(i, row + i * step);
    for (; row < p.rows; row += step) {
      Values<VEC> v[V], s(0.0f);
      [[maybe_unused]] const T* here = nullptr;
      if constexpr (kLines) {
        Slots::wait<kStages - 2>();
        line_barrier();   // all of the row is here, and the row before it has been read
        fetch(stage ? stage - 1 : kStages - 1, row + (kStages - 1) * step);
        here = lines.at(stage, static_cast<const T*>(p.x) + row * p.ld);
        stage = stage + 1 == kStages ? 0 : stage + 1;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!inside(i)) continue;
        float f[VEC];
        if constexpr (kLines) f[0] = (float)here[column(i)];
        else k[i].get(f);
        v[i] = Values<VEC>(f);
        s = s + v[i];
      }
      if constexpr (!kLines) fetch(0, row + step);   // on its way during the rest
      const float all = row_sum(total(s), red[threadIdx.y][0]), mean = fmaf(all, inv, all * rest);
      const Values<VEC> less(-mean);
      s = Values<VEC>(0.0f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!inside(i)) continue;
        v[i] = v[i] + less;
        s = fma(v[i], v[i], s);
      }
      const float r = inverse_root(row_sum(total(s), red[threadIdx.y][1]) * inv + p.eps);
      if (p.stats && threadIdx.x == 0) p.stats[row] = make_float2(mean, r);
      T* y = static_cast<T*>(p.y) + row * p.cols;
      const Values<VEC> rs(r);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!inside(i)) continue;
        const int at = kKeep ? i : 0;
        float f[VEC];
        if constexpr (!kKeep) fetch_params(i, 0);
        fma(v[i] * rs, kw[at], kb[at]).get(f);
        put<T, VEC>(y + column(i), f);
      }
    }
  });
}

// Rows that no block's registers hold: read three times, one value a thread.
template <typename T, typename P>
__global__ void __launch_bounds__(1024) forward_long_kernel(const Forward p) {
  __shared__ float red[2][32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ld;
  const P* w = static_cast<const P*>(p.w);
  const P* b = static_cast<const P*>(p.b);
  float s = 0.0f;
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) s += (float)x[c];
  const float mean = row_sum(s, red[0]) / p.cols;
  s = 0.0f;
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
    const float d = (float)x[c] - mean;
    s = fmaf(d, d, s);
  }
  const float r = inverse_root(row_sum(s, red[1]) / p.cols + p.eps);
  if (p.stats && threadIdx.x == 0) p.stats[row] = make_float2(mean, r);
  T* y = static_cast<T*>(p.y) + row * p.cols;
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
    float v = ((float)x[c] - mean) * r;
    if (w) v *= (float)w[c];
    if (b) v += (float)b[c];
    y[c] = narrow<T>(v);
  }
}

struct Backward {
  const void *x, *w, *dy;
  const float2* stats;
  void* dx;                   // or null
  float* part;                // [blocks][2][cols] sums of dy xh and dy, or null
  int64_t rows, ld, ld_dy;
  int cols;
};

// Sums of N values (2 or 4) over the threads of a row, for all of them.  Within
// a warp a lane keeps half of the values at each of the first steps, so that N
// sums take little more than one; red: [warps][N], where a row has several.
template <int N>
__device__ __forceinline__ void row_sums(float (&a)[N], float* red) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  float k[2] = {a[0], a[1]};
  if constexpr (N == 4) {
    const bool high = lane & 16;
    k[0] = (high ? a[2] : a[0]) + __shfl_xor_sync(0xffffffffu, high ? a[0] : a[2], 16);
    k[1] = (high ? a[3] : a[1]) + __shfl_xor_sync(0xffffffffu, high ? a[1] : a[3], 16);
  }
  constexpr int kBit = N == 4 ? 8 : 16;   // lane n * kBit ends up with value n
  const bool high = lane & kBit;
  float v = (high ? k[1] : k[0]) + __shfl_xor_sync(0xffffffffu, high ? k[0] : k[1], kBit);
#pragma unroll
  for (int o = kBit / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  int at = kBit;
  if (warps > 1) {
    if (lane % kBit == 0) red[(threadIdx.x >> 5) * N + lane / kBit] = v;
    asm volatile("bar.sync 1;" ::: "memory");   // warps may come from different calls of by_end
    v = 0.0f;   // lane n + N m: value n of warps m, m + 32 / N ...
    for (int i = lane; i < warps * N; i += 32) v += red[i];
#pragma unroll
    for (int o = N; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    at = 1;
  }
#pragma unroll
  for (int n = 0; n < N; ++n) a[n] = __shfl_sync(0xffffffffu, v, n * at);
}

// How the backward kernel takes its rows, two turns ahead: kRows at a time, in
// vectors through slots, single values through lines.
template <int VEC, int V>
struct Turn {
  static constexpr bool kLines = VEC == 1;
  static constexpr int kRows = !kLines && V <= 2 ? 2 : 1;
  static constexpr int kSlots = kRows * 2 * V;                          // x and dy, of a stage
  static constexpr int kBytes = kLines ? 0 : kStages * kSlots * 16;     // a thread
  static constexpr int kThreads = kLines && V <= 8 ? 1024 : 512;        // that an SM's registers hold
};

// A block takes rows in turns (a warp each, or the block one of each turn); its
// threads keep their columns' sums for the parameters, so x and dy are read
// once for dx, dw and db together.  8192 x 4096 bf16: 37.7 us, 5.3 TB/s, bounded
// like the forward pass.  Measured beside it: one row a turn with the next one in
// registers 47 us, one row a turn through a ring 59, x and dy kept in registers
// from the first use to the second 40 (and 52 once they spilled).  4096 x 8192
// f32, with its join: 72 us; 88 with xh as (x - mean) r.
//
// 8192 x 4095, forward and backward: 127 us bf16 (184 with single values in
// registers), 4096 x 8191 142 (303).
template <typename T, typename P, int VEC, int V, int THREADS>
__global__ void __launch_bounds__(512, Turn<VEC, V>::kThreads / 512) backward_kernel(const Backward p) {
  using U = Turn<VEC, V>;
  constexpr int R = U::kRows, S = kStages;
  extern __shared__ uint4 ring[];
  __shared__ float red[2][16 * 2 * R];
  const P* w = static_cast<const P*>(p.w);
  const float inv = 1.0f / p.cols;
  const Slots slots(ring);
  Lines<T> line_x, line_dy;
  line_x.template place<S>(ring, p.x, p.cols, 0, 2), line_dy.template place<S>(ring, p.dy, p.cols, 1, 2);
  auto column = [](int i) { return column_of<VEC, V, THREADS>(i); };
  by_rows<VEC, V, THREADS>(p.cols, [&](auto whole) {
    constexpr int kWhole = decltype(whole)::value;
    auto inside = [&](int i) { return i < kWhole || ((VEC > 1 || i < kWhole + 4) && column(i) < p.cols); };
    Values<VEC> kw[V], aw[V], ab[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = 1.0f;
      if (w && inside(i)) params<P, VEC>(w + column(i), v);
      kw[i] = Values<VEC>(v);
      aw[i] = ab[i] = Values<VEC>(0.0f);
    }
    const int64_t step = (int64_t)gridDim.x * blockDim.y * R;
    const int64_t first = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * R;
    float2 next[R];   // mean and r of the next rows
    auto fetch = [&](int stage, int64_t row) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (row + r >= p.rows) continue;
        const T* x = static_cast<const T*>(p.x) + (row + r) * p.ld;
        const T* dy = static_cast<const T*>(p.dy) + (row + r) * p.ld_dy;
        if constexpr (U::kLines) {
          line_x.copy(stage, x), line_dy.copy(stage, dy);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            if (!inside(i)) continue;
            const int c = column(i);
            slots.copy(stage * U::kSlots + r * 2 * V + i, x + c);
            slots.copy(stage * U::kSlots + r * 2 * V + V + i, dy + c);
          }
        }
      }
      slots.commit();
    };
    auto stats = [&](int64_t row) {
#pragma unroll
      for (int r = 0; r < R; ++r) next[r] = row + r < p.rows ? p.stats[row + r] : make_float2(0.0f, 0.0f);
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) fetch(i, first + i * step);
    stats(first);
    int stage = 0, turn = 0;
    for (int64_t row = first; row < p.rows; row += step, turn ^= 1) {   // blockDim.y > 1 only with a warp a row
      // xh = (x r + high) + low, high + low = -mean r: the rounding of that product
      // (by one fma, Dekker's TwoProduct) would otherwise be in all of the row's xh,
      // which it exceeds where x is near the mean and the mean far from 0
      float2 st[R];
      float high[R], low[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        st[r] = next[r];
        high[r] = -st[r].x * st[r].y, low[r] = fmaf(-st[r].x, st[r].y, -high[r]);
      }
      const int here = stage;
      slots.wait<S - 2>();
      if constexpr (U::kLines) line_barrier();   // all of the row is here, and the row before it has been used
      // into the stage whose rows the turn before this has used
      fetch(here ? here - 1 : S - 1, row + (S - 1) * step);
      stage = here + 1 == S ? 0 : here + 1;
      stats(row + step);
      const T* here_x = line_x.at(here, static_cast<const T*>(p.x) + row * p.ld);
      const T* here_dy = line_dy.at(here, static_cast<const T*>(p.dy) + row * p.ld_dy);
      // dy and xh - low, from shared memory both times that they are asked for
      // (registers that held them would be missing elsewhere)
      auto at = [&](int r, int i, Values<VEC>& d, Values<VEC>& xh) {
        Pack<T, VEC> kx, kd;
        if constexpr (U::kLines) {
          kx.raw = here_x[column(i)], kd.raw = here_dy[column(i)];
        } else {
          kx.raw = slots.read(here * U::kSlots + r * 2 * V + i);
          kd.raw = slots.read(here * U::kSlots + r * 2 * V + V + i);
        }
        float v[VEC];
        kd.get(v);
        d = Values<VEC>(v);
        kx.get(v);
        xh = fma(Values<VEC>(v), Values<VEC>(st[r].y), Values<VEC>(high[r]));
      };
      float sums[2 * R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        Values<VEC> s1(0.0f), s2(0.0f);
        if (r == 0 || row + r < p.rows) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            if (!inside(i)) continue;
            Values<VEC> d, xh;
            at(r, i, d, xh);
            xh = xh + Values<VEC>(low[r]);
            aw[i] = fma(d, xh, aw[i]);
            ab[i] = ab[i] + d;
            d = d * kw[i];
            s1 = s1 + d;
            s2 = fma(d, xh, s2);
          }
        }
        sums[2 * r] = total(s1), sums[2 * r + 1] = total(s2);
      }
      if (!p.dx) continue;
      row_sums(sums, red[turn]);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r && row + r >= p.rows) continue;
        const float mean_gx = -sums[2 * r + 1] * inv;
        const Values<VEC> m1(fmaf(low[r], mean_gx, -sums[2 * r] * inv)), m2(mean_gx), rs(st[r].y);
        T* dx = static_cast<T*>(p.dx) + (row + r) * p.cols;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (!inside(i)) continue;
          Values<VEC> d, xh;
          at(r, i, d, xh);
          float v[VEC];
          (fma(d, kw[i], fma(xh, m2, m1)) * rs).get(v);
          put<T, VEC>(dx + column(i), v);
        }
      }
    }
    launch_dependents();
    if (!p.part) return;
    float* part = p.part + (int64_t)blockIdx.x * 2 * p.cols;
    if (blockDim.y > 1) {
      // the warps add their sums one after the other, where the ring was
      float* sums = reinterpret_cast<float*>(ring);   // [2][cols]
      __syncthreads();
      for (int y = 0; y < blockDim.y; ++y) {
        if (threadIdx.y == y) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            if (!inside(i)) continue;
            const int c = column(i);
            float vw[VEC], vb[VEC];
            aw[i].get(vw), ab[i].get(vb);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              sums[c + j] = y ? sums[c + j] + vw[j] : vw[j];
              sums[p.cols + c + j] = y ? sums[p.cols + c + j] + vb[j] : vb[j];
            }
          }
        }
        __syncthreads();
      }
      for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < 2 * p.cols; c += blockDim.x * blockDim.y) part[c] = sums[c];
      return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (!inside(i)) continue;
      const int c = column(i);
      float vw[VEC], vb[VEC];
      aw[i].get(vw), ab[i].get(vb);
      if constexpr (VEC == 1) {
        part[c] = vw[0], part[p.cols + c] = vb[0];
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {   // cols is a multiple of VEC, so both halves lie on 16 bytes
          *reinterpret_cast<float4*>(part + c + j) = make_float4(vw[j], vw[j + 1], vw[j + 2], vw[j + 3]);
          *reinterpret_cast<float4*>(part + p.cols + c + j) = make_float4(vb[j], vb[j + 1], vb[j + 2], vb[j + 3]);
        }
      }
    }
  });
}

// Rows that no block's registers hold: dx, x and dy read twice.
template <typename T, typename P>
__global__ void __launch_bounds__(1024) backward_long_kernel(const Backward p) {
  __shared__ float red[2][32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ld;
  const T* dy = static_cast<const T*>(p.dy) + row * p.ld_dy;
  const P* w = static_cast<const P*>(p.w);
  const float2 st = p.stats[row];
  float s1 = 0.0f, s2 = 0.0f;
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
    const float g = (float)dy[c] * (w ? (float)w[c] : 1.0f);
    s1 += g;
    s2 = fmaf(g, ((float)x[c] - st.x) * st.y, s2);
  }
  s1 = row_sum(s1, red[0]) / p.cols;
  s2 = row_sum(s2, red[1]) / p.cols;
  T* dx = static_cast<T*>(p.dx) + row * p.cols;
  for (int c = threadIdx.x; c < p.cols; c += blockDim.x) {
    const float g = (float)dy[c] * (w ? (float)w[c] : 1.0f);
    dx[c] = narrow<T>(st.y * (g - s1 - ((float)x[c] - st.x) * st.y * s2));
  }
}

// Their sums for the parameters: a thread a column, a block every gridDim.y-th row.
template <typename T>
__global__ void __launch_bounds__(256) columns_kernel(const Backward p) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.cols) return;
  const T* x = static_cast<const T*>(p.x) + c;
  const T* dy = static_cast<const T*>(p.dy) + c;
  float aw = 0.0f, ab = 0.0f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float2 st = p.stats[row];
    const float d = (float)dy[row * p.ld_dy];
    aw = fmaf(d, ((float)x[row * p.ld] - st.x) * st.y, aw);
    ab += d;
  }
  float* part = p.part + (int64_t)blockIdx.y * 2 * p.cols;
  part[c] = aw, part[p.cols + c] = ab;
}

// Adds the blocks' sums, 32 neighbouring ones of [2][cols] a block, in an
// order that only their number decides.
template <typename P>
__global__ void __launch_bounds__(512) join_kernel(const float* __restrict__ part, int blocks, int cols, P* dw, P* db) {
  __shared__ float red[16][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane, n = 2 * (int64_t)cols;
  wait_prior_grid();
  float s = 0.0f;
  if (c < n)
    for (int b = warp; b < blocks; b += 16) s += part[b * n + c];
  red[warp][lane] = s;
  __syncthreads();
  if (warp) return;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += red[i][lane];
  if (c >= n) return;
  if (c < cols) {
    if (dw) dw[c] = narrow<P>(s);
  } else if (db) {
    db[c - cols] = narrow<P>(s);
  }
}

// ---------------------------------------------------------------- host side

// Features of rows that registers hold, 16 for each of 512 threads (in vectors
// the forward pass takes eight of them, 64 KB).
constexpr int kMost = 16 * 512;

Shape forward_shape(int cols, int vec) { return shape_of(cols, vec, 16, 512, 128); }

// Single values: a thread takes eight of rows that are two warps' otherwise, so
// that more of them wait at a time (training steps, f16: 333 x 711 12.7 us, with 16
// values 16; 32800 x 1023 156 and 183); longer rows fill an SM with 16, shorter
// ones are a warp's (127583 x 263: 153 us, with eight 387).
Shape backward_shape(int cols, int vec) {
  Shape s = shape_of(cols, vec, vec == 1 && cols > 512 && cols <= 1024 ? 8 : 16, 512, 256);
  if (s.threads > 32) s.rows = 1;
  return s;
}

// f(type of x, type of the parameters)
template <typename F>
void by_types(int dtype, int param_dtype, F f) {
  by_type(dtype, [&](auto t) {
    if (param_dtype == DS_F32) f(t, float());
    else f(t, t);
  });
}

// Blocks of the backward pass, each with its sums.
int backward_blocks(int64_t rows, const Shape& s) {
  const int turn = s.rows * (s.vec > 1 && s.v <= 2 ? 2 : 1);   // Turn::kRows
  const int threads = s.vec == 1 && s.v <= 8 ? 1024 : 512;             // Turn::kThreads
  const int64_t most = (int64_t)ds::sm_count() * std::max(1, threads / (s.threads * s.rows));
  return (int)std::min<int64_t>(most, (rows + turn - 1) / turn);
}

// Row groups of columns_kernel.
int column_blocks(int64_t rows, int cols) {
  const int64_t most = std::max<int64_t>(1, (int64_t)ds::sm_count() * 8 / ((cols + 255) / 256));
  return (int)std::min<int64_t>(most, rows);
}

int backward_parts(int64_t rows, int cols) {
  if (cols > kMost) return column_blocks(rows, cols);
  // whichever way the operands are aligned
  int n = 0;
  for (int vec : {1, 4, 8}) n = std::max(n, backward_blocks(rows, backward_shape(cols, vec)));
  return n;
}

int validate(int dtype, int param_dtype, int64_t rows, int64_t cols, int64_t ld, const char* what) {
  DS_REQUIRE(dtype == DS_F32 || dtype == DS_BF16 || dtype == DS_F16, DS_EINVAL, "%s: x must be f32, bf16 or f16", what);
  DS_REQUIRE(param_dtype == DS_F32 || param_dtype == dtype, DS_EINVAL,
             "%s: weight and bias must be f32 or of x's type", what);
  DS_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && cols >= 1 && cols <= (1 << 20), DS_ERANGE,
             "%s: rows must be in [0, 2^31), cols in [1, 2^20]", what);
  DS_REQUIRE(rows <= 1 || ld >= cols, DS_EINVAL, "%s: row stride of x below its columns", what);
  return DS_OK;
}

}  // namespace
}  // namespace norm
}  // namespace ds

using namespace ds::norm;
using ds::SmemOnce;

extern "C" int ds_layer_norm(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* weight,
                             const void* bias, int param_dtype, float eps, void* y, float* stats, void* stream) {
  int st = validate(dtype, param_dtype, rows, cols, ld, "layer_norm");
  if (st != DS_OK) return st;
  DS_REQUIRE(eps >= 0.0f && eps <= 3.4e38f, DS_EINVAL, "layer_norm: eps must be a number >= 0");
  if (rows == 0) return DS_OK;
  const int es = elements(dtype), ps = elements(param_dtype);
  DS_REQUIRE(x && y, DS_EINVAL, "layer_norm: null pointer");
  DS_REQUIRE(ds::aligned(x, es) && ds::aligned(y, es) && ds::aligned(weight, ps) && ds::aligned(bias, ps) &&
                 ds::aligned(stats, 8),
             DS_EALIGN, "layer_norm: operands must be aligned to their elements, stats to 8 bytes");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Forward p = {x, weight, bias, y, reinterpret_cast<float2*>(stats), rows, ld, (int)cols, eps};
  const bool vec = vectors(x, rows, cols, ld, es) && ds::aligned(y, 16) && ds::aligned(weight, 16) && ds::aligned(bias, 16);
  by_types(dtype, param_dtype, [&](auto t, auto pt) {
    using T = decltype(t);
    using P = decltype(pt);
    if (cols > (vec ? 64 * 1024 / es : kMost)) {
      forward_long_kernel<T, P><<<(unsigned)rows, 1024, 0, s>>>(p);
      return;
    }
    const Shape sh = forward_shape((int)cols, vec ? 16 / es : 1);
    by_shape<T, sizeof(T), 8, false>(sh, (int)cols, vec, [&](auto w, auto v, auto threads) {
      st = launch_rows<forward_kernel<T, P, decltype(w)::value, decltype(v)::value, decltype(threads)::value>>(
          sh, rows, vec ? 0 : kStages * Lines<T>::pitch_of((int)cols), s, p);
    });
  });
  if (st != DS_OK) return st;
  DS_CHECK_LAUNCH("layer_norm forward_kernel");
  return DS_OK;
}

extern "C" int ds_layer_norm_backward_workspace_size(int64_t rows, int64_t cols, size_t* bytes) {
  DS_REQUIRE(bytes && rows >= 0 && rows < ((int64_t)1 << 31) && cols >= 1 && cols <= (1 << 20), DS_EINVAL,
             "layer_norm_backward_workspace_size: rows in [0, 2^31), cols in [1, 2^20] and an output expected");
  *bytes = (size_t)backward_parts(rows, (int)cols) * 2 * cols * sizeof(float);
  return DS_OK;
}

extern "C" int ds_layer_norm_backward(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld,
                                      const void* weight, int param_dtype, const float* stats, const void* dy,
                                      int64_t ld_dy, void* dx, void* dweight, void* dbias, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  int st = validate(dtype, param_dtype, rows, cols, ld, "layer_norm_backward");
  if (st != DS_OK) return st;
  DS_REQUIRE(rows <= 1 || ld_dy >= cols, DS_EINVAL, "layer_norm_backward: row stride of dy below its columns");
  const int es = elements(dtype), ps = elements(param_dtype);
  const bool sums = dweight || dbias;
  DS_REQUIRE(rows == 0 || (x && dy && stats), DS_EINVAL, "layer_norm_backward: null pointer");
  DS_REQUIRE(ds::aligned(x, es) && ds::aligned(dy, es) && ds::aligned(dx, es) && ds::aligned(weight, ps) &&
                 ds::aligned(dweight, ps) && ds::aligned(dbias, ps) && ds::aligned(stats, 8) && ds::aligned(workspace, 256),
             DS_EALIGN, "layer_norm_backward: operands must be aligned to their elements, stats to 8 bytes, the workspace to 256");
  const size_t need = sums ? (size_t)backward_parts(rows, (int)cols) * 2 * cols * sizeof(float) : 0;
  DS_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), DS_EINVAL,
             "layer_norm_backward: workspace %zu bytes < required %zu", workspace_bytes, need);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float* part = sums ? static_cast<float*>(workspace) : nullptr;
  const Backward p = {x, weight, dy, reinterpret_cast<const float2*>(stats), dx, part, rows, ld, ld_dy, (int)cols};
  const bool vec = vectors(x, rows, cols, ld, es) && vectors(dy, rows, cols, ld_dy, es) && ds::aligned(dx, 16) &&
                   ds::aligned(weight, 16);
  int blocks = 0;
  if (rows > 0 && (dx || sums)) {
    by_types(dtype, param_dtype, [&](auto t, auto pt) {
      using T = decltype(t);
      using P = decltype(pt);
      if (cols > kMost) {
        if (dx) backward_long_kernel<T, P><<<(unsigned)rows, 1024, 0, s>>>(p);
        blocks = column_blocks(rows, (int)cols);
        if (sums) columns_kernel<T><<<dim3((unsigned)((cols + 255) / 256), (unsigned)blocks), 256, 0, s>>>(p);
        return;
      }
      const Shape sh = backward_shape((int)cols, vec ? 16 / es : 1);
      const dim3 block(sh.threads, sh.rows);
      blocks = backward_blocks(rows, sh);
      by_shape<T, sizeof(T), sizeof(T), false>(sh, (int)cols, vec, [&](auto w, auto v, auto threads) {
        constexpr int W = decltype(w)::value, V = decltype(v)::value;
        static SmemOnce once;
        const auto kernel = &backward_kernel<T, P, W, V, decltype(threads)::value>;
        const bool lines = Turn<W, V>::kLines;
        const int line = 2 * kStages * Lines<T>::pitch_of((int)cols);
        int smem = lines ? line * sh.rows : Turn<W, V>::kBytes * sh.threads * sh.rows;
        if (sh.rows > 1) smem = std::max(smem, (int)(2 * cols * sizeof(float)));
        if (smem > 40 * 1024 && (st = ds::allow_smem(&once, reinterpret_cast<const void*>(kernel), kMostSmem)) != DS_OK)
          return;
        kernel<<<blocks, block, smem, s>>>(p);
      });
    });
    if (st != DS_OK) return st;
    DS_CHECK_LAUNCH("layer_norm backward_kernel");
  }
  if (sums) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((2 * cols + 31) / 32));
    cfg.blockDim = dim3(512);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = blocks ? 1 : 0;
    cudaError_t e = cudaSuccess;
    by_type(param_dtype, [&](auto pt) {
      using P = decltype(pt);
      e = cudaLaunchKernelEx(&cfg, join_kernel<P>, (const float*)part, blocks, (int)cols, static_cast<P*>(dweight),
                             static_cast<P*>(dbias));
    });
    DS_CHECK_CUDA(e);
  }
  return DS_OK;
}
