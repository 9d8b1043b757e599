// Layer norm over the features of a token, forward and backward.
//
//   mean = sum x / H, var = sum (x - mean)^2 / H, r = 1 / sqrt(var + eps)
//   xh = (x - mean) r,  y = xh w + b
//   g = dy w,  dx = r (g - sum g / H - xh sum(g xh) / H)
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Bounded by memory.  A row stays in the registers of the threads that loaded
// it, so x and dy are read once.  Sums, mean and r are f32; the variance is
// summed from differences to the mean, so a mean far from 0 costs nothing.
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

struct Forward {
  const void *x, *w, *b;
  void* y;
  float2* stats;              // mean and r of every row, or null
  int64_t rows, ld;
  int cols;
  float eps;
};

// One row per blockDim.x threads, V times VEC values each.
template <typename T, typename P, int VEC, int V>
__global__ void __launch_bounds__(1024) forward_kernel(const Forward p) {
  __shared__ float red[2][32];
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;   // whole rows: a warp, or the block
  const T* x = static_cast<const T*>(p.x) + row * p.ld;
  const P* w = static_cast<const P*>(p.w);
  const P* b = static_cast<const P*>(p.b);
  float v[V][VEC];
  {
    Pack<T, VEC> k[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * VEC;
      if (c < p.cols) k[i].load(x + c);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * VEC;
      if (c < p.cols) {
        k[i].get(v[i]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = 0.0f;
      }
    }
  }
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) s += v[i][j];
  const float mean = row_sum(s, red[0]) / p.cols;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * VEC;
    if (c >= p.cols) continue;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      v[i][j] -= mean;
      s = fmaf(v[i][j], v[i][j], s);
    }
  }
  const float r = 1.0f / sqrtf(row_sum(s, red[1]) / p.cols + p.eps);
  if (p.stats && threadIdx.x == 0) p.stats[row] = make_float2(mean, r);
  T* y = static_cast<T*>(p.y) + row * p.cols;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * VEC;
    if (c >= p.cols) continue;
    float k[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[i][j] *= r;
    if (w) {
      params<P, VEC>(w + c, k);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] *= k[j];
    }
    if (b) {
      params<P, VEC>(b + c, k);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] += k[j];
    }
    put<T, VEC>(y + c, v[i]);
  }
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
  const float r = 1.0f / sqrtf(row_sum(s, red[1]) / p.cols + p.eps);
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

// A block takes rows blockIdx.x, + gridDim.x ... (a warp each, or the block
// one); its threads keep their columns' sums for the parameters, so x and dy
// are read once for dx, dw and db together.  The next row is on its way while
// this one is summed.
template <typename T, typename P, int VEC, int V>
__global__ void __launch_bounds__(512) backward_kernel(const Backward p) {
  extern __shared__ float sums[];   // blockDim.y > 1: [2][cols] of a warp
  __shared__ float2 red[2][32];
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  const P* w = static_cast<const P*>(p.w);
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const float inv = 1.0f / p.cols;
  float kw[V][VEC], aw[V][VEC], ab[V][VEC];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) aw[i][j] = ab[i][j] = 0.0f, kw[i][j] = 1.0f;
    if (w && c < p.cols) params<P, VEC>(w + c, kw[i]);
  }
  Pack<T, VEC> nx[V], nd[V];
  float2 nst = make_float2(0.0f, 0.0f);
  auto fetch = [&](int64_t row) {
    nst = p.stats[row];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * VEC;
      if (c >= p.cols) continue;
      nx[i].load(x + row * p.ld + c);
      nd[i].load(dy + row * p.ld_dy + c);
    }
  };
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row < p.rows) fetch(row);
  for (int turn = 0; row < p.rows; row += step, turn ^= 1) {   // blockDim.y > 1 only with a warp a row
    const float2 st = nst;
    float xh[V][VEC], g[V][VEC];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * VEC;
      if (c < p.cols) {
        nx[i].get(xh[i]);
        nd[i].get(g[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          xh[i][j] = (xh[i][j] - st.x) * st.y;
          aw[i][j] = fmaf(g[i][j], xh[i][j], aw[i][j]);
          ab[i][j] += g[i][j];
          g[i][j] *= kw[i][j];
          s1 += g[i][j];
          s2 = fmaf(g[i][j], xh[i][j], s2);
        }
      }
    }
    if (row + step < p.rows) fetch(row + step);
    if (!p.dx) continue;
    s1 = warp_sum(s1), s2 = warp_sum(s2);
    if (warps > 1) {
      if (lane == 0) red[turn][threadIdx.x >> 5] = make_float2(s1, s2);
      __syncthreads();
      const float2 o = lane < warps ? red[turn][lane] : make_float2(0.0f, 0.0f);
      s1 = warp_sum(o.x), s2 = warp_sum(o.y);
    }
    s1 *= inv, s2 *= inv;
    T* dx = static_cast<T*>(p.dx) + row * p.cols;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * VEC;
      if (c >= p.cols) continue;
#pragma unroll
      for (int j = 0; j < VEC; ++j) g[i][j] = st.y * (g[i][j] - s1 - xh[i][j] * s2);
      put<T, VEC>(dx + c, g[i]);
    }
  }
  launch_dependents();
  if (!p.part) return;
  float* part = p.part + (int64_t)blockIdx.x * 2 * p.cols;
  if (blockDim.y > 1) {
    // the warps add their sums one after the other
    for (int y = 0; y < blockDim.y; ++y) {
      if (threadIdx.y == y) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int c = (i * blockDim.x + threadIdx.x) * VEC;
          if (c >= p.cols) continue;
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            sums[c + j] = y ? sums[c + j] + aw[i][j] : aw[i][j];
            sums[p.cols + c + j] = y ? sums[p.cols + c + j] + ab[i][j] : ab[i][j];
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
    const int c = (i * blockDim.x + threadIdx.x) * VEC;
    if (c >= p.cols) continue;
    if constexpr (VEC == 1) {
      part[c] = aw[i][0], part[p.cols + c] = ab[i][0];
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {   // cols is a multiple of VEC, so both halves lie on 16 bytes
        *reinterpret_cast<float4*>(part + c + j) = make_float4(aw[i][j], aw[i][j + 1], aw[i][j + 2], aw[i][j + 3]);
        *reinterpret_cast<float4*>(part + p.cols + c + j) = make_float4(ab[i][j], ab[i][j + 1], ab[i][j + 2], ab[i][j + 3]);
      }
    }
  }
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

constexpr int kMostForward = 32 * 1024, kMostBackward = 16 * 512;

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
  const int64_t most = (int64_t)ds::sm_count() * std::max(1, 1024 / (s.threads * s.rows));
  return (int)std::min<int64_t>(most, (rows + s.rows - 1) / s.rows);
}

// Row groups of columns_kernel.
int column_blocks(int64_t rows, int cols) {
  const int64_t most = std::max<int64_t>(1, (int64_t)ds::sm_count() * 8 / ((cols + 255) / 256));
  return (int)std::min<int64_t>(most, rows);
}

int backward_parts(int64_t rows, int cols) {
  if (cols > kMostBackward) return column_blocks(rows, cols);
  // whichever way the operands are aligned
  int n = 0;
  for (int vec : {1, 4, 8}) n = std::max(n, backward_blocks(rows, shape_of(cols, vec, 16, 512)));
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

extern "C" int ds_layer_norm(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* weight,
                             const void* bias, int param_dtype, float eps, void* y, float* stats, void* stream) {
  int st = validate(dtype, param_dtype, rows, cols, ld, "layer_norm");
  if (st != DS_OK) return st;
  DS_REQUIRE(eps >= 0.0f, DS_EINVAL, "layer_norm: eps must be >= 0");
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
    if (cols > kMostForward) {
      forward_long_kernel<T, P><<<(unsigned)rows, 1024, 0, s>>>(p);
      return;
    }
    const Shape sh = shape_of((int)cols, vec ? 16 / es : 1, 16, 1024);
    const dim3 block(sh.threads, sh.rows);
    const unsigned grid = (unsigned)((rows + sh.rows - 1) / sh.rows);
    by_shape<T, 32>(sh, [&](auto w, auto v) {
      forward_kernel<T, P, decltype(w)::value, decltype(v)::value><<<grid, block, 0, s>>>(p);
    });
  });
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
      if (cols > kMostBackward) {
        if (dx) backward_long_kernel<T, P><<<(unsigned)rows, 1024, 0, s>>>(p);
        blocks = column_blocks(rows, (int)cols);
        if (sums) columns_kernel<T><<<dim3((unsigned)((cols + 255) / 256), (unsigned)blocks), 256, 0, s>>>(p);
        return;
      }
      const Shape sh = shape_of((int)cols, vec ? 16 / es : 1, 16, 512);
      const dim3 block(sh.threads, sh.rows);
      blocks = backward_blocks(rows, sh);
      const size_t smem = sh.rows > 1 ? 2 * cols * sizeof(float) : 0;
      by_shape<T, 16>(sh, [&](auto w, auto v) {
        backward_kernel<T, P, decltype(w)::value, decltype(v)::value><<<blocks, block, smem, s>>>(p);
      });
    });
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
