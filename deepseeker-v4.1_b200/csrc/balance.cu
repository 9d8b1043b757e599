// Balance loss of a router with its counts per expert, and its gradient.
//
// For a sequence of n valid tokens, k experts each, E experts in all:
//   c_e = times e was chosen, f_e = c_e E / (k n), P_e = sum_t p_te / n,
//   loss = sum_e f_e P_e,
// p_te = a_te / Z_t, Z_t = sum_e a_te, with a = exp(l - max l) or
// a = sqrt(softplus(l)).  With C_e = f_e / n (kept for the backward pass) and
// an upstream gradient g:
//   loss = sum_e C_e sum_t p_te,
//   dl_te = g (C_e - sum_e p_te C_e) / Z_t * da/dl,  da/dl = a (softmax; the
//   shift by the maximum cancels) or sigmoid(l) / (2 a).
//
// Bounded by memory: logits are read once forward, and once and written once
// backward.  A row lies in the registers of G lanes; the lanes' sums over
// rows are p's sums per expert.  Every sum has an order of its own that only
// sizes and offsets decide; counts are whole numbers.
//
// 65536 x 384 f32, sqrt-softplus: forward 38 us, backward 48 (2.6 and 4.2 TB/s).
// Neither memory (35 % busy) nor issue slots (62 and 72 % used) are full: a warp
// waits for its own arithmetic, one step of a score after the other, and an SM's 25
// warps do not cover all of that.  16384 x 256, softmax: 8.4 and 7.8 us, which are
// the starts and ends of launches.
#include <algorithm>
#include <cooperative_groups.h>
#include <type_traits>

#include "ds_common.cuh"
#include "ptx.cuh"
#include "route.cuh"
#include "rows.cuh"

namespace ds {
namespace balance {
namespace {

namespace cg = cooperative_groups;
using namespace ds::ptx;
using ds::rows::add2;
using ds::rows::fma2;
using ds::rows::mul2;
using ds::rows::split;
using ds::rows::two;

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct Params {
  const void* logits;
  int64_t tokens, ld;
  int experts, top_k;
  const int32_t* ids;
  const uint8_t* valid;        // or null: all are
  const void* offsets;         // [sequences + 1], or null: one sequence of all rows
  int wide;                    // offsets are int64
  int64_t sequences;
  int64_t rows_per_block;
  int lanes;                   // G: lanes of a row, a power of two
  // forward: records of (block, sequence), [2][experts] words and the valid rows
  uint32_t* records;
  float* loss;
  int32_t* counts;
  float* coef;                 // C
  int single;                  // one block and one sequence: no records
  // backward
  const float* dloss;
  void* dlogits;
};

// Row where sequence s begins (s = sequences: the last one's end), kept inside the matrix.
__device__ __forceinline__ int64_t offset_at(const Params& p, int64_t s) {
  if (!p.offsets) return s ? p.tokens : 0;
  const int64_t o = p.wide ? static_cast<const int64_t*>(p.offsets)[s] : static_cast<const int32_t*>(p.offsets)[s];
  return o < 0 ? 0 : o > p.tokens ? p.tokens : o;
}

// The last sequence that begins at or before `row`, or -1.
__device__ __forceinline__ int64_t sequence_of(const Params& p, int64_t row) {
  int64_t lo = -1, hi = p.sequences;   // offset(lo) <= row < offset(hi), as far as offsets ascend
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (offset_at(p, mid) <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int64_t record_words(const Params& p) { return 2 * (int64_t)p.experts + 1; }

// VEC neighbouring logits.
template <typename T, int VEC>
struct Pack {
  using Raw = std::conditional_t<VEC == 1, T, std::conditional_t<sizeof(T) == 4, uint4, uint2>>;
  Raw raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void get(float* v) const {
    if constexpr (VEC == 1) {
      v[0] = (float)raw;
    } else if constexpr (sizeof(T) == 4) {
      v[0] = __uint_as_float(raw.x), v[1] = __uint_as_float(raw.y);
      v[2] = __uint_as_float(raw.z), v[3] = __uint_as_float(raw.w);
    } else {
      const uint32_t w[2] = {raw.x, raw.y};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          v[2 * i] = f.x, v[2 * i + 1] = f.y;
        } else {
          v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
      }
    }
  }
};

template <typename T, int VEC>
__device__ __forceinline__ void put(T* p, const float* v) {
  if constexpr (std::is_same<T, float>::value) {
    if constexpr (VEC == 1) *p = v[0];
    else *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    T t[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if constexpr (std::is_same<T, __half>::value) t[i] = __float2half_rn(v[i]);
      else t[i] = __float2bfloat16_rn(v[i]);
    }
    if constexpr (VEC == 1) {
      *p = t[0];
    } else {
      uint2 w;
      memcpy(&w, t, 8);
      *reinterpret_cast<uint2*>(p) = w;
    }
  }
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// 2^x, sqrt(x), 1 / sqrt(x) and 1 / x of the special function unit, off by four
// units in the last place of f32 or less (results below 2^-126 become 0).
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_sqrt(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_rsqrt(float x) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_inverse(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// exp of both x (numbers, no infinities) as 2^t (1 + r): t is x log2 e in f32, a
// number as good as any near it, and r = x - t log 2 what it leaves of x, within
// 4e-6 where 2^t is not 0, so that exp(r) is 1 + r (Cody and Waite's reduction with
// t in the whole number's place).  2^t alone is off by the roundings of t and log2 e
// too, 58 units in the last place 60 below 0; this by 2^t's four, one of the
// product, and |t| / 30 for log 2 in f32.  A training step of 65536 x 384 takes 91
// us with it, 86 without.
__device__ __forceinline__ void exp_of(uint64_t x, float& a, float& b) {
  constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
  const uint64_t t = mul2(x, two(kLog2e, kLog2e));
  split(t, a, b);
  const uint64_t e = two(fast_exp2(a), fast_exp2(b));
  split(fma2(e, fma2(t, two(-kLn2, -kLn2), x), e), a, b);
}

// The larger of both, NaN where one is.
__device__ __forceinline__ float larger(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// log(1 + t) / t on [0, 1]: the polynomial of degree 8 with the least largest
// relative error (a fit in 64 bits: 3e-8; 3 units of f32 with its roundings).
__device__ __forceinline__ uint64_t log1p_ratio2(uint64_t t) {
  constexpr float k[9] = {0.9999999403953552f, -0.4999949336051941f, 0.3331909477710724f, -0.2484297752380371f,
                          0.1910598874092102f, -0.1366320699453354f, 0.07822549343109131f, -0.029504956677556038f,
                          0.005232623778283596f};
  uint64_t r = two(k[8], k[8]);
#pragma unroll
  for (int i = 7; i >= 0; --i) r = fma2(r, t, two(k[i], k[i]));
  return r;
}

// A row's logits -> a (in place), its slope da / dl where asked for.  Columns
// past the row hold -infinity, which gives a = 0 and slope 0 (exponents end at
// -200, far below where 2^t is 0, so that they stay numbers).  sqrt(softplus) takes
// 16 instructions and two of the special function unit a value, 20 and three with
// its slope (expf, log1pf, sqrtf and divisions: 50 to 70, and the passes over 65536
// x 384 three times as long as their memory).
template <bool SOFTMAX, bool SLOPE, int N>
__device__ __forceinline__ void scores(float (&v)[N], float (&slope)[SLOPE && !SOFTMAX ? N : 1], int lanes) {
  static_assert(N % 2 == 0, "pairs");
  constexpr float kLeast = -200.0f;
  if constexpr (SOFTMAX) {
    float m = v[0];
#pragma unroll
    for (int j = 1; j < N; ++j) m = fmaxf(m, v[j]);
    for (int o = 1; o < lanes; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (m == -INFINITY) m = 0.0f;   // no expert is left: every a is 0
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      float x, y;
      split(add2(two(v[j], v[j + 1]), two(-m, -m)), x, y);
      exp_of(two(larger(x, kLeast), larger(y, kLeast)), v[j], v[j + 1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      float h[2], s[2], t[2];
      // exp(-|l| / 2); what is no number stays none in the maximum below
      const uint64_t least = two(fmaxf(-fabsf(v[j]), 2.0f * kLeast), fmaxf(-fabsf(v[j + 1]), 2.0f * kLeast));
      exp_of(mul2(least, two(0.5f, 0.5f)), h[0], h[1]);
      const uint64_t h2 = two(h[0], h[1]), t2 = mul2(h2, h2);
      // softplus(l) = max(l, 0) + log(1 + exp(-|l|))
      split(fma2(t2, log1p_ratio2(t2), two(larger(v[j], 0.0f), larger(v[j + 1], 0.0f))), s[0], s[1]);
      split(t2, t[0], t[1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float l = v[j + i];
        const bool low = l < -17.0f;   // softplus(l) is exp(l) in f32, and its root stays above 0 for longer
        if constexpr (SLOPE) {
          const float root = fast_rsqrt(s[i]);
          v[j + i] = low ? h[i] : s[i] * root;
          slope[j + i] = low ? 0.5f * h[i] : (l >= 0.0f ? 0.5f : 0.5f * t[i]) * root * fast_inverse(1.0f + t[i]);
        } else {
          v[j + i] = low ? h[i] : fast_sqrt(s[i]);
        }
      }
    }
  }
}

// Calls visit(sequence or -1, first row, end) for the parts of rows begin .. end - 1,
// in order; ROWS_OUTSIDE: those of no sequence too.
template <bool OUTSIDE, typename F>
__device__ __forceinline__ void segments(const Params& p, int64_t begin, int64_t end, F visit) {
  int64_t row = begin;
  for (int64_t s = max(sequence_of(p, begin), (int64_t)0); s < p.sequences && row < end; ++s) {
    const int64_t from = max(row, min(offset_at(p, s), end)), to = min(offset_at(p, s + 1), end);
    if (OUTSIDE && from > row) visit((int64_t)-1, row, from);
    if (to > from) visit(s, from, to);
    row = max(from, to);
  }
  if (OUTSIDE && row < end) visit((int64_t)-1, row, end);
}

// Column of value j of lane l.
template <int VEC>
__device__ __forceinline__ int column(int j, int l, int lanes) {
  return (j / VEC * lanes + l) * VEC + j % VEC;
}

template <typename T, int VEC, int NV>
__device__ __forceinline__ void fetch(Pack<T, VEC> (&k)[NV], const T* row, int l, int lanes, int experts) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * lanes + l) * VEC;
    if (c < experts) k[i].load(row + c);
  }
}

template <typename T, int VEC, int NV>
__device__ __forceinline__ void unpack(const Pack<T, VEC> (&k)[NV], float (&v)[NV * VEC], int l, int lanes, int experts,
                                       bool live) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (live && (i * lanes + l) * VEC < experts) {
      k[i].get(&v[i * VEC]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i * VEC + j] = -INFINITY;
    }
  }
}

// E / (k n^2) of a sequence of n valid tokens, 0 without any.
__device__ __forceinline__ double factor_of(const Params& p, int n) {
  return n ? (double)p.experts / ((double)p.top_k * n * n) : 0.0;
}

// Stores count and coefficient of expert e; its part of the loss.
__device__ __forceinline__ double finish(const Params& p, int64_t s, int e, float sum, int count, double factor) {
  const double c = count * factor;
  p.counts[s * p.experts + e] = count;
  p.coef[s * p.experts + e] = (float)c;
  return c * sum;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Blocks of an SM, by the registers that a lane's values ask for.
__host__ __device__ constexpr int blocks_of(int vec, int nv) {
  const int n = vec == 1 ? 2 * nv : vec * nv;   // single values need their places too
  return n <= 12 ? 4 : n <= 16 ? 3 : n <= 32 ? 2 : 1;
}

template <typename T, bool SOFTMAX, int VEC, int NV>
__global__ void __launch_bounds__(kThreads, blocks_of(VEC, NV)) forward_kernel(const Params p) {
  constexpr int N = NV * VEC;
  extern __shared__ uint8_t smem[];
  float* sums = reinterpret_cast<float*>(smem);                       // [kWarps][experts]
  int* hist = reinterpret_cast<int*>(sums + kWarps * p.experts);      // [experts]
  __shared__ int valid_rows;
  __shared__ double losses[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = p.lanes, l = lane & (G - 1);
  const int per_pass = kThreads / G, slot = threadIdx.x / G;
  const T* logits = static_cast<const T*>(p.logits);
  const int64_t begin = blockIdx.x * p.rows_per_block, end = min(begin + p.rows_per_block, p.tokens);
  launch_dependents();
  segments<false>(p, begin, end, [&](int64_t s, int64_t from, int64_t to) {
    for (int e = threadIdx.x; e < p.experts; e += kThreads) hist[e] = 0;
    if (threadIdx.x == 0) valid_rows = 0;
    __syncthreads();
    uint64_t acc[N / 2] = {};
    int n = 0;
    Pack<T, VEC> next[NV];
    bool ok = false;
    auto ask = [&](int64_t row) {
      ok = row < to && (!p.valid || p.valid[row]);
      if (ok) fetch<T, VEC, NV>(next, logits + row * p.ld, l, G, p.experts);
    };
    ask(from + slot);
    // the chosen experts, while the first rows are on their way
    const int chosen = (int)((to - from) * p.top_k);
    const int32_t* ids = p.ids + from * p.top_k;
#pragma unroll 4
    for (int i = threadIdx.x; i < chosen; i += kThreads) {
      const int id = ids[i];
      if ((unsigned)id < (unsigned)p.experts && (!p.valid || p.valid[from + i / p.top_k])) atomicAdd(&hist[id], 1);
    }
    for (int64_t first = from; first < to; first += per_pass) {
      const int64_t row = first + slot;
      const bool live = ok;
      float v[N], none[1];
      unpack<T, VEC, NV>(next, v, l, G, p.experts, live);
      ask(row + per_pass);
      n += live && l == 0;
      scores<SOFTMAX, false, N>(v, none, G);
      uint64_t z2 = 0;
#pragma unroll
      for (int j = 0; j < N; j += 2) z2 = add2(z2, two(v[j], v[j + 1]));
      float z, y;
      split(z2, z, y);
      z = group_sum(z + y, G);
      const float inv = z == 0.0f ? 0.0f : 1.0f / z;   // a row without scores has no shares
#pragma unroll
      for (int j = 0; j < N; j += 2) acc[j / 2] = fma2(two(v[j], v[j + 1]), two(inv, inv), acc[j / 2]);
    }
    float part[N];
#pragma unroll
    for (int j = 0; j < N; j += 2) split(acc[j / 2], part[j], part[j + 1]);
    // lanes of the same column, then the warps
#pragma unroll
    for (int j = 0; j < N; ++j)
      for (int o = G; o < 32; o <<= 1) part[j] += __shfl_xor_sync(0xffffffffu, part[j], o);
    if (lane < G) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = column<VEC>(j, l, G);
        if (c < p.experts) sums[warp * p.experts + c] = part[j];
      }
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0 && n) atomicAdd(&valid_rows, n);
    __syncthreads();
    uint32_t* rec = p.records + (blockIdx.x + s) * record_words(p);
    const double factor = p.single ? factor_of(p, valid_rows) : 0.0;
    double loss = 0.0;
    for (int e = threadIdx.x; e < p.experts; e += kThreads) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) t += sums[w * p.experts + e];
      if (p.single) {
        loss += finish(p, 0, e, t, hist[e], factor);
      } else {
        rec[e] = __float_as_uint(t);
        rec[p.experts + e] = (uint32_t)hist[e];
      }
    }
    if (p.single) {
      loss = warp_sum(loss);
      if (lane == 0) losses[warp] = loss;
    } else if (threadIdx.x == 0) {
      rec[2 * p.experts] = (uint32_t)valid_rows;
    }
    __syncthreads();
    if (p.single && threadIdx.x == 0) {
      double t = 0.0;
      for (int w = 0; w < kWarps; ++w) t += losses[w];
      p.loss[0] = (float)t;
    }
  });
}

// Joins a sequence's records.  A cluster a sequence; a block takes a share of
// the experts, 32 at a time, its warps every sixteenth record.
constexpr int kJoinWarps = 16;
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const Params p) {
  __shared__ float sums[kJoinWarps][32];
  __shared__ int ints[kJoinWarps][33];
  __shared__ double part;
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t s = blockIdx.x / cluster.dim_blocks().x;
  const int rank = cluster.block_rank(), parts = cluster.dim_blocks().x, tiles = (p.experts + 31) / 32;
  const int64_t from = offset_at(p, s), to = offset_at(p, s + 1), R = p.rows_per_block, words = record_words(p);
  const int64_t b0 = from / R, b1 = to > from ? (to - 1) / R + 1 : b0;
  wait_prior_grid();
  const uint32_t* rec = p.records + s * words;   // + block * words
  int n = 0;
  double loss = 0.0, factor = 0.0;
  for (int tile = rank; tile < tiles; tile += parts) {
    const bool first = tile == rank;
    const int e = tile * 32 + lane;
    float t = 0.0f;
    int c = 0;
    if (first)   // beside the sums' loads
      for (int64_t b = b0 + threadIdx.x; b < b1; b += 32 * kJoinWarps) n += (int)rec[b * words + 2 * p.experts];
    if (e < p.experts) {
#pragma unroll 8
      for (int64_t b = b0 + warp; b < b1; b += kJoinWarps) {
        t += __uint_as_float(rec[b * words + e]);
        c += (int)rec[b * words + p.experts + e];
      }
    }
    sums[warp][lane] = t, ints[warp][lane] = c;
    if (first) {
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) ints[warp][32] = n;
    }
    __syncthreads();
    if (warp == 0) {
      if (first) {
        n = 0;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) n += ints[w][32];
        factor = factor_of(p, n);
      }
      t = 0.0f, c = 0;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) t += sums[w][lane], c += ints[w][lane];
      if (e < p.experts) loss += finish(p, s, e, t, c, factor);
    }
    __syncthreads();
  }
  if (warp == 0) {
    loss = warp_sum(loss);
    if (lane == 0) part = loss;
  }
  cluster.sync();
  if (rank == 0 && threadIdx.x == 0) {
    double t = 0.0;
    for (int r = 0; r < parts; ++r) t += *cluster.map_shared_rank(&part, r);
    p.loss[s] = (float)t;
  }
  cluster.sync();   // the parts stay until they have been read
}

template <typename T, bool SOFTMAX, int VEC, int NV>
__global__ void __launch_bounds__(kThreads, blocks_of(VEC, NV)) backward_kernel(const Params p) {
  constexpr int N = NV * VEC;
  const int lane = threadIdx.x & 31, G = p.lanes, l = lane & (G - 1);
  const int per_pass = kThreads / G, slot = threadIdx.x / G;
  const T* logits = static_cast<const T*>(p.logits);
  T* out = static_cast<T*>(p.dlogits);
  const int64_t begin = blockIdx.x * p.rows_per_block, end = min(begin + p.rows_per_block, p.tokens);
  segments<true>(p, begin, end, [&](int64_t s, int64_t from, int64_t to) {
    float c[N];
    float g = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = column<VEC>(j, l, G);
      c[j] = s >= 0 && e < p.experts ? p.coef[s * p.experts + e] : 0.0f;
    }
    if (s >= 0) g = p.dloss[s];
    Pack<T, VEC> next[NV];
    bool ok = false;
    auto ask = [&](int64_t row) {
      ok = s >= 0 && row < to && (!p.valid || p.valid[row]);
      if (ok) fetch<T, VEC, NV>(next, logits + row * p.ld, l, G, p.experts);
    };
    ask(from + slot);
    for (int64_t first = from; first < to; first += per_pass) {
      const int64_t row = first + slot;
      const bool live = ok;
      float v[N], slope[SOFTMAX ? 1 : N];
      unpack<T, VEC, NV>(next, v, l, G, p.experts, live);
      ask(row + per_pass);
      scores<SOFTMAX, true, N>(v, slope, G);
      uint64_t z2 = 0, d2 = 0;
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        const uint64_t a = two(v[j], v[j + 1]);
        z2 = add2(z2, a);
        d2 = fma2(a, two(c[j], c[j + 1]), d2);
      }
      float z, d, y;
      split(z2, z, y);
      z += y;
      split(d2, d, y);
      d += y;
      for (int o = 1; o < G; o <<= 1) {
        z += __shfl_xor_sync(0xffffffffu, z, o);
        d += __shfl_xor_sync(0xffffffffu, d, o);
      }
      if constexpr (!SOFTMAX) {
        // Roots that are all next to 0: neither their products with c nor g / Z need
        // be numbers of f32.  With Z below 2^-13 every logit is below -17 and a root
        // twice its slope, so both are taken 2^n times as large, Z in [1, 2).
        const bool small = z < 1.220703125e-4f && z > 0.0f;
        if (__any_sync(0xffffffffu, small)) {
          const float up = small ? __uint_as_float((254u - (__float_as_uint(z) >> 23)) << 23) : 1.0f;
          float e = 0.0f;
#pragma unroll
          for (int j = 0; j < N; ++j) {
            slope[j] *= up;
            e = fmaf(slope[j], c[j], e);
          }
          e = group_sum(e, G);
          if (small) z *= up, d = 2.0f * e;
        }
      }
      const float inv = z == 0.0f ? 0.0f : 1.0f / z, k = live ? g * inv : 0.0f;
      d *= inv;
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        const uint64_t a = SOFTMAX ? two(v[j], v[j + 1]) : two(slope[SOFTMAX ? 0 : j], slope[SOFTMAX ? 0 : j + 1]);
        split(mul2(mul2(two(k, k), a), add2(two(c[j], c[j + 1]), two(-d, -d))), v[j], v[j + 1]);
      }
      if (row < to) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int e = (i * G + l) * VEC;
          if (e < p.experts) put<T, VEC>(out + row * p.experts + e, &v[i * VEC]);
        }
      }
    }
  });
}

// ---------------------------------------------------------------- host side

// Vectors of four logits where rows allow it, and the lanes of a row: a lane
// takes up to 16 values (eight single ones) before a row gets more lanes, as
// fewer lanes meet in fewer shuffles.
struct Layout {
  int vec, nv, lanes;
};

Layout layout_of(int experts, bool vec) {
  Layout a;
  a.vec = vec ? 4 : 1;
  const int n = (experts + a.vec - 1) / a.vec, most = vec ? 4 : 8;
  a.lanes = 1;
  while (a.lanes < 32 && (n + a.lanes - 1) / a.lanes > most) a.lanes *= 2;
  a.nv = (n + a.lanes - 1) / a.lanes;
  // as by_layout rounds it up
  if (vec) a.nv = a.nv <= 4 ? a.nv : 8;
  else a.nv = a.nv <= 4 ? 4 : a.nv <= 8 ? 8 : a.nv <= 16 ? 16 : 32;
  return a;
}

template <typename F>
void by_layout(int dtype, int kind, const Layout& a, F f) {
  auto shape = [&](auto t, auto soft) {
    auto go = [&](auto vec, auto nv) { f(t, soft, vec, nv); };
    using std::integral_constant;
    if (a.vec == 4) {
      const integral_constant<int, 4> v;
      if (a.nv == 1) go(v, integral_constant<int, 1>());
      else if (a.nv == 2) go(v, integral_constant<int, 2>());
      else if (a.nv == 3) go(v, integral_constant<int, 3>());
      else if (a.nv == 4) go(v, integral_constant<int, 4>());
      else go(v, integral_constant<int, 8>());
    } else {
      const integral_constant<int, 1> v;
      if (a.nv <= 4) go(v, integral_constant<int, 4>());
      else if (a.nv <= 8) go(v, integral_constant<int, 8>());
      else if (a.nv <= 16) go(v, integral_constant<int, 16>());
      else go(v, integral_constant<int, 32>());
    }
  };
  auto type = [&](auto soft) {
    if (dtype == DS_F32) shape(float(), soft);
    else if (dtype == DS_F16) shape(__half(), soft);
    else shape(__nv_bfloat16(), soft);
  };
  if (kind == DS_ROUTE_SOFTMAX) type(std::true_type());
  else type(std::false_type());
}

bool vectors(const void* p, int experts, int64_t tokens, int64_t ld, int dtype) {
  return experts % 4 == 0 && (tokens <= 1 || ld % 4 == 0) && ds::aligned(p, dtype == DS_F32 ? 16 : 8);
}

// Rows of a block: whole passes, and as many blocks as are resident at a time.
int64_t rows_per_block(int64_t tokens, const Layout& a) {
  const int64_t pass = kThreads / a.lanes, most = (int64_t)ds::sm_count() * blocks_of(a.vec, a.nv);
  return ((tokens + most - 1) / most + pass - 1) / pass * pass;
}

size_t record_bytes(const DsBalance& d) {
  // whichever way the logits are aligned
  int64_t blocks = 1;
  for (bool vec : {false, true}) {
    const int64_t R = rows_per_block(std::max<int64_t>(d.tokens, 1), layout_of(d.experts, vec && d.experts % 4 == 0));
    blocks = std::max(blocks, (d.tokens + R - 1) / R);
  }
  return (size_t)(blocks + d.sequences) * (2 * d.experts + 1) * 4;
}

int validate(const DsBalance* d, const char* what) {
  DS_REQUIRE(d, DS_EINVAL, "%s: null descriptor", what);
  DS_REQUIRE(d->dtype == DS_F32 || d->dtype == DS_BF16 || d->dtype == DS_F16, DS_EINVAL,
             "%s: logits must be f32, bf16 or f16", what);
  DS_REQUIRE(d->kind == DS_ROUTE_SOFTMAX || d->kind == DS_ROUTE_SQRTSOFTPLUS, DS_EINVAL,
             "%s: kind must be softmax or sqrt-softplus", what);
  DS_REQUIRE(d->experts >= 1 && d->experts <= ds::route::kMaxExperts, DS_ERANGE, "%s: experts must be in [1, %d]", what,
             ds::route::kMaxExperts);
  DS_REQUIRE(d->top_k >= 1 && d->top_k <= ds::route::kMaxTopK, DS_ERANGE, "%s: top_k must be in [1, %d]", what,
             ds::route::kMaxTopK);
  DS_REQUIRE(d->tokens >= 0 && d->tokens < ((int64_t)1 << 31) && d->tokens * d->top_k < ((int64_t)1 << 31), DS_ERANGE,
             "%s: tokens x top_k must be below 2^31", what);
  DS_REQUIRE(d->sequences >= 0 && d->sequences <= (1 << 24) && (d->offsets || d->sequences == 1), DS_ERANGE,
             "%s: sequences must be in [0, 2^24], and 1 without offsets", what);
  DS_REQUIRE(d->tokens <= 1 || d->ld >= d->experts, DS_EINVAL, "%s: row stride of the logits below experts", what);
  DS_REQUIRE(d->tokens == 0 || d->logits, DS_EINVAL, "%s: null logits", what);
  DS_REQUIRE(ds::aligned(d->logits, d->dtype == DS_F32 ? 4 : 2) && ds::aligned(d->ids, 4) &&
                 ds::aligned(d->offsets, d->offsets_i64 ? 8 : 4),
             DS_EALIGN, "%s: operands must be aligned to their elements", what);
  return DS_OK;
}

Params params_of(const DsBalance& d, const Layout& a) {
  Params p = {};
  p.logits = d.logits, p.tokens = d.tokens, p.ld = d.ld, p.experts = d.experts, p.top_k = d.top_k, p.ids = d.ids;
  p.valid = d.valid, p.offsets = d.offsets, p.wide = d.offsets_i64, p.sequences = d.sequences;
  p.rows_per_block = rows_per_block(std::max<int64_t>(d.tokens, 1), a), p.lanes = a.lanes;
  return p;
}

}  // namespace
}  // namespace balance
}  // namespace ds

using namespace ds::balance;

extern "C" int ds_balance_loss_workspace_size(const DsBalance* desc, size_t* bytes) {
  const int st = validate(desc, "balance_loss_workspace_size");
  if (st != DS_OK) return st;
  DS_REQUIRE(bytes, DS_EINVAL, "balance_loss_workspace_size: null output");
  *bytes = record_bytes(*desc);
  return DS_OK;
}

extern "C" int ds_balance_loss(const DsBalance* desc, float* loss, int32_t* counts, float* coef, void* workspace,
                               size_t workspace_bytes, void* stream) {
  const int st = validate(desc, "balance_loss");
  if (st != DS_OK) return st;
  const DsBalance& d = *desc;
  if (d.sequences == 0) return DS_OK;
  DS_REQUIRE(d.tokens == 0 || d.ids, DS_EINVAL, "balance_loss: null ids");
  DS_REQUIRE(loss && counts && coef, DS_EINVAL, "balance_loss: null output");
  DS_REQUIRE(ds::aligned(loss, 4) && ds::aligned(counts, 4) && ds::aligned(coef, 4) && ds::aligned(workspace, 4),
             DS_EALIGN, "balance_loss: results and workspace must be aligned to 4 bytes");
  const size_t need = record_bytes(d);
  DS_REQUIRE(workspace && workspace_bytes >= need, DS_EINVAL, "balance_loss: workspace %zu bytes < required %zu",
             workspace_bytes, need);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Layout a = layout_of(d.experts, vectors(d.logits, d.experts, d.tokens, d.ld, d.dtype));
  Params p = params_of(d, a);
  p.records = static_cast<uint32_t*>(workspace), p.loss = loss, p.counts = counts, p.coef = coef;
  const int64_t blocks = (d.tokens + p.rows_per_block - 1) / p.rows_per_block;
  p.single = blocks == 1 && !d.offsets;
  if (blocks) {
    const size_t smem = (kWarps + 1) * (size_t)d.experts * 4;
    by_layout(d.dtype, d.kind, a, [&](auto t, auto soft, auto vec, auto nv) {
      forward_kernel<decltype(t), decltype(soft)::value, decltype(vec)::value, decltype(nv)::value>
          <<<(unsigned)blocks, kThreads, smem, s>>>(p);
    });
    DS_CHECK_LAUNCH("balance forward_kernel");
  }
  if (p.single) return DS_OK;
  const int parts = d.sequences <= 512 ? 8 : 1;   // a block alone takes the experts 32 after 32
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(d.sequences * parts));
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = blocks ? 2 : 1;
  DS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, join_kernel, p));
  return DS_OK;
}

extern "C" int ds_balance_loss_backward(const DsBalance* desc, const float* coef, const float* dloss, void* dlogits,
                                        void* stream) {
  const int st = validate(desc, "balance_loss_backward");
  if (st != DS_OK) return st;
  const DsBalance& d = *desc;
  if (d.tokens == 0) return DS_OK;
  DS_REQUIRE(dlogits && (d.sequences == 0 || (coef && dloss)), DS_EINVAL, "balance_loss_backward: null pointer");
  DS_REQUIRE(ds::aligned(coef, 4) && ds::aligned(dloss, 4) && ds::aligned(dlogits, d.dtype == DS_F32 ? 4 : 2), DS_EALIGN,
             "balance_loss_backward: operands must be aligned to their elements");
  const bool vec = vectors(d.logits, d.experts, d.tokens, d.ld, d.dtype) &&
                   vectors(dlogits, d.experts, d.tokens, d.experts, d.dtype);
  const Layout a = layout_of(d.experts, vec);
  Params p = params_of(d, a);
  p.coef = const_cast<float*>(coef), p.dloss = dloss, p.dlogits = dlogits;
  const int64_t blocks = (d.tokens + p.rows_per_block - 1) / p.rows_per_block;
  by_layout(d.dtype, d.kind, a, [&](auto t, auto soft, auto v, auto nv) {
    backward_kernel<decltype(t), decltype(soft)::value, decltype(v)::value, decltype(nv)::value>
        <<<(unsigned)blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  });
  DS_CHECK_LAUNCH("balance backward_kernel");
  return DS_OK;
}
