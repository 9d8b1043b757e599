// Dense gated feed-forward block over 16-bit weights, forward and backward:
//   g = x W1^T, u = x W3^T, h = silu(min(g, L)) * clip(u, -L, L), y = h W2^T
// and, from dy,
//   dh = dy W2, (dg, du) = dh * d h/d(g, u), dx = dg W1 + du W3,
//   dW1 = dg^T x, dW3 = du^T x, dW2 = dy^T h.
//
// Precision: products accumulate in f32 in tensor memory.  g and u are kept
// in f32 between the passes, so that the gated unit and its derivative see
// no rounded input; h, dg and du are rounded once to the 16-bit type, because
// they are tensor-core operands of the next product (one rounding there adds
// as much error as the rounding of the result itself).  With clamps, g and u
// too close to the limit for a f32 sum are settled in 64 bits (Near), as a
// derivative that is there or not depends on it: 900 us instead of 877 for a
// training step of 8192 x 4096 x 2048 with a limit of 10 (21 of them for the
// row norms), 940 with one of 1.5 and pre-activations of unit variance.
//
// Tile kernel (up to 128 rows): one CTA computes 128 features (the MMA's
// lanes) of all tokens over a slice of the contraction.
// The slices of one tile are the CTAs of a cluster: they leave their f32
// partial tiles in shared memory and each adds up a share of the columns
// through distributed shared memory, in slice order, so results do not
// depend on timing.  Weights on the lanes mean that one token costs a
// 16-wide MMA and the weights stream once: bounded by memory and by the start
// of two dependent launches (one token of 4096 / 2048: 17.7 us for 50 MB, of
// which memory needs 7.8; 64 tokens 23.6 us).  More rows: gated_pair.cuh.
#include <algorithm>
#include <cooperative_groups.h>
#include <initializer_list>

#include "gated_pair.cuh"

namespace ds {
namespace dense {
namespace {

namespace cg = cooperative_groups;

enum Mode { GATE_UP, PLAIN, DHID, DX };

template <int MODE>
struct ModeOf {
  static constexpr bool kAMn = MODE == DHID || MODE == DX;                 // A stored with m running fastest
  static constexpr int kMats = MODE == GATE_UP ? 2 : 1;                    // accumulators (W1 and W3 share x)
  static constexpr int kSegs = MODE == DX ? 2 : 1;                         // dg W1 and du W3 in one accumulator
};

struct TileParams {
  CUtensorMap a[2], b[2];      // GATE_UP: a = W1, W3; DX: segments
  int M, N;                    // features (lanes) and tokens
  void* out[2];                // out[n * ldo + m], 16 bit (DHID: dg, du)
  int64_t ldo;
  int K;                       // contraction of one segment
  int f16;
  float limit;
  float* g;                    // f32 pre-activations [n * ldp + m]: written (GATE_UP, may be null), read (DHID)
  float* u;
  int64_t ldp;
  Near near;                   // GATE_UP
  int* err;
};

__device__ int g_err;          // bit 1: a bounded wait gave up

template <int MODE, int NT>
struct TileShape {
  using Md = ModeOf<MODE>;
  static constexpr int kA = Md::kMats * 2 * kBoxBytes;
  static constexpr int kB = NT * 128;
  static constexpr int kStage = kA + kB;
  // up to 64 tokens a CTA takes less than half of an SM, so that the next
  // launch's CTAs join it and their weights are on their way while this one
  // finishes (one token of 4096 x 2048: 17.3 us, 23 with 200 KB each; above
  // half they do not join whatever the other launch takes)
  static constexpr int kStages = std::min(8, (NT == 128 ? 200 : 111) * 1024 / kStage);
  static constexpr int kSmem = 1024 + kStages * kStage;
  static constexpr int kCols = Md::kMats * NT < 32 ? 32 : Md::kMats * NT;
  static_assert(kStage % 1024 == 0 && kStages * kStage >= Md::kMats * NT * 128 * 4, "stages hold the partial tile");
};

constexpr int kTileThreads = 320;   // warp 0 copies, warp 1 MMA, warps 2-9 epilogue (two a lane quarter)

// What becomes of the elements (m, n0 .. n0 + J - 1) of the accumulator(s), nv
// of them inside the result (none for a feature outside; whole warps call).
// Lanes are features, so a warp's accesses are
// runs of 32; all reads come before the first write, which could alias them
// for all the compiler knows (one column after the other, the reads' latency
// made the hidden gradient of 1024 x 4096 x 2048 five times slower).
template <int MODE, int J>
__device__ __forceinline__ void tile_store(const TileParams& p, int m, int n0, int nv, const float (&v0)[J],
                                           const float (&v1)[J]) {
  uint16_t* out = static_cast<uint16_t*>(p.out[0]) + (int64_t)n0 * p.ldo + m;
  const int64_t at = (int64_t)n0 * p.ldp + m;
  if constexpr (MODE == DHID) {
    float g[J], u[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      g[j] = j < nv ? p.g[at + j * p.ldp] : 0.0f;
      u[j] = j < nv ? p.u[at + j * p.ldp] : 0.0f;
    }
    uint16_t* out1 = static_cast<uint16_t*>(p.out[1]) + (int64_t)n0 * p.ldo + m;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      gate_grad(g[j], u[j], v0[j], p.limit, g[j], u[j]);
      if (j < nv) {
        out[j * p.ldo] = to16(g[j], p.f16);
        out1[j * p.ldo] = to16(u[j], p.f16);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (j >= nv) continue;
      if (MODE == GATE_UP && p.g) {
        p.g[at + j * p.ldp] = v0[j];
        p.u[at + j * p.ldp] = v1[j];
      }
      out[j * p.ldo] = to16(MODE == GATE_UP ? gate_unit(v0[j], v1[j], p.limit) : v0[j], p.f16);
    }
    if constexpr (MODE == GATE_UP) {
      if (!p.near.x) return;
#pragma unroll 1
      for (int z = 0; z < 2; ++z) {
        const float nw = nv > 0 ? p.near.nw[z][m] : 0.0f;
        uint32_t near = 0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (j >= nv) continue;
          const float band = near_band(p.near, p.near.nx[n0 + j], nw);
          near |= (uint32_t)(z ? near_u(p.near, v1[j], band) : near_g(p.near, v0[j], band)) << j;
        }
        near_settle(p.near, z, near,
                    [&](int src, int bit, int64_t& t, int64_t& i) { t = n0 + bit, i = m - (int)(threadIdx.x & 31) + src; },
                    [&](int bit, float v) { (z ? p.u : p.g)[at + bit * p.ldp] = v; });
      }
    }
  }
}

// Sums this CTA's share of the columns over the partial tiles [mats][NT][128]
// of the cluster, in slice order.  The reads of four columns from all slices
// are in flight together.
template <int MODE, int NT, int SLICES>
__device__ __forceinline__ void tile_join(const TileParams& p, float* part, int slice, int turn, int m, int mi) {
  constexpr int kMats = ModeOf<MODE>::kMats;
  cg::cluster_group cluster = cg::this_cluster();
  const float* src[SLICES];
#pragma unroll
  for (int r = 0; r < SLICES; ++r) src[r] = cluster.map_shared_rank(part, r) + mi;
  const int share = (p.N + SLICES - 1) / SLICES, end = min(p.N, (slice + 1) * share);
  for (int n = slice * share + 4 * turn; n < end; n += 8) {
    float w[SLICES][kMats][4];
#pragma unroll
    for (int r = 0; r < SLICES; ++r)
#pragma unroll
      for (int t = 0; t < kMats; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) w[r][t][j] = src[r][(t * NT + min(n + j, end - 1)) * 128];
    float v[2][4] = {};
#pragma unroll
    for (int r = 0; r < SLICES; ++r)
#pragma unroll
      for (int t = 0; t < kMats; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[t][j] += w[r][t][j];
    tile_store<MODE>(p, m, n, m < p.M ? end - n : 0, v[0], v[1]);
  }
}

template <int MODE, int NT>
__global__ void __launch_bounds__(kTileThreads, NT == 128 ? 1 : 2) tile_kernel(const __grid_constant__ TileParams p) {
  using Md = ModeOf<MODE>;
  using C = TileShape<MODE, NT>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ __align__(8) uint64_t full[S], empty[S], accfull;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  cg::cluster_group cluster = cg::this_cluster();
  const int slices = cluster.dim_blocks().x, slice = cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = (blockIdx.x / slices) * 128;
  const int ksteps = (p.K + kBK - 1) / kBK;
  const int it0 = (int)((int64_t)Md::kSegs * ksteps * slice / slices);
  const int it1 = (int)((int64_t)Md::kSegs * ksteps * (slice + 1) / slices);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&accfull, 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tc5::alloc(&tmem_base, C::kCols);
  tc5::fence_before();
  __syncthreads();
  tc5::fence_after();
  const uint32_t tb = tmem_base;
  volatile int* abort = &abort_flag;
  launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      auto weights = [&](int g) {
        const int it = it0 + g, seg = it / ksteps, k0 = (it - seg * ksteps) * kBK;
        uint8_t* st = smem + g % S * C::kStage;
        uint64_t* bar = &full[g % S];
        mbar_arrive_expect_tx(bar, C::kStage);
        load_tile<Md::kAMn, 128>(st, &p.a[seg], m0, k0, bar);
        if (Md::kMats == 2) load_tile<Md::kAMn, 128>(st + 2 * kBoxBytes, &p.a[1], m0, k0, bar);
      };
      auto rows = [&](int g) {
        const int it = it0 + g, seg = it / ksteps, k0 = (it - seg * ksteps) * kBK;
        load_tile<false, NT>(smem + g % S * C::kStage + C::kA, &p.b[seg], 0, k0, &full[g % S]);
      };
      // The weights of the first stages need nothing of the launch before this
      // one in the stream: that is one of the same call, and the call's first
      // launch began after all earlier work had ended.
      const int n = it1 - it0, early = min(S, n);
      for (int g = 0; g < early; ++g) weights(g);
      wait_prior_grid();
      for (int g = 0; g < early; ++g) rows(g);
      int g = early;
      for (; g < n; ++g) {
        if (!ds::pair::wait(&empty[g % S], ((g / S) - 1) & 1, abort, p.err)) break;
        weights(g);
        rows(g);
      }
      // never leave with copies in flight into this CTA's shared memory
      for (int j = g - S < 0 ? 0 : g - S; j < g; ++j) mbar_wait_bounded(&full[j % S], (j / S) & 1, 200000000ull);
    }
  } else if (warp == 1) {
    const uint32_t idesc = idesc16(p.f16, Md::kAMn, false, 128, NT);
    const uint64_t a0 = tile_desc<Md::kAMn>(smem_u32(smem)), b0 = tile_desc<false>(smem_u32(smem) + C::kA);
    for (int g = 0; g < it1 - it0; ++g) {
      const int s = g % S;
      if (!ds::pair::wait_all(&full[s], (g / S) & 1, abort, p.err)) break;
      tc5::fence_after();
      if (elect_one()) {
        const uint64_t ad = a0 + (uint64_t)((s * C::kStage) >> 4), bd = b0 + (uint64_t)((s * C::kStage) >> 4);
#pragma unroll
        for (int kk = 0; kk < kBK / 16; ++kk) {
          tc5::mma_bf16(tb, ad + kk * kStep16<Md::kAMn>, bd + kk * kStep16<false>, idesc, (g | kk) != 0);
          if (Md::kMats == 2)
            tc5::mma_bf16(tb + NT, ad + ((2 * kBoxBytes) >> 4) + kk * kStep16<Md::kAMn>,
                          bd + kk * kStep16<false>, idesc, (g | kk) != 0);
        }
        tc5::commit(&empty[s]);
      }
      __syncwarp();
    }
    // all issued MMAs complete before the accumulators are read or released
    if (elect_one()) tc5::commit(&accfull);
    __syncwarp();
    ds::pair::wait_all(&accfull, 0, abort, p.err);
  } else {
    ds::pair::wait_all(&accfull, 0, abort, p.err);
  }
  tc5::fence_after();

  // ---- epilogue: thread = one feature (lane of tensor memory)
  wait_prior_grid();
  const int q = warp & 3, turn = (warp - 2) >> 2, mi = q * 32 + lane, m = m0 + mi;
  float* part = reinterpret_cast<float*>(smem);   // [mats][NT][128]
  if (warp >= 2) {
    for (int c0 = 16 * turn; c0 < p.N; c0 += 32) {
      float v[Md::kMats][16];
#pragma unroll
      for (int t = 0; t < Md::kMats; ++t) tc5::ld_x16_nowait(tc5::lane_quarter(tb + t * NT + c0, q), v[t]);
      tc5::wait_ld();
      if (slices > 1) {
#pragma unroll
        for (int t = 0; t < Md::kMats; ++t)
#pragma unroll
          for (int j = 0; j < 16; ++j) part[(t * NT + c0 + j) * 128 + mi] = v[t][j];
      } else {
        tile_store<MODE>(p, m, c0, m < p.M ? p.N - c0 : 0, v[0], v[Md::kMats - 1]);
      }
    }
  }
  if (slices > 1) {
    cluster.sync();
    if (warp >= 2) {
      if (slices == 8) tile_join<MODE, NT, 8>(p, part, slice, turn, m, mi);
      else if (slices == 4) tile_join<MODE, NT, 4>(p, part, slice, turn, m, mi);
      else tile_join<MODE, NT, 2>(p, part, slice, turn, m, mi);
    }
    cluster.sync();   // partial tiles stay until every CTA has read them
  }
  tc5::fence_before();
  __syncthreads();
  if (warp == 1) {
    tc5::fence_after();
    tc5::dealloc(tb, C::kCols);
  }
}

// ---------------------------------------------------------------- operand copies

// Copies strided 16-bit matrices into rows of ldd (a multiple of 8) elements,
// zeros behind the columns: the form that the tensor maps need of an operand
// whose base or row stride is no multiple of 16 bytes.  All operands of a call
// in one launch (blockIdx.y).
struct PackParams {
  const uint16_t* src[5];
  uint16_t* dst[5];
  int64_t rows[5], lds[5];
  int cols[5];
};

__global__ void __launch_bounds__(256) pack_kernel(const PackParams p) {
  const int z = blockIdx.y, cols = p.cols[z], ldd = (cols + 7) / 8 * 8;
  const int64_t lds = p.lds[z], n = p.rows[z] * (ldd / 8);
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / (ldd / 8);
    const int c = (int)(i - r * (ldd / 8)) * 8;
    const uint16_t* src = p.src[z] + r * lds + c;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < cols) w[j >> 1] |= (uint32_t)src[j] << (16 * (j & 1));
    *reinterpret_cast<uint4*>(p.dst[z] + r * ldd + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---------------------------------------------------------------- values close to the limit

// 2-norms of the rows of x, W1 and W3, a warp a row, rather 2^-10 too large
// than too small: how far a sum may be off (Near).  Memory-bound: 100 MB in 21
// us for 8192 x 4096 x 2048.  Empties the list.
struct NormParams {
  const uint16_t* p[3];
  int64_t ld[3];
  int64_t end[3];              // rows so far, in the order of the norms
  int K, f16;
  float* out;
  unsigned long long* count;
};

__device__ __forceinline__ float sum_squares(const uint16_t* row, int K, int f16, float scale) {
  const int lane = threadIdx.x & 31;
  float s = 0.0f;
#pragma unroll 4
  for (int k = lane * 8; k + 8 <= K; k += 256) {
    const uint4 v = *reinterpret_cast<const uint4*>(row + k);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = from16(w[j] & 0xFFFFu, f16) * scale, b = from16(w[j] >> 16, f16) * scale;
      s = fmaf(a, a, fmaf(b, b, s));
    }
  }
  const int k = K / 8 * 8 + lane;   // an uneven end
  if (k < K) {
    const float a = from16(row[k], f16) * scale;
    s = fmaf(a, a, s);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

__global__ void __launch_bounds__(256) norm_kernel(const NormParams p) {
  launch_dependents();
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.count = 0ull;
  const int64_t r = blockIdx.x * (int64_t)8 + (threadIdx.x >> 5);
  if (r >= p.end[2]) return;
  const uint16_t* row = r < p.end[0]   ? p.p[0] + r * p.ld[0]
                        : r < p.end[1] ? p.p[1] + (r - p.end[0]) * p.ld[1]
                                       : p.p[2] + (r - p.end[1]) * p.ld[2];
  float s = 0.0f, scale = 1.0f;
  // a sum past f32's range (either end): again with the row brought inside
  for (int pass = 0; pass < 2; ++pass) {
    s = sum_squares(row, p.K, p.f16, scale);
    if (pass || (s >= 1e-30f && s <= 1e37f)) break;
    scale = s < 1e-30f ? 0x1p70f : 0x1p-70f;
  }
  if ((threadIdx.x & 31) == 0) p.out[r] = sqrtf(s) / scale * (1.0f + 0x1p-10f);
}

// The listed values, a warp each, into the kept pre-activations [2][rows][ldp].
// More than the list holds: each warp goes through whole rows.
__global__ void __launch_bounds__(256) settle_kernel(const Near p, float* pre, int64_t ldp, int rows, int cols) {
  launch_dependents();
  wait_prior_grid();
  const int lane = threadIdx.x & 31;
  const int64_t plane = rows * ldp, warp = blockIdx.x * (int64_t)8 + (threadIdx.x >> 5), warps = gridDim.x * (int64_t)8;
  const unsigned long long n = *p.count;
  if (n <= p.room) {
    for (int64_t e = warp; e < (int64_t)n; e += warps) {
      const uint64_t v = p.list[e];
      const int64_t t = (int64_t)(v >> 32), i = (int64_t)(v & 0x7FFFFFFFu);
      const int z = (int)(v >> 31 & 1);
      const float settled = near_round(near_sum(p, z, t, i), p.limit);
      if (lane == 0) pre[z * plane + t * ldp + i] = settled;
    }
    return;
  }
  for (int64_t e = warp; e < 2 * (int64_t)rows; e += warps) {
    const int z = e >= rows;
    const int64_t row = e - (z ? rows : 0);
    const float nx = p.nx[row], *nw = z ? p.nw[1] : p.nw[0];
    for (int c0 = 0; c0 < cols; c0 += 32) {
      const int c = c0 + lane;
      float* at = pre + z * plane + row * ldp + c;
      uint32_t near = 0;
      if (c < cols) near = z ? near_u(p, *at, near_band(p, nx, nw[c])) : near_g(p, *at, near_band(p, nx, nw[c]));
      near_settle(p, z, near, [&](int src, int, int64_t& t, int64_t& i) { t = row, i = c0 + src; },
                  [&](int, float v) { *at = v; });
    }
  }
}

// ---------------------------------------------------------------- host side

int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }

bool direct(const void* p, int64_t ld) { return ds::aligned(p, 16) && ld % 8 == 0; }

struct Operand {
  const void* p;
  int64_t rows, cols, ld;
};

// Bytes a packed copy of the operand takes (0: read in place).
size_t copy_bytes(const Operand& o) {
  return direct(o.p, o.ld) ? 0 : grouped::up((size_t)o.rows * up8(o.cols) * 2, 256);
}

// Replaces the operands that need one by their packed copies in the workspace.
int place(std::initializer_list<Operand*> operands, char*& ws, cudaStream_t s) {
  PackParams p = {};
  int n = 0;
  int64_t most = 0;
  for (Operand* o : operands) {
    const size_t bytes = copy_bytes(*o);
    if (bytes == 0) continue;
    p.src[n] = static_cast<const uint16_t*>(o->p);
    p.dst[n] = reinterpret_cast<uint16_t*>(ws);
    p.rows[n] = o->rows, p.lds[n] = o->ld, p.cols[n] = (int)o->cols;
    most = std::max<int64_t>(most, o->rows * (up8(o->cols) / 8));
    o->p = ws;
    o->ld = up8(o->cols);
    ws += bytes;
    ++n;
  }
  if (n == 0) return DS_OK;
  const int grid = (int)std::min<int64_t>((most + 255) / 256, (int64_t)ds::sm_count() * 16);
  pack_kernel<<<dim3(grid, n), 256, 0, s>>>(p);
  DS_CHECK_LAUNCH("pack_kernel");
  return DS_OK;
}

int* err_word() {
  static SymbolOnce known;
  return ds::symbol_address(&known, &g_err);
}

template <int MODE, int NT>
int launch_tiles(const TileParams& p, int slices, cudaStream_t s, bool chained) {
  using C = TileShape<MODE, NT>;
  static SmemOnce once;
  const int st = ds::allow_smem(&once, reinterpret_cast<const void*>(&tile_kernel<MODE, NT>), C::kSmem);
  if (st != DS_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.M + 127) / 128 * slices));
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)slices;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = chained ? 2 : 1;
  DS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, tile_kernel<MODE, NT>, p));
  return DS_OK;
}

// Box rows of the token-side operand for a given token count, and the slices
// of the contraction: enough to give every SM a CTA, at least four stages each.
int token_tile(int64_t n) { return n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : 128; }

int slices_for(int64_t tiles, int ksteps) {
  int s = 1;
  while (s < 8 && tiles * s * 2 <= ds::sm_count() && ksteps / (s * 2) >= 4) s *= 2;
  return s;
}

template <int MODE>
int run_tiles(const TileParams& p, int nt, cudaStream_t s, bool chained) {
  const int64_t tiles = (p.M + 127) / 128;
  const int slices = slices_for(tiles, ModeOf<MODE>::kSegs * ((p.K + kBK - 1) / kBK));
  if (nt == 16) return launch_tiles<MODE, 16>(p, slices, s, chained);
  if (nt == 32) return launch_tiles<MODE, 32>(p, slices, s, chained);
  if (nt == 64) return launch_tiles<MODE, 64>(p, slices, s, chained);
  return launch_tiles<MODE, 128>(p, slices, s, chained);
}

// ---- pair kernel

// The pair kernel takes the products of at least this many rows, where its 256
// are half full (at 96 rows the two are even on 4096 x 2048 and 1024 x 1024,
// 34 and 16 us, and the tile kernel is ahead on uneven widths and in the
// backward pass, 51 against 59 us; at 129 it would need a second tile of
// rows); weight gradients always.
constexpr int kPairRows = 129;

int64_t tiles_of(const Problem& q, int nt) {
  const int c = pair::tile_cols(q.epi, nt);
  return (q.M + 255) / 256 * (int64_t)((q.N + c - 1) / c);
}

// Adds the problem c = a b^T to a launch (k: the contraction).  Problems of
// one contraction form a group; the longer one is given first.
Problem* add(PairParams& p, int epi, int64_t M, int64_t N, int64_t k, int segs, void* c, int64_t ldc) {
  Problem& q = p.pr[p.n++];
  q.epi = epi, q.M = (int)M, q.N = (int)N;
  q.ksteps = (int)((k + kBK - 1) / kBK), q.segs = segs;
  q.c = c, q.ldc = ldc;
  return &q;
}

// One of a launch's problems with its operands; W3's map of a gate / up
// product in b1.
struct Sides {
  Problem* q;
  Operand a0, b0, a1, b1;
};

// Time of a launch in tensor cycles for tiles of nt columns: a stage takes 2 nt
// of them, or what its bytes take at the ~70 bytes a cycle that an SM gets
// from L2; a tile's epilogue is hidden but for the last; whole tiles per pair.
int64_t cycles_of(const PairParams& p, int nt, int pairs) {
  const int64_t stage = nt == 256 ? 512 : nt == 128 ? 350 : 300;
  int64_t work = 0, longest = 0, tiles = 0;
  for (int z = 0; z < p.n; ++z) {
    const int64_t its = (int64_t)p.pr[z].ksteps * p.pr[z].segs, n = tiles_of(p.pr[z], nt), tile = its * stage + 400;
    work += n * tile;
    tiles += n;
    longest = std::max(longest, tile);
  }
  const int64_t level = (work + pairs - 1) / pairs;
  return p.split == p.n ? (tiles + pairs - 1) / pairs * longest : std::max(longest, level + longest / 4);
}

template <int EPI, int NT>
int launch_pairs(PairParams& p, Sides* sides, cudaStream_t s, bool chained) {
  using C = pair::Shape<EPI, NT>;
  int64_t tiles = 0;
  for (int z = 0; z < p.n; ++z) {
    Problem& q = p.pr[z];
    const Sides& d = sides[z];
    auto side = [&](CUtensorMap* m, const Operand& o, int mn, int rows) {
      return !o.p || map16(m, o.p, o.rows, o.cols, o.ld, mn ? 64 : rows);
    };
    q.boxed = q.epi == STORE && direct(q.c, q.ldc);
    const bool ok = side(&q.a[0], d.a0, q.a_mn, 128) && side(&q.a[1], d.a1, q.a_mn, 128) &&
                    side(&q.b[0], d.b0, q.b_mn, NT / 2) && side(&q.b[1], d.b1, q.b_mn, NT / 2) &&
                    (!q.boxed || map16(&q.out, q.c, q.M, q.N, q.ldc, 32));
    DS_REQUIRE(ok, DS_ECUDA, "gated_ffn: tensor map encoding failed");
    tiles += tiles_of(q, NT);
    DS_REQUIRE(tiles < ((int64_t)1 << 31), DS_ERANGE, "gated_ffn: too many tiles");
    q.tiles = (int)tiles;
  }
  static SmemOnce once;
  const int st = ds::allow_smem(&once, reinterpret_cast<const void*>(&pair::pair_kernel<EPI, NT>), C::kSmem);
  if (st != DS_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, ds::sm_count() / 2)));
  cfg.blockDim = dim3(pair::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = chained ? 1 : 0;
  DS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, pair::pair_kernel<EPI, NT>, p));
  return DS_OK;
}

// Runs the problems with the tile width that takes least time.
template <int EPI>
int run_pairs(PairParams& p, Sides* sides, cudaStream_t s, bool chained) {
  if (p.split == 0) p.split = p.n;
  const int pairs = ds::sm_count() / 2;
  const int64_t t256 = cycles_of(p, 256, pairs), t128 = cycles_of(p, 128, pairs), t64 = cycles_of(p, 64, pairs);
  if (t256 <= t128 && t256 <= t64) return launch_pairs<EPI, 256>(p, sides, s, chained);
  if (t128 <= t64) return launch_pairs<EPI, 128>(p, sides, s, chained);
  return launch_pairs<EPI, 64>(p, sides, s, chained);
}

int validate(const DsGatedFfn* d) {
  DS_REQUIRE(d != nullptr, DS_EINVAL, "gated_ffn: null descriptor");
  DS_REQUIRE(d->tokens >= 0 && d->tokens <= (1 << 22), DS_ERANGE, "gated_ffn: tokens must be in [0, 2^22]");
  DS_REQUIRE(d->hidden >= 1 && d->hidden <= (1 << 17) && d->inter >= 1 && d->inter <= (1 << 17), DS_ERANGE,
             "gated_ffn: hidden and inter must be in [1, 2^17]");
  DS_REQUIRE(d->dtype == DS_BF16 || d->dtype == DS_F16, DS_EINVAL, "gated_ffn: dtype must be bf16 or f16");
  DS_REQUIRE(d->limit >= 0.0f, DS_EINVAL, "gated_ffn: limit must be >= 0 (0: no clamps)");
  DS_REQUIRE(d->ld_x >= d->hidden && d->ld_w1 >= d->hidden && d->ld_w3 >= d->hidden && d->ld_w2 >= d->inter,
             DS_EINVAL, "gated_ffn: row strides must cover the rows");
  return DS_OK;
}

int validate_call(const DsGatedFfn* d, const void* ws, size_t ws_bytes, size_t need, const char* what) {
  DS_REQUIRE(d->x && d->w1 && d->w3 && d->w2, DS_EINVAL, "%s: null operand", what);
  DS_REQUIRE(ds::aligned(d->x, 2) && ds::aligned(d->w1, 2) && ds::aligned(d->w3, 2) && ds::aligned(d->w2, 2),
             DS_EALIGN, "%s: operands must be 2-byte aligned", what);
  DS_REQUIRE(ws_bytes >= need && (need == 0 || ws), DS_EINVAL, "%s: workspace %zu bytes < required %zu", what,
             ws_bytes, need);
  DS_REQUIRE(ds::aligned(ws, 256), DS_EALIGN, "%s: workspace must be 256-byte aligned", what);
  DS_REQUIRE(grouped::encode_fn() != nullptr, DS_ECUDA, "%s: cuTensorMapEncodeTiled unavailable", what);
  return DS_OK;
}

struct Parts {
  Operand x, w1, w3, w2;
};

Parts parts_of(const DsGatedFfn* d) {
  return {{d->x, d->tokens, d->hidden, d->ld_x},
          {d->w1, d->inter, d->hidden, d->ld_w1},
          {d->w3, d->inter, d->hidden, d->ld_w3},
          {d->w2, d->hidden, d->inter, d->ld_w2}};
}

size_t mid_bytes(const DsGatedFfn* d) { return grouped::up((size_t)d->tokens * up8(d->inter) * 2, 256); }

// The operands' packed copies.
size_t packed_bytes(const DsGatedFfn* d) {
  const Parts o = parts_of(d);
  return copy_bytes(o.x) + copy_bytes(o.w1) + copy_bytes(o.w3) + copy_bytes(o.w2);
}

// Values close to the limit that are listed before they are settled: one in
// 32, far more than data leaves there by chance; none for the tile kernel.
size_t near_room(const DsGatedFfn* d) {
  return d->tokens < kPairRows ? 0 : std::min<size_t>((size_t)d->tokens * d->inter / 32, 1u << 30);
}

size_t norm_bytes(const DsGatedFfn* d) {
  return grouped::up((size_t)(d->tokens + 2 * (int64_t)d->inter) * 4, 256);
}

// With clamps: row norms of x, W1 and W3, the list and its length.
size_t near_bytes(const DsGatedFfn* d) {
  return d->limit > 0.0f ? norm_bytes(d) + 256 + grouped::up(near_room(d) * 8, 256) : 0;
}

size_t forward_bytes(const DsGatedFfn* d, bool own_h) {
  return packed_bytes(d) + near_bytes(d) + (own_h ? mid_bytes(d) : 0);
}

size_t backward_bytes(const DsGatedFfn* d, const void* dy, int64_t ld_dy) {
  const Operand g = {dy, d->tokens, d->hidden, ld_dy};
  return packed_bytes(d) + copy_bytes(g) + 2 * mid_bytes(d);
}

// What settles the kept pre-activations that lie close to the limit; the
// launch that writes them is chained to the one of the norms.
int prepare_near(Near& p, const DsGatedFfn* d, const Parts& o, char* ws, cudaStream_t s) {
  const int64_t T = d->tokens, I = d->inter;
  float* norms = reinterpret_cast<float*>(ws);
  p.count = reinterpret_cast<unsigned long long*>(ws + norm_bytes(d));
  p.list = reinterpret_cast<uint64_t*>(ws + norm_bytes(d) + 256);
  p.room = (uint32_t)near_room(d);
  NormParams n = {};
  const Operand* const rows[3] = {&o.x, &o.w1, &o.w3};
  for (int z = 0; z < 3; ++z) {
    n.p[z] = static_cast<const uint16_t*>(rows[z]->p), n.ld[z] = rows[z]->ld;
    n.end[z] = T + z * I;
  }
  n.K = d->hidden, n.f16 = d->dtype == DS_F16, n.out = norms, n.count = p.count;
  norm_kernel<<<(unsigned)((n.end[2] + 7) / 8), 256, 0, s>>>(n);
  DS_CHECK_LAUNCH("norm_kernel");
  p.x = n.p[0], p.w[0] = n.p[1], p.w[1] = n.p[2];
  p.ldx = n.ld[0], p.ldw[0] = n.ld[1], p.ldw[1] = n.ld[2];
  p.nx = norms, p.nw[0] = norms + T, p.nw[1] = norms + T + I;
  p.K = n.K, p.f16 = n.f16, p.limit = d->limit;
  p.per = (float)((d->hidden + 15) / 16 + 1) * 0x1p-23f;
  return DS_OK;
}

// Settles what the launch before has listed.
int settle_listed(const Near& p, float* pre, int64_t ldp, int rows, int cols, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>((p.room + 7) / 8, (int64_t)ds::sm_count() * 8));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  DS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, settle_kernel, p, pre, ldp, rows, cols));
  return DS_OK;
}

}  // namespace
}  // namespace dense
}  // namespace ds

using namespace ds::dense;

extern "C" int ds_gated_ffn_workspace_size(const DsGatedFfn* desc, int keeps_h, size_t* bytes) {
  int st = validate(desc);
  if (st != DS_OK) return st;
  DS_REQUIRE(bytes != nullptr, DS_EINVAL, "gated_ffn_workspace_size: null output");
  *bytes = forward_bytes(desc, !keeps_h);
  return DS_OK;
}

extern "C" int ds_gated_ffn(const DsGatedFfn* desc, void* y, void* h, float* pre, void* workspace,
                            size_t workspace_bytes, void* stream) {
  int st = validate(desc);
  if (st != DS_OK) return st;
  if (desc->tokens == 0) return DS_OK;
  if ((st = validate_call(desc, workspace, workspace_bytes, forward_bytes(desc, h == nullptr), "gated_ffn")) != DS_OK)
    return st;
  DS_REQUIRE(y && ds::aligned(y, 2) && ds::aligned(h, 16) && ds::aligned(pre, 16), DS_EALIGN,
             "gated_ffn: y must be 2-byte, h and pre 16-byte aligned");
  const int T = (int)desc->tokens, H = desc->hidden, I = desc->inter;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  Parts o = parts_of(desc);
  if ((st = place({&o.x, &o.w1, &o.w3, &o.w2}, ws, s)) != DS_OK) return st;
  Near near = {};
  const bool clamped = pre && desc->limit > 0.0f;
  if (clamped && (st = prepare_near(near, desc, o, ws, s)) != DS_OK) return st;
  ws += near_bytes(desc);
  if (!h) h = ws;
  const int64_t ldm = up8(I);
  int* err = err_word();
  DS_REQUIRE(err != nullptr, DS_ECUDA, "gated_ffn: error word unavailable");
  const int f16 = desc->dtype == DS_F16;
  float* pre_u = pre ? pre + (int64_t)T * ldm : nullptr;
  const Operand oh = {h, T, I, ldm}, none = {};

  if (T >= kPairRows) {
    PairParams p = {};
    p.f16 = f16, p.limit = desc->limit, p.err = err, p.keep = pre != nullptr, p.near = near;
    Sides up[1] = {{add(p, GATED, T, I, H, 1, h, ldm), o.x, o.w1, none, o.w3}};
    DS_REQUIRE(map_slim(&p.h, h, T, I, ldm) &&
                   (!pre || (map32(&p.g, pre, T, I, ldm) && map32(&p.u, pre_u, T, I, ldm))),
               DS_ECUDA, "gated_ffn: tensor map encoding failed (h, pre-activations)");
    if ((st = run_pairs<GATED>(p, up, s, clamped)) != DS_OK) return st;
    if (near.room && (st = settle_listed(near, pre, ldm, T, I, s)) != DS_OK) return st;
    PairParams d = {};
    d.f16 = f16, d.err = err;
    Sides down[1] = {{add(d, STORE, T, H, I, 1, y, H), oh, o.w2, none, none}};
    return run_pairs<STORE>(d, down, s, true);
  }
  const int nt = token_tile(T);
  TileParams p = {};
  p.f16 = f16, p.limit = desc->limit, p.err = err;
  bool ok = map16(&p.a[0], o.w1.p, I, H, o.w1.ld, 128) && map16(&p.a[1], o.w3.p, I, H, o.w3.ld, 128) &&
            map16(&p.b[0], o.x.p, T, H, o.x.ld, nt);
  DS_REQUIRE(ok, DS_ECUDA, "gated_ffn: tensor map encoding failed (gate / up)");
  p.M = I, p.N = T, p.K = H;
  p.out[0] = h, p.ldo = ldm;
  p.g = pre, p.u = pre_u, p.ldp = ldm, p.near = near;
  if ((st = run_tiles<GATE_UP>(p, nt, s, clamped)) != DS_OK) return st;
  ok = map16(&p.a[0], o.w2.p, H, I, o.w2.ld, 128) && map16(&p.b[0], h, T, I, ldm, nt);
  DS_REQUIRE(ok, DS_ECUDA, "gated_ffn: tensor map encoding failed (down)");
  p.M = H, p.K = I;
  p.out[0] = y, p.ldo = H;
  return run_tiles<PLAIN>(p, nt, s, true);
}

extern "C" int ds_gated_ffn_backward_workspace_size(const DsGatedFfn* desc, const void* dy, int64_t ld_dy,
                                                    size_t* bytes) {
  int st = validate(desc);
  if (st != DS_OK) return st;
  DS_REQUIRE(bytes != nullptr && ld_dy >= desc->hidden, DS_EINVAL,
             "gated_ffn_backward_workspace_size: null output or row stride of dy below hidden");
  *bytes = backward_bytes(desc, dy, ld_dy);
  return DS_OK;
}

extern "C" int ds_gated_ffn_backward(const DsGatedFfn* desc, const void* h, const float* pre, const void* dy,
                                     int64_t ld_dy, void* dx, void* dw1, void* dw3, void* dw2, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  int st = validate(desc);
  if (st != DS_OK) return st;
  DS_REQUIRE(ld_dy >= desc->hidden, DS_EINVAL, "gated_ffn_backward: row stride of dy below hidden");
  const int T = (int)desc->tokens, H = desc->hidden, I = desc->inter;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (T == 0) {   // sums over no tokens
    if (dw1) DS_CHECK_CUDA(cudaMemsetAsync(dw1, 0, (size_t)I * H * 2, s));
    if (dw3) DS_CHECK_CUDA(cudaMemsetAsync(dw3, 0, (size_t)I * H * 2, s));
    if (dw2) DS_CHECK_CUDA(cudaMemsetAsync(dw2, 0, (size_t)I * H * 2, s));
    return DS_OK;
  }
  if ((st = validate_call(desc, workspace, workspace_bytes, backward_bytes(desc, dy, ld_dy),
                          "gated_ffn_backward")) != DS_OK)
    return st;
  DS_REQUIRE(h && pre && dy, DS_EINVAL, "gated_ffn_backward: null saved tensor or gradient");
  DS_REQUIRE(ds::aligned(h, 16) && ds::aligned(pre, 16) && ds::aligned(dy, 2) && ds::aligned(dx, 2) &&
                 ds::aligned(dw1, 2) && ds::aligned(dw3, 2) && ds::aligned(dw2, 2),
             DS_EALIGN, "gated_ffn_backward: h and pre must be 16-byte, gradients 2-byte aligned");
  char* ws = static_cast<char*>(workspace);
  Parts o = parts_of(desc);
  Operand gy = {dy, T, H, ld_dy};
  if ((st = place({&o.x, &o.w1, &o.w3, &o.w2, &gy}, ws, s)) != DS_OK) return st;
  const int64_t ldm = up8(I);
  void* dg = ws;
  void* du = ws + mid_bytes(desc);
  int* err = err_word();
  DS_REQUIRE(err != nullptr, DS_ECUDA, "gated_ffn_backward: error word unavailable");
  const int f16 = desc->dtype == DS_F16;
  float* g = const_cast<float*>(pre);
  float* u = g + (int64_t)T * ldm;
  const Operand og = {dg, T, I, ldm}, ou = {du, T, I, ldm}, oh = {h, T, I, ldm}, none = {};
  const bool need_mid = dx || dw1 || dw3, wide = T >= kPairRows;
  auto grad = [&](PairParams& p, Sides* sd, void* dw, int64_t M, int64_t N, const Operand& dy_, const Operand& act) {
    Problem* q = add(p, STORE, M, N, T, 1, dw, N);   // dw [M, N] = dy_^T act
    q->a_mn = q->b_mn = 1;
    sd[p.n - 1] = {q, dy_, act, none, none};
  };
  bool chained = false;

  if (wide) {
    // first launch: dg and du from dy, and beside them dW2, which needs neither
    PairParams p = {};
    p.f16 = f16, p.limit = desc->limit, p.err = err;
    Sides sd[3];
    for (int k = 0; k < 2; ++k) {
      if ((k == 0) == (T >= H)) {
        if (dw2) grad(p, sd, dw2, H, I, gy, oh);
      } else if (need_mid) {
        Problem* q = add(p, HIDDEN, T, I, H, 1, dg, ldm);
        q->b_mn = 1;
        sd[p.n - 1] = {q, gy, o.w2, none, none};
      }
      if (k == 0) p.split = p.n;
    }
    if (p.n) {
      DS_REQUIRE(map32(&p.g, g, T, I, ldm) && map32(&p.u, u, T, I, ldm) && map_slim(&p.dg, dg, T, I, ldm) &&
                     map_slim(&p.du, du, T, I, ldm),
                 DS_ECUDA, "gated_ffn_backward: tensor map encoding failed (pre-activations)");
      if ((st = run_pairs<HIDDEN>(p, sd, s, false)) != DS_OK) return st;
      chained = true;
    }
  } else {
    const int nt = token_tile(T);
    TileParams p = {};
    p.f16 = f16, p.limit = desc->limit, p.err = err;
    p.N = T, p.g = g, p.u = u, p.ldp = ldm;
    if (need_mid) {
      const bool ok = map16(&p.a[0], o.w2.p, H, I, o.w2.ld, 64) && map16(&p.b[0], gy.p, T, H, gy.ld, nt);
      DS_REQUIRE(ok, DS_ECUDA, "gated_ffn_backward: tensor map encoding failed (hidden gradient)");
      p.M = I, p.K = H;
      p.out[0] = dg, p.out[1] = du, p.ldo = ldm;
      if ((st = run_tiles<DHID>(p, nt, s, false)) != DS_OK) return st;
      chained = true;
    }
    if (dx) {
      const bool ok = map16(&p.a[0], o.w1.p, I, H, o.w1.ld, 64) && map16(&p.a[1], o.w3.p, I, H, o.w3.ld, 64) &&
                      map16(&p.b[0], dg, T, I, ldm, nt) && map16(&p.b[1], du, T, I, ldm, nt);
      DS_REQUIRE(ok, DS_ECUDA, "gated_ffn_backward: tensor map encoding failed (dx)");
      p.M = H, p.K = I;
      p.out[0] = dx, p.ldo = H;
      if ((st = run_tiles<DX>(p, nt, s, chained)) != DS_OK) return st;
    }
  }
  // last launch: dW1 and dW3, and beside them dx, or dW2 of few rows
  PairParams p = {};
  p.f16 = f16, p.err = err;
  Sides sd[3];
  for (int k = 0; k < 2; ++k) {
    if (!wide || (k == 0) == (T >= 2 * I)) {
      if (k == 1 && !wide) break;
      if (dw1) grad(p, sd, dw1, I, H, og, o.x);
      if (dw3) grad(p, sd, dw3, I, H, ou, o.x);
      if (dw2 && !wide) grad(p, sd, dw2, H, I, gy, oh);
    } else if (dx) {
      Problem* q = add(p, STORE, T, H, I, 2, dx, H);
      q->b_mn = 1;
      sd[p.n - 1] = {q, og, o.w1, ou, o.w3};
    }
    if (k == 0) p.split = p.n;
  }
  return p.n ? run_pairs<STORE>(p, sd, s, chained) : DS_OK;
}

extern "C" int ds_gated_ffn_status(int32_t* err, void* stream) {
  DS_REQUIRE(err != nullptr, DS_EINVAL, "gated_ffn_status: null output");
  int* w = err_word();
  DS_REQUIRE(w != nullptr, DS_ECUDA, "gated_ffn_status: error word unavailable");
  return ds::take_error_word(w, err, static_cast<cudaStream_t>(stream));
}
