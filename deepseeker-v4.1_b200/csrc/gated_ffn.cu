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
// as much error as the rounding of the result itself).
//
// Tile kernel (every product of every size): one CTA computes 128 features
// (the MMA's lanes) x NT tokens or columns over a slice of the contraction.
// The slices of one tile are the CTAs of a cluster: they leave their f32
// partial tiles in shared memory and each adds up a share of the columns
// through distributed shared memory, in slice order, so results do not
// depend on timing.  Weights on the lanes mean that one token costs a
// 16-wide MMA and the weights stream once.
#include <algorithm>
#include <cooperative_groups.h>
#include <string.h>

#include "gated_pair.cuh"

namespace ds {
namespace dense {
namespace {

namespace cg = cooperative_groups;

enum Mode { GATE_UP, PLAIN, DHID, DX, DW };

template <int MODE>
struct ModeOf {
  static constexpr bool kAMn = MODE == DHID || MODE == DX || MODE == DW;   // A stored with m running fastest
  static constexpr bool kBMn = MODE == DW;
  static constexpr int kMats = MODE == GATE_UP ? 2 : 1;                      // accumulators (W1 and W3 share x)
  static constexpr int kSegs = MODE == DX ? 2 : 1;                         // dg W1 and du W3 in one accumulator
  static constexpr int kProblems = MODE == DW ? 3 : 1;
};

struct TileParams {
  CUtensorMap a[3], b[3];
  int M[3], N[3];              // features (lanes) and tokens / columns of each problem
  void* out[3];                // out[n * ldo + m], 16 bit
  int64_t ldo[3];
  int K;                       // contraction of one segment
  int f16;
  float limit;
  float* g;                    // f32 pre-activations [n * ldp + m]: written (GATED, may be null), read (DHID)
  float* u;
  int64_t ldp;
  int* err;
};

__device__ int g_err;          // bit 1: a bounded wait gave up

template <int MODE, int NT>
struct TileShape {
  using Md = ModeOf<MODE>;
  static constexpr int kA = Md::kMats * 2 * kBoxBytes;
  static constexpr int kB = NT * 128;
  static constexpr int kStage = kA + kB;
  static constexpr int kStages = std::min(8, 200 * 1024 / kStage);
  static constexpr int kSmem = 1024 + kStages * kStage;
  static constexpr int kCols = Md::kMats * NT < 32 ? 32 : Md::kMats * NT;
  static_assert(kStage % 1024 == 0 && kStages * kStage >= Md::kMats * NT * 128 * 4, "stages hold the partial tile");
  static_assert(!Md::kBMn || NT % 64 == 0, "MN-major tiles come in boxes of 64");
};

constexpr int kTileThreads = 192;   // warp 0 copies, warp 1 MMA, warps 2-5 epilogue

// What becomes of one element (m, n) of the accumulator(s).
template <int MODE>
__device__ __forceinline__ void tile_store(const TileParams& p, int z, int m, int n, float v0, float v1) {
  uint16_t* out = static_cast<uint16_t*>(p.out[z]) + (int64_t)n * p.ldo[z] + m;
  if constexpr (MODE == GATE_UP) {
    if (p.g) {
      p.g[(int64_t)n * p.ldp + m] = v0;
      p.u[(int64_t)n * p.ldp + m] = v1;
    }
    *out = to16(gate_unit(v0, v1, p.limit), p.f16);
  } else if constexpr (MODE == DHID) {
    float dg, du;
    gate_grad(p.g[(int64_t)n * p.ldp + m], p.u[(int64_t)n * p.ldp + m], v0, p.limit, dg, du);
    *out = to16(dg, p.f16);
    static_cast<uint16_t*>(p.out[1])[(int64_t)n * p.ldo[1] + m] = to16(du, p.f16);
  } else {
    *out = to16(v0, p.f16);
  }
}

template <int MODE, int NT>
__global__ void __launch_bounds__(kTileThreads, 1) tile_kernel(const __grid_constant__ TileParams p) {
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
  const int z = blockIdx.z;
  const int m0 = (blockIdx.x / slices) * 128, n0 = blockIdx.y * NT;
  if (m0 >= p.M[z] || n0 >= p.N[z]) return;   // the whole cluster: its CTAs share m0 and n0
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
  wait_prior_grid();

  if (warp == 0) {
    if (lane == 0) {
      int g = 0;
      for (int it = it0; it < it1; ++it, ++g) {
        const int s = g % S;
        if (g >= S && !grouped::wait_or_abort(&empty[s], ((g / S) - 1) & 1, abort, p.err)) break;
        const int seg = it / ksteps, k0 = (it - seg * ksteps) * kBK;
        uint8_t* st = smem + s * C::kStage;
        mbar_arrive_expect_tx(&full[s], C::kStage);
        load_tile<Md::kAMn, 128>(st, &p.a[z + seg], m0, k0, &full[s]);
        if (Md::kMats == 2) load_tile<Md::kAMn, 128>(st + 2 * kBoxBytes, &p.a[1], m0, k0, &full[s]);
        load_tile<Md::kBMn, NT>(st + C::kA, &p.b[z + seg], n0, k0, &full[s]);
      }
      // never leave with copies in flight into this CTA's shared memory
      for (int j = g - S < 0 ? 0 : g - S; j < g; ++j) mbar_wait_bounded(&full[j % S], (j / S) & 1, 200000000ull);
    }
  } else if (warp == 1) {
    const uint32_t idesc = idesc16(p.f16, Md::kAMn, Md::kBMn, 128, NT);
    const uint64_t a0 = tile_desc<Md::kAMn>(smem_u32(smem)), b0 = tile_desc<Md::kBMn>(smem_u32(smem) + C::kA);
    for (int g = 0; g < it1 - it0; ++g) {
      const int s = g % S;
      if (!grouped::warp_wait(&full[s], (g / S) & 1, abort, p.err)) break;
      tc5::fence_after();
      if (elect_one()) {
        const uint64_t ad = a0 + (uint64_t)((s * C::kStage) >> 4), bd = b0 + (uint64_t)((s * C::kStage) >> 4);
#pragma unroll
        for (int kk = 0; kk < kBK / 16; ++kk) {
          tc5::mma_bf16(tb, ad + kk * kStep16<Md::kAMn>, bd + kk * kStep16<Md::kBMn>, idesc, (g | kk) != 0);
          if (Md::kMats == 2)
            tc5::mma_bf16(tb + NT, ad + ((2 * kBoxBytes) >> 4) + kk * kStep16<Md::kAMn>,
                          bd + kk * kStep16<Md::kBMn>, idesc, (g | kk) != 0);
        }
        tc5::commit(&empty[s]);
      }
      __syncwarp();
    }
    // all issued MMAs complete before the accumulators are read or released
    if (elect_one()) tc5::commit(&accfull);
    __syncwarp();
    grouped::warp_wait(&accfull, 0, abort, p.err);
  } else {
    grouped::warp_wait(&accfull, 0, abort, p.err);
  }
  tc5::fence_after();

  // ---- epilogue: thread = one feature (lane of tensor memory)
  const int q = warp & 3, mi = q * 32 + lane, m = m0 + mi;
  const int nv = min(NT, p.N[z] - n0);
  float* part = reinterpret_cast<float*>(smem);   // [mats][NT][128]
  if (warp >= 2) {
    for (int c0 = 0; c0 < nv; c0 += 16) {
      float v[Md::kMats][16];
#pragma unroll
      for (int t = 0; t < Md::kMats; ++t) tc5::ld_x16_nowait(tc5::lane_quarter(tb + t * NT + c0, q), v[t]);
      tc5::wait_ld();
      if (slices > 1) {
#pragma unroll
        for (int t = 0; t < Md::kMats; ++t)
#pragma unroll
          for (int j = 0; j < 16; ++j) part[(t * NT + c0 + j) * 128 + mi] = v[t][j];
      } else if (m < p.M[z]) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c0 + j < nv) tile_store<MODE>(p, z, m, n0 + c0 + j, v[0][j], v[Md::kMats - 1][j]);
      }
    }
  }
  if (slices > 1) {
    cluster.sync();
    if (warp >= 2 && m < p.M[z]) {
      for (int n = slice; n < nv; n += slices) {
        float v0 = 0.0f, v1 = 0.0f;
        for (int r = 0; r < slices; ++r) {
          const float* src = cluster.map_shared_rank(part, r);
          v0 += src[n * 128 + mi];
          if (Md::kMats == 2) v1 += src[(NT + n) * 128 + mi];
        }
        tile_store<MODE>(p, z, m, n0 + n, v0, v1);
      }
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

// Copies a strided 16-bit matrix into rows of ldd (a multiple of 8) elements,
// zeros behind the columns: the form that the tensor maps need of an operand
// whose base or row stride is no multiple of 16 bytes.
__global__ void __launch_bounds__(256) pack_kernel(const uint16_t* __restrict__ src, int64_t rows, int cols,
                                                   int64_t lds, uint16_t* __restrict__ dst, int ldd) {
  const int64_t n = rows * (ldd / 8);
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / (ldd / 8);
    const int c = (int)(i - r * (ldd / 8)) * 8;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < cols) w[j >> 1] |= (uint32_t)src[r * lds + c + j] << (16 * (j & 1));
    *reinterpret_cast<uint4*>(dst + r * ldd + c) = make_uint4(w[0], w[1], w[2], w[3]);
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

// Replaces the operand by its packed copy in the workspace where it needs one.
int place(Operand& o, char*& ws, cudaStream_t s) {
  const size_t bytes = copy_bytes(o);
  if (bytes == 0) return DS_OK;
  const int ldd = (int)up8(o.cols);
  const int64_t work = o.rows * (ldd / 8);
  const int grid = (int)std::min<int64_t>((work + 255) / 256, (int64_t)ds::sm_count() * 16);
  pack_kernel<<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(o.p), o.rows, (int)o.cols, o.ld,
                                   reinterpret_cast<uint16_t*>(ws), ldd);
  DS_CHECK_LAUNCH("pack_kernel");
  o.p = ws;
  o.ld = ldd;
  ws += bytes;
  return DS_OK;
}

int* err_word() {
  void* p = nullptr;
  return cudaGetSymbolAddress(&p, g_err) == cudaSuccess ? static_cast<int*>(p) : nullptr;
}

template <int MODE, int NT>
int launch_tiles(const TileParams& p, int max_m, int max_n, int slices, cudaStream_t s, bool chained) {
  using C = TileShape<MODE, NT>;
  DS_CHECK_CUDA(cudaFuncSetAttribute(tile_kernel<MODE, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((max_m + 127) / 128 * slices), (unsigned)((max_n + NT - 1) / NT),
                     ModeOf<MODE>::kProblems);
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
  using Md = ModeOf<MODE>;
  int max_m = 0, max_n = 0;
  int64_t tiles = 0;
  for (int z = 0; z < Md::kProblems; ++z) {
    max_m = std::max(max_m, p.M[z]);
    max_n = std::max(max_n, p.N[z]);
    tiles += (int64_t)((p.M[z] + 127) / 128) * ((p.N[z] + nt - 1) / nt);
  }
  const int slices = slices_for(tiles, Md::kSegs * ((p.K + kBK - 1) / kBK));
  if constexpr (MODE != DW) {
    if (nt == 16) return launch_tiles<MODE, 16>(p, max_m, max_n, slices, s, chained);
    if (nt == 32) return launch_tiles<MODE, 32>(p, max_m, max_n, slices, s, chained);
    if (nt == 64) return launch_tiles<MODE, 64>(p, max_m, max_n, slices, s, chained);
  }
  return launch_tiles<MODE, 128>(p, max_m, max_n, slices, s, chained);
}

// ---- pair kernel

// Tiles of an [M, N] result in the pair kernel.
int64_t pair_tiles(int epi, int64_t M, int64_t N) {
  const int c = pair::tile_cols(epi);
  return (M + 255) / 256 * ((N + c - 1) / c);
}

// The pair kernel takes the products with at least this many tiles.
constexpr int kPairMin = 37;

// Adds the problem c = a b^T (a and b given with their own layouts; k the
// contraction) to a launch.
Problem* add(PairParams& p, int epi, int64_t M, int64_t N, int64_t k, void* c, int64_t ldc) {
  Problem& q = p.pr[p.n++];
  q.epi = epi, q.M = (int)M, q.N = (int)N;
  q.ksteps = (int)((k + kBK - 1) / kBK), q.segs = 1;
  q.c[0] = c, q.ldc = ldc;
  q.tiles = (int)(pair_tiles(epi, M, N) + (p.n > 1 ? p.pr[p.n - 2].tiles : 0));
  return &q;
}

// Boxes of the result where its rows allow them.
bool box_result(Problem& q) {
  q.boxed = q.epi == STORE && direct(q.c[0], q.ldc);
  return !q.boxed || map16(&q.out, q.c[0], q.M, q.N, q.ldc, 32);
}

// Operand maps: box rows by the way the operand is stored.
bool side(CUtensorMap* m, const Operand& o, int mn) { return map16(m, o.p, o.rows, o.cols, o.ld, mn ? 64 : 128); }

template <int EPI>
int run_pairs(PairParams& p, cudaStream_t s, bool chained) {
  if (p.split == 0) p.split = p.n;
  DS_CHECK_CUDA(cudaFuncSetAttribute(pair::pair_kernel<EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, pair::kSmem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * std::min(p.pr[p.n - 1].tiles, ds::sm_count() / 2)));
  cfg.blockDim = dim3(pair::kThreads);
  cfg.dynamicSmemBytes = pair::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = chained ? 1 : 0;
  DS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, pair::pair_kernel<EPI>, p));
  return DS_OK;
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

size_t forward_bytes(const DsGatedFfn* d, bool own_h) {
  const Parts o = parts_of(d);
  return copy_bytes(o.x) + copy_bytes(o.w1) + copy_bytes(o.w3) + copy_bytes(o.w2) + (own_h ? mid_bytes(d) : 0);
}

size_t backward_bytes(const DsGatedFfn* d, const void* dy, int64_t ld_dy) {
  const Operand g = {dy, d->tokens, d->hidden, ld_dy};
  return forward_bytes(d, false) + copy_bytes(g) + 2 * mid_bytes(d);
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
  for (Operand* q : {&o.x, &o.w1, &o.w3, &o.w2})
    if ((st = place(*q, ws, s)) != DS_OK) return st;
  if (!h) h = ws;
  const int64_t ldm = up8(I);
  int* err = err_word();
  DS_REQUIRE(err != nullptr, DS_ECUDA, "gated_ffn: error word unavailable");
  const int f16 = desc->dtype == DS_F16;
  float* pre_u = pre ? pre + (int64_t)T * ldm : nullptr;
  const int nt = token_tile(T);

  if (pair_tiles(GATED, T, I) >= kPairMin) {
    PairParams p = {};
    p.f16 = f16, p.limit = desc->limit, p.err = err, p.keep = pre != nullptr;
    Problem& q = *add(p, GATED, T, I, H, h, ldm);
    const bool ok = side(&q.a[0], o.x, 0) && side(&q.b[0], o.w1, 0) && side(&q.b[1], o.w3, 0) &&
                    (!pre || (map32(&p.g, pre, T, I, ldm) && map32(&p.u, pre_u, T, I, ldm)));
    DS_REQUIRE(ok, DS_ECUDA, "gated_ffn: tensor map encoding failed (gate / up)");
    st = run_pairs<GATED>(p, s, false);
  } else {
    TileParams p = {};
    p.f16 = f16, p.limit = desc->limit, p.err = err;
    const bool ok = map16(&p.a[0], o.w1.p, I, H, o.w1.ld, 128) && map16(&p.a[1], o.w3.p, I, H, o.w3.ld, 128) &&
                    map16(&p.b[0], o.x.p, T, H, o.x.ld, nt);
    DS_REQUIRE(ok, DS_ECUDA, "gated_ffn: tensor map encoding failed (gate / up)");
    p.M[0] = I, p.N[0] = T, p.K = H;
    p.out[0] = h, p.ldo[0] = ldm;
    p.g = pre, p.u = pre_u, p.ldp = ldm;
    st = run_tiles<GATE_UP>(p, nt, s, false);
  }
  if (st != DS_OK) return st;

  const Operand oh = {h, T, I, ldm};
  if (pair_tiles(STORE, T, H) >= kPairMin) {
    PairParams p = {};
    p.f16 = f16, p.err = err;
    Problem& q = *add(p, STORE, T, H, I, y, H);
    const bool ok = side(&q.a[0], oh, 0) && side(&q.b[0], o.w2, 0) && box_result(q);
    DS_REQUIRE(ok, DS_ECUDA, "gated_ffn: tensor map encoding failed (down)");
    return run_pairs<STORE>(p, s, true);
  }
  TileParams p = {};
  p.f16 = f16, p.err = err;
  const bool ok = map16(&p.a[0], o.w2.p, H, I, o.w2.ld, 128) && map16(&p.b[0], h, T, I, ldm, nt);
  DS_REQUIRE(ok, DS_ECUDA, "gated_ffn: tensor map encoding failed (down)");
  p.M[0] = H, p.N[0] = T, p.K = I;
  p.out[0] = y, p.ldo[0] = H;
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
  for (Operand* q : {&o.x, &o.w1, &o.w3, &o.w2, &gy})
    if ((st = place(*q, ws, s)) != DS_OK) return st;
  const int64_t ldm = up8(I);
  void* dg = ws;
  void* du = ws + mid_bytes(desc);
  int* err = err_word();
  DS_REQUIRE(err != nullptr, DS_ECUDA, "gated_ffn_backward: error word unavailable");
  const int f16 = desc->dtype == DS_F16;
  float* g = const_cast<float*>(pre);
  float* u = g + (int64_t)T * ldm;
  const int nt = token_tile(T);
  const Operand og = {dg, T, I, ldm}, ou = {du, T, I, ldm}, oh = {h, T, I, ldm};
  const bool need_mid = dx || dw1 || dw3;
  const int64_t wtiles = pair_tiles(STORE, H, I);
  bool ok = true, chained = false;

  // first launch: dg and du from dy, and beside them dW2, which needs neither
  const bool mid_pair = need_mid && pair_tiles(HIDDEN, T, I) >= kPairMin;
  const bool dw2_pair = dw2 && wtiles * ((dw1 != nullptr) + (dw3 != nullptr) + 1) >= kPairMin;
  if (mid_pair || dw2_pair) {
    PairParams p = {};
    p.f16 = f16, p.limit = desc->limit, p.err = err;
    const bool long_first = T >= H;   // the longer tiles are dealt first
    for (int k = 0; k < 2; ++k) {
      if ((k == 0) == long_first) {
        if (!dw2_pair) continue;
        Problem& q = *add(p, STORE, H, I, T, dw2, I);
        q.a_mn = q.b_mn = 1;
        ok = ok && side(&q.a[0], gy, 1) && side(&q.b[0], oh, 1) && box_result(q);
      } else if (mid_pair) {
        Problem& q = *add(p, HIDDEN, T, I, H, dg, ldm);
        q.c[1] = du, q.b_mn = 1;
        ok = ok && side(&q.a[0], gy, 0) && side(&q.b[0], o.w2, 1) && map32(&p.g, g, T, I, ldm) &&
             map32(&p.u, u, T, I, ldm);
      }
      if (k == 0) p.split = p.n;
    }
    DS_REQUIRE(ok, DS_ECUDA, "gated_ffn_backward: tensor map encoding failed (hidden gradient)");
    if ((st = run_pairs<HIDDEN>(p, s, false)) != DS_OK) return st;
    chained = true;
  }
  if (need_mid && !mid_pair) {
    TileParams p = {};
    p.f16 = f16, p.limit = desc->limit, p.err = err;
    ok = map16(&p.a[0], o.w2.p, H, I, o.w2.ld, 64) && map16(&p.b[0], gy.p, T, H, gy.ld, nt);
    DS_REQUIRE(ok, DS_ECUDA, "gated_ffn_backward: tensor map encoding failed (hidden gradient)");
    p.M[0] = I, p.N[0] = T, p.K = H;
    p.out[0] = dg, p.out[1] = du, p.ldo[0] = p.ldo[1] = ldm;
    p.g = g, p.u = u, p.ldp = ldm;
    if ((st = run_tiles<DHID>(p, nt, s, chained)) != DS_OK) return st;
    chained = true;
  }

  // second launch: dW1 and dW3, and beside them dx
  void* const dw[2] = {dw1, dw3};
  const Operand* const mid[2] = {&og, &ou};
  const int64_t w13 = wtiles * ((dw1 != nullptr) + (dw3 != nullptr));
  const bool dx_pair = dx && pair_tiles(STORE, T, H) >= kPairMin, dw_pair = w13 >= kPairMin;
  if (dx_pair || dw_pair) {
    PairParams p = {};
    p.f16 = f16, p.err = err;
    const bool long_first = T >= 2 * I;
    for (int k = 0; k < 2; ++k) {
      if ((k == 0) == long_first) {
        for (int z = 0; z < 2 && dw_pair; ++z) {
          if (!dw[z]) continue;
          Problem& q = *add(p, STORE, I, H, T, dw[z], H);
          q.a_mn = q.b_mn = 1;
          ok = ok && side(&q.a[0], *mid[z], 1) && side(&q.b[0], o.x, 1) && box_result(q);
        }
      } else if (dx_pair) {
        Problem& q = *add(p, STORE, T, H, I, dx, H);
        q.b_mn = 1, q.segs = 2;
        ok = ok && side(&q.a[0], og, 0) && side(&q.a[1], ou, 0) && side(&q.b[0], o.w1, 1) && side(&q.b[1], o.w3, 1) &&
             box_result(q);
      }
      if (k == 0) p.split = p.n;
    }
    DS_REQUIRE(ok, DS_ECUDA, "gated_ffn_backward: tensor map encoding failed (dx, dW1, dW3)");
    if ((st = run_pairs<STORE>(p, s, chained)) != DS_OK) return st;
    chained = true;
  }
  if (dx && !dx_pair) {
    TileParams p = {};
    p.f16 = f16, p.err = err;
    ok = map16(&p.a[0], o.w1.p, I, H, o.w1.ld, 64) && map16(&p.a[1], o.w3.p, I, H, o.w3.ld, 64) &&
         map16(&p.b[0], dg, T, I, ldm, nt) && map16(&p.b[1], du, T, I, ldm, nt);
    DS_REQUIRE(ok, DS_ECUDA, "gated_ffn_backward: tensor map encoding failed (dx)");
    p.M[0] = H, p.N[0] = T, p.K = I;
    p.out[0] = dx, p.ldo[0] = H;
    if ((st = run_tiles<DX>(p, nt, s, chained)) != DS_OK) return st;
    chained = true;
  }
  // what weight gradients are left: dW1 and dW3 [I, H] from x against dg and du, dW2 [H, I] from h against dy
  void* const left[3] = {dw_pair ? nullptr : dw1, dw_pair ? nullptr : dw3, dw2_pair ? nullptr : dw2};
  if (left[0] || left[1] || left[2]) {
    const Operand grads[3] = {og, ou, gy}, acts[3] = {o.x, o.x, oh};
    TileParams p = {};
    p.f16 = f16, p.err = err, p.K = T;
    for (int z = 0; z < 3; ++z) {
      if (!left[z]) continue;     // M = 0: the problem's CTAs return at once
      p.M[z] = (int)acts[z].cols, p.N[z] = (int)grads[z].cols;
      p.out[z] = left[z], p.ldo[z] = acts[z].cols;
      ok = map16(&p.a[z], acts[z].p, T, acts[z].cols, acts[z].ld, 64) &&
           map16(&p.b[z], grads[z].p, T, grads[z].cols, grads[z].ld, 64);
      DS_REQUIRE(ok, DS_ECUDA, "gated_ffn_backward: tensor map encoding failed (weight gradients)");
    }
    return run_tiles<DW>(p, 128, s, chained);
  }
  return DS_OK;
}

extern "C" int ds_gated_ffn_status(int32_t* err, void* stream) {
  DS_REQUIRE(err != nullptr, DS_EINVAL, "gated_ffn_status: null output");
  int* w = err_word();
  DS_REQUIRE(w != nullptr, DS_ECUDA, "gated_ffn_status: error word unavailable");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DS_CHECK_CUDA(cudaMemcpyAsync(err, w, sizeof(int), cudaMemcpyDefault, s));
  DS_CHECK_CUDA(cudaMemsetAsync(w, 0, sizeof(int), s));
  return DS_OK;
}
