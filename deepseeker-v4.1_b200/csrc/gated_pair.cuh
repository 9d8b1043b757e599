// Pair kernel of the dense gated block: the products of many rows.
//
// A cluster of two CTAs computes 256 rows x 256 columns with one
// tcgen05.mma.cta_group::2 (M = 256, N = 256, K = 16): each CTA stages its
// 128 rows of A and half of B's 256 rows and holds its rows' accumulators, so
// a stage of 64 along k costs each SM 32 KB of L2 reads per 512 tensor
// cycles (a CTA alone on 128 x 256 would need 48 KB).  In the gate / up
// product the halves of B are 128 rows of W1 and the same 128 rows of W3, so
// every CTA ends up with g and u of the same features.
//
// Persistent, one cluster per two SMs, 320 threads a CTA: warp 0 copies
// (both CTAs signal the leader's barrier), warp 1 of the leader issues the
// MMAs, warps 2-9 empty one 256-column accumulator while the other fills.
// Lanes are rows here, so a thread owns runs of 32 columns of its row and
// stores them 16 bytes at a time.
#pragma once

#include "dense16.cuh"

namespace ds {
namespace dense {

enum Mode { GATED, PLAIN, DHID, DX, DW };

struct PairParams {
  CUtensorMap a[3], b[3];      // GATED: b = W1, W3; DX: segments; DW: three problems
  int M[3], N[3];              // rows and columns of each problem's result
  void* out[3];                // out[m * ldo + n], 16 bit (DHID: dg, du)
  int64_t ldo[3];
  int tiles[3];                // tiles of the problems up to and with this one
  int K;                       // contraction of one segment
  int f16;
  float limit;
  float* g;                    // f32 pre-activations [m * ldp + n]: written (GATED, may be null), read (DHID)
  float* u;
  int64_t ldp;
  int* err;
};

namespace pair {

constexpr int kStages = 6;
constexpr int kOperand = 2 * kBoxBytes;          // 128 rows x 64
constexpr int kStage = 2 * kOperand;
constexpr int kSmem = 1024 + kStages * kStage;
constexpr int kThreads = 320;
constexpr int kEpiWarps = 8;

template <int MODE>
struct Shape {
  static constexpr bool kAMn = MODE == DW;
  static constexpr bool kBMn = MODE == DHID || MODE == DX || MODE == DW;
  static constexpr int kSegs = MODE == DX ? 2 : 1;
  static constexpr int kProblems = MODE == DW ? 3 : 1;
  static constexpr int kCols = MODE == GATED ? 128 : 256;   // result columns of a tile
};

__device__ __forceinline__ uint32_t leader_addr(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}

// A tile load whose bytes are counted on the leader's barrier.
template <bool MN>
__device__ __forceinline__ void load_half(uint8_t* dst, const CUtensorMap* map, int r0, int k0, uint32_t bar) {
#pragma unroll
  for (int b = 0; b < (MN ? 2 : 1); ++b)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
        "[%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst + b * kBoxBytes)),
        "l"(map), "r"(MN ? r0 + 64 * b : k0), "r"(MN ? k0 : r0), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrives on this barrier of both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

__device__ __forceinline__ void arrive_leader(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

__device__ __forceinline__ void ld_x32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// 32 columns of one row, n of them inside the result; vec: 16-byte stores.
__device__ __forceinline__ void store16(uint16_t* dst, const float (&v)[32], int n, bool vec, int f16) {
  if (vec && n >= 32) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = pack16(v[8 * c + 2 * j], v[8 * c + 2 * j + 1], f16);
      *reinterpret_cast<uint4*>(dst + 8 * c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < n) dst[j] = to16(v[j], f16);
  }
}

// f32 rows of the saved pre-activations: their stride is a multiple of 8, so
// whole groups of four may be moved where at least one column is inside.
__device__ __forceinline__ void store_pre(float* dst, const float (&v)[32], int n) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (4 * c < n) *reinterpret_cast<float4*>(dst + 4 * c) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
}

__device__ __forceinline__ void load_pre(const float* src, float (&v)[32], int n) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const float4 t = 4 * c < n ? *reinterpret_cast<const float4*>(src + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
    v[4 * c] = t.x, v[4 * c + 1] = t.y, v[4 * c + 2] = t.z, v[4 * c + 3] = t.w;
  }
}

// A tile: problem z, first row and first column of the result.  Rows run
// fastest inside bands of 16 row tiles, so the CTAs at work at one time share
// both operands in L2.
template <int MODE>
__device__ __forceinline__ void locate(const PairParams& p, int tile, int& z, int& m0, int& n0) {
  z = 0;
  if (Shape<MODE>::kProblems > 1)
    while (z < Shape<MODE>::kProblems - 1 && tile >= p.tiles[z]) ++z;
  if (z) tile -= p.tiles[z - 1];
  const int mt = (p.M[z] + 255) / 256, nt = (p.N[z] + Shape<MODE>::kCols - 1) / Shape<MODE>::kCols;
  const int band = tile / (16 * nt), in = tile - band * 16 * nt, rows = min(16, mt - 16 * band);
  n0 = (in / rows) * Shape<MODE>::kCols;
  m0 = (16 * band + in % rows) * 256;
}

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1) pair_kernel(const __grid_constant__ PairParams p) {
  using C = Shape<MODE>;
  constexpr int S = kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ __align__(8) uint64_t full[S], empty[S], accfull[2], accempty[2];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1, pairs = gridDim.x >> 1, first = blockIdx.x >> 1;
  const int n_tiles = p.tiles[C::kProblems - 1];
  const int ksteps = (p.K + kBK - 1) / kBK, its = C::kSegs * ksteps;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accfull[b], 1);
      mbar_init(&accempty[b], 2 * kEpiWarps);
    }
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_base))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc5::fence_before();
  __syncthreads();
  cluster_sync();   // both CTAs' barriers exist before either signals the other
  tc5::fence_after();
  const uint32_t tb = tmem_base;
  volatile int* abort = &abort_flag;
  launch_dependents();
  wait_prior_grid();

  if (warp == 0) {
    // ------------------------------------------------------------ copies
    if (lane == 0) {
      int g = 0;
      for (int tile = first; tile < n_tiles; tile += pairs) {
        int z, m0, n0;
        locate<MODE>(p, tile, z, m0, n0);
        for (int it = 0; it < its; ++it, ++g) {
          const int s = g % S;
          if (g >= S && !grouped::wait_or_abort(&empty[s], ((g / S) - 1) & 1, abort, p.err)) goto drain;
          const int seg = C::kSegs > 1 && it >= ksteps ? 1 : 0, k0 = (it - seg * ksteps) * kBK;
          uint8_t* st = smem + s * kStage;
          const uint32_t bar = leader_addr(&full[s]);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kStage);
          load_half<C::kAMn>(st, &p.a[z + seg], m0 + 128 * rank, k0, bar);
          load_half<C::kBMn>(st + kOperand, &p.b[MODE == GATED ? rank : z + seg],
                             MODE == GATED ? n0 : n0 + 128 * rank, k0, bar);
        }
      }
    drain:
      // every stage has been read by the MMAs, and the signal of that has
      // arrived, before this CTA's shared memory goes
      for (int j = g - S < 0 ? 0 : g - S; j < g; ++j) mbar_wait_bounded(&empty[j % S], (j / S) & 1, 200000000ull);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMAs, by the leader
    if (rank == 0) {
      const uint32_t idesc = idesc16(p.f16, C::kAMn, C::kBMn, 256, 256);
      const uint64_t a0 = tile_desc<C::kAMn>(smem_u32(smem)), b0 = tile_desc<C::kBMn>(smem_u32(smem) + kOperand);
      int g = 0, li = 0;
      for (int tile = first; tile < n_tiles; tile += pairs, ++li) {
        const int b = li & 1;
        if (li >= 2 && !grouped::warp_wait(&accempty[b], ((li >> 1) - 1) & 1, abort, p.err)) break;
        tc5::fence_after();
        for (int it = 0; it < its; ++it, ++g) {
          const int s = g % S;
          if (!grouped::warp_wait(&full[s], (g / S) & 1, abort, p.err)) goto mma_out;
          tc5::fence_after();
          if (elect_one()) {
            const uint64_t ad = a0 + (uint64_t)((s * kStage) >> 4), bd = b0 + (uint64_t)((s * kStage) >> 4);
#pragma unroll
            for (int kk = 0; kk < kBK / 16; ++kk)
              mma(tb + b * 256, ad + kk * kStep16<C::kAMn>, bd + kk * kStep16<C::kBMn>, idesc, (it | kk) != 0);
            commit(&empty[s]);
          }
          __syncwarp();
        }
        if (elect_one()) commit(&accfull[b]);
        __syncwarp();
      }
    mma_out:;
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t bar[2] = {leader_addr(&accempty[0]), leader_addr(&accempty[1])};
    int li = 0;
    for (int tile = first; tile < n_tiles; tile += pairs, ++li) {
      int z, m0, n0;
      locate<MODE>(p, tile, z, m0, n0);
      const int b = li & 1;
      const int m = m0 + 128 * rank + 32 * q + lane;
      const bool row = m < p.M[z];
      const uint32_t acc = tc5::lane_quarter(tb + b * 256, q);
      uint16_t* out = static_cast<uint16_t*>(p.out[z]) + (int64_t)m * p.ldo[z];
      const bool vec = ((reinterpret_cast<uintptr_t>(p.out[z]) | (uintptr_t)(p.ldo[z] * 2)) & 15) == 0;
      constexpr int kPer = C::kCols / 2;                    // columns of this warp
      if constexpr (MODE == DHID) {
        // the first pre-activations are on their way while the MMAs still run
        const int n = n0 + half * kPer;
        if (row && n < p.N[0]) {
          asm volatile("prefetch.global.L2 [%0];" ::"l"(p.g + (int64_t)m * p.ldp + n));
          asm volatile("prefetch.global.L2 [%0];" ::"l"(p.u + (int64_t)m * p.ldp + n));
        }
      }
      if (!grouped::warp_wait(&accfull[b], (li >> 1) & 1, abort, p.err)) break;
      tc5::fence_after();
#pragma unroll 1
      for (int c = 0; c < kPer; c += 32) {
        const int col = half * kPer + c, n = n0 + col, left = p.N[z] - n;
        const bool in = row && left > 0;
        __syncwarp();
        if (MODE == GATED) {
          float gv[32], uv[32];
          ld_x32(acc + col, gv);
          ld_x32(acc + 128 + col, uv);
          tc5::wait_ld();
          if (in) {
            if (p.g) {
              store_pre(p.g + (int64_t)m * p.ldp + n, gv, left);
              store_pre(p.u + (int64_t)m * p.ldp + n, uv, left);
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) gv[j] = gate_unit(gv[j], uv[j], p.limit);
            store16(out + n, gv, left, vec, p.f16);
          }
        } else if (MODE == DHID) {
          float v[32], gv[32], uv[32];
          if (in) {
            load_pre(p.g + (int64_t)m * p.ldp + n, gv, left);
            load_pre(p.u + (int64_t)m * p.ldp + n, uv, left);
          }
          ld_x32(acc + col, v);
          tc5::wait_ld();
          if (in) {
#pragma unroll
            for (int j = 0; j < 32; ++j) gate_grad(gv[j], uv[j], v[j], p.limit, gv[j], uv[j]);
            store16(out + n, gv, left, vec, p.f16);
            store16(static_cast<uint16_t*>(p.out[1]) + (int64_t)m * p.ldo[1] + n, uv, left, vec, p.f16);
          }
        } else {
          float v[32];
          ld_x32(acc + col, v);
          tc5::wait_ld();
          if (in) store16(out + n, v, left, vec, p.f16);
        }
      }
      tc5::fence_before();
      __syncwarp();
      if (lane == 0) arrive_leader(bar[b]);
    }
  }
  tc5::fence_before();
  __syncthreads();
  cluster_sync();   // no CTA leaves while the other may still signal it
  if (warp == 1) {
    tc5::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tb) : "memory");
  }
}

}  // namespace pair
}  // namespace dense
}  // namespace ds
