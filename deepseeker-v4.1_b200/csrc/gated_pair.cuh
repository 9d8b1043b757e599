// Pair kernel of the dense gated block: the products of many rows.
//
// A cluster of two CTAs computes 256 rows x NT columns (256, or 128 or 64
// where that would leave SMs without a tile) with one tcgen05.mma.cta_group::2
// (M = 256, N = NT, K = 16): each CTA stages its 128 rows of A and half of B's
// NT rows and holds its rows' accumulators, so at NT = 256 a stage of 64
// along k costs each SM 32 KB of L2 reads per 512 tensor cycles (a CTA alone
// on 128 x 256 would need 48 KB).  In the gate / up product the halves of B
// are NT / 2 rows of W1 and the same rows of W3, so every CTA ends up with g
// and u of the same features.
//
// Persistent, one cluster per two SMs, 320 threads a CTA: warp 0 copies
// (both CTAs signal the leader's barrier), warp 1 of the leader issues the
// MMAs, warps 2-9 empty one NT-column accumulator while the other fills.
// Lanes are rows here.  What the epilogue moves beside the accumulator goes
// through boxes of 32 rows in shared memory: a thread's own 16-byte accesses
// touch 32 rows at a time, and with them the gate / up launch that keeps g and
// u took 227 us instead of 200 (8192 x 4096 x 2048; 110 instead of 66 at a
// hidden size of 1024), the launch of dg and du 107 instead of 92 (hidden size
// 1024; with 4096 they are even, as the boxes cost that launch a stage).
//
// Bounded by the tensor cores under the power cap: forward and backward of
// 8192 x 4096 x 2048 take 878 us (1.41 PFLOP/s; nine plain library products of
// those sizes 844 us), 1.02 ms after seconds of load (984).
//
// A launch may hold two groups of problems with different contractions (the
// gradient of W2 beside that of the hidden values; those of W1 and W3 beside
// dx), so that the last wave of tiles is one of the shorter ones.
#pragma once

#include "dense16.cuh"
#include "pair.cuh"

namespace ds {
namespace dense {

enum Epilogue { STORE, GATED, HIDDEN };   // plain result; h (and g, u); dg and du

struct Problem {
  CUtensorMap a[2], b[2];      // operands of the segments; GATED: b = W1, W3
  CUtensorMap out;             // STORE with boxed = 1: the result in boxes of 64 columns x 32 rows
  void* c;                     // result [m * ldc + n], 16 bit
  int64_t ldc;
  int M, N;                    // rows and columns of the result
  int ksteps, segs;            // stages of one segment, segments
  int a_mn, b_mn;              // operand stored with m / n running fastest
  int epi, boxed;
  int tiles;                   // filled by the launch
};

struct PairParams {
  Problem pr[3];
  int n, split;                // problems; the first `split` form group 0
  CUtensorMap g, u;            // f32 pre-activations, boxes of 32 x 32
  CUtensorMap dg, du, h;       // results of HIDDEN and GATED, boxes of 32 x 32
  int keep;                    // GATED: write them
  Near near;
  int f16;
  float limit;
  int* err;
};

namespace pair {

using namespace ds::pair;

constexpr int kOperand = 2 * kBoxBytes;          // 128 rows x 64
constexpr int kEpiWarps = 8;
constexpr int kThreads = 32 * (2 + kEpiWarps);

template <int EPI, int NT>
struct Shape {
  // half of B: NT / 2 rows x 64; MN-major boxes are 64 wide whatever NT
  static constexpr int kHalf = NT == 256 ? kOperand : kBoxBytes;
  static constexpr int kStage = kOperand + kHalf;
  // per epilogue warp two boxes of 128-byte lines, for dg and du two of 64 more
  static constexpr int kBoxes = (EPI == HIDDEN ? 3 : 2) * kBox;
  static constexpr int kStages = (NT == 256 ? 5 : 6) - (EPI == HIDDEN ? 1 : 0);
  static constexpr int kSmem = 1024 + kStages * kStage + kEpiWarps * kBoxes;
  static_assert(kSmem <= 226 * 1024, "shared memory of an SM");
};

// Result columns of a tile.
__host__ __device__ constexpr int tile_cols(int epi, int nt) { return epi == GATED ? nt / 2 : nt; }

// ROWS of them; a K-major box holds them all, MN-major ones 64 each (of 32
// rows the rest of the box is not used).
template <bool MN, int ROWS>
__device__ __forceinline__ void load_half(uint8_t* dst, const CUtensorMap* map, int r0, int k0, uint32_t bar) {
  if (MN) {
    load_box(dst, map, r0, k0, bar);
    if (ROWS > 64) load_box(dst + kBoxBytes, map, r0 + 64, k0, bar);
  } else {
    load_box(dst, map, k0, r0, bar);
  }
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 columns of a row (lane = row) into a box of 64-byte lines, 16-byte pieces
// swizzled by line pairs.
__device__ __forceinline__ void slim_put(uint8_t* box, int lane, const float (&v)[32], int f16) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<uint4*>(box + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(pack16(v[8 * c], v[8 * c + 1], f16), pack16(v[8 * c + 2], v[8 * c + 3], f16),
                   pack16(v[8 * c + 4], v[8 * c + 5], f16), pack16(v[8 * c + 6], v[8 * c + 7], f16));
}

// Lists the values of 32 rows (lane = row, from m0 on) and `cols` columns (from
// n0 on) that lie close to the limit.  The distance goes by the largest weight
// norm of the columns.
__device__ __forceinline__ void near_find(const Near& p, int lane, const float (&g)[32], const float (&u)[32], int m0,
                                          int rows, int n0, int cols) {
  const bool row = m0 + lane < rows;
  const float nx = row ? p.nx[m0 + lane] : 0.0f;
  uint32_t near[2] = {0u, 0u};
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    // bits of non-negative values (and of NaN above them) order as the values
    const uint32_t w = lane < cols ? __float_as_uint(p.nw[z][n0 + lane]) : 0u;
    const float band = near_band(p, nx, __uint_as_float(__reduce_max_sync(0xffffffffu, w)));
#pragma unroll
    for (int j = 0; j < 32; ++j) near[z] |= (uint32_t)(z ? near_u(p, u[j], band) : near_g(p, g[j], band)) << j;
    near[z] &= cols < 32 ? (1u << cols) - 1u : 0xffffffffu;
    if (!row) near[z] = 0u;
  }
  near_list(p, near, m0 + lane, n0);
}

// The i-th tile of pair c.  Group 0 is dealt round robin.  A tile of group 1
// goes to the pair that is free first (ties: fewer tiles of group 0, then the
// lower index), which a pair can tell for itself: x pairs have one tile of
// group 0 more than the others, a tile of group 0 takes `a` stages and one of
// group 1 `b`, so the m-th tile of one of the y others comes after m * y + c'
// of theirs and the ceil(m - a / b) * x that start before it, and so on.
// Returns -1 after the last.
struct Dealer {
  int t0, t1, pairs, c, own0;
  int64_t a, b;
  __device__ __forceinline__ Dealer(const PairParams& p, int pairs_, int c_) : pairs(pairs_), c(c_) {
    t0 = p.pr[p.split - 1].tiles;
    t1 = p.pr[p.n - 1].tiles - t0;
    a = (int64_t)p.pr[0].ksteps * p.pr[0].segs;
    b = (int64_t)p.pr[p.n - 1].ksteps * p.pr[p.n - 1].segs;
    own0 = t0 / pairs + (c < t0 % pairs ? 1 : 0);
  }
  __device__ __forceinline__ int tile(int i) const {
    if (i < own0) return c + i * pairs;
    const int64_t m = i - own0, x = t0 % pairs, y = pairs - x;
    int64_t rank;
    if (c < x) rank = m * x + c + ((m * b + a) / b + 1) * y;
    else rank = m * y + (c - x) + (m * b > a ? (m * b - a + b - 1) / b : 0) * x;
    return rank < t1 ? t0 + (int)rank : -1;
  }
};

// A tile's problem, first row and first column of its result.  Rows run
// fastest inside bands of 16 row tiles, so the pairs at work at one time
// share both operands in L2.
template <int NT>
__device__ __forceinline__ int locate(const PairParams& p, int tile, int& m0, int& n0) {
  int z = 0;
  while (z < p.n - 1 && tile >= p.pr[z].tiles) ++z;
  if (z) tile -= p.pr[z - 1].tiles;
  const Problem& q = p.pr[z];
  const int cols = tile_cols(q.epi, NT), mt = (q.M + 255) / 256, nt = (q.N + cols - 1) / cols;
  const int band = tile / (16 * nt), in = tile - band * 16 * nt, rows = min(16, mt - 16 * band);
  n0 = (in / rows) * cols;
  m0 = (16 * band + in % rows) * 256;
  return z;
}

struct Rings {
  uint64_t *full, *empty;
  uint8_t* smem;
  volatile int* abort;
  int* err;
};

// The copies of one tile, stages g on.  False: a wait gave up.
template <bool AMN, bool BMN, int EPI, int NT>
__device__ __forceinline__ bool copy_tile(const Rings& r, const Problem& q, int rank, int m0, int n0, int& g) {
  using C = Shape<EPI, NT>;
  constexpr bool GATE = EPI == GATED;
  constexpr uint32_t kBytes = kOperand + (BMN ? (NT == 256 ? 2 : 1) * kBoxBytes : NT / 2 * 128);
  const int ksteps = q.ksteps, its = ksteps * q.segs, am = m0 + 128 * rank, bn = GATE ? n0 : n0 + NT / 2 * rank;
  for (int it = 0; it < its; ++it, ++g) {
    const int s = g % C::kStages;
    if (g >= C::kStages && !wait(&r.empty[s], ((g / C::kStages) - 1) & 1, r.abort, r.err)) return false;
    const int seg = it >= ksteps ? 1 : 0, k0 = (it - seg * ksteps) * kBK;
    uint8_t* st = r.smem + s * C::kStage;
    const uint32_t bar = leader_addr(&r.full[s]);
    if (rank == 0) mbar_arrive_expect_tx(&r.full[s], 2 * kBytes);
    load_half<AMN, 128>(st, &q.a[seg], am, k0, bar);
    load_half<BMN, NT / 2>(st + kOperand, &q.b[GATE ? rank : seg], bn, k0, bar);
  }
  return true;
}

// The MMAs of one tile, issued by an elected lane of a warp-uniform loop with
// descriptors that differ by constants (held in uniform registers; operand
// layouts read at run time instead made the 64 stages of a tile a fifth slower).
template <bool AMN, bool BMN, int EPI, int NT>
__device__ __forceinline__ bool mma_tile(const Rings& r, int its, int f16, uint32_t acc, int& g) {
  using C = Shape<EPI, NT>;
  const uint32_t idesc = idesc16(f16, AMN, BMN, 256, NT);
  const uint64_t a0 = tile_desc<AMN>(smem_u32(r.smem)), b0 = tile_desc<BMN>(smem_u32(r.smem) + kOperand);
  for (int it = 0; it < its; ++it, ++g) {
    const int s = g % C::kStages;
    if (!wait_all(&r.full[s], (g / C::kStages) & 1, r.abort, r.err)) return false;
    tc5::fence_after();
    if (elect_one()) {
      const uint64_t ad = a0 + (uint64_t)((s * C::kStage) >> 4), bd = b0 + (uint64_t)((s * C::kStage) >> 4);
#pragma unroll
      for (int kk = 0; kk < kBK / 16; ++kk) mma(acc, ad + kk * kStep16<AMN>, bd + kk * kStep16<BMN>, idesc, (it | kk) != 0);
      commit(&r.empty[s]);
    }
    __syncwarp();
  }
  return true;
}

// EPI: the launch's epilogue beside STORE.
template <int EPI, int NT>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1) pair_kernel(const __grid_constant__ PairParams p) {
  using C = Shape<EPI, NT>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ __align__(8) uint64_t full[S], empty[S], accfull[2], accempty[2], boxfull[kEpiWarps];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1;
  const Dealer dealer(p, gridDim.x >> 1, blockIdx.x >> 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accfull[b], 1);
      mbar_init(&accempty[b], 2 * kEpiWarps);
    }
    for (int w = 0; w < kEpiWarps; ++w) mbar_init(&boxfull[w], 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    alloc512(&tmem_base);
  }
  tc5::fence_before();
  __syncthreads();
  cluster_sync();   // both CTAs' barriers exist before either signals the other
  tc5::fence_after();
  const uint32_t tb = tmem_base;
  volatile int* abort = &abort_flag;
  launch_dependents();
  wait_prior_grid();

  const Rings r = {full, empty, smem, abort, p.err};

  if (warp == 0) {
    // ------------------------------------------------------------ copies
    if (lane == 0) {
      int g = 0;
      bool ok = true;
      for (int i = 0, tile; ok && (tile = dealer.tile(i)) >= 0; ++i) {
        int m0, n0;
        const Problem& q = p.pr[locate<NT>(p, tile, m0, n0)];
        if (EPI == GATED) ok = copy_tile<false, false, EPI, NT>(r, q, rank, m0, n0, g);
        else if (q.a_mn) ok = copy_tile<true, true, EPI, NT>(r, q, rank, m0, n0, g);
        else if (q.b_mn) ok = copy_tile<false, true, EPI, NT>(r, q, rank, m0, n0, g);
        else ok = copy_tile<false, false, EPI, NT>(r, q, rank, m0, n0, g);
      }
      // every stage has been read by the MMAs, and the signal of that has
      // arrived, before this CTA's shared memory goes
      for (int j = g - S < 0 ? 0 : g - S; j < g; ++j) mbar_wait_bounded(&empty[j % S], (j / S) & 1, 200000000ull);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMAs, by the leader
    if (rank == 0) {
      int g = 0;
      bool ok = true;
      for (int i = 0, tile; ok && (tile = dealer.tile(i)) >= 0; ++i) {
        int m0, n0;
        const Problem& q = p.pr[locate<NT>(p, tile, m0, n0)];
        const int its = q.ksteps * q.segs, b = i & 1;
        if (i >= 2 && !wait_all(&accempty[b], ((i >> 1) - 1) & 1, abort, p.err)) break;
        tc5::fence_after();
        const uint32_t acc = tb + b * NT;
        if (EPI != GATED && q.a_mn) ok = mma_tile<true, true, EPI, NT>(r, its, p.f16, acc, g);
        else if (EPI != GATED && q.b_mn) ok = mma_tile<false, true, EPI, NT>(r, its, p.f16, acc, g);
        else ok = mma_tile<false, false, EPI, NT>(r, its, p.f16, acc, g);
        if (ok && elect_one()) commit(&accfull[b]);
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int q4 = warp & 3, half = (warp - 2) >> 2;
    uint8_t* box0 = smem + S * C::kStage + (warp - 2) * C::kBoxes;
    uint8_t* box1 = box0 + kBox;
    uint8_t* slim = box1 + kBox;   // HIDDEN: boxes of dg and du
    uint64_t* loaded = &boxfull[warp - 2];
    int loads = 0, turn = 0;
    for (int i = 0, tile; (tile = dealer.tile(i)) >= 0; ++i) {
      int m0, n0;
      const Problem& q = p.pr[locate<NT>(p, tile, m0, n0)];
      const int b = i & 1, mw = m0 + 128 * rank + 32 * q4;
      const bool hidden = EPI == HIDDEN && q.epi == HIDDEN;
      const uint32_t acc = tc5::lane_quarter(tb + b * NT, q4);
      // the two warps of a lane quarter take turns at the columns inside the result
      const int nc = mw < q.M ? min(tile_cols(EPI, NT), q.N - n0) : 0;
      // the pre-activations of 32 columns come in while the accumulator of
      // the previous ones (or the MMAs) are still at work
      auto fetch = [&](int c) {
        if (lane == 0) {
          mbar_arrive_expect_tx(loaded, 2 * kBox);
          tma_load_2d(box0, &p.g, n0 + c, mw, loaded);
          tma_load_2d(box1, &p.u, n0 + c, mw, loaded);
        }
      };
      if (hidden && half * 32 < nc) fetch(half * 32);
      if (!wait_all(&accfull[b], (i >> 1) & 1, abort, p.err)) {
        if (hidden && half * 32 < nc && lane == 0) mbar_wait_bounded(loaded, loads & 1, 200000000ull);
        break;
      }
      tc5::fence_after();
      if (EPI == GATED) {
#pragma unroll 1
        for (int c = half * 32; c < nc; c += 64) {
          float gv[32], uv[32];
          __syncwarp();
          ld_x32(acc + c, gv);
          ld_x32(acc + NT / 2 + c, uv);
          tc5::wait_ld();
          if (p.keep) {
            if (lane == 0) box_wait_read<0>();
            __syncwarp();
            box_put(box0, lane, gv);
            box_put(box1, lane, uv);
            if (p.near.x) near_find(p.near, lane, gv, uv, mw, q.M, n0 + c, nc - c);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              box_store(&p.g, n0 + c, mw, box0);
              box_store(&p.u, n0 + c, mw, box1);
              box_commit();
            }
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) gv[j] = gate_unit(gv[j], uv[j], p.limit);
          if (lane == 0) box_wait_read<0>();   // g has left box 0
          __syncwarp();
          slim_put(box0, lane, gv, p.f16);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            box_store(&p.h, n0 + c, mw, box0);
            box_commit();
          }
        }
      } else if (hidden) {
#pragma unroll 1
        for (int c = half * 32; c < nc; c += 64) {
          float v[32], gv[32], uv[32];
          if (!wait_all(loaded, loads & 1, abort, p.err)) break;
          ++loads;
          box_get(box0, lane, gv);
          box_get(box1, lane, uv);
          // every lane's reads are done before the next boxes may land (without
          // the fence, reads still queued met the newer values)
          fence_proxy_async_smem();
          __syncwarp();
          if (c + 64 < nc) fetch(c + 64);
          __syncwarp();
          ld_x32(acc + c, v);
          tc5::wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) gate_grad(gv[j], uv[j], v[j], p.limit, gv[j], uv[j]);
          if (lane == 0) box_wait_read<0>();   // the previous columns have left
          __syncwarp();
          slim_put(slim, lane, gv, p.f16);
          slim_put(slim + kBox / 2, lane, uv, p.f16);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            box_store(&p.dg, n0 + c, mw, slim);
            box_store(&p.du, n0 + c, mw, slim + kBox / 2);
            box_commit();
          }
        }
      } else if (q.boxed) {
#pragma unroll 1
        for (int c = half * 64; c < nc; c += 128) {
          uint8_t* box = turn++ & 1 ? box1 : box0;   // the store before the last has read its box
          if (lane == 0) box_wait_read<1>();
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v[32];
            ld_x32(acc + c + 32 * e, v);
            tc5::wait_ld();
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *box_at(box, lane, 4 * e + k) =
                  make_uint4(pack16(v[8 * k], v[8 * k + 1], p.f16), pack16(v[8 * k + 2], v[8 * k + 3], p.f16),
                             pack16(v[8 * k + 4], v[8 * k + 5], p.f16), pack16(v[8 * k + 6], v[8 * k + 7], p.f16));
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            box_store(&q.out, n0 + c, mw, box);
            box_commit();
          }
        }
      } else {
        if (lane == 0) box_wait_read<0>();   // a boxed result may still leave from here
#pragma unroll 1
        for (int c = half * 32; c < nc; c += 64) {
          float v[32];
          __syncwarp();
          ld_x32(acc + c, v);
          tc5::wait_ld();
          by_rows(box0, lane, v, [&](int r, float y) {
            if (mw + r < q.M && c + lane < nc)
              static_cast<uint16_t*>(q.c)[(int64_t)(mw + r) * q.ldc + n0 + c + lane] = to16(y, p.f16);
          });
        }
      }
      // the boxes are free again before a later tile's loads overwrite them
      if (EPI == HIDDEN && !hidden) {
        if (lane == 0) box_wait_read<0>();
        fence_proxy_async_smem();
      }
      tc5::fence_before();
      __syncwarp();
      if (lane == 0) arrive_leader(leader_addr(&accempty[b]));
    }
    if (lane == 0) box_wait_all();
  }
  tc5::fence_before();
  __syncthreads();
  cluster_sync();   // no CTA leaves while the other may still signal it
  if (warp == 1) {
    tc5::fence_after();
    dealloc512(tb);
  }
}

}  // namespace pair
}  // namespace dense
}  // namespace ds
