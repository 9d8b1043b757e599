// Pair kernel of the microscaled 4-bit products: many rows of x.
//
// A pair computes 256 rows x 256 columns with tcgen05.mma.cta_group::2
// kind::mxf4 (M = 256, N = 256, K = 64).  A stage is 256 codes along k (one
// 128-byte line): 16 KB of x and 16 KB of weights a CTA per 512 tensor cycles.
// Scales: a CTA needs those of its own 128 rows of x and of all 256 weight
// rows, six atoms a stage, which the leader copies into both tensor memories
// (tcgen05.cp, ordered before the MMAs that read them).  In the gated product
// the weight halves are 128 rows of W1 and the same rows of W3.
//
// Tensor memory: 256 accumulator columns and two sets of 24 scale columns
// leave no room for a second accumulator.  So the epilogue first takes the
// accumulator into registers (128 columns a thread), hands it back, and only
// then rounds and stores while the next tile's MMAs run: the tensor cores
// wait for a few hundred cycles a tile, where tiles of 128 columns (with two
// accumulators) would ask 94 bytes a cycle of L2 for each SM instead of 64.
// Lanes are rows: a thread holds whole blocks of h and quantises them alone.
//
// 16384 x 4096 to 4096: 107 us, 5.1 PFLOP/s; gate / up of 16384 x 4096 x 2048:
// 110 us.  A tile takes 12.4 k cycles for 8.2 k of MMAs: about 1.5 k are the
// accumulator's hand-over, the rest stages that arrive late (1.17 GB from L2, 11
// TB/s; what L2 could give has not been measured apart).
#pragma once

#include "mx4.cuh"
#include "pair.cuh"

namespace ds {
namespace mx4 {

struct PairParams {
  CUtensorMap a, b[2];         // codes of x; of W (gated: W1, W3)
  CUtensorMap sa, sb[2];       // their scale atoms as lines of 512 bytes, boxes of two
  CUtensorMap out;             // linear with boxed = 1: result boxes of 128 bytes x 32 rows
  void* y;                     // linear: y[m * ldy + n]
  int64_t ldy;
  int out_dtype, boxed;
  uint8_t* hq;                 // gated: codes and atoms of h
  uint8_t* hs;
  float limit;
  int M, N;                    // rows of x, columns of the result
  int blocks;                  // blocks of 32 along the contraction
  int* err;
};

namespace pairs {

using namespace ds::pair;

constexpr int kOps = 32768;                       // 128 rows of x and of W, 128 bytes each
constexpr int kSf = 6 * kAtom;                    // x: two atoms along k; W: 2 x two
constexpr int kStage = kOps + kSf;                // 35 KB
constexpr int kSfCols = 24;

// As many stages as fit beside a result box per epilogue warp (the gated
// product stores h from registers).  The gated epilogue's arithmetic is as
// long as a tile's 16 stages, so it gets sixteen warps (with eight the block
// over 16384 x 4096 x 2048 took 128 us in this launch).
template <bool GATED>
struct Shape {
  static constexpr int kEpiWarps = GATED ? 16 : 8;
  static constexpr int kThreads = 32 * (2 + kEpiWarps);
  static constexpr int kStages = GATED ? 6 : 5;
  static constexpr int kSmem = 1024 + kStages * kStage + (GATED ? 0 : kEpiWarps * kBox);
  static_assert(kStage % 1024 == 0 && kSmem <= 226 * 1024, "shared memory of an SM");
};

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                    uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
      : "memory");
}

// An atom of each CTA's shared memory into four columns of its tensor memory.
__device__ __forceinline__ void copy_atom2(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Instruction descriptor: M = 256, N = 256, e2m1 operands, ue8m0 scales; sf_id
// (0 or 2): the pair of scale bytes that a step of 64 uses.
__device__ __forceinline__ constexpr uint32_t idesc(uint32_t sf_id) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | (32u << 17) | (1u << 23) | (16u << 24) | (sf_id << 29);
}

// The MMAs of a stage: steps of 64 codes, two an atom.
template <int STEPS>
__device__ __forceinline__ void stage_mmas(uint32_t acc, uint32_t tsf, uint64_t ops, uint64_t sf, bool first) {
#pragma unroll
  for (int a = 0; a < (STEPS + 1) / 2; ++a) {
    copy_atom2(tsf + 4 * a, sf + a * (kAtom >> 4));                              // x
    copy_atom2(tsf + 8 + 8 * a, sf + (2 + a) * (kAtom >> 4));                    // weight rows 0 .. 127
    copy_atom2(tsf + 12 + 8 * a, sf + (4 + a) * (kAtom >> 4));                   // 128 .. 255
  }
#pragma unroll
  for (int kk = 0; kk < STEPS; ++kk)
    mma(acc, ops + 2 * kk, ops + (16384 >> 4) + 2 * kk, idesc(kk & 1 ? 2 : 0), tsf + 4 * (kk >> 1),
        tsf + 8 + 8 * (kk >> 1), !(first && kk == 0));
}

// Rows run fastest inside bands of 16 row tiles (shared operands in L2).
template <bool GATED>
__device__ __forceinline__ void locate(const PairParams& p, int tile, int& m0, int& n0) {
  constexpr int cols = GATED ? 128 : 256;
  const int mt = (p.M + 255) / 256, nt = (p.N + cols - 1) / cols;
  const int band = tile / (16 * nt), in = tile - band * 16 * nt, rows = min(16, mt - 16 * band);
  n0 = (in / rows) * cols;
  m0 = (16 * band + in % rows) * 256;
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool f16) {
  if (f16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// One block of h: its 16 bytes of codes and its scale byte.
__device__ __forceinline__ uint4 quantize_block(const float* h, int& s) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) top = max(top, __float_as_uint(h[j]) & 0x7FFFFFFFu);
  s = scale_byte(top);
  const float inv = inv_scale(s);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = h[8 * i + j] * inv;
    w[i] = s == 255 ? 0u : e2m1x8(v);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool GATED>
__global__ void __launch_bounds__(Shape<GATED>::kThreads, 1) __cluster_dims__(2, 1, 1)
    pair_kernel(const __grid_constant__ PairParams p) {
  constexpr int S = Shape<GATED>::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ __align__(8) uint64_t full[S], empty[S], accfull, accempty;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1, pairs = gridDim.x >> 1, first = blockIdx.x >> 1;
  constexpr int cols = GATED ? 128 : 256;
  const int n_tiles = (p.M + 255) / 256 * ((p.N + cols - 1) / cols);
  const int chunks = (p.blocks + 3) / 4, its = (chunks + 1) / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&accfull, 1);
    mbar_init(&accempty, 2 * Shape<GATED>::kEpiWarps);
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) alloc512(&tmem_base);
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
        int m0, n0;
        locate<GATED>(p, tile, m0, n0);
        const int am = m0 + 128 * rank, bn = GATED ? n0 : n0 + 128 * rank;
        const int ra = (am >> 7) * chunks, rb = (n0 >> 7) * chunks;   // first atom lines
        for (int it = 0; it < its; ++it, ++g) {
          const int s = g % S;
          if (g >= S && !wait(&empty[s], ((g / S) - 1) & 1, abort, p.err)) goto drain;
          uint8_t* st = smem + s * kStage;
          const uint32_t bar = leader_addr(&full[s]);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kStage);
          load_box(st, &p.a, 128 * it, am, bar);
          load_box(st + 16384, &p.b[GATED ? rank : 0], 128 * it, bn, bar);
          // past the last atom the boxes read zeros (a scale, not NaN)
          load_box(st + kOps, &p.sa, 0, ra + 2 * it, bar);
          load_box(st + kOps + 2 * kAtom, &p.sb[0], 0, rb + 2 * it, bar);
          load_box(st + kOps + 4 * kAtom, &p.sb[GATED ? 1 : 0], 0, rb + 2 * it + (GATED ? 0 : chunks), bar);
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
      const uint64_t ops = tc5::sdesc_sw128(smem_u32(smem));
      const uint64_t sf0 = (uint64_t)(((smem_u32(smem) + kOps) >> 4) & 0x3FFFu) | (uint64_t)8 << 32 | (uint64_t)1 << 46;
      const int last = min(4, (p.blocks - 8 * (its - 1) + 1) / 2);   // steps of a tile's last stage
      int g = 0, li = 0;
      for (int tile = first; tile < n_tiles; tile += pairs, ++li) {
        if (li && !wait_all(&accempty, (li - 1) & 1, abort, p.err)) break;
        tc5::fence_after();
        for (int it = 0; it < its; ++it, ++g) {
          const int s = g % S;
          if (!wait_all(&full[s], (g / S) & 1, abort, p.err)) goto mma_out;
          tc5::fence_after();
          if (elect_one()) {
            const uint64_t od = ops + (uint64_t)((s * kStage) >> 4), sd = sf0 + (uint64_t)((s * kStage) >> 4);
            const uint32_t tsf = tb + 256 + (g & 1) * kSfCols;
            if (it < its - 1 || last == 4) stage_mmas<4>(tb, tsf, od, sd, it == 0);
            else if (last == 3) stage_mmas<3>(tb, tsf, od, sd, it == 0);
            else if (last == 2) stage_mmas<2>(tb, tsf, od, sd, it == 0);
            else stage_mmas<1>(tb, tsf, od, sd, it == 0);
            commit(&empty[s]);
          }
          __syncwarp();
        }
        if (elect_one()) commit(&accfull);
        __syncwarp();
      }
    mma_out:;
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3, part = (warp - 2) >> 2;
    uint8_t* box = smem + S * kStage + (warp - 2) * kBox;
    const uint32_t bar = leader_addr(&accempty), acc = tc5::lane_quarter(tb, q);
    int li = 0;
    for (int tile = first; tile < n_tiles; tile += pairs, ++li) {
      int m0, n0;
      locate<GATED>(p, tile, m0, n0);
      const int mw = m0 + 128 * rank + 32 * q, m = mw + lane;
      if (!wait_all(&accfull, li & 1, abort, p.err)) break;
      tc5::fence_after();
      // linear: columns part * 128 .. + 127; gated: features part * 32 .. + 31, gate and up
      float v[GATED ? 2 : 4][32];
      if (GATED) {
        ld_x32(acc + part * 32, v[0]);
        ld_x32(acc + 128 + part * 32, v[1]);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) ld_x32(acc + part * 128 + 32 * c, v[c]);
      }
      tc5::wait_ld();
      tc5::fence_before();
      __syncwarp();
      if (lane == 0) arrive_leader(bar);

      if constexpr (GATED) {
        const int blocks = (p.N + 31) / 32, hchunks = (blocks + 3) / 4, b = (n0 >> 5) + part, left = p.N - b * 32;
        // features past the result read unset scales: no part of the block
#pragma unroll
        for (int j = 0; j < 32; ++j) v[0][j] = j < left ? gate_unit(v[0][j], v[1][j], p.limit) : 0.0f;
        int s;
        const uint4 codes = quantize_block(v[0], s);
        if (m < p.M) {
          if (b < blocks) *reinterpret_cast<uint4*>(p.hq + ((int64_t)m * blocks + b) * 16) = codes;
          p.hs[atom_at(m, b, hchunks)] = (uint8_t)s;   // a tile is a chunk of four blocks
        }
      } else if (p.boxed) {
        const int per = p.out_dtype == DS_F32 ? 32 : 64;   // columns of a box
        const bool f16 = p.out_dtype == DS_F16;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int n = n0 + part * 128 + 32 * c;
          if (mw >= p.M || n >= p.N) continue;
          const bool opens = per == 32 || (c & 1) == 0, closes = per == 32 || (c & 1) || n + 32 >= p.N;
          if (opens) {
            if (lane == 0) box_wait_read<0>();   // the last store has read the box
            __syncwarp();
          }
          if (per == 32) {
            box_put(box, lane, v[c]);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *box_at(box, lane, 4 * (c & 1) + k) =
                  make_uint4(pack16(v[c][8 * k], v[c][8 * k + 1], f16), pack16(v[c][8 * k + 2], v[c][8 * k + 3], f16),
                             pack16(v[c][8 * k + 4], v[c][8 * k + 5], f16), pack16(v[c][8 * k + 6], v[c][8 * k + 7], f16));
          }
          if (closes) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              box_store(&p.out, per == 32 ? n : n - 32 * (c & 1), mw, box);
              box_commit();
            }
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int n = n0 + part * 128 + 32 * c;
          if (mw >= p.M || n >= p.N) continue;
          by_rows(box, lane, v[c], [&](int r, float y) {
            if (mw + r >= p.M || n + lane >= p.N) return;
            const int64_t at = (int64_t)(mw + r) * p.ldy + n + lane;
            if (p.out_dtype == DS_F32) static_cast<float*>(p.y)[at] = y;
            else if (p.out_dtype == DS_F16) static_cast<__half*>(p.y)[at] = __float2half_rn(y);
            else static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(y);
          });
        }
      }
      __syncwarp();
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

}  // namespace pairs
}  // namespace mx4
}  // namespace ds
