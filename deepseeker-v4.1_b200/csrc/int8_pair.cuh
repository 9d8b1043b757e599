// Pair kernel of the 8-bit integer product: many rows of x.
//
// A pair computes 256 rows x NT columns (256, 128 or 64) with
// tcgen05.mma.cta_group::2 kind::i8 (M = 256, N = NT, K = 32).  A stage is 128
// codes along k (one 128-byte line): 16 KB of x and NT / 2 lines of weights a
// CTA.  Persistent, one cluster per two SMs: warp 0 copies, warp 1 of the
// leader issues the MMAs, warps 2-9 empty one accumulator while the other
// fills.  Lanes are rows: a thread multiplies its row's sums by the row's and
// the columns' scales and rounds once.
//
// 16384 x 4096 to 4096: 154 to 163 us, 3.4 to 3.6 POP/s, bounded by the tensor
// cores under the power cap (pipe 92 % active at 1.6 GHz; 64 bytes a cycle of L2
// for each SM at 256 columns).  A tile's epilogue is 1.5 k cycles of its 16 k.
#pragma once

#include "int8.cuh"

namespace ds {
namespace int8 {

struct PairParams {
  CUtensorMap a, b;            // codes of x, of W
  CUtensorMap out;             // boxed = 1: result boxes of 128 bytes x 32 rows
  const float *sx, *sw;
  void* y;                     // y[m * ldy + n]
  int64_t ldy;
  int out_dtype, boxed;
  int M, N;                    // rows of x, columns of the result
  int ksteps;                  // stages of 128 codes
  int* err;
};

namespace pairs {

using namespace ds::pair;

constexpr int kEpiWarps = 8;
constexpr int kThreads = 32 * (2 + kEpiWarps);

template <int NT>
struct Shape {
  static constexpr int kStage = 16384 + NT / 2 * 128;
  // as many as fit beside a result box and the scales of 32 columns per epilogue warp
  static constexpr int kStages = NT == 256 ? 6 : NT == 128 ? 8 : 9;
  static constexpr int kSmem = 1024 + kStages * kStage + kEpiWarps * kBox;
  static_assert(kStage % 1024 == 0 && kSmem + kEpiWarps * 32 * 4 + 512 <= 227 * 1024, "shared memory of an SM");
};

// Rows run fastest inside bands of 16 row tiles (shared operands in L2).
template <int NT>
__device__ __forceinline__ void locate(const PairParams& p, int tile, int& m0, int& n0) {
  const int mt = (p.M + 255) / 256, nt = (p.N + NT - 1) / NT;
  const int band = tile / (16 * nt), in = tile - band * 16 * nt, rows = min(16, mt - 16 * band);
  n0 = (in / rows) * NT;
  m0 = (16 * band + in % rows) * 256;
}

// 32 columns of the accumulator times their scales; s: the columns' scales in shared memory.
__device__ __forceinline__ void take(uint32_t acc, float sx, const float* s, float (&v)[32]) {
  ld_x32(acc, v);
  tc5::wait_ld();
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const float4 w = *reinterpret_cast<const float4*>(s + j);
    v[j] = scaled(__float_as_int(v[j]), sx, w.x), v[j + 1] = scaled(__float_as_int(v[j + 1]), sx, w.y);
    v[j + 2] = scaled(__float_as_int(v[j + 2]), sx, w.z), v[j + 3] = scaled(__float_as_int(v[j + 3]), sx, w.w);
  }
}

template <int NT>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1) pair_kernel(const __grid_constant__ PairParams p) {
  using C = Shape<NT>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ __align__(8) uint64_t full[S], empty[S], accfull[2], accempty[2];
  __shared__ __align__(16) float scales[kEpiWarps][32];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1, pairs = gridDim.x >> 1, first = blockIdx.x >> 1;
  const int n_tiles = (p.M + 255) / 256 * ((p.N + NT - 1) / NT), its = p.ksteps;

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
        locate<NT>(p, tile, m0, n0);
        const int am = m0 + 128 * rank, bn = n0 + NT / 2 * rank;
        for (int it = 0; it < its; ++it, ++g) {
          const int s = g % S;
          if (g >= S && !wait(&empty[s], ((g / S) - 1) & 1, abort, p.err)) goto drain;
          uint8_t* st = smem + s * C::kStage;
          const uint32_t bar = leader_addr(&full[s]);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::kStage);
          load_box(st, &p.a, 128 * it, am, bar);
          load_box(st + 16384, &p.b, 128 * it, bn, bar);
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
      constexpr uint32_t id = idesc(256, NT);
      int g = 0, li = 0;
      for (int tile = first; tile < n_tiles; tile += pairs, ++li) {
        const int b = li & 1;
        if (li >= 2 && !wait_all(&accempty[b], ((li >> 1) - 1) & 1, abort, p.err)) break;
        tc5::fence_after();
        const uint32_t acc = tb + b * NT;
        for (int it = 0; it < its; ++it, ++g) {
          const int s = g % S;
          if (!wait_all(&full[s], (g / S) & 1, abort, p.err)) goto mma_out;
          tc5::fence_after();
          if (elect_one()) {
            const uint64_t ad = ops + (uint64_t)((s * C::kStage) >> 4), bd = ad + (16384 >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) mma2(acc, ad + 2 * kk, bd + 2 * kk, id, (it | kk) != 0);
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
    uint8_t* box = smem + S * C::kStage + (warp - 2) * kBox;
    float* sc = scales[warp - 2];
    const bool f16 = p.out_dtype == DS_F16;
    int li = 0;
    for (int tile = first; tile < n_tiles; tile += pairs, ++li) {
      int m0, n0;
      locate<NT>(p, tile, m0, n0);
      const int b = li & 1, mw = m0 + 128 * rank + 32 * q;
      const uint32_t acc = tc5::lane_quarter(tb + b * NT, q);
      const int nc = mw < p.M ? min(NT, p.N - n0) : 0;   // columns inside the result
      const float sx = mw + lane < p.M ? p.sx[mw + lane] : 0.0f;
      if (!wait_all(&accfull[b], (li >> 1) & 1, abort, p.err)) break;
      tc5::fence_after();
      // 32 columns of results from column c on
      auto results = [&](int c, float (&v)[32]) {
        __syncwarp();
        sc[lane] = c + lane < nc ? p.sw[n0 + c + lane] : 0.0f;
        __syncwarp();
        take(acc + c, sx, sc, v);
      };
      auto box_free = [&] {   // the last store has read the box
        if (lane == 0) box_wait_read<0>();
        __syncwarp();
      };
      auto send = [&](int c) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          box_store(&p.out, n0 + c, mw, box);
          box_commit();
        }
      };
      // the two warps of a lane quarter take turns at the columns
      if (p.boxed && p.out_dtype != DS_F32) {
#pragma unroll 1
        for (int c = half * 64; c < nc; c += 128) {
          box_free();
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v[32];
            results(c + 32 * e, v);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *box_at(box, lane, 4 * e + k) =
                  make_uint4(pack16(v[8 * k], v[8 * k + 1], f16), pack16(v[8 * k + 2], v[8 * k + 3], f16),
                             pack16(v[8 * k + 4], v[8 * k + 5], f16), pack16(v[8 * k + 6], v[8 * k + 7], f16));
          }
          send(c);
        }
      } else {
#pragma unroll 1
        for (int c = half * 32; c < nc; c += 64) {
          float v[32];
          results(c, v);
          box_free();
          if (p.boxed) {
            box_put(box, lane, v);
            send(c);
          } else {
            by_rows(box, lane, v, [&](int r, float y) {
              if (mw + r >= p.M || c + lane >= nc) return;
              const int64_t at = (int64_t)(mw + r) * p.ldy + n0 + c + lane;
              if (p.out_dtype == DS_F32) static_cast<float*>(p.y)[at] = y;
              else if (f16) static_cast<__half*>(p.y)[at] = __float2half_rn(y);
              else static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(y);
            });
          }
        }
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

}  // namespace pairs
}  // namespace int8
}  // namespace ds
