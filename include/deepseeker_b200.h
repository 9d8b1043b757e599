/*
 * deepseeker_b200 -- C ABI of the B200 (sm_100a) routed-expert MoE hot path.
 *
 * Every entry point:
 *   - returns an int status (DS_OK = 0); the message of the last failure on
 *     the calling thread is available from ds_last_error_string();
 *   - takes DEVICE pointers for tensors (caller owns every buffer) unless the
 *     name says otherwise, plain integer sizes, and a cudaStream_t passed as
 *     `void* stream` (NULL = legacy default stream);
 *   - launches asynchronously on that stream and never synchronises it;
 *   - allocates nothing: scratch comes from a caller-provided workspace whose
 *     size a matching *_workspace_size() call reports (ds_moe_decode_noalloc
 *     uses a static device array instead).
 * The library is stateless and reentrant across distinct streams.
 *
 * Layout conventions (all row-major, K = input features contiguous):
 *   FP4  : packed [N, K/2] u8, two e2m1 codes per byte, LOW nibble = even
 *          element; scales [N, K/32] u8 (ue8m0: 2^(b-127), 0xFF = NaN).
 *   Q3   : words [N, K*3/32] u32, scales / biases [N, K/64] f16;
 *          w = f32(scale)*q + f32(bias).  One 64-element group = six
 *          little-endian u32 words: word w (0..3) holds the low two bits of
 *          elements 16w+i at bits [2i, 2i+2) (i = 0..15); word 4+h holds
 *          bit 2 of the codes: element 16(2h+v)+j at bit 8v+j and element
 *          16(2h+v)+8+j at bit 16+8v+j (v in {0,1}, j = 0..7).
 *   BF16 : [N, K] bf16.
 *   Expert banks stack E experts: [E, N, ...] with the per-expert layout above.
 */
#ifndef DEEPSEEKER_B200_H
#define DEEPSEEKER_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ------------------------------------------------------ */
#define DS_OK 0
#define DS_EINVAL 1   /* bad shape / dtype / argument                       */
#define DS_EALIGN 2   /* pointer not aligned as the call requires            */
#define DS_ERANGE 3   /* index out of range (host check or device guard)     */
#define DS_ECUDA 4    /* CUDA runtime error                                  */
#define DS_ETIMEOUT 5 /* a bounded device-side wait gave up                  */
#define DS_ENOTSUP 6  /* unsupported combination                            */

/* ---- element types ----------------------------------------------------- */
#define DS_F32 0
#define DS_BF16 1
#define DS_F16 2
#define DS_U8 3
#define DS_I8 4

/* ---- weight formats ---------------------------------------------------- */
#define DS_FMT_FP4 0
#define DS_FMT_Q3 1
#define DS_FMT_BF16 2

/* ---- routing kinds ----------------------------------------------------- */
#define DS_ROUTE_SOFTMAX 0      /* softmax over experts, top-k, renormalised  */
#define DS_ROUTE_SQRTSOFTPLUS 1 /* sqrt(softplus(s)), top-k of s+bias, *scale */
#define DS_ROUTE_SCORES 2       /* input already scores s: top-k of s+bias     */

/* Message of the last failed call on this thread ("" if none). */
const char* ds_last_error_string(void);

/* Library ABI version (major*10000 + minor*100 + patch). */
int ds_version(void);

/* ------------------------------------------------------------------------
 * FP4 e2m1 dequantisation, bit-exact with the reference table.
 * Replaces metal_fp4.metal_dequant / the three Metal kernels
 *   (reference: src/deepseeker/metal_fp4.py:28-66, 139-155) and
 *   mlx_weights.dequant_fp4_rowmajor (src/deepseeker/mlx_weights.py:148-166).
 * out[e] = FP4_TABLE[nibble(e)] * scale[e / 32] in f32 (round-to-nearest,
 * no flush-to-zero), then stored as f32 or bf16 (RNE).
 *   packed     : n_bytes u8 (n = 2*n_bytes elements)
 *   scales     : n_scales entries, f32 (scale_kind = DS_F32) or raw ue8m0
 *                bytes (scale_kind = DS_U8); n_scales must be ceil(n/32)
 *   out        : n elements of out_dtype (DS_F32 or DS_BF16)
 * ------------------------------------------------------------------------ */
int ds_fp4_dequant(const uint8_t* packed, int64_t n_bytes, const void* scales,
                   int scale_kind, int64_t n_scales, void* out, int out_dtype,
                   void* stream);

/* FP8 e4m3 with one ue8m0 scale per 32x32 block -> f32.
 * Replaces mlx_weights.dequant_fp8_block (src/deepseeker/mlx_weights.py:82-89).
 *   packed [rows, cols] u8, scales [rows/32, cols/32] u8, out [rows, cols] f32 */
int ds_fp8_block_dequant(const uint8_t* packed, int64_t rows, int64_t cols,
                         const uint8_t* scales, float* out, void* stream);

/* 3-bit affine (group 64) dequantisation: out = f32(scale)*q + f32(bias)
 * (multiply, then add: two roundings).  Replaces mx.dequantize(bits=3,
 * group_size=64) at src/deepseeker/mlx_forward.py:99-101 and
 * tests/test_q3.py:100-105.  cols % 64 == 0.
 *   words [rows, cols*3/32] u32, scales/biases [rows, cols/64] f16,
 *   out [rows, cols] of out_dtype (DS_F32 or DS_BF16) */
int ds_q3_dequant(const uint32_t* words, const uint16_t* scales,
                  const uint16_t* biases, int64_t rows, int64_t cols,
                  void* out, int out_dtype, void* stream);

/* 3-bit affine quantiser (builder rule: per-64 min/max, scale=(max-min)/7,
 * bias=min, both rounded to f16, q=clamp(rint((w-bias)/scale),0,7)).
 * Replaces mx.quantize(group_size=64, bits=3) in
 * scripts/requant_experts_3bit.py:69-83 (convert_tensor).
 *   w [rows, cols] f32 -> words [rows, cols*3/32], scales, biases [rows, cols/64] */
int ds_q3_quantize(const float* w, int64_t rows, int64_t cols, uint32_t* words,
                   uint16_t* scales, uint16_t* biases, void* stream);

/* FP4 quantiser for synthetic weights (builder rule: per-32 block
 * e = ceil(log2(amax/6)) clamped to [-127,127], RNE onto the e2m1 grid with
 * ties to the even code).  The reference consumes pre-quantised checkpoints
 * (no counterpart); used to build resident banks for tests and benches.
 *   w [rows, cols] f32 -> packed [rows, cols/2] u8, scales [rows, cols/32] u8 */
int ds_fp4_quantize(const float* w, int64_t rows, int64_t cols, uint8_t* packed,
                    uint8_t* scales, void* stream);

/* ------------------------------------------------------------------------
 * Router: per row, choose top_k experts and their gates.
 *   kind = DS_ROUTE_SOFTMAX: softmax over n_experts logits, top-k (ties to the
 *          lower id), gates renormalised to sum 1;
 *   kind = DS_ROUTE_SQRTSOFTPLUS: s = sqrt(softplus(logit)), top-k of s+bias,
 *          gates = s/(sum s + 1e-20) * route_scale
 *          (src/deepseeker/mlx_forward.py:62-81, sqrtsoftplus_scores/route_topk);
 *   kind = DS_ROUTE_SCORES: as SQRTSOFTPLUS with the input already the scores
 *          s (route_topk alone, mlx_forward.py:68-81).
 * Slots are written in descending selection-score order.
 *   logits [rows, n_experts] f32; bias [n_experts] f32 or NULL;
 *   ids [rows, top_k] i32; weights [rows, top_k] f32.  n_experts <= 1024,
 *   top_k <= 32. */
int ds_route_topk(const float* logits, const float* bias, int64_t rows,
                  int n_experts, int top_k, int kind, float route_scale,
                  int32_t* ids, float* weights, void* stream);

/* ------------------------------------------------------------------------
 * Expert banks and the fused routed-expert MoE layer.
 * ------------------------------------------------------------------------ */
typedef struct DsExpertBank {
  int32_t format;     /* DS_FMT_FP4, DS_FMT_Q3 or DS_FMT_BF16                 */
  int32_t n_experts;  /* E                                                    */
  int32_t rows;       /* N: output features                                  */
  int32_t cols;       /* K: input features                                   */
  const void* data;   /* FP4 [E,N,K/2] u8 | Q3 [E,N,K*3/32] u32 | BF16 [E,N,K] */
  const void* scales; /* FP4 [E,N,K/32] u8 | Q3 [E,N,K/64] f16 | BF16 NULL     */
  const void* biases; /* Q3 [E,N,K/64] f16 | otherwise NULL                   */
  const void* scales_tc; /* FP4 only, optional: the scales re-laid into tensor-
                            core atoms by ds_fp4_scale_atoms; when w1, w3 and w2
                            all carry them, ds_moe_decode runs its tcgen05
                            kernels.  NULL otherwise.                         */
} DsExpertBank;

typedef struct DsMoeDesc {
  int32_t hidden;       /* H                                                  */
  int32_t inter;        /* I (routed intermediate size)                       */
  int32_t n_experts;    /* E                                                  */
  int32_t top_k;        /* k                                                  */
  DsExpertBank w1;      /* gate: N = I, K = H                                 */
  DsExpertBank w3;      /* up  : N = I, K = H                                 */
  DsExpertBank w2;      /* down: N = H, K = I                                 */
  /* optional shared expert, BF16 (NULL pointers = none)                      */
  const void* shared_w1; /* [shared_inter, H] bf16                            */
  const void* shared_w3; /* [shared_inter, H] bf16                            */
  const void* shared_w2; /* [H, shared_inter] bf16                            */
  int32_t shared_inter;
  float swiglu_limit;    /* > 0: g = min(g, L), u = clip(u, -L, L); else none */
  int32_t route_before_down; /* 1: h *= gate before the down projection
                                (moe_layer, mlx_forward.py:404-405);
                                0: y *= gate after it (grouped.py:50-53)       */
  int32_t out_f32;       /* ds_moe_decode with bf16 x: 1 writes the layer
                            output in f32 without the final rounding (partial
                            sums that another rank adds to), 0 = x's dtype.
                            Served by FP4 banks with scale atoms, by one
                            token over FP4 banks with swiglu_limit > 0, and
                            by Q3 banks; DS_ENOTSUP otherwise.               */
} DsMoeDesc;

/* Workspace bytes ds_moe_decode needs for `tokens` rows.  The first 4096
 * bytes of a workspace are reserved (error word, control words of the
 * single-token kernel): zero them once before the first call with that
 * workspace (e.g. allocate it zero-filled); every call that completes leaves
 * the control words zero, so layers and token counts may share it.  After a
 * call that reported a bounded-wait timeout, zero it again. */
int ds_moe_decode_workspace_size(const DsMoeDesc* desc, int64_t tokens,
                                 size_t* bytes);

/* Fused routed-expert MoE layer for decode (tokens <= 8): for every distinct
 * routed expert e (ascending id), h = silu(min(x W1e^T, L)) * clip(x W3e^T, ±L)
 * (f32, weights dequantised in registers), scaled by the token's gate, then
 * out += h W2e^T; plus the shared expert (its output rounded to bf16 before
 * the add, as the reference does); out has the dtype of x.
 * Replaces moe_layer's expert loop + qmm + shared add
 *   (src/deepseeker/mlx_forward.py:84-103, 388-419;
 *    src/deepseeker/mlx_runner.py:776-781).
 *   x [tokens, H] of x_dtype (DS_BF16, or DS_F32 for the f32 oracle config);
 *   topk_ids [tokens, k] i32 (-1 = dropped slot); topk_w [tokens, k] f32;
 *   out [tokens, H] of x_dtype. */
int ds_moe_decode(const DsMoeDesc* desc, const void* x, int x_dtype, int64_t tokens,
                  const int32_t* topk_ids, const float* topk_w, void* out,
                  void* workspace, size_t workspace_bytes, void* stream);

/* Router + decode layer in one call: ds_route_topk(logits, route_bias, tokens,
 * n_experts, top_k, route_kind, route_scale) into topk_ids / topk_w (OUTPUTS
 * here, [tokens, k]), then ds_moe_decode with that routing.  Same results as
 * the two calls, bit for bit.  On the tcgen05 kernels (FP4 banks with scale
 * atoms, bf16 x) the routing is computed inside the decode's first kernel
 * (one launch fewer per layer); otherwise the router runs first.
 * Replaces route_topk + the moe_layer expert loop
 *   (src/deepseeker/mlx_forward.py:62-81, 388-419).
 *   logits [tokens, n_experts] f32, route_bias [n_experts] f32 or NULL;
 *   n_experts <= 1024, top_k <= 32; workspace as for ds_moe_decode. */
int ds_moe_decode_route(const DsMoeDesc* desc, const void* x, int x_dtype, int64_t tokens,
                        const float* logits, const float* route_bias, int route_kind,
                        float route_scale, int32_t* topk_ids, float* topk_w, void* out,
                        void* workspace, size_t workspace_bytes, void* stream);

/* One compressed matrix times a batch of activations: out[r, n] =
 * sum_k x[r, k] * W[n, k], W dequantised in registers (exactly: FP4 codes times
 * their ue8m0 scale; Q3 as f32(scale)*q + f32(bias)), f32 accumulate.
 * Replaces qmm (src/deepseeker/mlx_forward.py:84-103: mx.quantized_matmul with
 * mode="mxfp4", or bits=3 / group 64 with biases).
 *   w   : one matrix (n_experts = 1), DS_FMT_FP4 or DS_FMT_Q3, [N = rows, K = cols]
 *   x   : [rows, K] f32 (DS_F32) or bf16 (DS_BF16), 16-byte aligned
 *   out : [rows, N] f32.  K <= 6144 (eight x rows staged in shared memory). */
int ds_qmm(const DsExpertBank* w, const void* x, int x_dtype, int64_t rows, float* out, void* stream);

/* ---- host-fed decode steps: staging without the copy engines ------------ */

/* Device address of pinned host memory (cudaHostGetDevicePointer).  DS_EINVAL
 * when the memory is not pinned and mapped.  No reference counterpart: the
 * reference's MLX arrays live in unified memory. */
int ds_host_device_pointer(const void* host, void** device);

/* Copies n (1..4) byte ranges dst[k] <- src[k] in one kernel launch on
 * `stream`.  Pointers are device addresses (device memory, or pinned host
 * memory through ds_host_device_pointer), 16-byte aligned; bytes[k] is a
 * multiple of 16.  A host-fed decode step stages its inputs in and its
 * output out with it: a copy-engine transfer of a few kilobytes costs
 * several microseconds of latency on the step's critical path, this one
 * launch about as much as one.  No reference counterpart (see above). */
int ds_copy_ranges(int n, void* const* dst, const void* const* src, const size_t* bytes, void* stream);

/* ---- sort-and-pad of routed pairs by expert ---------------------------- */

/* Output capacities ds_moe_align needs for topk_ids [m, k] over n_experts:
 * sorted_cap = m*k + min(n_experts, m*k) * (block - 1), blocks_cap =
 * sorted_cap / block. */
int ds_moe_align_capacity(int64_t m, int k, int n_experts, int block,
                          int64_t* sorted_cap, int64_t* blocks_cap);

/* align_block_size on the device (src/deepseeker/moe_align.py:21-46):
 * flat positions of topk_ids [m, k] (i32, device) grouped by expert in
 * stable order, each expert's run padded with the sentinel m*k to a multiple
 * of block, experts in id order.  Writes sorted_ids (i32), expert_ids (i32,
 * one per block) and *n_pad (device i32, the padded length; -1 when an id is
 * outside [0, n_experts), in which case the other outputs are undefined).
 * n_experts <= 1024. */
int ds_moe_align(const int32_t* topk_ids, int64_t m, int k, int n_experts, int block,
                 int32_t* sorted_ids, int64_t sorted_cap, int32_t* expert_ids,
                 int64_t blocks_cap, int32_t* n_pad, void* stream);

/* ---- batched grouped expert FFN (FP4 banks, tcgen05) ------------------- */

/* FP4 bank scales [E, rows, cols/32] (ue8m0) -> tensor-core scale atoms
 * [E][rows/128][cols/128][512 B]: byte (r%32)*16 + (r/32)*4 + b of an atom is
 * the scale of row r, k-block b of that 128 x 128 tile.  rows and cols must be
 * multiples of 128; atoms holds E*rows*cols/32 bytes (the size of the scales).
 * Run once per resident bank; set DsExpertBank.scales_tc to the result. */
int ds_fp4_scale_atoms(const void* scales, int64_t n_experts, int rows, int cols, void* atoms,
                       void* stream);

/* Bytes of the re-laid-out block scales the grouped kernels read: W1 and W3
 * together (w13_bytes) and W2 (w2_bytes); same totals as the bank scales. */
int ds_grouped_scales_size(const DsMoeDesc* desc, size_t* w13_bytes, size_t* w2_bytes);

/* Re-lay the FP4 bank scales of desc (w1, w3, w2) into the tensor-core scale
 * atoms: for every 128 weight rows and 128-wide K chunk, 512 bytes where byte
 * (r%32)*16 + (r/32)*4 + b is the scale of row r, k-block b.  Run once per
 * resident bank (replaces no reference function: the reference reads the
 * checkpoint scales directly, mlx_weights.py:92-110). */
int ds_grouped_prepare_scales(const DsMoeDesc* desc, void* w13_sf, void* w2_sf, void* stream);

int ds_grouped_ffn_workspace_size(const DsMoeDesc* desc, int64_t tokens, size_t* bytes);

/* Routed-expert SwiGLU FFN for a batch of tokens (prefill / MTP verify):
 * pairs sorted by expert on the device, gate/up and down projections as
 * tcgen05 block-scaled MMAs, f32 accumulate, combine in top-k order.
 * Replaces grouped_swiglu and the moe_layer expert loop / banked gather
 * (src/deepseeker/grouped.py:34-56, src/deepseeker/mlx_forward.py:159-210,
 * 388-419).  FP4 banks: weights as e2m1 operands, activations as exact e4m3
 * pieces.  Q3 banks: the 3-bit codes become exact e4m3 operands in shared
 * memory and each 64-group's f16 scale and bias are applied after the MMA
 * (w13_sf / w2_sf unused, may be null).  Hidden and inter multiples of 128,
 * x bf16 [tokens, hidden], no shared expert (add it separately); topk_ids
 * [tokens, k] (-1 = dropped slot); out [tokens, hidden] of out_dtype (DS_BF16,
 * or DS_F32 for partial sums that are combined later, as the
 * expert-parallel path does).  desc->route_before_down selects where the
 * route weight is applied. */
int ds_grouped_ffn(const DsMoeDesc* desc, const void* w13_sf, const void* w2_sf,
                   const void* x, int x_dtype, int64_t tokens, const int32_t* topk_ids,
                   const float* topk_w, void* out, int out_dtype, void* workspace,
                   size_t workspace_bytes, void* stream);

/* FP4 throughput mode of the grouped FFN: FP4 banks with their scale atoms
 * (DsExpertBank.scales_tc, ds_fp4_scale_atoms) times activations rounded to
 * FP4 as well -- x and h become one e2m1 value per element with a per-32
 * ue8m0 scale that maps the block maximum into (3, 6] -- on tcgen05
 * kind::mxf4 MMAs (K = 64 per instruction, one MMA per weight byte instead of
 * one per activation piece).  The result carries the FP4 rounding of x and h
 * (relative L2 of order 0.1 against the exact layer); it equals, to f32
 * accumulation order, the layer evaluated on the FP4-rounded x and h.  No
 * reference counterpart: the reference's grouped path keeps f32 / bf16
 * activations (src/deepseeker/grouped.py:34-56).  Hidden and inter multiples
 * of 256; other arguments as ds_grouped_ffn. */
int ds_grouped_ffn_fp4_workspace_size(const DsMoeDesc* desc, int64_t tokens, size_t* bytes);
int ds_grouped_ffn_fp4(const DsMoeDesc* desc, const void* x, int x_dtype, int64_t tokens,
                       const int32_t* topk_ids, const float* topk_w, void* out, int out_dtype,
                       void* workspace, size_t workspace_bytes, void* stream);

/* ---- dense-weight pair FFN (grouped_swiglu / naive_swiglu with dense experts) */

int ds_dense_swiglu_workspace_size(int64_t n_pairs, int hidden, size_t* bytes);

/* y_p = w_p * (silu(x_r gate_e) * (x_r up_e)) down_e for every pair p = (r, e)
 * (f32; gate/up [E, H, I], down [E, I, H]; w_p = 1 when pair_weight is NULL;
 * swiglu_limit > 0 clamps as moe_layer does), then out[t] = sum of y_p over
 * the pairs row_ptr[t] .. row_ptr[t+1]-1 in that order
 * (src/deepseeker/grouped.py:34-81). */
int ds_dense_swiglu(const float* x, int64_t tokens, int hidden, int inter, int n_experts,
                    const float* gate, const float* up, const float* down, int64_t n_pairs,
                    const int32_t* pair_row, const int32_t* pair_expert, const float* pair_weight,
                    const int32_t* row_ptr, float swiglu_limit, float* out, void* workspace,
                    size_t workspace_bytes, void* stream);

/* ds_moe_decode without a workspace.  No counterpart in the reference (its
 * MLX runtime owns all scratch); added for callers that may not allocate
 * device memory at all while decoding, e.g. a serving loop whose device memory
 * is carved up once by its own pool.  Scratch comes from a static device array
 * of ds_moe_decode_noalloc_max_scratch() bytes (8 MiB) per device.
 *   - Kernels: exactly those ds_moe_decode runs when given a workspace of
 *     that size (the fastest path whose scratch fits: tcgen05 for FP4 banks
 *     with scale atoms, the single-token register-dequant kernel for one
 *     token over FP4 banks without them, the q3 kernels for Q3 banks, else
 *     the generic ones),
 *     so results equal ds_moe_decode's bit for bit whenever
 *     ds_moe_decode_workspace_size() <= the limit, and stay within the
 *     decode tolerance (rel-L2 <= 1e-3 of the f32 oracle) otherwise.
 *   - Limit: a layer whose generic-path scratch (4096 + (min(tokens*k, E) + 1)
 *     * tokens * max(inter, shared_inter) * 4 bytes, rounded up to 256) exceeds
 *     the array is rejected with DS_ERANGE.
 *   - The first call on each device resolves the array's address (setup,
 *     cudaGetSymbolAddress with that device current); make that first call
 *     before any stream capture and before any latency-sensitive phase.
 *   - Each call clears the array's 4096-byte reserved head (error word and
 *     control words) on `stream` (cudaMemsetAsync); nothing else has to start
 *     at zero.  ds_moe_decode_noalloc_status reads
 *     the word back: bit 0 = an expert id >= n_experts was skipped, bit 1 = a
 *     bounded device wait gave up (outputs of that call are then undefined).
 *   - All calls on one device share the array: two calls that may overlap
 *     (different streams, or host threads without ordering) race on it and
 *     corrupt each other's results.  Serialise them on one stream. */
size_t ds_moe_decode_noalloc_max_scratch(void);
int ds_moe_decode_noalloc(const DsMoeDesc* desc, const void* x, int x_dtype, int64_t tokens,
                          const int32_t* topk_ids, const float* topk_w, void* out,
                          void* stream);
/* Copy the no-allocation scratch's error word of the current device into *err
 * (host or device memory; one cudaMemcpyAsync on `stream`, read it after the
 * stream has finished).  No counterpart in the reference. */
int ds_moe_decode_noalloc_status(int32_t* err, void* stream);

/* ---------------------------------------------------------------------------
 * Expert-parallel decode over NVLink peer memory.
 *
 * Replaces, across G ranks (one process per GPU), the per-layer MoE call of a
 * decode step (src/deepseeker/mlx_runner.py:765-985 Runner.moe ->
 * src/deepseeker/mlx_forward.py:257-419 moe_layer).  Rank r holds experts
 * [first_expert, first_expert + desc->n_experts) of every layer and decodes
 * `rows` tokens per step; the token rows are exchanged and the partial
 * outputs summed by the library's own kernels through CUDA IPC mappings of
 * every rank's region (no collective library on the data path, so a step
 * captures into a CUDA graph).
 *
 * Setup, on every rank with its device current:
 *   ds_ep_create -> ds_ep_ipc_handle -> (exchange the world handles, e.g.
 *   torch.distributed.all_gather_object) -> ds_ep_connect(all handles, in
 *   rank order) -> a barrier, so that no rank writes into a peer before the
 *   peer has connected.
 * Step: every rank calls ds_ep_decode for the same layers in the same order
 * with the same `rows`.  Device waits give up after `timeout_ms`; the error
 * word then holds bit 2 (ds_ep_status), and later calls of that
 * communicator return without exchanging (outputs undefined).
 * Limits: world <= 8, world * max_rows <= 8; FP4 banks with scale atoms,
 * hidden and inter multiples of 1024 (the tcgen05 decode kernels), or Q3
 * banks, hidden and inter multiples of 128 (the CUDA-core q3 kernels). */
#define DS_EP_HANDLE_BYTES 64
typedef struct DsEp DsEp;
int ds_ep_create(int world, int rank, int max_rows, int hidden, int top_k, int timeout_ms, DsEp** ep);
size_t ds_ep_region_bytes(int world, int max_rows, int hidden, int top_k);
int ds_ep_ipc_handle(DsEp* ep, void* handle /* DS_EP_HANDLE_BYTES */);
int ds_ep_connect(DsEp* ep, const void* handles /* world * DS_EP_HANDLE_BYTES, rank order */);
/* Same as ds_ep_connect for communicators created by ONE process (one per
 * device, or several on one device: the single-device form exists to test
 * the bounded waits, since ranks sharing a GPU must not wait on each other).
 * all[world] in rank order, all[rank] == ep; peer access is enabled between
 * distinct devices. */
int ds_ep_connect_peers(DsEp* ep, DsEp* const* all);
int ds_ep_decode_workspace_size(DsEp* ep, const DsMoeDesc* desc, int64_t rows, size_t* bytes);
/* x [rows, hidden] bf16, topk_ids [rows, top_k] GLOBAL expert ids (-1 =
 * none), topk_w [rows, top_k] f32 -> out [rows, hidden] bf16: routed experts
 * of all ranks (route weight before the down projection) plus this layer's
 * shared expert (desc->shared_*, the full matrices on every rank: rank r
 * evaluates intermediate slice r of it for all ranks' rows when
 * shared_inter is a multiple of 256 * world, else all of it for its own
 * rows; its output is rounded to bf16 before it joins the routed sum). */
int ds_ep_decode(DsEp* ep, const DsMoeDesc* desc, int32_t first_expert, const void* x, int64_t rows,
                 const int32_t* topk_ids, const float* topk_w, void* out, void* workspace,
                 size_t workspace_bytes, void* stream);
int ds_ep_status(DsEp* ep, int32_t* err);
int ds_ep_destroy(DsEp* ep);

/* ---------------------------------------------------------------------------
 * Dense gated feed-forward block over 16-bit weights, forward and backward
 * (the shared expert of a layer, or a layer without routing; the reference's
 * is four separate products, src/deepseeker/mlx_runner.py:776-781, and has no
 * backward pass):
 *   g = x W1^T, u = x W3^T, h = silu(min(g, L)) * clip(u, -L, L), y = h W2^T.
 * Products accumulate in f32; h and the gradients of g and u are rounded once
 * to the 16-bit type (in f16 beyond 65,504 to an infinity, which h cannot reach
 * with L <= 255), g and u are kept in f32 between the passes.  NaN passes
 * through the clamps.  A clamped value has no gradient, one that equals the
 * limit has one, and the exact sums decide: with clamps, kept values of g and u
 * that f32 sums cannot place are summed up in 64 bits and stored on the side of
 * the limit where they belong.  Any sizes, row strides and 2-byte alignments; operands
 * whose base is no multiple of 16 bytes or whose row stride is no multiple of
 * 8 elements are first copied into the workspace.  Results do not depend on
 * timing (no atomics). */
typedef struct DsGatedFfn {
  int64_t tokens;             /* T, 0 <= T <= 2^22                                 */
  int32_t hidden, inter;      /* H, I, 1 .. 2^17                                   */
  int32_t dtype;              /* DS_BF16 or DS_F16: x, weights, y, gradients        */
  float limit;                /* L > 0, or 0: no clamps                            */
  const void* x;              /* [T, H], rows ld_x elements apart                   */
  const void* w1;             /* [I, H] gate                                       */
  const void* w3;             /* [I, H] up                                         */
  const void* w2;             /* [H, I] down                                       */
  int64_t ld_x, ld_w1, ld_w3, ld_w2;
} DsGatedFfn;

/* Workspace bytes of ds_gated_ffn; keeps_h: the call gets an h buffer. */
int ds_gated_ffn_workspace_size(const DsGatedFfn* desc, int keeps_h, size_t* bytes);
/* y [T, H] contiguous.  For a later backward pass: h [T, Ip] 16 bit and
 * pre [2][T, Ip] f32 (g, then u), Ip = inter rounded up to a multiple of 8
 * (columns from inter on hold nothing); both NULL otherwise. */
int ds_gated_ffn(const DsGatedFfn* desc, void* y, void* h, float* pre, void* workspace,
                 size_t workspace_bytes, void* stream);

/* Backward pass from dy [T, H] (rows ld_dy elements apart) and the h and pre
 * that ds_gated_ffn left: dx [T, H], dw1 and dw3 [I, H], dw2 [H, I], each
 * contiguous and 16 bit; NULL skips one, with the products only it needs. */
int ds_gated_ffn_backward_workspace_size(const DsGatedFfn* desc, const void* dy, int64_t ld_dy, size_t* bytes);
int ds_gated_ffn_backward(const DsGatedFfn* desc, const void* h, const float* pre, const void* dy,
                          int64_t ld_dy, void* dx, void* dw1, void* dw3, void* dw2, void* workspace,
                          size_t workspace_bytes, void* stream);
/* Copies the current device's error word of these calls into *err (host or
 * device memory; read it after the stream has finished) and clears it, in one
 * step: a call on another stream that gives up meanwhile is in this answer or in
 * the next.  Bit 1: a bounded device wait gave up, and that call's outputs are undefined. */
int ds_gated_ffn_status(int32_t* err, void* stream);

/* ---------------------------------------------------------------------------
 * Microscaled 4-bit dense operators over the FP4 layout above (the reference
 * only dequantises such weights, src/deepseeker/metal_fp4.py:28-66; products
 * of two quantised matrices have no counterpart there).
 * A row of K values is ceil(K / 32) blocks: 16 bytes of codes (zeros behind an
 * uneven end) and one ue8m0 scale each, the smallest power of two that brings
 * the block's largest magnitude to 6 or less (1 for zeros; the rule of
 * ds_fp4_quantize).  Rounding is to nearest, ties to the even code; 0 has one
 * code.  A block with a NaN or an infinity gets scale 255 (NaN), so products
 * with it are NaN.  Magnitudes that round to 2^128 (above 2.9e38) stand for a
 * value outside f32.
 * Beside the scales, the tensor cores read them as atoms
 * [ceil(rows/128)][ceil(K/128)][512 B]: byte (r%32)*16 + (r/32)*4 + b is the
 * scale of row r, block b of a 128 x 128 tile (as ds_fp4_scale_atoms, for any
 * sizes; rows past the matrix are not written). */
int ds_mx4_atoms_size(int64_t rows, int64_t cols, size_t* bytes);
/* x [rows, cols] f32, bf16 or f16, rows ld elements apart -> packed
 * [rows, 16 ceil(cols/32)], scales [rows, ceil(cols/32)], atoms (or NULL). */
int ds_mx4_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ld, uint8_t* packed,
                    uint8_t* scales, uint8_t* atoms, void* stream);
/* The values that codes and scales stand for, out [rows, cols] f32 or bf16
 * contiguous (both exact; scale 255 gives NaN). */
int ds_mx4_dequantize(const uint8_t* packed, const uint8_t* scales, int64_t rows, int64_t cols, void* out,
                      int out_dtype, void* stream);
/* Atoms of stored scales [rows, ceil(cols/32)]: once per weight matrix. */
int ds_mx4_scale_atoms(const uint8_t* scales, int64_t rows, int64_t cols, uint8_t* atoms, void* stream);

typedef struct DsMx4 {
  const uint8_t* packed;
  const uint8_t* atoms;
  int64_t rows, cols;         /* 1 .. 2^20 each */
} DsMx4;

/* out [rows, w->rows] (f32, bf16 or f16, contiguous) = x W^T, f32 accumulate.
 * x_dtype f32 / bf16 / f16: x [rows, w->cols], rows ld elements apart, is
 * quantised into the workspace first, or up to 16 rows by the product itself
 * without one (x_atoms NULL); DS_U8: x is codes and x_atoms its atoms, and no
 * workspace is needed.  rows in [0, 2^22]. */
int ds_mx4_linear_workspace_size(int64_t rows, int64_t cols, size_t* bytes);
int ds_mx4_linear(const void* x, const uint8_t* x_atoms, int x_dtype, int64_t rows, int64_t ld, const DsMx4* w,
                  void* out, int out_dtype, void* workspace, size_t workspace_bytes, void* stream);

/* The gated block (ds_gated_ffn's formula) over quantised weights: x is
 * quantised (or given as codes), h = silu(min(g, limit)) * clip(u, +-limit) is
 * computed from the f32 sums and quantised in the product's epilogue; limit 0:
 * no clamps.  out [rows, hidden] f32, bf16 or f16. */
int ds_mx4_gated_ffn_workspace_size(int64_t rows, int64_t hidden, int64_t inter, size_t* bytes);
int ds_mx4_gated_ffn(const void* x, const uint8_t* x_atoms, int x_dtype, int64_t rows, int64_t ld, const DsMx4* w1,
                     const DsMx4* w3, const DsMx4* w2, float limit, void* out, int out_dtype, void* workspace,
                     size_t workspace_bytes, void* stream);
/* As ds_gated_ffn_status, for the calls of this group. */
int ds_mx4_status(int32_t* err, void* stream);

/* ---------------------------------------------------------------------------
 * Layer norm over the last dimension, forward and backward (the reference has
 * an RMS norm only, src/deepseeker/mlx_forward.py:45, and no backward pass):
 *   mean = sum x / H, r = 1 / sqrt(sum (x - mean)^2 / H + eps),
 *   xh = (x - mean) r, y = xh w + b.
 * x, y, dy, dx are f32, bf16 or f16; weight and bias (either may be NULL: 1
 * and 0) and their gradients f32 or of x's type.  Sums and statistics are f32,
 * results rounded once.  Squares of differences to the mean have to stay
 * inside f32 (magnitudes up to about 1e19 / sqrt(H)).  Any sizes, row strides
 * and alignments to the element.  Results do not depend on timing. */
/* x [rows, cols], rows ld elements apart, rows in [0, 2^31), cols in [1, 2^20]
 * -> y contiguous.  stats [rows, 2] f32 (mean, r) is what a backward pass
 * reads; NULL where none follows. */
int ds_layer_norm(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* weight,
                  const void* bias, int param_dtype, float eps, void* y, float* stats, void* stream);
/* From dy (rows ld_dy elements apart) and the forward pass's stats: dx
 * contiguous, dweight and dbias [cols] of param_dtype; NULL skips one.  The
 * workspace is needed for dweight and dbias only. */
int ds_layer_norm_backward_workspace_size(int64_t rows, int64_t cols, size_t* bytes);
int ds_layer_norm_backward(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* weight,
                           int param_dtype, const float* stats, const void* dy, int64_t ld_dy, void* dx,
                           void* dweight, void* dbias, void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Balance loss of a router, its counts per expert and its gradient (the
 * reference only serves; its routers, src/deepseeker/mlx_forward.py:62-81, are
 * ds_route_topk).  Per sequence, over its n valid tokens:
 *   c_e = how often e was chosen, P_e = 1/n sum_t p_te,
 *   loss = sum_e (c_e E / (k n)) P_e   (1 when both are even),
 * p_te = softmax(l_t)_e, or s_te / sum_e s_te with s = sqrt(softplus(l)).  The
 * gradient takes c_e as given.  Sums of p are f32; results do not depend on
 * timing.  Scores below 2^-126 are 0, and a row of none but such (logits of
 * -infinity; for the root of softplus, about exp(l / 2) there, of -174.7 and
 * less) has p = 0 and no gradient. */
typedef struct DsBalance {
  const void* logits;         /* [T, E], rows ld elements apart                      */
  int64_t tokens, ld;         /* T: T * top_k < 2^31                                  */
  int32_t dtype;              /* DS_F32, DS_BF16, DS_F16: logits and their gradient   */
  int32_t experts, top_k;     /* E in [1, 1024], k in [1, 32]                         */
  int32_t kind;               /* DS_ROUTE_SOFTMAX or DS_ROUTE_SQRTSOFTPLUS            */
  const int32_t* ids;         /* [T, k] contiguous; outside [0, E): no expert         */
  const uint8_t* valid;       /* [T] or NULL; 0: the row is not looked at             */
  const void* offsets;        /* [sequences + 1] ascending rows; NULL: one sequence   */
  int32_t offsets_i64;        /* offsets are int64, else int32                        */
  int64_t sequences;          /* S in [0, 2^24], 1 without offsets                    */
} DsBalance;

int ds_balance_loss_workspace_size(const DsBalance* desc, size_t* bytes);
/* loss [S] (0 for a sequence without valid tokens), counts [S, E], and coef
 * [S, E] = c_e E / (k n^2), which the backward pass reads. */
int ds_balance_loss(const DsBalance* desc, float* loss, int32_t* counts, float* coef, void* workspace,
                    size_t workspace_bytes, void* stream);
/* dlogits [T, E] contiguous, of the logits' type, from dloss [S]: 0 in rows
 * that are not valid or belong to no sequence.  ids is not read. */
int ds_balance_loss_backward(const DsBalance* desc, const float* coef, const float* dloss, void* dlogits,
                             void* stream);

/* ---------------------------------------------------------------------------
 * 8-bit integer dense operators, one f32 scale per row of either operand (a
 * token's activations, an output channel's weights; the reference has no
 * product in this format).  Of a row of K < 2^17 values: s = max |x| * (1 / 127)
 * in f32 (factor and product rounded), code q = the whole number nearest to the
 * exact x / s, the even one of two, clipped to +-127 (0 where s is 0).  (The
 * rounded quotient max |x| / 127 is a unit of the last place away in about one row
 * of twenty, where half of the maximum can have another code; the operators that
 * take codes take either.)  A row with a NaN or an infinity has scale NaN and codes
 * 0, so products with it are NaN.  Codes of a row lie together, rows `pitch` bytes
 * apart, a multiple of 16 (what lies between is neither read as a value nor
 * written). */
int ds_int8_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ld, int8_t* codes, int64_t pitch,
                     float* scales, void* stream);
/* out [rows, cols] f32, bf16 or f16 contiguous = code * scale, rounded to f32
 * and then to out's type. */
int ds_int8_dequantize(const int8_t* codes, int64_t pitch, const float* scales, int64_t rows, int64_t cols, void* out,
                       int out_dtype, void* stream);

typedef struct DsInt8 {
  const int8_t* codes;        /* 16-byte aligned                                    */
  const float* scales;        /* [rows]                                             */
  int64_t rows, cols;         /* 1 .. 2^20, 1 .. 2^17 - 1                           */
  int64_t pitch;              /* bytes from row to row, a multiple of 16            */
} DsInt8;

/* out [rows, w->rows] (f32, bf16 or f16, contiguous) = x W^T: the sum of
 * products of codes, exact in 32-bit integers, converted to f32, times both
 * scales (the one nearer to 0 first), rounded to out's type.  x_dtype f32 / bf16 / f16:
 * x [rows, w->cols], rows ld elements apart, is quantised into the workspace
 * first (x_scales NULL; a single row by the product itself, without one);
 * DS_I8: x is codes, rows ld bytes apart (a multiple of 16), x_scales their
 * scales, and no workspace is needed.  rows in [0, 2^22]. */
int ds_int8_linear_workspace_size(int64_t rows, int64_t cols, size_t* bytes);
int ds_int8_linear(const void* x, const float* x_scales, int x_dtype, int64_t rows, int64_t ld, const DsInt8* w,
                   void* out, int out_dtype, void* workspace, size_t workspace_bytes, void* stream);
/* As ds_gated_ffn_status, for the calls of this group. */
int ds_int8_status(int32_t* err, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DEEPSEEKER_B200_H */
