/*
 * julia1_hip_ops.h — the individual gfx950 kernels of the encoder forward,
 * callable on caller-owned device memory.
 *
 * These are the launch wrappers jh_forward uses, exported so each kernel can
 * be parity-tested and timed on its own (the GEMM sweep runs through
 * jh_op_gemm).  All pointers are device pointers; `stream` is a hipStream_t
 * (NULL = the null stream).  Calls enqueue work and return; they do not
 * synchronise.  Shape errors return JH_ERR_INVALID before anything is
 * launched.  Element types: f32 = float, bf16 = uint16_t bit patterns.
 *
 * Each entry point names the reference kernel or library call it stands in
 * for; the reference launches its own versions from src/cuda/mod.rs:400-521.
 */
#ifndef JULIA1_HIP_OPS_H
#define JULIA1_HIP_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Epilogues of jh_op_gemm: what happens to each FP32 accumulator tile of out = X · Wᵀ. */
enum {
    JH_EPI_STORE_BF16 = 0,      /* out bf16 = acc                                         */
    JH_EPI_ROPE_BF16 = 1,       /* out bf16 = acc, rotate-half RoPE applied to the columns  */
                                /*   below rope_cols (q and k of a packed qkv row)          */
    JH_EPI_GEGLU_BF16 = 2,      /* W rows interleaved per 32 (see jh_op_interleave_geglu):  */
                                /*   out[:, n/2] bf16 = gelu(gate) * up                     */
    JH_EPI_RESID_F32 = 3,       /* out f32 += acc (+ bias if given)                         */
    JH_EPI_BIAS_BF16 = 4,       /* out bf16 = acc + bias                                    */
    JH_EPI_BIAS_RELU_BF16 = 5,  /* out bf16 = max(acc + bias, 0)                            */
    JH_EPI_BIAS_F32 = 6         /* out f32 = acc + bias                                     */
};

/*
 * out[r, col + n] = epi( Σ_k X[row(r), k] · W[n, k] ) for r < rows, n < N.
 *  X bf16 with row stride ldx; row(r) = gather ? gather[r] : r.
 *  W bf16 [N, K] row-major (PyTorch Linear layout).
 *  out has row stride ldo (elements), written from column `col`.
 *  bias f32 [N] (NULL allowed for RESID_F32).
 *  ROPE: pos[r] is the row's position; cos/sin are [positions, 32] f32 tables;
 *        columns < rope_cols are rotated per 64-wide head.
 * Requirements: K % 64 == 0, N % 64 == 0, K <= 8192; x, w and out 16-byte aligned,
 * and out's rows and column `col` on 16-byte boundaries.  Replaces cuBLAS gemm_ex
 * (src/cuda/mod.rs:347-375) plus the separate geglu/bias_act kernels
 * (src/cuda/kernels.cu:137-172) and the residual add of ln_bf16 (:97-109).
 */
int jh_op_gemm(int epilogue, const void* x, size_t ldx, const int32_t* gather, size_t rows,
               const void* w, size_t n, size_t k, void* out, size_t ldo, size_t col,
               const float* bias, const int32_t* pos, const float* cos_t, const float* sin_t,
               size_t rope_cols, void* stream);

/*
 * jh_op_gemm with split-K: K is cut into `splits` chunks (0 = chosen from the
 * tile count, as the backend does for small batches) whose FP32 partial sums
 * go to `workspace` (splits · rows · N floats must fit `workspace_bytes`;
 * fewer splits are used otherwise), then one more kernel sums them in chunk
 * order and applies the epilogue.  With splits 0, shapes that a one-launch
 * kernel serves better (few tokens; K = 384, 768 or 1152 from some hundreds of
 * tokens up) run on it without the workspace.  Deterministic.  Same
 * requirements as jh_op_gemm.  No reference counterpart (cuBLAS chooses its own split-K).
 */
int jh_op_gemm_splitk(int epilogue, const void* x, size_t ldx, const int32_t* gather, size_t rows,
                      const void* w, size_t n, size_t k, void* out, size_t ldo, size_t col,
                      const float* bias, const int32_t* pos, const float* cos_t, const float* sin_t,
                      size_t rope_cols, void* workspace, size_t workspace_bytes, int splits, void* stream);

/*
 * jh_op_gemm_splitk without the workspace argument: the FP32 partial sums live
 * in a fixed 16 MiB device array inside the library (one per GPU, held until
 * the process ends), so the call allocates nothing (no hipMalloc, hipFree or
 * allocating library call).  For callers that cannot allocate: code under HIP
 * graph capture, tight serving loops, harnesses that forbid hipMalloc.
 * `splits` as jh_op_gemm_splitk: 0 picks the split count that fits the array,
 * a forced count whose partials (splits x rows x N floats) exceed 16 MiB is
 * rejected with JH_ERR_INVALID.  Calls that overlap on one GPU (two streams,
 * or two threads) share the array and race; serialise them.  Results equal
 * jh_op_gemm_splitk's with the same split count.  No reference counterpart.
 */
int jh_op_gemm_splitk_noalloc(int epilogue, const void* x, size_t ldx, const int32_t* gather,
                              size_t rows, const void* w, size_t n, size_t k, void* out, size_t ldo,
                              size_t col, const float* bias, const int32_t* pos, const float* cos_t,
                              const float* sin_t, size_t rope_cols, int splits, void* stream);

/*
 * jh_op_gemm whose X operand is bf16(LayerNorm(xf[r]; ln_w, ln_b, eps)), the
 * normalisation computed in the small-batch kernel's prologue exactly as
 * jh_op_layer_norm computes it (the same bits).  xf f32 [rows, k] with row
 * stride ldx floats (ldx % 4 == 0, 16-byte aligned); ln_w f32 [k], ln_b f32 [k]
 * or NULL.  k = hidden in {128, 256, 384, 512, 768}; epilogues STORE_BF16,
 * ROPE_BF16 and GEGLU_BF16; one workgroup per 64 x 32 output tile, so it is
 * meant for the few-token batches the backend runs on the small-batch kernel.
 * Replaces ln_bf16 (src/cuda/kernels.cu:97-109) followed by cuBLAS gemm_ex
 * (src/cuda/mod.rs:347-375) for those batches.
 */
int jh_op_gemm_ln(int epilogue, const float* xf, size_t ldx, size_t rows, const void* w, size_t n,
                  size_t k, void* out, size_t ldo, size_t col, const int32_t* pos, const float* cos_t,
                  const float* sin_t, size_t rope_cols, const float* ln_w, const float* ln_b, float eps,
                  void* stream);

/*
 * jh_op_gemm on the weight-stationary kernel: each workgroup (one per CU)
 * keeps a slab of W resident (registers and LDS) and streams 16-token blocks
 * of X through LDS, so only X moves from L2 during the multiply.  w_packed
 * is W (as jh_op_gemm takes it, [n, k] bf16; the GEGLU interleave for Wi) in
 * the fragment order jh_op_pack_ws writes.  Shapes: K == 768 with N % 256 ==
 * 0 (256-row slabs, every epilogue), or K == 1152 with N % 128 == 0 and
 * JH_EPI_RESID_F32 only (128-row slabs, K split between partner waves whose
 * two half sums are added lower half first); no row gather; rows of X and of
 * the output under 2^28 bytes.  Other arguments as jh_op_gemm.  The same bf16 products as jh_op_gemm, summed in FP32 in K
 * order in steps of 32 (jh_op_gemm: 16), so outputs agree to FP32 rounding.
 * jh_forward uses it for the K = 768 GEMMs and the MLP-out projection
 * (K = intermediate = 1152) outside the small-batch path.  Replaces cuBLAS
 * gemm_ex (src/cuda/mod.rs:347-375) for those shapes.
 */
int jh_op_gemm_ws(int epilogue, const void* x, size_t ldx, size_t rows, const void* w_packed, size_t n,
                  size_t k, void* out, size_t ldo, size_t col, const float* bias, const int32_t* pos,
                  const float* cos_t, const float* sin_t, size_t rope_cols, void* stream);

/*
 * Host: reorder a bf16 W [n, k] (row-major) into jh_op_gemm_ws's fragment
 * order (n*k elements; k % 32 == 0 and n % 256 == 0, or n % 128 == 0 at
 * k == 1152, whose layout is the K-split kernel's).  No reference counterpart
 * (a one-time weight layout, as the reference's BF16 conversion at upload,
 * src/cuda/mod.rs:36-39).
 */
int jh_op_pack_ws(const void* w, size_t n, size_t k, void* out);

/* Reorder a host FP32 Wi [2*inter, k] into the gate/up interleave JH_EPI_GEGLU_BF16 expects. */
void jh_op_interleave_geglu(const float* wi, size_t inter, size_t k, float* out);

/*
 * x[t] = LayerNorm(table[ids[t]]; w, no bias, eps) (f32), xn[t] = bf16(x[t]).
 * table f32 [vocab, hidden].  Replaces embed_ln (src/cuda/kernels.cu:66-75).
 */
int jh_op_embed_ln(const uint32_t* ids, size_t rows, const float* table, const float* w,
                   float eps, size_t hidden, float* x, void* xn, void* stream);

/*
 * out[r] = bf16(LayerNorm(x[r]; w, b, eps)), b may be NULL.
 * Replaces ln_bf16 (src/cuda/kernels.cu:97-109) without its residual add,
 * which the producing GEMM's RESID_F32 epilogue performs instead.
 */
int jh_op_layer_norm(const float* x, size_t rows, const float* w, const float* b, float eps,
                     size_t hidden, void* out, void* stream);

/*
 * Encoder final norm fused with the question-type embedding and the first
 * head layer's norm1: x[t] = LN(x[t]; fw, eps) + type_emb[qtype(t)];
 * out[t] = bf16(LN(x[t]; hw, hb, 1e-5)).  tok_meta[t] packs the token's
 * position (bits 0..15) and its sequence's qtype (bits 16..23).
 * Replaces final_norm (src/cuda/kernels.cu:113-132).
 */
int jh_op_final_norm(float* x, size_t rows, const float* fw, const float* type_emb,
                     const uint32_t* tok_meta, const float* hw, const float* hb, float eps,
                     size_t hidden, void* out, void* stream);

/*
 * dst[r] = src[idx[r]] for f32 rows of `hidden`.  Replaces gather_rows
 * (src/cuda/kernels.cu:175-183) for the FP32 residual; bf16 marker gathers
 * are folded into jh_op_gemm's `gather` argument instead.
 */
int jh_op_gather_f32(const float* src, const int32_t* idx, size_t rows, size_t hidden,
                     float* dst, void* stream);

/*
 * score[r] = Σ_i gelu(z[r, i]) · w2[i] + b2 (z already includes scorer.1's bias).
 * Replaces scorer (src/cuda/kernels.cu:186-194).
 */
int jh_op_scorer(const float* z, size_t rows, size_t hidden, const float* w2, float b2,
                 float* out, void* stream);

/*
 * Attention work item: `nq` query rows starting at absolute row `q_row` attend
 * to `kv_len` key/value rows starting at `kv_row`; the first query sits at
 * sequence position `q_pos` (keys are at positions 0..kv_len-1), which is what
 * the sliding window measures against.  nq <= 128.
 */
typedef struct jh_attn_tile {
    int32_t q_row, nq, kv_row, kv_len, q_pos;
} jh_attn_tile;

/*
 * FlashAttention-2 forward, one workgroup per (tile, head): MFMA QKᵀ and PV,
 * K/Vᵀ staged in LDS, online softmax of scale·QKᵀ over keys with
 * |q_pos - k_pos| <= window (window < 0: all keys of the sequence).
 * q/k/v bf16 with row strides ldq/ldkv; head h reads columns [64h, 64h+64)
 * of each; out bf16 row stride ldo.  `tiles` is a device array; work items
 * are dispatched in list order with heads varying fastest, so listing the
 * costliest tiles first (as the backend does) balances the CUs.  Few work
 * items (at most one for every two CUs, or two per CU over long rows) have
 * their keys split over two or four groups of waves where kv_len is 513 or
 * more, which adds such a query's partial sums in another order; rows of up to
 * 512 keys get the same bits in any launch.
 * Replaces attention_rope/attention_plain (src/cuda/kernels.cu:274-391); RoPE
 * is applied by the producing GEMM's ROPE epilogue instead of on every load.
 */
int jh_op_attention(const void* q, size_t ldq, const void* k, const void* v, size_t ldkv,
                    void* out, size_t ldo, const jh_attn_tile* tiles, size_t ntiles,
                    size_t heads, int window, float scale, void* stream);

/*
 * jh_op_attention with work items of up to 256 queries (tiles of nq <= 256):
 * eight waves per (tile, head), each staged K/V tile shared by twice the
 * queries, or two 128-query workgroups per tile where those leave fewer CUs
 * idle (and on window layers).  The backend uses it for the global layers of
 * sequences of 4096 tokens or more.  Keys are split over few items as in
 * jh_op_attention.  No separate counterpart in the reference (part of
 * attention_rope/attention_plain, src/cuda/kernels.cu:274-391).
 */
int jh_op_attention_wide(const void* q, size_t ldq, const void* k, const void* v, size_t ldkv,
                         void* out, size_t ldo, const jh_attn_tile* tiles, size_t ntiles,
                         size_t heads, int window, float scale, void* stream);

/*
 * jh_op_attention (wide = 0) or jh_op_attention_wide (wide != 0) with no key
 * split: every query's keys are added by one wave in one order, so a row gets the
 * same bits whatever else is in the launch, and from both item sizes where they
 * cut the row at multiples of 128 and 256.  What the backend runs after
 * jh_set_splitk(model, 0).  No reference counterpart.
 */
int jh_op_attention_unsplit(const void* q, size_t ldq, const void* k, const void* v, size_t ldkv,
                            void* out, size_t ldo, const jh_attn_tile* tiles, size_t ntiles,
                            size_t heads, int window, float scale, int wide, void* stream);

/* ------------------------------------------------------------------------
 * The feed-forward block of models that normalise by the root mean square and
 * gate their projections: norm -> gated projections -> projection with the
 * residual's addition, in bf16 or f16 with every gradient, and with e4m3
 * operands for serving.  No reference counterpart (the reference's encoder has
 * LayerNorm and runs GEGLU as two kernels, src/cuda/kernels.cu:97-172).
 *
 * Element types of these operators, and activations.  e4m3 is OCP FP8 E4M3
 * (largest magnitude 448), held one byte per value with an f32 scale per row:
 * the value is code * scale.
 */
enum { JH_F32 = 0, JH_BF16 = 1, JH_F16 = 2, JH_E4M3 = 3 };
enum {
    JH_ACT_NONE = 0,
    JH_ACT_RELU = 1,
    JH_ACT_GELU = 2,       /* z * normal cdf(z)                                  */
    JH_ACT_GELU_TANH = 3,  /* z/2 * (1 + tanh(sqrt(2/pi) * (z + 0.044715 z^3)))  */
    JH_ACT_SILU = 4        /* z * sigmoid(z)                                     */
};

/*
 * Rules common to them.  Matrices are row-major with a row stride in elements;
 * pointers and rows lie on 16-byte boundaries (e4m3 rows that rms_norm and
 * quantize_rows write: 8), row strides are at most 4 MiB.  f32 vectors
 * (weights of norms, biases, scales, rstd) need 4-byte alignment only.  Feature
 * counts are multiples of 8, or of 16 where they are the contraction of e4m3
 * operands; the number of rows is free, 0 included (at most 2^30 for products),
 * and the stride of one row is not used.  An output or a workspace may not overlap
 * an input or another output (JH_ERR_INVALID) except where said.  Memory is the
 * current device's, whose stream the call is put on; nothing is allocated, so calls
 * can be captured into graphs.  A workspace is scratch of one call at a time: calls
 * that may run at once, replays of graphs among them, have one each.  Sums,
 * statistics and activations are FP32 (but for sums of e4m3 products with a bf16 output,
 * see jh_op_linear), results are rounded once, and every sum
 * has a fixed order: the same call gives the same bits.  GELU and SiLU are good to
 * (8 + E) 2^-23 of their value, E = z^2 and |z| (the tanh form: 4 times the argument
 * of its exponential), down to 2^-119.  A row's bits may depend
 * on the number of rows in the call (kernels are chosen by size).  Squares are
 * summed as they are: rows whose sum of squares passes 3.4e38 are not normalised, nor,
 * with eps = 0, rows whose squares vanish in FP32.
 */

/*
 * s = x + resid (s = x where resid is NULL), rounded to resid's type and stored
 * to resid_out; out = s / sqrt(mean(s^2) + eps) * w, computed from the rounded
 * s.  x is f32, bf16 or f16; resid and resid_out are f32 or x's type, and may be
 * the same memory (NULL together).  hidden is at most 16384; w f32 [hidden].
 * out is bf16 or f16 (x's type where that is a 16-bit one), or e4m3 with
 * scales[rows]: scale = max|out| / 448 per row, and each code is the e4m3 value
 * nearest to the exact quotient of 448 s w by its row's max|s w| (ties to even),
 * so that codes do not depend on how sums are ordered.  A row of zeros has scale
 * 0, whatever eps (its 16-bit output with eps = 0 is 0 / 0); a NaN gives NaN codes; a row
 * with an infinity has no finite scale.
 * rstd[rows] (or NULL) receives 1 / sqrt(mean(s^2) + eps) for the backward pass.
 */
int jh_op_rms_norm(int x_type, const void* x, size_t ldx, int resid_type, const void* resid, size_t ldr,
                   void* resid_out, size_t ldro, size_t rows, size_t hidden, const float* w, float eps,
                   int out_type, void* out, size_t ldo, float* scales, float* rstd, void* stream);

/*
 * Gradients of jh_op_rms_norm with a 16-bit or f32 output: s is what it stored (or
 * x without a residual), rstd what it wrote, dy the gradient of out, dres (or
 * NULL) the gradient that reaches s past the norm.
 *   g = w dy, n = s rstd:  ds = rstd (g - n mean(g n)) + dres,  dw = sum over rows of dy n.
 * ds is the gradient of s, thus of x and of resid.  dy is f32, bf16 or f16; s, and
 * dres with ds, are f32 or dy's type.  ds may be dres, or dy or s where it has
 * their type and stride.  dw f32 [hidden], or NULL; it needs a workspace of
 * jh_op_rms_norm_backward_workspace(rows, hidden) bytes, 16-byte aligned.
 */
int jh_op_rms_norm_backward(int dy_type, const void* dy, size_t lddy, int s_type, const void* s, size_t lds,
                            size_t rows, size_t hidden, const float* w, const float* rstd, int ds_type,
                            const void* dres, size_t lddr, void* ds, size_t ldds, float* dw, void* workspace,
                            size_t workspace_bytes, void* stream);
size_t jh_op_rms_norm_backward_workspace(size_t rows, size_t hidden);

/*
 * q[r] = e4m3 codes of x[r] with scales[r] = max|x[r]| / 448, each code the value
 * nearest to the exact quotient of 448 x by the row's maximum (ties to even).  x is
 * f32, bf16 or f16, cols at most 16384.  Quantises activations for, and (once) the
 * rows of W of, jh_op_linear and jh_op_gated_ffn.
 */
int jh_op_quantize_rows(int x_type, const void* x, size_t ldx, size_t rows, size_t cols, void* q, size_t ldq,
                        float* scales, void* stream);

/*
 * out = act(z) + resid, z[r, j] = x_scale[r] w_scale[j] sum_k x[r, k] w[j, k] + bias[j].
 * type (of x and w): bf16, f16 or e4m3.  w [n, k] row-major without padding.
 * x_scale[rows] and w_scale[n] belong to e4m3 (NULL: ones); bias f32 [n] or NULL.
 * out and resid (or NULL) have out_type: f32, or type (bf16 for e4m3); resid may
 * be out itself, with its stride.  pre [rows, n] of type (16-bit types; or NULL)
 * receives z for the backward pass.  With e4m3 operands and a bf16 output the 8-bit
 * matrix instruction drops of every product the bits below 2^-13 of the largest one that it
 * adds with it: a sum is off by less than k 2^-13 of its largest |x w|, so where large
 * products cancel, small ones may be lost whole.  (Of normally distributed operands sums
 * came out within 1.5e-5 of their norm, 1/100 of the rounding to bf16.)  With an f32 output they
 * are FP32 sums of exact products, at half the rate.
 */
int jh_op_linear(int type, const void* x, size_t ldx, const float* x_scale, size_t rows, const void* w,
                 const float* w_scale, size_t n, size_t k, const float* bias, int act, const void* resid,
                 size_t ldr, int out_type, void* out, size_t ldo, void* pre, size_t ldp, void* stream);

/*
 * Gradients of jh_op_linear (bf16 or f16): dz = dy act'(pre), rounded to type;
 * dx = dz w, dw = dz^T x [n, k] without padding, dbias = column sums of dz before
 * its rounding, f32 [n].  The gradient of resid is dy.  Each of dx, dw, dbias may
 * be NULL; x is read for dw, w for dx, pre where act is not JH_ACT_NONE.  dx has
 * type, dw grad_type (type or f32).  rows = 0 writes zeros to dw and dbias.  The
 * workspace has jh_op_linear_backward_workspace(rows, n, k, act) bytes (0 where a
 * size is refused).
 */
int jh_op_linear_backward(int type, const void* dy, size_t lddy, const void* x, size_t ldx, size_t rows,
                          const void* w, size_t n, size_t k, int act, const void* pre, size_t ldp, void* dx,
                          size_t lddx, int grad_type, void* dw, float* dbias, void* workspace,
                          size_t workspace_bytes, void* stream);
size_t jh_op_linear_backward_workspace(size_t rows, size_t n, size_t k, int act);

/*
 * out = act(x Wg^T) * (x Wu^T) in one kernel: wi [2 inter, k] holds Wg's rows and then
 * Wu's, as jh_encoder_layer.wi does (JH_EPI_GEGLU_BF16's interleave is not needed).
 * type as for jh_op_linear, wi_scale [2 inter]; out has type (bf16 for e4m3, whose sums
 * are as jh_op_linear's with a bf16 output).  gu
 * [rows, 2 inter] of type (16-bit types; or NULL) receives both projections for
 * the backward pass.
 */
int jh_op_gated_ffn(int type, const void* x, size_t ldx, const float* x_scale, size_t rows, const void* wi,
                    const float* wi_scale, size_t inter, size_t k, int act, void* out, size_t ldo, void* gu,
                    size_t ldgu, void* stream);

/*
 * Gradients of jh_op_gated_ffn (bf16 or f16): dg = dh u act'(g), du = dh act(g), rounded to
 * type; dx = [dg du] wi, dwi = [dg du]^T x [2 inter, k] without padding.  dx has type,
 * dwi grad_type (type or f32); either may be NULL.  The workspace has
 * jh_op_gated_ffn_backward_workspace(rows, inter, k) bytes (0 where a size is refused).
 */
int jh_op_gated_ffn_backward(int type, const void* dh, size_t lddh, const void* gu, size_t ldgu, const void* x,
                             size_t ldx, size_t rows, const void* wi, size_t inter, size_t k, int act, void* dx,
                             size_t lddx, int grad_type, void* dwi, void* workspace, size_t workspace_bytes,
                             void* stream);
size_t jh_op_gated_ffn_backward_workspace(size_t rows, size_t inter, size_t k);

/*
 * Which kernels a product runs on, as the calls above choose them by size: jh_op_linear's
 * (LINEAR; n, k as there), jh_op_gated_ffn's (GATED; n its inter) and the gradients' dx and dw (DX, DW;
 * n and k as in jh_op_linear_backward, n = 2 inter for the gated projections').  Two launches
 * where the first takes whole rounds of 256 x 256 tiles and the second the other rows, else
 * launches[1].rows is 0.  rows counts the output's (DW: n of them in all), parts the pieces
 * of the contraction that are summed by one more kernel.  Needs no device.
 */
enum { JH_PRODUCT_LINEAR = 0, JH_PRODUCT_GATED = 1, JH_PRODUCT_DX = 2, JH_PRODUCT_DW = 3 };
enum {
    JH_KERNEL_SMALL = 0,   /* 64 x 64 tiles                            */
    JH_KERNEL_DEEP = 1,    /* 128 x 128, one tile to a CU              */
    JH_KERNEL_PAIR = 2,    /* 128 x 128, two to a CU                   */
    JH_KERNEL_TALL = 3,    /* 256 rows x 128 columns                   */
    JH_KERNEL_WIDE = 4,    /* 256 x 256                                */
    JH_KERNEL_STREAM = 5   /* up to 16 rows, w streams past them       */
};
typedef struct {
    int kernel, parts;
    size_t rows;
} jh_linear_launch;
int jh_op_linear_plan(int product, int type, int out_type, size_t rows, size_t n, size_t k, jh_linear_launch launches[2]);

#ifdef __cplusplus
}
#endif

#endif /* JULIA1_HIP_OPS_H */
