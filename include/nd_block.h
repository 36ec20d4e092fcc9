/*
 * nd_block.h -- C ABI of libnd_block.so: the operators of a transformer block over image tokens on MI355X (gfx950).
 *
 * They stand beside the attention and 1x1-convolution entry points of nd_hip.h and take the rows those produce: NHWC maps
 * are [batch, token, channel] rows here, and every tensor has its own element strides, so the q / k / v parts of a packed
 * qkv row are passed as they lie.  They form a library of their own so that a change here leaves the build id of
 * libnd_hip.so, and with it the measured kernel choices of the convolutions, as they are.
 *
 * Conventions (those of nd_hip.h): caller-owned device pointers; every launch is asynchronous on `stream`, allocation-free
 * and sync-free (a caller may capture it); scratch memory is the caller's, sized by the *_workspace_* functions; return
 * value 0 or ND_E_*, message via nd_block_last_error() (thread-local); nothing throws.  `dtype` (ND_DT_F32 / ND_DT_BF16) is
 * the type of every tensor and parameter of a call unless stated otherwise; sums and softmax statistics are fp32.
 */
#ifndef ND_BLOCK_H
#define ND_BLOCK_H

#include "nd_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

const char* nd_block_build_id(void);   /* hash of the library's sources */
const char* nd_block_last_error(void); /* thread-local message of the last failing call */

/* ---- RMS norm of each query / key head and rotation by position, one pass ------------------------------------------- */

#define ND_ROPE_INTERLEAVED 1 /* rotated pairs are channels (2i, 2i+1); default: (i, i + R/2) */

/* q [B, T, Hq, D], k [B, T, Hk, D] (Hk may be 0) with element strides (batch, token, head), channels contiguous; an output may be
 * its input itself (same pointer and strides), and overlaps nothing else (refused).  weights [D] or NULL.  cos / sin: fp32
 * [T][R/2] rows, batch stride table_sb (0 = shared by the batch); the first R channels are rotated (R even, 0 = none).  D even, at
 * most 512. */
int nd_qk_norm_rope(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh,
                    const void* q_weight, const void* k_weight, const float* cos, const float* sin, int64_t table_sb, void* q_out,
                    int64_t qo_sb, int64_t qo_st, int64_t qo_sh, void* k_out, int64_t ko_sb, int64_t ko_st, int64_t ko_sh, int B, int T,
                    int Hq, int Hk, int D, int R, float eps, int flags, int dtype, nd_stream_t stream);

/* Whether a [B, T, Ha, D] and b [B, T, Hb, D] (element strides; es: bytes of an element) have an address in common; b NULL: whether
 * rows of a meet each other.  Exact where both have the same strides (views of one packed row), else 1 if their ranges meet. */
int nd_rows_overlap(const void* a, int64_t a_sb, int64_t a_st, int64_t a_sh, int Ha, const void* b, int64_t b_sb, int64_t b_st, int64_t b_sh,
                    int Hb, int B, int T, int D, int es);

/* gradients: dq, dk (own strides) and, where dq_weight / dk_weight is not NULL, the weights' (needs the workspace) */
int nd_qk_norm_rope_bwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh,
                        const void* q_weight, const void* k_weight, const float* cos, const float* sin, int64_t table_sb,
                        const void* dq_out, int64_t dqo_sb, int64_t dqo_st, int64_t dqo_sh, const void* dk_out, int64_t dko_sb,
                        int64_t dko_st, int64_t dko_sh, void* dq, int64_t dq_sb, int64_t dq_st, int64_t dq_sh, void* dk, int64_t dk_sb,
                        int64_t dk_st, int64_t dk_sh, void* dq_weight, void* dk_weight, float* workspace, int B, int T, int Hq, int Hk,
                        int D, int R, float eps, int flags, int dtype, nd_stream_t stream);
int64_t nd_qk_norm_rope_bwd_workspace_floats(int B, int T, int Hq, int Hk, int D);

/* ---- differential attention --------------------------------------------------------------------------------------------- */

#define ND_ATTN_CAUSAL 1 /* query t sees the keys up to t + length - Tq */

/* out = (softmax(scale q1 k1^T) - lam softmax(scale q2 k2^T)) v with lam = exp(lq1 . lk1) - exp(lq2 . lk2) + lambda_init
 * q [B, Tq, H, 2D], k [B, Tk, Hk, 2D] (channels 0 .. D-1: first map, D .. 2D-1: second), v [B, Tk, Hk, Dv], element strides
 * (batch, token, head), channels contiguous, rows 16-byte aligned.  Query heads h use key head h / (H / Hk).  D, Dv multiples of
 * 8, at most 128 / 256.  lambda vectors [D] (lambda_sh 0) or [H, D] (lambda_sh D).  key_lengths [B] on the device or NULL: keys
 * at or past it are neither used nor read as numbers; a query that sees no key gives a zero row.  out [B, Tq, H, Dv] contiguous.
 * Training: out1, out2 (the two maps' own outputs, like out) and lse [2][B, Tq, H], all or none. */
int nd_diff_attention(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh,
                      const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh, const void* lambda_q1, const void* lambda_k1,
                      const void* lambda_q2, const void* lambda_k2, int64_t lambda_sh, float lambda_init, const int* key_lengths,
                      void* out, void* out1, void* out2, float* lse, float* workspace, int B, int Tq, int Tk, int H, int Hk, int D, int Dv,
                      float scale, int flags, int dtype, nd_stream_t stream);
int64_t nd_diff_attention_workspace_floats(int B, int Tq, int Tk, int H, int Hk, int D, int Dv, int dtype); /* may be 0 */

/* gradients of nd_diff_attention from its out1, out2 and lse: dq [B, Tq, H, 2D], dk [B, Tk, Hk, 2D], dv [B, Tk, Hk, Dv]
 * contiguous; the lambda vectors' (laid out like them) where not NULL.  dout [B, Tq, H, Dv] with its own strides. */
int nd_diff_attention_bwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh,
                          const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh, const void* lambda_q1, const void* lambda_k1,
                          const void* lambda_q2, const void* lambda_k2, int64_t lambda_sh, float lambda_init, const int* key_lengths,
                          const void* out1, const void* out2, const float* lse, const void* dout, int64_t do_sb, int64_t do_st,
                          int64_t do_sh, void* dq, void* dk, void* dv, void* dlambda_q1, void* dlambda_k1, void* dlambda_q2,
                          void* dlambda_k2, float* workspace, int B, int Tq, int Tk, int H, int Hk, int D, int Dv, float scale, int flags,
                          int dtype, nd_stream_t stream);
int64_t nd_diff_attention_bwd_workspace_floats(int B, int Tq, int Tk, int H, int Hk, int D, int Dv, int dtype);

/* ---- gated feed-forward block ----------------------------------------------------------------------------------------- */

#define ND_ACT_SILU 0
#define ND_ACT_GELU 1      /* a Phi(a), with the error function */
#define ND_ACT_GELU_TANH 2 /* its tanh form */

/* y = residual + (act(x w_in[:F]^T + b_in[:F]) * (x w_in[F:]^T + b_in[F:])) w_out^T + b_out
 * x [M, C] (row stride ldx), w_in [2F, C], b_in [2F] or NULL, w_out [C, F], b_out [C] or NULL, residual [M, C] (ldr) or NULL,
 * y [M, C] (ldy; may be the residual's memory).  C, F multiples of 8; rows and pointers 16-byte aligned.  h [M, F]: scratch,
 * and what the backward pass reads; au [M, 2F]: the pre-activations for the backward pass, or NULL. */
int nd_gated_ffn(const void* x, int64_t ldx, const void* w_in, const void* b_in, const void* w_out, const void* b_out, const void* residual,
                 int64_t ldr, void* y, int64_t ldy, void* h, void* au, float* workspace, int M, int C, int F, int act, int dtype,
                 nd_stream_t stream);
int64_t nd_gated_ffn_workspace_floats(int M, int C, int F, int dtype); /* may be 0: workspace NULL */

/* gradients of nd_gated_ffn (any of dx [M, C], dw_in, db_in, dw_out, db_out may be NULL; that of the residual is dy); dau
 * [M, 2F] is scratch for the first three */
int nd_gated_ffn_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w_in, const void* w_out, const void* au,
                     const void* h, void* dx, void* dw_in, void* db_in, void* dw_out, void* db_out, void* dau, float* workspace, int M,
                     int C, int F, int act, int dtype, nd_stream_t stream);
int64_t nd_gated_ffn_bwd_workspace_floats(int M, int C, int F, int dtype);

/* ---- one array of arguments ------------------------------------------------------------------------------------------- */

#define ND_CALL_QK_NORM_ROPE 0
#define ND_CALL_QK_NORM_ROPE_BWD 1
#define ND_CALL_DIFF_ATTENTION 2
#define ND_CALL_DIFF_ATTENTION_BWD 3
#define ND_CALL_GATED_FFN 4
#define ND_CALL_GATED_FFN_BWD 5

/* The call above with its arguments (all but the stream) as 8-byte words in their order: pointers and integers as they are, floats as
 * doubles.  For callers through a foreign-function interface, whose cost is per argument. */
int nd_block_packed(int call, const int64_t* words, int count, nd_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif
