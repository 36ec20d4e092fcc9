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

/* q [B, T, Hq, D], k [B, T, Hk, D] (Hk may be 0) with element strides (batch, token, head), channels contiguous; outputs may
 * be the inputs themselves (same pointer and strides).  weights [D] or NULL.  cos / sin: fp32 [T][R/2] rows, batch stride
 * table_sb (0 = shared by the batch); the first R channels are rotated (R even, 0 = none).  D even, at most 512. */
int nd_qk_norm_rope(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh,
                    const void* q_weight, const void* k_weight, const float* cos, const float* sin, int64_t table_sb, void* q_out,
                    int64_t qo_sb, int64_t qo_st, int64_t qo_sh, void* k_out, int64_t ko_sb, int64_t ko_st, int64_t ko_sh, int B, int T,
                    int Hq, int Hk, int D, int R, float eps, int flags, int dtype, nd_stream_t stream);

/* gradients: dq, dk (own strides) and, where dq_weight / dk_weight is not NULL, the weights' (needs the workspace) */
int nd_qk_norm_rope_bwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh,
                        const void* q_weight, const void* k_weight, const float* cos, const float* sin, int64_t table_sb,
                        const void* dq_out, int64_t dqo_sb, int64_t dqo_st, int64_t dqo_sh, const void* dk_out, int64_t dko_sb,
                        int64_t dko_st, int64_t dko_sh, void* dq, int64_t dq_sb, int64_t dq_st, int64_t dq_sh, void* dk, int64_t dk_sb,
                        int64_t dk_st, int64_t dk_sh, void* dq_weight, void* dk_weight, float* workspace, int B, int T, int Hq, int Hk,
                        int D, int R, float eps, int flags, int dtype, nd_stream_t stream);
int64_t nd_qk_norm_rope_bwd_workspace_floats(int B, int T, int Hq, int Hk, int D);

#ifdef __cplusplus
}
#endif
#endif
