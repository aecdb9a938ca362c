/*
 * flux_hip_tune.h — C ABI of libfluxhip.so, second part: what fine-tuning a block and serving one block to many requests
 * need beside the operators of flux_hip.h, whose conventions (device pointers, strides in elements, streams, return values,
 * flux_last_error, dtype codes) hold here too. None of these calls stands for an interface of the reference.
 */
#ifndef FLUX_HIP_TUNE_H
#define FLUX_HIP_TUNE_H

#include "flux_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FLUX_TUNE_ABI_VERSION 1
int flux_tune_abi_version(void);

/* ---------------------------------------------------------------------------------------------
 * Layer norm with weights.   h = (x - mean) * rstd,  y = h * w + b,  rounded once.
 * x is [batch, seq, n] with element strides (sb, sl, 1), y contiguous. w and b are [n] vectors: one for all rows (groups 1), or one for
 * each batch element (groups == batch), w_sb and b_sb elements apart. w null: the factor is 1, b null: nothing is added. plus_one != 0:
 * the factor is 1 + w (adaLN's scale).
 * mean and rstd (both or neither null) receive the fp32 statistics of every row, for the backward pass.
 * w and b may be FLUX_F32 while x is FLUX_BF16. Statistics, factors and sums are fp32.
 * ------------------------------------------------------------------------------------------- */
typedef struct flux_layer_norm_fwd_args {
    const void* x; const void* w; const void* b; void* y;
    float* mean; float* rstd;
    int64_t batch, seq, x_sb, x_sl, groups, w_sb, b_sb;
    int32_t n, x_dtype, w_dtype, plus_one;
    float eps;
} flux_layer_norm_fwd_args;
int flux_layer_norm(const flux_layer_norm_fwd_args* args, void* stream);

/* Its gradients. With g = dy * w (or dy * (1 + w)):
 *   dx = rstd * (g - mean_n(g) - h * mean_n(g * h)),  dw = sum over the rows of a weight of dy * h,  db = the same of dy.
 * x and dy have strides of their own, dx is contiguous. dw and db are contiguous [groups, n] in w_dtype; each of
 * dx, dw and db may be null. Sums over rows are formed in fp32 in a fixed order, whose parts go through the
 * workspace (flux_layer_norm_bwd_workspace_bytes, 0 where neither dw nor db is wanted; it need not be cleared), and rounded once. */
typedef struct flux_layer_norm_bwd_args {
    const void* dy; const void* x; const void* w; const float* mean; const float* rstd;
    void* dx; void* dw; void* db;
    int64_t batch, seq, dy_sb, dy_sl, x_sb, x_sl, groups, w_sb;
    int32_t n, x_dtype, w_dtype, plus_one;
} flux_layer_norm_bwd_args;
int64_t flux_layer_norm_bwd_workspace_bytes(const flux_layer_norm_bwd_args* args);
int flux_layer_norm_bwd(const flux_layer_norm_bwd_args* args, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* FLUX_HIP_TUNE_H */
