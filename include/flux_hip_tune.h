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
 * each batch element (groups == batch, 65535 at most), w_sb and b_sb elements apart. w null: the factor is 1, b null: nothing is added. plus_one != 0:
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
 * workspace (flux_layer_norm_bwd_workspace_bytes, 0 for few rows and where neither dw nor db is wanted; it need not be cleared), and rounded once. */
typedef struct flux_layer_norm_bwd_args {
    const void* dy; const void* x; const void* w; const float* mean; const float* rstd;
    void* dx; void* dw; void* db;
    int64_t batch, seq, dy_sb, dy_sl, x_sb, x_sl, groups, w_sb;
    int32_t n, x_dtype, w_dtype, plus_one;
} flux_layer_norm_bwd_args;
int64_t flux_layer_norm_bwd_workspace_bytes(const flux_layer_norm_bwd_args* args);
int flux_layer_norm_bwd(const flux_layer_norm_bwd_args* args, void* workspace, int64_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Rotary positions of several axes, straight from the tokens' ids.
 * A row has P = sum(axes_dim) / 2 pairs (x[2i], x[2i+1]); the first axes_dim[0] / 2 of them belong to axis 0, and so on. Pair j of an axis of
 * d values turns by the angle ids[b, l, axis] * theta^(-2j/d), formed in 64 bits.
 * ids is [B, L, n_axes] with element strides (ids_sb, ids_sl, ids_sa), ids_sb = 0 for one list of positions for all batch elements.
 * ------------------------------------------------------------------------------------------- */
enum flux_ids_dtype { FLUX_IDS_F32 = 0, FLUX_IDS_F64 = 1, FLUX_IDS_I32 = 2, FLUX_IDS_I64 = 3 };
enum { FLUX_ROPE_MOST_AXES = 8, FLUX_ROPE_MOST_DIM = 512 };
typedef struct flux_rope_ids {
    const void* ids; int64_t sb, sl, sa;
    double theta;
    int32_t dtype, n_axes, axes_dim[8];
} flux_rope_ids;

/* q_out = q and k_out = k with every pair turned by its angle ((x0 c - x1 s, x0 s + x1 c); inverse != 0: by the negative one, which is the
 * backward pass). q is [B, Hq, L, D] and k [B, Hk, L, D] with strides as in flux_src4, D = 2 P; the outputs are contiguous. Either may be
 * absent (null pointers and no heads), B is 65535 at most. fp32 arithmetic, rounded once; sines and cosines of an angle of a radians are within
 * 2^-23 + |a| (3 |log2 theta| + d / 5 + 5) 2^-53 of the exact ones, d the values of its axis; the second term is the smaller one up to positions of ten million. */
typedef struct flux_rope_nd_args {
    flux_src4 q, k;
    void* q_out; void* k_out;
    flux_rope_ids at;
    int64_t B, Hq, Hk, L;
    int32_t D, dtype, inverse;
} flux_rope_nd_args;
int flux_rope_nd(const flux_rope_nd_args* args, void* stream);

/* The rotation matrices themselves, as flux_qkv_prep and the q/k epilogue of flux_linear_bf16 take them:
 * out[b, l, pair] = [[c, -s], [s, c]], fp32, contiguous [B, L, P, 2, 2]. */
int flux_rope_table(const flux_rope_ids* at, float* out, int64_t B, int64_t L, void* stream);

/* ---------------------------------------------------------------------------------------------
 * A projection shared by many requests, each with a low-rank adapter of its own:
 *   y[m] = act(x[m] W^T + bias + s_i (x[m] a_i^T) b_i^T),  i = adapter[m / (M / requests)]
 * x [M, K] (row stride ldx), w [N, K] (row stride ldw), bias [N] or null, y [M, N] (row stride ldy) as in flux_linear_bf16, bf16; act
 * is FLUX_ACT_NONE or FLUX_ACT_GELU_TANH. lora_a is [adapters, rank, K], lora_b [adapters, N, rank], contiguous bf16, with rank up to
 * FLUX_LORA_MOST_RANK; scaling is fp32 [adapters] or null (1). adapter holds one number for each of `requests` groups of M / requests rows that
 * follow one another, int32 or (wide_ids) int64; a number outside [0, adapters) means no adapter, whatever lora_a and lora_b hold.
 * fp32 sums, y rounded once; s_i x a_i^T goes between the two products as a bf16 number and another one for what that leaves over, 2^-16 of its
 * value off. What is not finite in an adapter reaches rows of its own requests only, as the formula has it: +inf and -inf by the signs, NaN for
 * NaN, for 0 * inf and for infinities of both signs, whatever else is in the call.
 * The workspace (flux_linear_lora_workspace_bytes; 256-byte aligned, the launch's own until it has run) holds s_i x a_i^T and, where K is cut
 * over workgroups, partial sums; flux_linear_lora_least_bytes is what the call cannot do without. Beyond rank 16 that may have no room for the second
 * numbers of s_i x a_i^T, which is then off by 2^-8 of its value; twice that many bytes have it.
 * ------------------------------------------------------------------------------------------- */
#define FLUX_LORA_MOST_RANK 256
typedef struct flux_linear_lora_args {
    const void* x; const void* w; const void* bias; void* y;
    const void* lora_a; const void* lora_b; const void* adapter; const float* scaling;
    int64_t M, N, K, ldx, ldw, ldy, requests;
    int32_t adapters, rank, wide_ids, act;
} flux_linear_lora_args;
int64_t flux_linear_lora_workspace_bytes(const flux_linear_lora_args* args);
int64_t flux_linear_lora_least_bytes(const flux_linear_lora_args* args);
int flux_linear_lora_bf16(const flux_linear_lora_args* args, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* FLUX_HIP_TUNE_H */
