/*
 * flux_hip_serve.h — C ABI of libfluxhip.so, third part: serving a block with less to read and less to multiply. Products with weights held in 4
 * bits, and attention over the blocks of keys that a cheap score selects. The conventions of flux_hip.h (device pointers, strides in elements,
 * streams, return values, flux_last_error, dtype codes) hold here too. None of these calls stands for an interface of the reference.
 */
#ifndef FLUX_HIP_SERVE_H
#define FLUX_HIP_SERVE_H

#include "flux_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FLUX_SERVE_ABI_VERSION 2
int flux_serve_abi_version(void);

/* ---------------------------------------------------------------------------------------------
 * Weights in 4 bits.  W[n, k] = (q[n, k] - z[n, k / group]) * s[n, k / group], q and z in 0 .. 15, s bf16, z null: 8 everywhere; group 32, 64 or 128,
 * K a multiple of it. In memory (N up to a multiple of 16, K of 128, what is behind them q = z = s = 0):
 *   q      tiles of 16 rows x 128 columns, [ceil(N / 16)][ceil(K / 128)][4][16][16 bytes]: 16 bytes at [g][r] are row r's columns 32 j + 8 g + e
 *          (j 0 .. 3 the 32-bit word, e 0 .. 7), e at bits 4 (e / 2) + 16 (e mod 2) of its word
 *   s, z   [ceil(N / 16)][ceil(K / 128)][16][128 / group], two bytes and one byte each
 * ------------------------------------------------------------------------------------------- */
typedef struct flux_w4 {
    const void* q; const void* s; const void* z;
    int64_t N, K;
    int32_t group;
} flux_w4;

/* y[m] = act(f(x[m]) W^T + bias): x [M, K] bf16 (row stride ldx), bias [N] bf16 or null, y [M, N] bf16 (row stride ldy); act is FLUX_ACT_NONE or
 * FLUX_ACT_GELU_TANH, in_act FLUX_ACT_NONE or (up to 8 rows) FLUX_ACT_SILU, f(x) = x sigmoid(x). fp32 sums, rounded once; f(x) is held to 2^-16 of its
 * value. Up to 128 rows a group's sum is that of (q + 16) x less that of (z + 16) x, both in fp32: what they lose is some 2^-23 of the group's sum of (32 + q + z) |x| s,
 * also where q = z leaves nothing of the largest x. Beyond them each weight is rounded to bf16 once (2^-8 of it), and ldx is at least K: some hundreds of rows of thousands of outputs take them in registers, others lay them
 * out in the workspace (flux_linear_w4_workspace_bytes, 0 for all the others; 256-byte aligned, the launch's own until it has run) in front of flux_linear_bf16. */
typedef struct flux_linear_w4_args {
    const void* x; const void* bias; void* y;
    flux_w4 w;
    int64_t M, ldx, ldy;
    int32_t act, in_act;
} flux_linear_w4_args;
int64_t flux_linear_w4_workspace_bytes(const flux_linear_w4_args* args);
int flux_linear_w4_bf16(const flux_linear_w4_args* args, void* workspace, int64_t workspace_bytes, void* stream);

/* The weights themselves, out [N, K] bf16, contiguous, rounded once. */
int flux_w4_unpack(const flux_w4* w, void* out, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Which blocks of keys a block of queries attends to.
 * q [B, Hq, Lq, D] and k [B, Hk, Lk, D] bf16 with strides as in flux_src4, Hq a multiple of Hk (query head h reads key head h / (Hq / Hk)), D 64 or 128. For each
 * block of FLUX_QUERY_BLOCK queries (the last may be shorter) the scores of the blocks of FLUX_KEY_BLOCK keys are mean(q) . mean(k), formed in 64 bits;
 * the `keep` largest (or all, where there are no more) are chosen, the lower number among equals, a NaN below everything, the first `always` blocks (up to `keep` of them) in any case.
 * lengths (int32 [B], or null): keys from lengths[b] on are not there; below 0 counts as 0, beyond Lk as Lk. q_lengths (the same for q and Lq): queries from
 * q_lengths[b] on are in no mean, and a block of none but them names nothing, -1 throughout. Without it all Lq rows of q are in their blocks' means.
 * blocks receives int32 [B, Hq, ceil(Lq / 128), min(keep, ceil(Lk / 64))]: the chosen numbers in ascending order, -1 behind them.
 * The workspace (flux_select_blocks_workspace_bytes; 256-byte aligned) holds the means, 8 D bytes a block and head, and beyond 1024 blocks of keys scores: 64 KB
 * for each of them, less where there are fewer than 8192 query blocks and heads.
 * ------------------------------------------------------------------------------------------- */
enum { FLUX_QUERY_BLOCK = 128, FLUX_KEY_BLOCK = 64, FLUX_SELECT_MOST_BLOCKS = 16384 };
typedef struct flux_select_blocks_args {
    flux_src4 q, k;
    const int32_t* lengths; int32_t* blocks;
    int64_t B, Hq, Hk, Lq, Lk, keep, always;
    int32_t D;
    const int32_t* q_lengths;
} flux_select_blocks_args;
int64_t flux_select_blocks_workspace_bytes(const flux_select_blocks_args* args);
int flux_select_blocks(const flux_select_blocks_args* args, void* workspace, int64_t workspace_bytes, void* stream);

/* Attention of every block of queries over the blocks of keys that its list names:
 *   o[i] = sum_j p_j v[j],  p = softmax(sm_scale q[i] . k[j]) over the tokens j of those blocks, j < min(lengths[b], Lk).
 * q, o [B, Hq, Lq, D], k, v [B, Hk, Lk, D] bf16. blocks is int32 [B, Hq, ceil(Lq / 128), count], contiguous; numbers that are no block of the sequence
 * name nothing, a number that stands there twice counts twice. Rows that see no token at all are 0. sm_scale is finite.
 * The workspace (flux_sparse_attention_workspace_bytes, 0 where lists are not cut; 256-byte aligned) holds partial results; without it lists stay whole. */
typedef struct flux_sparse_attention_args {
    flux_src4 q, k, v;
    void* o; int64_t o_sb, o_sh, o_sl;
    const int32_t* blocks; const int32_t* lengths;
    int64_t B, Hq, Hk, Lq, Lk, count;
    int32_t D; float sm_scale;
} flux_sparse_attention_args;
int64_t flux_sparse_attention_workspace_bytes(const flux_sparse_attention_args* args);
int flux_sparse_attention_bf16(const flux_sparse_attention_args* args, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* FLUX_HIP_SERVE_H */
