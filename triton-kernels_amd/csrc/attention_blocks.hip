// Attention of blocks of 128 queries over the blocks of 64 keys that a list names for each.
//
//   o[i] = sum_j p_j v[j],  p = softmax(scale q[i] . k[j]),  j over the tokens of the list of i's block
//
// 4 D operations for each pair of a query and a listed key: bound by the matrix cores, and for single tokens by the bytes of k and v. The 32-row kernel of
// attention_pipe.h with a block of the list for a tile: a workgroup of four waves takes one block of queries, so its list is one list for all its rows, and every
// tile of keys is read by all of them. Where lists are long and query blocks few, a list is cut over several workgroups.
// us: 24 heads of 128, 4608 tokens, 18 of 72 blocks 81 (65 GFLOP: 0.80 PFLOP/s, four workgroups on some CUs and three on others), 32760 tokens, 64 of 512 blocks 1604 (1.03
// PFLOP/s); all blocks at 4608 tokens take the kernels for all keys 200.
#include "attention_pipe.h"
#include "../../include/flux_hip_serve.h"
#include <algorithm>
#include <math.h>

namespace flux {

template <int D>
__global__ __launch_bounds__(256, 2) void attn_blocks_kernel(AttnParams p, ListedKeys from) {
    __shared__ __attribute__((aligned(1024))) char lds[pipe_lds_bytes(D, 64)];
    attn_pipe<D, 1, 64, false, true, false>(p, lds, gridDim.x, nullptr, 1, 0, from);
}

template <int D>
__global__ __launch_bounds__(256, 2) void attn_blocks_parts_kernel(AttnParams p, ListedKeys from, float* ws, int splits, int part_entries) {
    __shared__ __attribute__((aligned(1024))) char lds[pipe_lds_bytes(D, 64)];
    attn_pipe<D, 1, 64, true, true, false>(p, lds, gridDim.x, ws, splits, part_entries, from);
}

// O = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s over the parts of a row's list, in their order; rows whose parts have no key (m_s = -inf, l_s = 0) are 0. A wave
// takes 32 rows x 32 columns, in the layout attn_pipe leaves them in.
template <int D>
__global__ __launch_bounds__(256) void attn_blocks_combine_kernel(AttnParams p, const float* ws, int splits, int blocks) {
    constexpr int DB = D / 32, BPG = 4 / DB;   // blocks of 32 rows per workgroup
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, frow = lane & 31, fhalf = lane >> 5;
    const int64_t blk = static_cast<int64_t>(blockIdx.x) * BPG + wave / DB;
    const int db = wave % DB, per_bh = p.n_qtiles * 4;
    if (blk >= blocks) return;
    const int bh = static_cast<int>(blk / per_bh), row0 = static_cast<int>(blk % per_bh) * 32, row = row0 + frow;
    if (row0 >= p.L) return;
    const f32x2* const ml = reinterpret_cast<const f32x2*>(ws + static_cast<int64_t>(splits) * blocks * (32 * D)) + blk * 32 + frow;
    const Vec16<float>* const part = reinterpret_cast<const Vec16<float>*>(ws) + (blk * (8 * D) + db * 256 + lane);
    float m = -INFINITY, l = 0.0f, acc[16] = {};
    bool seen = false;
    for (int s = 0; s < splits; ++s) {
        const f32x2 t = ml[static_cast<int64_t>(s) * blocks * 32];
        m = fmaxf(m, t.x);
        seen |= t.y != 0.0f;
    }
#pragma unroll 2
    for (int s = 0; s < splits; ++s) {
        const f32x2 t = ml[static_cast<int64_t>(s) * blocks * 32];
        // a part without a key, or with scores of -inf only beside others, adds nothing; NaNs stay in l_s and O_s
        const float w = t.x == -INFINITY ? 0.0f : t.x == m ? 1.0f : __builtin_amdgcn_exp2f(t.x - m);
        l += t.y * w;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const Vec16<float> a = part[static_cast<int64_t>(s) * blocks * (8 * D) + g * 64];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[g * 4 + e] = __builtin_fmaf(a.v[e], w, acc[g * 4 + e]);
        }
    }
    if (row >= p.L) return;
    const float inv = seen ? 1.0f / l : 0.0f;
    bf16_t* const orow = p.o + (bh / p.H) * p.o_sb + (bh % p.H) * p.o_sh + row * p.o_sl + db * 32 + fhalf * 4;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        u32x2 y;
        y.x = pack2_bf16(acc[g * 4 + 0] * inv, acc[g * 4 + 1] * inv);
        y.y = pack2_bf16(acc[g * 4 + 2] * inv, acc[g * 4 + 3] * inv);
        *reinterpret_cast<u32x2*>(orow + g * 8) = y;
    }
}

// Parts that lists are cut in where their workgroups leave CUs idle. A workgroup alone on its CU takes 1.03 us a block (0.68 at head dim 64); two on one CU take twice
// that, so more than 256 gain nothing. The second launch and the parts' results cost some 2.3 us (1.0), 0.6 a part and 0.027 a workgroup of 128 rows, less with fewer.
// us whole and in the parts that this takes: heads of 128, one token of 24 heads, 32 blocks 37.7 and 17.7 (8 parts), of 4 x 24 heads 39.1 and 27.5 (2), 8 x 1000 rows, 18 blocks
// 25.8 and 22.6 (4), 24 x 640 rows, 18 blocks 26.4 and 24.8 (2), 24 x 512 rows, 6 blocks 13.4 (whole; 19.0 in 2); heads of 64, one token of 24 heads, 16 blocks 15.9 and 11.0 (5).
static int sparse_splits(int64_t groups, int64_t rows, int64_t count, int D, int& part_entries) {
    const double tile_us = D == 128 ? 1.03 : 0.68, fixed_us = D == 128 ? 2.3 : 1.0, group_us = 0.027 * static_cast<double>((std::min<int64_t>(rows, 128) + 31) / 32) / 4.0;
    double gained = 0.5;
    part_entries = static_cast<int>(count);
    for (int64_t s = 2; s <= 16 && s * groups <= 256 && s <= count; ++s) {
        const int64_t part = (count + s - 1) / s;
        const double gain = tile_us * static_cast<double>(count - part) - (fixed_us + 0.6 * static_cast<double>(s) + group_us * static_cast<double>(groups * s));
        if (gain <= gained) continue;
        gained = gain;
        part_entries = static_cast<int>(part);
    }
    return count == 0 ? 1 : static_cast<int>((count + part_entries - 1) / part_entries);   // (no part is empty)
}
static int64_t sparse_bytes(int64_t groups, int D, int splits) { return splits > 1 ? splits * groups * 128 * (D + 2) * 4 : 0; }

template <int D>
static void sparse_launch(AttnParams& p, const ListedKeys& from, int64_t groups, void* ws, int64_t ws_bytes, hipStream_t st) {
    int part_entries, splits = sparse_splits(groups, p.L, from.count, D, part_entries);
    if (splits > 1 && ws_bytes < sparse_bytes(groups, D, splits)) splits = 1;
    p.total_tiles = static_cast<int>(groups * splits);
    const dim3 grid((p.total_tiles + 7) / 8 * 8);
    if (splits == 1) {
        hipLaunchKernelGGL(attn_blocks_kernel<D>, grid, dim3(256), 0, st, p, from);
        return;
    }
    hipLaunchKernelGGL(attn_blocks_parts_kernel<D>, grid, dim3(256), 0, st, p, from, static_cast<float*>(ws), splits, part_entries);
    const int blocks = static_cast<int>(groups) * 4, per_group = 128 / D;
    hipLaunchKernelGGL(attn_blocks_combine_kernel<D>, dim3((blocks + per_group - 1) / per_group), dim3(256), 0, st, p, static_cast<const float*>(ws), splits, blocks);
}

}  // namespace flux

using namespace flux;

static bool sparse_view_ok(const void* ptr, int64_t sb, int64_t sh, int64_t sl) {
    return ptr != nullptr && aligned16(ptr) && sb % 8 == 0 && sh % 8 == 0 && sl % 8 == 0;
}

// Checks a call and turns it into the kernels' parameters; `nothing`: there are no rows.
static int read_sparse_args(const flux_sparse_attention_args* a, AttnParams& p, ListedKeys& from, bool& nothing) {
    const char* const what = "flux_sparse_attention_bf16";
    nothing = false;
    if (!a) return fail(FLUX_E_NULL, "%s: null args", what);
    if (a->B < 0 || a->Hq <= 0 || a->Hk <= 0 || a->Hq % a->Hk != 0 || a->Lq < 0 || a->Lk < 0 || a->count < 0)
        return fail(FLUX_E_SHAPE, "%s: bad shape B=%lld Hq=%lld Hk=%lld Lq=%lld Lk=%lld, lists of %lld", what, (long long)a->B, (long long)a->Hq, (long long)a->Hk, (long long)a->Lq,
                    (long long)a->Lk, (long long)a->count);
    if (a->D != 64 && a->D != 128) return fail(FLUX_E_UNSUPPORTED, "%s: head dim %d not supported (64, 128)", what, a->D);
    const float scale = a->sm_scale * 1.4426950408889634f;
    if (!(fabsf(scale) < INFINITY)) return fail(FLUX_E_UNSUPPORTED, "%s: sm_scale is not finite", what);
    nothing = a->B == 0 || a->Lq == 0;
    if (nothing) return FLUX_OK;
    const int64_t tiles = (a->Lq + FLUX_QUERY_BLOCK - 1) / FLUX_QUERY_BLOCK;
    if (a->Lq > 0x7fffffff / 64 || a->Lk > 0x7fffffff / 64 || a->B > 0x7fffffff / 64 || a->Hq > 0x7fffffff / 64 / a->B || a->B * a->Hq > 0x7fffffff / 256 / tiles || a->count > 0x7fffffff / 64)
        return fail(FLUX_E_SHAPE, "%s: problem too large", what);
    const bool keys = a->Lk > 0 && a->count > 0;   // without any, k, v and blocks are not looked at
    if (!sparse_view_ok(a->q.ptr, a->q.sb, a->q.sh, a->q.sl) || !sparse_view_ok(a->o, a->o_sb, a->o_sh, a->o_sl) ||
        (keys && (!sparse_view_ok(a->k.ptr, a->k.sb, a->k.sh, a->k.sl) || !sparse_view_ok(a->v.ptr, a->v.sb, a->v.sh, a->v.sl))))
        return fail(FLUX_E_ALIGN, "%s: q/k/v/o must be non-null, 16-byte aligned, with strides that are multiples of 8", what);
    if (keys && !a->blocks) return fail(FLUX_E_NULL, "%s: null lists", what);
    if (a->k.sl * 2 * 64 >= 0x7fffffffLL || a->v.sl * 2 * 64 >= 0x7fffffffLL || a->k.sl < 0 || a->v.sl < 0) return fail(FLUX_E_SHAPE, "%s: row stride too large", what);
    p = {};
    p.q = static_cast<const bf16_t*>(a->q.ptr); p.k = static_cast<const bf16_t*>(a->k.ptr);
    p.v = static_cast<const bf16_t*>(a->v.ptr); p.o = static_cast<bf16_t*>(a->o);
    p.q_sb = a->q.sb; p.q_sh = a->q.sh; p.q_sl = a->q.sl;
    p.k_sb = a->k.sb; p.k_sh = a->k.sh; p.k_sl = a->k.sl;
    p.v_sb = a->v.sb; p.v_sh = a->v.sh; p.v_sl = a->v.sl;
    p.o_sb = a->o_sb; p.o_sh = a->o_sh; p.o_sl = a->o_sl;
    p.H = static_cast<int>(a->Hq); p.L = static_cast<int>(a->Lq);
    p.n_qtiles = static_cast<int>(tiles);
    // the sign goes into Q, and so does a scale of 0: masked scores of -inf stay what they are
    p.scale_log2 = scale > 0.0f ? 1.0f : scale < 0.0f ? -1.0f : 0.0f;
    from = {a->blocks, a->lengths, keys ? static_cast<int>(a->count) : 0, static_cast<int>(a->Hq / a->Hk), static_cast<int>(a->Lk), scale == 0.0f ? 1.0f : fabsf(scale)};
    return FLUX_OK;
}

extern "C" int64_t flux_sparse_attention_workspace_bytes(const flux_sparse_attention_args* a) {
    if (!a || a->B <= 0 || a->Hq <= 0 || a->Lq <= 0 || a->Lk <= 0 || a->count <= 0 || (a->D != 64 && a->D != 128)) return 0;
    const int64_t tiles = (a->Lq + FLUX_QUERY_BLOCK - 1) / FLUX_QUERY_BLOCK;
    if (a->B > 1024 || a->Hq > 1024 || tiles > 1024) return 0;   // (never few)
    int part_entries;
    return sparse_bytes(a->B * a->Hq * tiles, a->D, sparse_splits(a->B * a->Hq * tiles, a->Lq, a->count, a->D, part_entries));
}

extern "C" int flux_sparse_attention_bf16(const flux_sparse_attention_args* a, void* workspace, int64_t workspace_bytes, void* stream) {
    AttnParams p;
    ListedKeys from;
    bool nothing;
    const int rc = read_sparse_args(a, p, from, nothing);
    if (rc != FLUX_OK || nothing) return rc;
    if (workspace_bytes < 0 || (workspace_bytes > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)))
        return fail(FLUX_E_NULL, "flux_sparse_attention_bf16: workspace must be 256-byte aligned memory");
    const int64_t groups = a->B * a->Hq * p.n_qtiles;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->D == 128) sparse_launch<128>(p, from, groups, workspace, workspace_bytes, st);
    else sparse_launch<64>(p, from, groups, workspace, workspace_bytes, st);
    return check_launch("flux_sparse_attention_bf16");
}
