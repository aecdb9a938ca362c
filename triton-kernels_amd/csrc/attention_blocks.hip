// Attention of blocks of 128 queries over the blocks of 64 keys that a list names for each.
//
// The 32-row kernel of attention_pipe.h with a block of the list for a tile: a workgroup of four waves takes one block of queries, so its list is one list
// for all its rows, and every tile of keys is read by all of them. Where lists are long and query blocks few, a list is cut over several workgroups, whose
// results attn_blocks_combine_kernel adds up as it does for all keys.
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

extern "C" int64_t flux_sparse_attention_workspace_bytes(const flux_sparse_attention_args*) { return 0; }

extern "C" int flux_sparse_attention_bf16(const flux_sparse_attention_args* a, void*, int64_t, void* stream) {
    AttnParams p;
    ListedKeys from;
    bool nothing;
    const int rc = read_sparse_args(a, p, from, nothing);
    if (rc != FLUX_OK || nothing) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    p.total_tiles = static_cast<int>(a->B * a->Hq * p.n_qtiles);
    const dim3 grid((p.total_tiles + 7) / 8 * 8);
    if (a->D == 128) hipLaunchKernelGGL(attn_blocks_kernel<128>, grid, dim3(256), 0, st, p, from);
    else hipLaunchKernelGGL(attn_blocks_kernel<64>, grid, dim3(256), 0, st, p, from);
    return check_launch("flux_sparse_attention_bf16");
}
