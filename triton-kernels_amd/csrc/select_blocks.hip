// Which blocks of 64 keys each block of 128 queries attends to: the means of the blocks, their products as scores, the largest of each row.
//
//   mq[i] = mean of block i's queries, mk[j] = mean of block j's keys, score[i, j] = mq[i] . mk[j]
//
// Everything behind the reads of q and k is formed in 64 bits: a row's scores lie close together, and which of two neighbours in their order is chosen must not
// go with the order of a sum. That is cheap: the sums of the means are an addition a value beside its two bytes, and the products 2 D operations for 64 x 128 x D of
// the attention itself, on the matrix cores (16x16x4). Bound by reading q and k once.
#include "common.h"
#include "../../include/flux_hip_serve.h"
#include <algorithm>

namespace flux {

struct SelectParams {
    flux_src4 q, k;
    const int32_t* lengths; int32_t* blocks;
    double* mq; double* mk; double* scores;
    int B, Hq, Hk, Lq, Lk, nq, nk, keep, width, always;   // width: entries of a list
    int64_t groups;                                      // of 16 query blocks of a (batch, head)
};

__device__ __forceinline__ int select_length(const SelectParams& p, int b) { return p.lengths ? min(max(p.lengths[b], 0), p.Lk) : p.Lk; }

// A workgroup takes one block of tokens; a thread 8 columns of every (2048 / D)th row, all requested at once.
template <int D>
__global__ __launch_bounds__(256) void block_means_kernel(SelectParams p) {
    constexpr int CH = D / 8, RG = 256 / CH;
    __shared__ double fold[RG][D];
    const int64_t q_blocks = static_cast<int64_t>(p.B) * p.Hq * p.nq;
    const bool is_q = static_cast<int64_t>(blockIdx.x) < q_blocks;
    const int64_t at = is_q ? blockIdx.x : blockIdx.x - q_blocks;
    const int n = is_q ? p.nq : p.nk, H = is_q ? p.Hq : p.Hk, size = is_q ? FLUX_QUERY_BLOCK : FLUX_KEY_BLOCK;
    const int blk = static_cast<int>(at % n), h = static_cast<int>(at / n % H), b = static_cast<int>(at / n / H);
    const int rows = min(size, (is_q ? p.Lq : select_length(p, b)) - blk * size);
    if (rows <= 0) return;   // (a block of keys that is not there)
    const flux_src4 src = is_q ? p.q : p.k;
    const int c = threadIdx.x % CH, rg = threadIdx.x / CH;
    const bf16_t* const base = static_cast<const bf16_t*>(src.ptr) + b * src.sb + h * src.sh + static_cast<int64_t>(blk) * size * src.sl + c * 8;
    double sum[8] = {};
    constexpr int U = FLUX_KEY_BLOCK / RG;
    for (int r0 = rg; r0 < rows; r0 += U * RG) {
        Vec16<bf16_t> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = ld16(base + static_cast<int64_t>(min(r0 + u * RG, rows - 1)) * src.sl);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r0 + u * RG < rows)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += static_cast<double>(bf2f(v[u].v[e]));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) fold[rg][c * 8 + e] = sum[e];
    __syncthreads();
    if (threadIdx.x < D) {
        double t = 0.0;
        for (int i = 0; i < RG; ++i) t += fold[i][threadIdx.x];
        (is_q ? p.mq : p.mk)[at * D + threadIdx.x] = t / rows;
    }
}

typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));

// A double as a whole number of the same order; a NaN is below everything.
__device__ __forceinline__ uint64_t select_rank(double s) {
    if (s != s) return 0;
    const uint64_t u = __builtin_bit_cast(uint64_t, s + 0.0);   // (-0 becomes 0)
    return (u >> 63) ? ~u : u | (uint64_t{1} << 63);
}

// The numbers of the `keep` largest of key[0 .. n) in ascending order, the lower number among equals, by one wave. The keep-th largest is found bit by bit: the
// count of keys at or above a candidate says whether that bit is one of its own. Most rows are done once as many keys as are wanted are left.
template <typename Keys>
__device__ __forceinline__ void select_largest(const Keys key, int n, int keep, int lane, int32_t* out, int width) {
    uint64_t floor_ = 0;
    bool exact = n <= keep;   // whether the keys at or above floor_ are what is wanted
    for (int bit = 63; bit >= 0 && !exact; --bit) {
        const uint64_t candidate = floor_ | (uint64_t{1} << bit);
        int count = 0;
        for (int i = 0; i < n; i += 64) count += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i + lane < n && key[i + lane] >= candidate));
        if (count >= keep) floor_ = candidate;
        exact = count == keep;
    }
    int ties = 0x7fffffff;   // how many of the keys equal to floor_
    if (!exact) {
        ties = keep;
        for (int i = 0; i < n; i += 64) ties -= __builtin_popcountll(__builtin_amdgcn_ballot_w64(i + lane < n && key[i + lane] > floor_));
    }
    int written = 0;
    const uint64_t below = (uint64_t{1} << lane) - 1;
    for (int i = 0; i < n; i += 64) {
        const uint64_t k = i + lane < n ? key[i + lane] : 0;
        const uint64_t equal = __builtin_amdgcn_ballot_w64(i + lane < n && k == floor_);
        const bool mine = i + lane < n && (k > floor_ || (k == floor_ && __builtin_popcountll(equal & below) < ties));
        ties -= ties == 0x7fffffff ? 0 : min(ties, __builtin_popcountll(equal));
        const uint64_t chosen = __builtin_amdgcn_ballot_w64(mine);
        if (mine) out[written + __builtin_popcountll(chosen & below)] = i + lane;
        written += __builtin_popcountll(chosen);
    }
    for (int i = written + lane; i < width; i += 64) out[i] = -1;
}

// A workgroup of eight waves takes 16 query blocks of a (batch, head): their scores against all blocks of keys, 16 blocks a wave at a time, then the lists, two rows a
// wave. The scores stay in LDS as whole numbers, or beyond 1024 blocks in memory of the workgroup's own.
// The contraction is taken in an order of its own, so that a lane reads whole stretches of a mean: step s of lane group g is column g D/4 + s.
// MOST: blocks of keys that there is room for in LDS, 0: none.
template <int D, int MOST>
__global__ __launch_bounds__(512) void select_rows_kernel(SelectParams p) {
    __shared__ uint64_t lds[16 * MOST + 1];
    constexpr int S = D / 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
    const int per_head = (p.nq + 15) / 16, padded = (p.nk + 15) / 16 * 16;
    uint64_t* const keys = MOST == 0 ? reinterpret_cast<uint64_t*>(p.scores) + static_cast<int64_t>(blockIdx.x) * 16 * padded : lds;
    for (int64_t at = blockIdx.x; at < p.groups; at += gridDim.x) {
        const int64_t bh = at / per_head;
        const int i0 = static_cast<int>(at % per_head) * 16, b = static_cast<int>(bh / p.Hq), h = static_cast<int>(bh % p.Hq);
        const int have = (select_length(p, b) + FLUX_KEY_BLOCK - 1) / FLUX_KEY_BLOCK;
        const double* const mq = p.mq + (bh * p.nq + min(i0 + l16, p.nq - 1)) * D + g * S;
        const double* const mk = p.mk + (static_cast<int64_t>(b) * p.Hk + h / (p.Hq / p.Hk)) * p.nk * D + g * S;
        f64x2 a[S / 2];
#pragma unroll
        for (int s = 0; s < S / 2; ++s) a[s] = *reinterpret_cast<const f64x2*>(mq + 2 * s);
        for (int j0 = wave * 16; j0 < have; j0 += 128) {
            const double* const row = mk + static_cast<int64_t>(min(j0 + l16, have - 1)) * D;
            f64x4 t = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
            for (int s = 0; s < S / 2; ++s) {
                const f64x2 v = *reinterpret_cast<const f64x2*>(row + 2 * s);
                t = __builtin_amdgcn_mfma_f64_16x16x4f64(a[s].x, v.x, t, 0, 0, 0);
                t = __builtin_amdgcn_mfma_f64_16x16x4f64(a[s].y, v.y, t, 0, 0, 0);
            }
            const int j = j0 + l16;   // the lane's column; its rows are g, 4 + g, 8 + g and 12 + g
#pragma unroll
            for (int r = 0; r < 4; ++r) keys[(4 * r + g) * padded + j] = j < p.always ? ~uint64_t{0} : select_rank(t[r]);
        }
        __syncthreads();
        for (int r = wave; r < 16 && i0 + r < p.nq; r += 8)
            select_largest(keys + r * padded, have, p.keep, lane, p.blocks + (bh * p.nq + i0 + r) * p.width, p.width);
        __syncthreads();
    }
}

constexpr int kSelectNear = 1024, kSelectFarGroups = 512;

static int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

// Checks a call and turns it into the kernels' parameters; `nothing`: there are no lists. `need`: bytes of the workspace.
static int read_select_args(const flux_select_blocks_args* a, SelectParams& p, bool& nothing, int64_t& need) {
    const char* const what = "flux_select_blocks";
    need = 0;
    nothing = false;
    if (!a) return fail(FLUX_E_NULL, "%s: null args", what);
    if (a->B < 0 || a->Hq <= 0 || a->Hk <= 0 || a->Hq % a->Hk != 0 || a->Lq < 0 || a->Lk < 0 || a->keep < 0 || a->always < 0)
        return fail(FLUX_E_SHAPE, "%s: bad shape B=%lld Hq=%lld Hk=%lld Lq=%lld Lk=%lld, keep %lld, always %lld", what, (long long)a->B, (long long)a->Hq, (long long)a->Hk, (long long)a->Lq,
                    (long long)a->Lk, (long long)a->keep, (long long)a->always);
    if (a->D != 64 && a->D != 128) return fail(FLUX_E_UNSUPPORTED, "%s: head dim %d not supported (64, 128)", what, a->D);
    if (a->Lq > 0x7fffffff / 64 || a->Lk > 0x7fffffff / 64) return fail(FLUX_E_SHAPE, "%s: problem too large", what);
    const int64_t nq = (a->Lq + FLUX_QUERY_BLOCK - 1) / FLUX_QUERY_BLOCK, nk = (a->Lk + FLUX_KEY_BLOCK - 1) / FLUX_KEY_BLOCK, width = std::min(a->keep, nk);
    nothing = a->B == 0 || nq == 0 || width == 0;
    if (nothing) return FLUX_OK;
    if (nk > FLUX_SELECT_MOST_BLOCKS) return fail(FLUX_E_UNSUPPORTED, "%s: %lld blocks of keys, at most %d", what, (long long)nk, FLUX_SELECT_MOST_BLOCKS);
    if (a->B > 0x7fffffff / 64 || a->Hq > 0x7fffffff / 64 / a->B || a->B * a->Hq > 0x7fffffff / 512 / (nq + nk)) return fail(FLUX_E_SHAPE, "%s: problem too large", what);
    p = {a->q, a->k, a->lengths, a->blocks, nullptr, nullptr, nullptr, (int)a->B, (int)a->Hq, (int)a->Hk, (int)a->Lq, (int)a->Lk, (int)nq, (int)nk, (int)width, (int)width,
         (int)std::min(a->always, nk), a->B * a->Hq * ((nq + 15) / 16)};
    need = round256(a->B * a->Hq * nq * a->D * 8) + round256(a->B * a->Hk * nk * a->D * 8);
    if (nk > kSelectNear) need += std::min<int64_t>(p.groups, kSelectFarGroups) * 16 * ((nk + 15) / 16 * 16) * 8;
    return FLUX_OK;
}

template <int D>
static void select_launch(SelectParams p, char* ws, hipStream_t st) {
    p.mq = reinterpret_cast<double*>(ws);
    ws += round256(static_cast<int64_t>(p.B) * p.Hq * p.nq * D * 8);
    p.mk = reinterpret_cast<double*>(ws);
    ws += round256(static_cast<int64_t>(p.B) * p.Hk * p.nk * D * 8);
    p.scores = reinterpret_cast<double*>(ws);
    const int64_t blocks = static_cast<int64_t>(p.B) * (static_cast<int64_t>(p.Hq) * p.nq + static_cast<int64_t>(p.Hk) * p.nk);
    hipLaunchKernelGGL(block_means_kernel<D>, dim3((unsigned)blocks), dim3(256), 0, st, p);
    const dim3 groups((unsigned)p.groups), far_groups((unsigned)std::min<int64_t>(p.groups, kSelectFarGroups));
    if (p.nk <= 256) hipLaunchKernelGGL((select_rows_kernel<D, 256>), groups, dim3(512), 0, st, p);
    else if (p.nk <= 512) hipLaunchKernelGGL((select_rows_kernel<D, 512>), groups, dim3(512), 0, st, p);   // (two workgroups a CU)
    else if (p.nk <= kSelectNear) hipLaunchKernelGGL((select_rows_kernel<D, kSelectNear>), groups, dim3(512), 0, st, p);
    else hipLaunchKernelGGL((select_rows_kernel<D, 0>), far_groups, dim3(512), 0, st, p);
}

}  // namespace flux

using namespace flux;

extern "C" int64_t flux_select_blocks_workspace_bytes(const flux_select_blocks_args* a) {
    SelectParams p;
    bool nothing;
    int64_t need;
    return read_select_args(a, p, nothing, need) == FLUX_OK ? need : 0;
}

extern "C" int flux_select_blocks(const flux_select_blocks_args* a, void* ws, int64_t ws_bytes, void* stream) {
    const char* const what = "flux_select_blocks";
    SelectParams p;
    bool nothing;
    int64_t need;
    const int rc = read_select_args(a, p, nothing, need);
    if (rc != FLUX_OK || nothing) return rc;
    if (!a->blocks) return fail(FLUX_E_NULL, "%s: null lists", what);
    for (const flux_src4& s : {a->q, a->k})
        if (!s.ptr || !aligned16(s.ptr) || s.sb % 8 != 0 || s.sh % 8 != 0 || s.sl % 8 != 0)
            return fail(FLUX_E_ALIGN, "%s: q and k must be non-null, 16-byte aligned, with strides that are multiples of 8", what);
    if (!ws || reinterpret_cast<uintptr_t>(ws) % 256 != 0 || ws_bytes < need) return fail(FLUX_E_SHAPE, "%s: needs %lld bytes of 256-byte aligned workspace", what, (long long)need);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->D == 128) select_launch<128>(p, static_cast<char*>(ws), st);
    else select_launch<64>(p, static_cast<char*>(ws), st);
    return check_launch(what);
}
