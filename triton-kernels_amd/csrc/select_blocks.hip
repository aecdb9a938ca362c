// Which blocks of 64 keys each block of 128 queries attends to: the means of the blocks, their products as scores, the largest of each row.
//
//   mq[i] = mean of block i's queries, mk[j] = mean of block j's keys, score[i, j] = mq[i] . mk[j]
//
// over the queries and keys in front of their sequences' ends.
//
// Everything behind the reads of q and k is formed in 64 bits: a row's scores lie close together, and which of two neighbours in their order is chosen must not
// go with the order of a sum. That is cheap: the sums of the means are an addition a value beside its two bytes, and the products 2 D operations for 64 x 128 x D of
// the attention itself, on the matrix cores (16x16x4). Bound by reading q and k once.
#include "common.h"
#include "../../include/flux_hip_serve.h"
#include <algorithm>
#include <math.h>

namespace flux {

struct SelectParams {
    flux_src4 q, k;
    const int32_t* lengths; const int32_t* q_lengths; int32_t* blocks;
    double* mq; double* mk; double* scores;
    int B, Hq, Hk, Lq, Lk, nq, nk, keep, width, always;   // width: entries of a list
    int64_t groups;                                      // of 16 query blocks of a (batch, head)
};

__device__ __forceinline__ int select_length(const int32_t* lengths, int b, int most) { return lengths ? min(max(lengths[b], 0), most) : most; }

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
    const int rows = min(size, select_length(is_q ? p.q_lengths : p.lengths, b, is_q ? p.Lq : p.Lk) - blk * size);
    if (rows <= 0) return;   // (a block that is not there)
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

// The numbers of the first `always` scores and of the largest of the others, `keep` in all, of score[0 .. n) in ascending order to `out`, -1 behind them, by one wave.
struct SelectRow {
    int32_t* out;
    int n, keep, always, width, lane;
    int written = 0;
    __device__ __forceinline__ void take(int i, bool mine) {   // of the 64 scores from i on
        const uint64_t chosen = __builtin_amdgcn_ballot_w64(mine);
        if (mine) out[written + __builtin_popcountll(chosen & ((uint64_t{1} << lane) - 1))] = i + lane;
        written += __builtin_popcountll(chosen);
    }
    __device__ __forceinline__ void rest() const {
        for (int i = written + lane; i < width; i += 64) out[i] = -1;
    }
};

// Among equals the lower number. The rest-th largest score is found bit by bit: the count of scores at or above a candidate says whether that bit is one of its own.
__device__ __forceinline__ void select_by_bits(SelectRow row, const double* score) {
    const int rest = row.keep - row.always, lane = row.lane;
    auto rank = [&](int i) { return i + lane >= row.always && i + lane < row.n ? select_rank(score[i + lane]) : 0; };
    auto there = [&](int i) { return i + lane >= row.always && i + lane < row.n; };
    uint64_t floor_ = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const uint64_t candidate = floor_ | (uint64_t{1} << bit);
        int count = 0;
        for (int i = 0; i < row.n; i += 64) count += __builtin_popcountll(__builtin_amdgcn_ballot_w64(there(i) && rank(i) >= candidate));
        if (count >= rest) floor_ = candidate;
    }
    int ties = rest;   // how many of those equal to floor_
    for (int i = 0; i < row.n; i += 64) ties -= __builtin_popcountll(__builtin_amdgcn_ballot_w64(there(i) && rank(i) > floor_));
    for (int i = 0; i < row.n; i += 64) {
        const uint64_t equal = __builtin_amdgcn_ballot_w64(there(i) && rank(i) == floor_);
        const bool tied = (equal >> lane & 1) && __builtin_popcountll(equal & ((uint64_t{1} << lane) - 1)) < ties;
        row.take(i, i + lane < row.always || (there(i) && rank(i) > floor_) || tied);
        ties -= min(ties, __builtin_popcountll(equal));
    }
    row.rest();
}

// The same for up to 64 V scores, which a lane holds rounded to fp32. Rounding keeps their order, so a bound that as many of them reach as are wanted parts the
// scores themselves, and halving the range finds one in a dozen steps (512 scores: 64 bits one by one took 5 us a row). Where two scores on either side of the border
// are one number in fp32, or something is not finite, there is no such bound.
template <int V>
__device__ __forceinline__ void select_by_bound(SelectRow row, const double* score) {
    const int rest = row.keep - row.always, lane = row.lane;
    float f[V];
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int i = v * 64 + lane;
        const bool there = i >= row.always && i < row.n;
        f[v] = there ? static_cast<float>(score[there ? i : 0]) : -INFINITY;
        if (there) {
            lo = fminf(lo, f[v]);
            hi = fmaxf(hi, f[v]);
        }
    }
    auto across = [&](auto permuted) {
        lo = fminf(lo, permuted(lo));
        hi = fmaxf(hi, permuted(hi));
    };
    across([](float v) { return dpp_f32<0xB1>(v); });
    across([](float v) { return dpp_f32<0x4E>(v); });
    across([](float v) { return dpp_f32<0x141>(v); });
    across([](float v) { return dpp_f32<0x140>(v); });
    across([](float v) { return __shfl_xor(v, 16, 64); });
    across([](float v) { return __shfl_xor(v, 32, 64); });
    bool found = false;
    float bound = lo;
    for (int step = 0; step < 40 && !found; ++step) {
        bound = lo + (hi - lo) * 0.5f;
        if (!(bound > lo)) break;   // (nothing between them, or no number)
        int count = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) count += __builtin_popcountll(__builtin_amdgcn_ballot_w64(f[v] >= bound));
        found = count == rest;
        if (count > rest) lo = bound;
        else hi = bound;
    }
    if (!found) {
        select_by_bits(row, score);
        return;
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (v * 64 < row.n) row.take(v * 64, v * 64 + lane < row.always || f[v] >= bound);
    row.rest();
}

// A workgroup takes 16 query blocks of a (batch, head): their scores against all blocks of keys, 16 blocks a wave at a time, then the lists, one or two rows a
// wave. The scores stay in LDS, or beyond 1024 blocks in memory of the workgroup's own.
// The contraction is taken in an order of its own, so that the four lanes of a mean read 64 bytes of it that lie together: steps 2 s and 2 s + 1 of lane group g are columns
// 8 s + 2 g and the next (with a stretch of a mean for each lane a load was 64 pieces of 16 bytes: 512 x 256 blocks of 24 heads 71 us).
// MOST: blocks of keys that there is room for in LDS, 0: none.
template <int D, int MOST, int WAVES>
__global__ __launch_bounds__(64 * WAVES, MOST > 512 ? 2 : 4) void select_rows_kernel(SelectParams p) {
    __shared__ double lds[16 * MOST + 1];
    constexpr int S = D / 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
    const int per_head = (p.nq + 15) / 16, padded = (p.nk + 15) / 16 * 16;
    double* const scores = MOST == 0 ? p.scores + static_cast<int64_t>(blockIdx.x) * 16 * padded : lds;
    // (the groups of a head of keys share an XCD, whose L2 keeps its means)
    const int64_t per_xcd = gridDim.x / 8;
    for (int64_t at = blockIdx.x % 8 * per_xcd + blockIdx.x / 8; at < p.groups; at += gridDim.x) {
        const int64_t bh = at / per_head;
        const int i0 = static_cast<int>(at % per_head) * 16, b = static_cast<int>(bh / p.Hq), h = static_cast<int>(bh % p.Hq);
        const int have = (select_length(p.lengths, b, p.Lk) + FLUX_KEY_BLOCK - 1) / FLUX_KEY_BLOCK, queries = select_length(p.q_lengths, b, p.Lq);
        const double* const mq = p.mq + (bh * p.nq + min(i0 + l16, p.nq - 1)) * D + g * 2;
        const double* const mk = p.mk + (static_cast<int64_t>(b) * p.Hk + h / (p.Hq / p.Hk)) * p.nk * D + g * 2;
        const int always = min(p.always, min(p.keep, have));
        const bool all = have <= p.keep || always == p.keep;   // the first ones, whatever their scores are
        if (!all) {
            f64x2 a[S / 2];
#pragma unroll
            for (int s = 0; s < S / 2; ++s) a[s] = *reinterpret_cast<const f64x2*>(mq + 8 * s);
            for (int j0 = wave * 16; j0 < have; j0 += 16 * WAVES) {
                const double* const row = mk + static_cast<int64_t>(min(j0 + l16, have - 1)) * D;
                f64x4 t = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
                for (int s = 0; s < S / 2; ++s) {
                    const f64x2 v = *reinterpret_cast<const f64x2*>(row + 8 * s);
                    t = __builtin_amdgcn_mfma_f64_16x16x4f64(a[s].x, v.x, t, 0, 0, 0);
                    t = __builtin_amdgcn_mfma_f64_16x16x4f64(a[s].y, v.y, t, 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) scores[(4 * r + g) * padded + j0 + l16] = t[r];   // (the lane's rows are g, 4 + g, 8 + g and 12 + g)
            }
        }
        __syncthreads();
        for (int r = wave; r < 16 && i0 + r < p.nq; r += WAVES) {
            SelectRow row = {p.blocks + (bh * p.nq + i0 + r) * p.width, have, p.keep, always, p.width, lane};
            if ((i0 + r) * FLUX_QUERY_BLOCK >= queries) {   // (its mean was not written: a row of the product that goes nowhere)
                row.rest();
            } else if (all) {
                for (int i = 0; i < min(have, p.keep); i += 64) row.take(i, i + lane < min(have, p.keep));
                row.rest();
            } else if constexpr (MOST == 0) {
                select_by_bits(row, scores + r * padded);
            } else {
                select_by_bound<MOST / 64>(row, scores + r * padded);
            }
        }
        __syncthreads();
    }
}

constexpr int kSelectNear = 1024, kSelectFarGroups = 512;

static int64_t mean_bytes(int64_t blocks, int D) { return (blocks * D * 8 + 255) / 256 * 256; }

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
    p = {a->q, a->k, a->lengths, a->q_lengths, a->blocks, nullptr, nullptr, nullptr, (int)a->B, (int)a->Hq, (int)a->Hk, (int)a->Lq, (int)a->Lk, (int)nq, (int)nk, (int)width, (int)width,
         (int)std::min(a->always, nk), a->B * a->Hq * ((nq + 15) / 16)};
    need = mean_bytes(a->B * a->Hq * nq, a->D) + mean_bytes(a->B * a->Hk * nk, a->D);
    if (nk > kSelectNear) need += std::min<int64_t>((p.groups + 7) / 8 * 8, kSelectFarGroups) * 16 * ((nk + 15) / 16 * 16) * 8;
    return FLUX_OK;
}

template <int D>
static void select_launch(SelectParams p, char* ws, hipStream_t st) {
    p.mq = reinterpret_cast<double*>(ws);
    ws += mean_bytes(static_cast<int64_t>(p.B) * p.Hq * p.nq, D);
    p.mk = reinterpret_cast<double*>(ws);
    ws += mean_bytes(static_cast<int64_t>(p.B) * p.Hk * p.nk, D);
    p.scores = reinterpret_cast<double*>(ws);
    const int64_t blocks = static_cast<int64_t>(p.B) * (static_cast<int64_t>(p.Hq) * p.nq + static_cast<int64_t>(p.Hk) * p.nk);
    hipLaunchKernelGGL(block_means_kernel<D>, dim3((unsigned)blocks), dim3(256), 0, st, p);
    const dim3 groups((unsigned)((p.groups + 7) / 8 * 8)), far_groups((unsigned)std::min<int64_t>((p.groups + 7) / 8 * 8, kSelectFarGroups));
    // (sixteen waves, a row each, where there are few workgroups: 72 x 36 blocks of 24 heads 10.7 -> 9.9 us; eight where two workgroups fit a CU)
#define CALL(MOST, WAVES, GROUPS) hipLaunchKernelGGL((select_rows_kernel<D, MOST, WAVES>), GROUPS, dim3(64 * WAVES), 0, st, p)
    if (p.nk <= 128) CALL(128, 16, groups);
    else if (p.nk <= 256) CALL(256, 16, groups);
    else if (p.nk <= 512) CALL(512, 8, groups);
    else if (p.nk <= kSelectNear) CALL(kSelectNear, 8, groups);
    else CALL(0, 8, far_groups);
#undef CALL
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
