// The eight-wave tiles (gemm_pair.hip says what they are made for), for the launches that multiply and for those that add an adapter's product to
// the same tile (gemm_lora_pair.hip).
#pragma once

#include "gemm_common.h"

namespace flux {

constexpr int kPairThreads = 512;

// ahead(): loads of the caller's own, requested behind those of the first slabs; they have landed on return.
template <int FM, int FN, int ST, bool KTAIL, int G, typename Ahead>
__device__ __forceinline__ void gemm_pair_slabs(const GemmParams& p, char* lds, int m0, int n0, int kb, int ke, int turn, int turns, int w4, int lane, f32x4 (&acc)[FM][FN], Ahead ahead) {
    constexpr int BM = 32 * FM, BN = 32 * FN, BK = 64, ROWB = BK * 2;
    constexpr int SLAB = (BM + BN) * ROWB;       // A rows, then W rows
    constexpr int NL = (FM + FN + 1 - G) / 2;    // loads of this wave per slab: passes of 32 rows, every other one
    constexpr int WROWS = 16 * FM, WCOLS = 16 * FN;
    constexpr int READS = FM + FN, MFMAS = FM * FN;
    constexpr int BS = READS / 4;                // slots in front of the barrier
    static_assert(2 * (READS - BS) >= READS && READS - BS >= NL && MFMAS >= READS, "schedule shape");
    static_assert(ST >= 3 && (ST - 1) * NL <= 63 && ST * SLAB <= 160 * 1024, "ring shape");
    const int wm = w4 >> 1, wn = w4 & 1;

    const int lrow = w4 * 8 + (lane >> 3);
    const int lchunk = (lane & 7) ^ ((lrow >> 1) & 7);
    const int rows_a = min(p.M - m0, BM), rows_b = min(p.N - n0, BN);
    const int64_t a0 = row_of_a(p, m0);
    bf16_t* const base_a = const_cast<bf16_t*>(p.A + a0);
    bf16_t* const base_b = const_cast<bf16_t*>(p.W + static_cast<int64_t>(n0) * p.ldw);
    const int bytes_a = static_cast<int>((row_of_a(p, m0 + rows_a - 1) - a0 + p.K) * 2);
    const int bytes_b = static_cast<int>(((rows_b - 1) * p.ldw + p.K) * 2);
    uint32_t voff[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) {
        const int pass = 2 * j + G;
        if (pass < FM) {
            const int r = pass * 32 + lrow;
            voff[j] = r < rows_a ? static_cast<uint32_t>((row_of_a(p, m0 + r) - a0 + lchunk * 8) * 2) : kOutOfRange;
        } else {
            const int r = (pass - FM) * 32 + lrow;
            voff[j] = r < rows_b ? static_cast<uint32_t>((r * p.ldw + lchunk * 8) * 2) : kOutOfRange;
        }
    }
    // slabs from ke on read as zeros, which keeps the number of loads in flight the same to the last slab
    auto load = [&](int soff, int j, int kt) {
        const int pass = 2 * j + G;
        const bool in = kt < ke;
        const uint32_t v = KTAIL && kt * BK + lchunk * 8 >= p.K ? kOutOfRange : voff[j];
        if (pass < FM) load_chunk(__builtin_amdgcn_make_buffer_rsrc(base_a, 0, in ? bytes_a : 0, kRsrcFlags), lds + soff + pass * 4096 + w4 * 1024, v, kt * ROWB);
        else load_chunk(__builtin_amdgcn_make_buffer_rsrc(base_b, 0, in ? bytes_b : 0, kRsrcFlags), lds + soff + pass * 4096 + w4 * 1024, v, kt * ROWB);
    };

    const int frow = lane & 15, fq = lane >> 4;
    const int ko = ((G * 4 + fq) ^ ((frow >> 1) & 7)) * 16;
    const int koff_a = (wm * WROWS + frow) * ROWB + ko;
    const int koff_w = BM * ROWB + (wn * WCOLS + frow) * ROWB + ko;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = 0.0f;

    bf16x8 xa[2][FM], wb[2][FN];
    auto read_frag = [&](int buf, int soff, int r) {
        if (r == 0) xa[buf][0] = *reinterpret_cast<const bf16x8*>(lds + (soff + koff_a));
        else if (r <= FN) wb[buf][r - 1] = *reinterpret_cast<const bf16x8*>(lds + (soff + koff_w) + (r - 1) * 16 * ROWB);
        else xa[buf][r - FN] = *reinterpret_cast<const bf16x8*>(lds + (soff + koff_a) + (r - FN) * 16 * ROWB);
    };
    auto mfma_one = [&](int buf, int idx) {
        const int i = idx / FN, j = (i & 1) ? FN - 1 - idx % FN : idx % FN;
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[buf][j], xa[buf][i], acc[i][j], 0, 0, 0);
    };
    // slab number i in the order of this tile; those of a last, shorter group in turn
    const bool rotated = turns > 1;
    auto slab_at = [&](int i) { return ((i - kb) | (turns - 1)) < ke - kb ? kb + ((i - kb) ^ turn) : i; };
    // k: the slab that is requested; cur: stage of the one that is multiplied (its fragments are in buffer `buf`), nxt: of the one behind it
    auto slab = [&](auto bufc, int k, int cur, int nxt) {
        constexpr int buf = decltype(bufc)::value;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < READS; ++r) {
            const int lo = r * MFMAS / READS, hi = (r + 1) * MFMAS / READS;
            if (r == BS) {
                wait_loads_and_barrier<(ST - 2) * NL>();   // slab kt + 1 has landed; every wave holds its fragments of slab kt
                __builtin_amdgcn_sched_barrier(0);
            }
            if (r >= BS) {
                const int f0 = 2 * (r - BS);
                for (int f = f0; f < f0 + 2 && f < READS; ++f) read_frag(buf ^ 1, nxt, f);
            }
            mfma_one(buf, lo);
            __builtin_amdgcn_sched_barrier(0);
            if (r >= BS && r - BS < NL) load(cur, r - BS, k);
#pragma unroll
            for (int m = lo + 1; m < hi; ++m) mfma_one(buf, m);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

#pragma unroll
    for (int s = 0; s < ST; ++s) {
        const int k = rotated ? slab_at(kb + s) : kb + s;
#pragma unroll
        for (int j = 0; j < NL; ++j) load(s * SLAB, j, k);
    }
    ahead();
    wait_loads_and_barrier<(ST - 1) * NL>();
#pragma unroll
    for (int r = 0; r < READS; ++r) read_frag(0, 0, r);
    __builtin_amdgcn_sched_barrier(0);
    int cur = 0;
    auto after = [](int s) { return s + SLAB == ST * SLAB ? 0 : s + SLAB; };
    for (int kt = kb; kt < ke; kt += 2) {
        const int n1 = after(cur), n2 = after(n1);
        int k0 = kt + ST, k1 = kt + ST + 1;
        if (rotated) {
            k0 = slab_at(k0);
            k1 = slab_at(k1);
        }
        slab(ic<0>(), k0, cur, n1);
        if (kt + 1 < ke) slab(ic<1>(), k1, n1, n2);
        cur = n2;
    }
    wait_vmem_all();
}

// A workgroup's tile, or its part of one. `tail` adds to the sums of a wave's fragment rows before their epilogue (finish) and may ask for what that
// takes in front of the first slabs (begin) and behind them (touch). lane(): the lane's number behind finish. NoTail: nothing.
struct NoTail {
    static __device__ __forceinline__ int lane(int known) { return known; }
    template <int ROWS, int FN> struct Ahead {};
    template <int ROWS, int FN> __device__ __forceinline__ void begin(Ahead<ROWS, FN>&, int, const GemmParams&) const {}
    template <int ROWS, int FN> __device__ __forceinline__ void touch(Ahead<ROWS, FN>&, int, int, const GemmParams&) const {}
    template <int ROWS, int FN> __device__ __forceinline__ void finish(f32x4 (&)[ROWS][FN], Ahead<ROWS, FN>&, int, int, const GemmParams&) const {}
};
template <int FM, int FN, int ST, bool KTAIL, bool SPLIT, typename Tail>
__global__ __launch_bounds__(kPairThreads) void gemm_nt_pair_kernel(GemmLaunch L, Tail tail) {
    constexpr int BM = 32 * FM, BN = 32 * FN, BK = 64;
    constexpr int R0 = (FM + 1) / 2, R1 = FM - R0;   // fragment rows that group 0 / group 1 finishes
    __shared__ __attribute__((aligned(1024))) char lds[ST * (BM + BN) * BK * 2];
    static_assert(4 * FM * FN * 1024 <= ST * (BM + BN) * BK * 2 && 2 * rect_epilogue_lds(FN) <= ST * (BM + BN) * BK * 2, "exchange and epilogue must fit the ring");
    int t = 0, split = 0, tm, tn;
    if constexpr (SPLIT) {   // the parts of a tile are `tiles` places apart in the sequence
        t = (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
        if (t >= L.tiles_m * L.tiles_n * L.splits) return;
        split = t / (L.tiles_m * L.tiles_n);
        t -= split * (L.tiles_m * L.tiles_n);
        tile_at(L, t, tm, tn);
    } else {
        if (FN == 8 && L.p[0].qk_cols > 0 ? !tile_of_block_qk(L, BN, tm, tn) : !tile_of_block(L, tm, tn)) return;
    }
    int turn = 0, turns = 1;
    if (L.take_turns) {
        const int tiles = min(L.tiles_m - tm / L.group_m * L.group_m, L.group_m);
        turns = tiles > 2 ? 4 : tiles;
        turn = (tm % L.group_m + tn) & (turns - 1);
    }
    const GemmParams p = L.p[product_of_tile(L, tm)];
    const int m0 = tm * BM, n0 = tn * BN;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w4 = wave & 3;
    const int kb = split * L.slabs_per_split, ke = min((p.K + BK - 1) / BK, kb + L.slabs_per_split);
    f32x4* const ex = reinterpret_cast<f32x4*>(lds) + w4 * (FM * FN * 64) + lane;   // exchange: 64 lanes x 16 bytes per fragment
    const int wm0 = m0 + (w4 >> 1) * (16 * FM), wn0 = n0 + (w4 & 1) * (16 * FN);
    auto finish = [&](auto gc, f32x4 (&acc)[FM][FN], auto& have) {
        constexpr int G = decltype(gc)::value, OWN0 = G == 0 ? 0 : R0, OWN = G == 0 ? R0 : R1, GIVE0 = G == 0 ? R0 : 0, GIVE = FM - OWN;
        __syncthreads();                       // everyone is done with the ring
#pragma unroll
        for (int i = 0; i < GIVE; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) ex[((GIVE0 + i) * FN + j) * 64] = acc[GIVE0 + i][j];
        __syncthreads();
        f32x4 own[OWN][FN];
#pragma unroll
        for (int i = 0; i < OWN; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) own[i][j] = acc[OWN0 + i][j] + ex[((OWN0 + i) * FN + j) * 64];
        if constexpr (SPLIT) {
            f32x4* dst = reinterpret_cast<f32x4*>(L.partial) + ((static_cast<int64_t>(split) * (L.tiles_m * L.tiles_n) + t) * 4 + w4) * (FM * FN * 64) + lane;
#pragma unroll
            for (int i = 0; i < OWN; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) dst[((OWN0 + i) * FN + j) * 64] = own[i][j];
        } else {
            tail.finish(own, have, wm0 + OWN0 * 16, wn0, p);
            __syncthreads();                   // the exchange has been read: its LDS is the epilogue's now
            gemm_finish_rect<FM, FN, OWN, FN != 8>(p, own, lds + G * (ST * (BM + BN) * BK), m0, n0, OWN0, w4, tail.lane(lane));
        }
    };
    f32x4 acc[FM][FN];
    if (wave < 4) {
        typename Tail::template Ahead<R0, FN> have;
        if (!SPLIT) tail.begin(have, wm0, p);
        gemm_pair_slabs<FM, FN, ST, KTAIL, 0>(p, lds, m0, n0, kb, ke, turn, turns, w4, lane, acc, [&]() { if (!SPLIT) tail.touch(have, wm0, wn0, p); });
        finish(ic<0>(), acc, have);
    } else {
        typename Tail::template Ahead<R1, FN> have;
        if (!SPLIT) tail.begin(have, wm0 + R0 * 16, p);
        gemm_pair_slabs<FM, FN, ST, KTAIL, 1>(p, lds, m0, n0, kb, ke, turn, turns, w4, lane, acc, [&]() { if (!SPLIT) tail.touch(have, wm0 + R0 * 16, wn0, p); });
        finish(ic<1>(), acc, have);
    }
}

// Second half of a split-K launch: a workgroup per (tile, fragment row) adds the parts in order and runs
// the epilogue on that fragment row of its four waves' sub-tiles.
template <int FM, int FN, typename Tail>
__global__ __launch_bounds__(kGemmThreads) void gemm_reduce_kernel(GemmLaunch L, Tail tail) {
    constexpr int BM = 32 * FM, BN = 32 * FN;
    __shared__ __attribute__((aligned(16))) char lds[rect_epilogue_lds(FN)];
    const int tiles = L.tiles_m * L.tiles_n;
    const int t = blockIdx.x / FM, row = blockIdx.x - t * FM;
    int tm, tn;
    tile_at(L, t, tm, tn);
    const GemmParams p = L.p[product_of_tile(L, tm)];
    const int m0 = tm * BM, n0 = tn * BN;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm0 = m0 + (wave >> 1) * (16 * FM) + row * 16, wn0 = n0 + (wave & 1) * (16 * FN);
    typename Tail::template Ahead<1, FN> have;
    tail.begin(have, wm0, p);
    const f32x4* src = reinterpret_cast<const f32x4*>(L.partial) + (static_cast<int64_t>(t) * 4 + wave) * (FM * FN * 64) + row * (FN * 64) + lane;
    const int64_t part = static_cast<int64_t>(tiles) * 4 * (FM * FN * 64);
    f32x4 acc[1][FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[0][j] = src[j * 64];
    tail.touch(have, wm0, wn0, p);
    for (int s = 1; s < L.splits; ++s) {
        src += part;
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[0][j] += src[j * 64];
    }
    tail.finish(acc, have, wm0, wn0, p);
    gemm_finish_rect<FM, FN, 1, FN != 8>(p, acc, lds, m0, n0, row, wave, lane);
}

}  // namespace flux
