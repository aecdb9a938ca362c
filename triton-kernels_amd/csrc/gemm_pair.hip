// Linear layer on the matrix cores, middle sizes: a few hundred to a few thousand rows.
#include "gemm_eight_waves.h"

#include <climits>

namespace flux {

// ------------------------------------------------------------------------------------------------
// Middle sizes: eight waves on a (32*FM) x (32*FN) tile, two per SIMD, as two groups of four. Both groups
// hold accumulators of the whole tile; of every K = 64 slab group 0 multiplies the first K = 32 step and
// group 1 the second, and the two sums are added through LDS at the end. A single wave per SIMD issues in
// order, and on tiles that are small enough for a few hundred rows its fragment reads (18 cycles each) and
// LDS-writing loads (34 to 64) take longer than its MFMAs; two waves that share the slab, and with it the
// LDS traffic, fill each other's gaps. ST slabs of LDS, round-robin: fragments of slab kt + 1 are read
// while slab kt is multiplied, so behind the barrier of slab kt its buffer takes slab kt + ST, and
// ST - 1 slabs are in flight or waiting.
// What bounds it: the bytes a CU can have in flight. With everything but the loads taken out 320 x 21504 x
// 3072 (160 x 192 tiles) takes 50 us with W coming from HBM and 32 us from the Infinity Cache, 50 and 38 us
// as it is, 30 us with neither loads nor fragment reads; a CU's loads stop at about 55 bytes per ns from HBM and
// 104 from the caches however many slabs are in flight. So the tile shape is chosen for few bytes per
// product. Measured (weights from HBM, before -> now): 320 x 3072 x 15360 75 -> 45 us, 768 x 3072 x 12288
// 138 -> 62 us, 1280 x 3072 x 12288 141 -> 93 us, 512 x 3072 x 3072 28 -> 21 us; a four-wave workgroup on the
// same tiles: 50, 78, 120 and 21 us.
// ------------------------------------------------------------------------------------------------
// Slabs out of turn. Tiles that share columns of W run side by side and ask for the same slab at the same time, so each of them waits for it to
// come from HBM. Where W is too large to be found in the Infinity Cache, the tiles of a column take every two or four slabs of K (`turns`, as many as there
// are tiles, or one more than three) in an order of their own, slab i ^ turn: each is the first at some of a group and finds the others in the L2, where its
// neighbours have brought them. The same goes for A among the tiles of a row. us, W from HBM, in turn -> so: 320 x 21504 x 3072 50.4 -> 47.3, 320 x 3072 x
// 15360 45.2 -> 44.5, 640 65.7 -> 63.9, 1024 101.7 -> 92.3, 1600 154.9 -> 135.4, 1900 169.3 -> 154.4, 2048 177.4 -> 158.5. A W of more than a third of
// that cache that is found there all the same costs 40.0 -> 40.4, 39.9 -> 40.5, 60.0 -> 61.6, 86.9 -> 89.4, 126.8 -> 127.9, 145.1 -> 148.4 and 150.2 -> 153.7 us; a smaller one is walked in turn.
// The order has to be cheap: rotated by additions, a branch at the end of a group and a division at the head of the kernel, all tiles in turn took 3 % longer at 1600 and 1900
// rows (130.6 and 148.9 us from the cache; 139.5 and 159.2 rotated, from HBM), and inside a slab instead of between two the order took 1 % of 512 x 3072 x 3072.
// Two products in a launch gain nothing (1024 + 256 x 3072 x 12288 99.6 and 100.2): the second's one row of tiles has nobody to share with and ends
// last. Groups of two and four times as many slabs: 48.0 and 49.2 us at the first size, 46.8 so. From four tile rows on the last one has to be three quarters full: one of
// mostly padding runs ahead of its neighbours and is then the first at every slab (K = 15360, hardly filled: 1152 rows 102.8 -> 106.1, 1402 118.4 -> 121.1, 1750
// 149.0 -> 154.2, 2100 170.8 -> 175.6, in turn now).
GemmLaunch make_pair_launch(const GemmSet& g, int fm, int fn) {
    GemmLaunch L = make_launch(g, 32 * fm, 32 * fn);
    L.take_turns = g.n == 1 && weights_from_hbm(g) && (L.tiles_m < 4 || 4 * (g.p[0].M - (L.tiles_m - 1) * 32 * fm) >= 3 * 32 * fm);
    return L;
}

// K in parts (whole slabs only): the parts' sums, which gemm_reduce_kernel adds up; nothing where there would be one part.
template <int FM, int FN, int ST>
static GemmLaunch launch_parts(const GemmSet& g, int splits, float* partial, hipStream_t st) {
    const int K = g.p[0].K;
    GemmLaunch L = make_pair_launch(g, FM, FN);
    L.slabs_per_split = (K / 64 + splits - 1) / splits;
    L.splits = (K / 64 + L.slabs_per_split - 1) / L.slabs_per_split;
    L.partial = partial;
    if (L.splits > 1) hipLaunchKernelGGL((gemm_nt_pair_kernel<FM, FN, ST, false, true, NoTail>), dim3(grid_of(L)), dim3(kPairThreads), 0, st, L, NoTail());
    return L;
}

template <int FM, int FN, int ST>
static void launch_pair(const GemmSet& g, int splits, float* partial, hipStream_t st) {
    const GemmLaunch L = splits > 1 ? launch_parts<FM, FN, ST>(g, splits, partial, st) : make_pair_launch(g, FM, FN);
    if (L.splits > 1) {
        hipLaunchKernelGGL((gemm_reduce_kernel<FM, FN, NoTail>), dim3((unsigned)(L.tiles_m * L.tiles_n * FM)), dim3(kGemmThreads), 0, st, L, NoTail());
    } else if (g.p[0].K % 64 == 0) {
        hipLaunchKernelGGL((gemm_nt_pair_kernel<FM, FN, ST, false, false, NoTail>), dim3(grid_of(L)), dim3(kPairThreads), 0, st, L, NoTail());
    } else {
        hipLaunchKernelGGL((gemm_nt_pair_kernel<FM, FN, ST, true, false, NoTail>), dim3(grid_of(L)), dim3(kPairThreads), 0, st, L, NoTail());
    }
}

void launch_pair_tiles(int fm, int fn, const GemmSet& g, int splits, float* partial, hipStream_t st) {
#define FLUX_PAIR(FM, FN, ST) if (fm == FM && fn == FN) return launch_pair<FM, FN, ST>(g, splits, partial, st)
    FLUX_PAIR(5, 6, 3); FLUX_PAIR(6, 6, 3); FLUX_PAIR(4, 6, 3); FLUX_PAIR(8, 4, 3); FLUX_PAIR(7, 4, 3); FLUX_PAIR(6, 4, 4);
    FLUX_PAIR(5, 4, 4); FLUX_PAIR(5, 3, 4); FLUX_PAIR(4, 3, 4); FLUX_PAIR(3, 3, 4); FLUX_PAIR(2, 3, 4);
    FLUX_PAIR(2, 2, 6); FLUX_PAIR(4, 8, 3);
#undef FLUX_PAIR
}

GemmLaunch launch_pair_parts(int fm, int fn, const GemmSet& g, int splits, float* partial, hipStream_t st) {
#define FLUX_PAIR(FM, FN, ST) if (fm == FM && fn == FN) return launch_parts<FM, FN, ST>(g, splits, partial, st)
    FLUX_PAIR(5, 6, 3); FLUX_PAIR(6, 6, 3); FLUX_PAIR(4, 6, 3); FLUX_PAIR(8, 4, 3); FLUX_PAIR(7, 4, 3); FLUX_PAIR(6, 4, 4);
    FLUX_PAIR(5, 4, 4); FLUX_PAIR(5, 3, 4); FLUX_PAIR(4, 3, 4); FLUX_PAIR(3, 3, 4); FLUX_PAIR(2, 3, 4);
    FLUX_PAIR(2, 2, 6);
#undef FLUX_PAIR
    return GemmLaunch();
}

}  // namespace flux
