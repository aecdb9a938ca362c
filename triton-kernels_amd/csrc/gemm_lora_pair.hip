// Low-rank adapters beside a shared projection (gemm_lora.h) on the eight-wave tiles. With K in parts the adapter's product is added where the
// parts are.
#include "gemm_eight_waves.h"
#include "gemm_lora.h"

namespace flux {

template <int FM, int FN, int ST>
static void launch_pair(const GemmSet& g, int splits, float* partial, const LoraTail& tail, hipStream_t st) {
    const GemmLaunch L = splits > 1 ? launch_pair_parts(FM, FN, g, splits, partial, st) : make_pair_launch(g, FM, FN);
    if (L.splits > 1) {
        hipLaunchKernelGGL((gemm_reduce_kernel<FM, FN, LoraTail>), dim3((unsigned)(L.tiles_m * L.tiles_n * FM)), dim3(kGemmThreads), 0, st, L, tail);
        return;
    }
    if (g.p[0].K % 64 == 0) hipLaunchKernelGGL((gemm_nt_pair_kernel<FM, FN, ST, false, false, LoraTail>), dim3(grid_of(L)), dim3(kPairThreads), 0, st, L, tail);
    else hipLaunchKernelGGL((gemm_nt_pair_kernel<FM, FN, ST, true, false, LoraTail>), dim3(grid_of(L)), dim3(kPairThreads), 0, st, L, tail);
}

void launch_lora_pair(int fm, int fn, const GemmSet& g, int splits, float* partial, const LoraTail& tail, hipStream_t st) {
#define FLUX_PAIR(FM, FN, ST) if (fm == FM && fn == FN) return launch_pair<FM, FN, ST>(g, splits, partial, tail, st)
    FLUX_PAIR(5, 6, 3); FLUX_PAIR(6, 6, 3); FLUX_PAIR(4, 6, 3); FLUX_PAIR(8, 4, 3); FLUX_PAIR(7, 4, 3); FLUX_PAIR(6, 4, 4);
    FLUX_PAIR(5, 4, 4); FLUX_PAIR(5, 3, 4); FLUX_PAIR(4, 3, 4); FLUX_PAIR(3, 3, 4); FLUX_PAIR(2, 3, 4);
    FLUX_PAIR(2, 2, 6);
#undef FLUX_PAIR
}

}  // namespace flux
