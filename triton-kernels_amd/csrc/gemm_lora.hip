// Low-rank adapters beside a shared projection (gemm_lora.h): the first launch, and the second one on the four-wave tiles, on row vectors and for
// operands that no tile can address.
#include "gemm_lora.h"
#include "gemm_tiles.h"
#include <algorithm>

namespace flux {

// low[m] = s_i x[m] a_i^T for the rows of a tile of 16 that belong to one adapter: blockIdx.y says which of the tile's adapters, in rising order;
// there are fewer of them than that in most tiles, and a workgroup without one leaves at once. The waves take every n-th 64 of K and add up
// their sums through LDS. NF * 16 columns of the rank from blockIdx.z on. Bound by x coming from HBM once (M x K) and by a_i coming from the L2 once
// a tile.
constexpr int kLowThreads = 1024;
template <int NF>
__global__ __launch_bounds__(kLowThreads) void lora_low_kernel(LoraLow p) {
    __shared__ float part[kLowThreads / 64][NF * 256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int frow = lane & 15, fq = lane >> 4;
    const int m0 = blockIdx.x * 16, m = min(m0 + frow, p.M - 1);
    const int64_t request = m / p.rows_per_request;
    const int64_t id = p.wide_ids ? static_cast<const int64_t*>(p.adapter)[request] : static_cast<const int32_t*>(p.adapter)[request];
    const int own = id >= 0 && id < p.adapters ? static_cast<int>(id) : -1;
    if (blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x < 16 && m0 + frow < p.M) p.owner[m0 + frow] = own;
    constexpr int kNone = 0x7fffffff;
    int a = -1;
    for (unsigned i = 0; i <= blockIdx.y; ++i) {
        a = LoraTail::first_of_rows(own > a ? own : kNone);
        if (a == kNone) return;   // (alike in every wave)
    }
    const int r0 = blockIdx.z * (NF * 16);
    const bf16_t* const xr = p.x + m * p.lda;
    const bf16_t* const ar = p.a + static_cast<int64_t>(a) * p.rank * p.K;
    f32x4 acc[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto piece = [&](const bf16_t* row, int k, bool ok) -> bf16x8 {
        Vec16<bf16_t> v;
        if (p.vec) {   // (K is a multiple of 8)
            ok = ok && k < p.K;
            v = ld16(row + (ok ? k : 0));
            if (!ok) v = Vec16<bf16_t>{};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v.v[e] = ok && k + e < p.K ? row[k + e] : static_cast<bf16_t>(0);
        }
        return __builtin_bit_cast(bf16x8, v);
    };
    constexpr int STEPS = 4;   // of 32 of K whose operands are requested at once
    for (int k0 = wave * 64; k0 < p.K; k0 += waves * (STEPS * 32)) {
        bf16x8 xf[STEPS], af[STEPS][NF];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int k = k0 + (s / 2) * (waves * 64) + (s % 2) * 32 + fq * 8;
            xf[s] = piece(xr, k, true);
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const int r = r0 + f * 16 + frow;
                af[s][f] = piece(ar + static_cast<int64_t>(r < p.rank ? r : 0) * p.K, k, r < p.rank);
            }
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int f = 0; f < NF; ++f) acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[s][f], xf[s], acc[f], 0, 0, 0);
    }
#pragma unroll
    for (int f = 0; f < NF; ++f) *reinterpret_cast<f32x4*>(&part[wave][f * 256 + lane * 4]) = acc[f];
    __syncthreads();
    const float scale = p.scaling != nullptr ? p.scaling[a] : 1.0f;
    for (int t = threadIdx.x; t < NF * 256; t += blockDim.x) {   // lane l of fragment f holds row l % 16 and ranks 16 f + l / 16 * 4 ...
        const int row = (t >> 2) & 15, r = r0 + (t >> 8) * 16 + ((t & 255) >> 6) * 4 + (t & 3);
        float sum = 0.0f;
        for (int w = 0; w < waves; ++w) sum += part[w][t];
        const bool mine = __shfl(own, row) == a;
        if (mine && m0 + row < p.M && r < p.width) p.low[static_cast<int64_t>(m0 + row) * p.width + r] = r < p.rank ? f2bf(sum * scale) : static_cast<bf16_t>(0);
    }
}

void launch_lora_low(const LoraLow& p, hipStream_t st) {
    const int tiles = (p.M + 15) / 16;
    // adapters a tile can hold: requests that touch 16 rows
    const int64_t requests = p.rows_per_request % 16 == 0 ? 1 : std::min<int64_t>(16, 14 / p.rows_per_request + 2);
    const unsigned slots = static_cast<unsigned>(std::min<int64_t>(requests, p.adapters));
    const unsigned threads = tiles >= 512 ? 256 : tiles >= 128 ? 512 : kLowThreads;
    if (p.width <= 32) hipLaunchKernelGGL((lora_low_kernel<2>), dim3((unsigned)tiles, slots), dim3(threads), 0, st, p);
    else hipLaunchKernelGGL((lora_low_kernel<4>), dim3((unsigned)tiles, slots, (unsigned)((p.width + 63) / 64)), dim3(threads), 0, st, p);
}

// The four-wave tiles of gemm_bf16.hip with the adapter's product in front of their epilogue.
template <bool KTAIL>
__global__ __launch_bounds__(kGemmThreads) void lora_ring_kernel(GemmLaunch L, LoraTail tail) {
    constexpr int MI = 4, BM = 64 * MI, BK = 64, NU = 5, UNIT = BM * BK * 2;
    __shared__ __attribute__((aligned(1024))) char lds[NU * UNIT];
    int tm, tn;
    if (!tile_of_block(L, tm, tn)) return;
    const GemmParams& p = L.p[0];
    const int m0 = tm * BM, n0 = tn * BM;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    f32x4 acc[2 * MI][2 * MI];
    gemm_tile_slabs<MI, KTAIL>(p, lds, m0, n0, (p.K + BK - 1) / BK, acc);
    tail(acc, m0 + (wave >> 1) * (32 * MI), n0 + (wave & 1) * (32 * MI), p);
    gemm_epilogue<MI, MI>(p, acc, lds, m0, n0, wave, lane);
}

template <int FM, int FN, bool KTAIL>
__global__ __launch_bounds__(kGemmThreads) void lora_rect_kernel(GemmLaunch L, LoraTail tail) {
    constexpr int BM = 32 * FM, BN = 32 * FN, BK = 64;
    __shared__ __attribute__((aligned(1024))) char lds[(3 * BM + 2 * BN) * BK * 2];
    int tm, tn;
    if (!tile_of_block(L, tm, tn)) return;
    const GemmParams p = L.p[0];
    const int m0 = tm * BM, n0 = tn * BN;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    f32x4 acc[FM][FN];
    gemm_rect_slabs<FM, FN, KTAIL>(p, lds, m0, n0, (p.K + BK - 1) / BK, acc);
    tail(acc, m0 + (wave >> 1) * (16 * FM), n0 + (wave & 1) * (16 * FN), p);
    gemm_finish_rect<FM, FN, FM, false>(p, acc, lds, m0, n0, 0, wave, lane);
}

void launch_lora_square(const GemmSet& g, const LoraTail& tail, hipStream_t st) {
    const GemmLaunch L = make_launch(g, 256, 256);
    if (g.p[0].K % 64 == 0) hipLaunchKernelGGL((lora_ring_kernel<false>), dim3(grid_of(L)), dim3(kGemmThreads), 0, st, L, tail);
    else hipLaunchKernelGGL((lora_ring_kernel<true>), dim3(grid_of(L)), dim3(kGemmThreads), 0, st, L, tail);
}

template <int FM, int FN>
static void launch_rect(const GemmSet& g, const LoraTail& tail, hipStream_t st) {
    const GemmLaunch L = make_launch(g, 32 * FM, 32 * FN);
    if (g.p[0].K % 64 == 0) hipLaunchKernelGGL((lora_rect_kernel<FM, FN, false>), dim3(grid_of(L)), dim3(kGemmThreads), 0, st, L, tail);
    else hipLaunchKernelGGL((lora_rect_kernel<FM, FN, true>), dim3(grid_of(L)), dim3(kGemmThreads), 0, st, L, tail);
}

void launch_lora_rect(int fm, int fn, const GemmSet& g, const LoraTail& tail, hipStream_t st) {
    if (fm == 9) launch_rect<9, 6>(g, tail, st);
    else if (fm == 8 && fn == 7) launch_rect<8, 7>(g, tail, st);
    else if (fm == 8) launch_rect<8, 6>(g, tail, st);
    else if (fn == 9) launch_rect<7, 9>(g, tail, st);
    else if (fn == 6) launch_rect<7, 6>(g, tail, st);
    else launch_rect<7, 8>(g, tail, st);
}

// Row vectors: the loops over K of launch_gemv (gemm_bf16.hip) that fit any K; W keeps the non-temporal hint where it is large.
template <int MM, bool LDS, int U, bool ONCE>
__global__ __launch_bounds__(256) void lora_rows_kernel(GemmParams p, LoraTail t) {
    extern __shared__ __attribute__((aligned(16))) char act_lds[];
    LoraRowTail<MM> tail;
    tail.t = t;
    gemv_small_m<MM, LDS, U, false, ONCE>(p, static_cast<int>(blockIdx.x), act_lds, tail);
}

template <int MM>
static void launch_rows_of(const GemmParams& p, const LoraTail& tail, hipStream_t st) {
    const dim3 grid((unsigned)((p.N + 4 * kGemvCols - 1) / (4 * kGemvCols)));
    const size_t act_bytes = static_cast<size_t>(MM) * p.K * 2;
    const bool once = static_cast<int64_t>(p.N) * p.K * 2 <= (int64_t{128} << 20);
    constexpr int U = MM <= 2 ? 6 : 3;
#define CALL(LDS, ONCE, BYTES) hipLaunchKernelGGL((lora_rows_kernel<MM, LDS, U, ONCE>), grid, dim3(256), BYTES, st, p, tail)
    if (act_bytes <= kGemvSiluLds) {
        if (once) CALL(true, true, act_bytes);
        else CALL(true, false, act_bytes);
    } else {
        if (once) CALL(false, true, 0);
        else CALL(false, false, 0);
    }
#undef CALL
}

void launch_lora_rows(const GemmParams& p, const LoraTail& tail, hipStream_t st) {
    switch (p.M) {
        case 1: launch_rows_of<1>(p, tail, st); break;
        case 2: launch_rows_of<2>(p, tail, st); break;
        case 3: launch_rows_of<3>(p, tail, st); break;
        case 4: launch_rows_of<4>(p, tail, st); break;
        case 5: launch_rows_of<5>(p, tail, st); break;
        case 6: launch_rows_of<6>(p, tail, st); break;
        case 7: launch_rows_of<7>(p, tail, st); break;
        default: launch_rows_of<8>(p, tail, st); break;
    }
}

// Operands without 16-byte rows: a thread an output.
__global__ __launch_bounds__(256) void lora_scalar_kernel(GemmParams p, LoraTail t) {
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (idx >= static_cast<int64_t>(p.M) * p.N) return;
    const int m = static_cast<int>(idx / p.N), n = static_cast<int>(idx % p.N), own = t.owner[m];
    const bf16_t* a = p.A + static_cast<int64_t>(m) * p.lda;
    const bf16_t* w = p.W + static_cast<int64_t>(n) * p.ldw;
    float sum = 0.0f;
    for (int k = 0; k < p.K; ++k) sum += bf2f(a[k]) * bf2f(w[k]);
    if (own >= 0) {
        const bf16_t* b = t.b + (static_cast<int64_t>(own) * p.N + n) * t.rank;
        for (int r = 0; r < t.rank; ++r) sum += bf2f(t.low[static_cast<int64_t>(m) * t.width + r]) * bf2f(b[r]);
    }
    sum += p.bias ? bf2f(p.bias[n]) : 0.0f;
    if (p.act == FLUX_ACT_GELU_TANH) sum = gelu_tanh_f32(sum);
    p.Y[static_cast<int64_t>(m) * p.ldy + n] = f2bf(sum);
}

void launch_lora_scalar(const GemmParams& p, const LoraTail& tail, hipStream_t st) {
    hipLaunchKernelGGL(lora_scalar_kernel, dim3((unsigned)((static_cast<int64_t>(p.M) * p.N + 255) / 256)), dim3(256), 0, st, p, tail);
}

}  // namespace flux
