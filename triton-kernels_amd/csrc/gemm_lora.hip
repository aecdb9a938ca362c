// Low-rank adapters beside a shared projection (gemm_lora.h): the first launch, and the second one on the four-wave tiles, on row vectors and for
// operands that no tile can address.
#include "gemm_lora.h"
#include "gemm_tiles.h"
#include <algorithm>

namespace flux {

// low[m] = s_i x[m] a_i^T for the rows of a tile of 16 that belong to one adapter: blockIdx.y says which of the tile's adapters, in rising order;
// there are fewer of them than that in most tiles, and a workgroup without one leaves at once. NF * 16 columns of the rank from blockIdx.z on.
// The waves take every n-th 64 of K, each through LDS of its own and without a barrier, and add up their sums at the end.
// Bound by the loads: x comes from HBM once, a_i from the L2 once a tile. They go to LDS eight rows of 128 bytes at a time: straight to the
// registers of the matrix instructions, whose lanes side by side belong to rows, each lane's 16 bytes are a cache line of their own to the
// address unit (4608 x 3072, rank 64: 34 us).
template <int R>           // row fragments of a tile: R * 16 rows
struct LowOfTile {
    int own[R], a;         // the adapters of this lane's rows, and the one of this workgroup; a < 0: none is left for it
    int row0;
};
template <int R>
__device__ __forceinline__ LowOfTile<R> low_of_tile(const LoraLow& p) {
    const int frow = threadIdx.x & 15;
    LowOfTile<R> t;
    t.row0 = blockIdx.x * (R * 16);
    t.a = -1;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int m = t.row0 + i * 16 + frow;
        const int64_t request = min(m, p.M - 1) / p.rows_per_request;
        const int64_t id = p.wide_ids ? static_cast<const int64_t*>(p.adapter)[request] : static_cast<const int32_t*>(p.adapter)[request];
        t.own[i] = id >= 0 && id < p.adapters ? static_cast<int>(id) : -1;
        if (blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x < 16 && m < p.M) p.owner[m] = t.own[i];
    }
    constexpr int kNone = 0x7fffffff;
    for (unsigned n = 0; n <= blockIdx.y; ++n) {
        int next = kNone;
#pragma unroll
        for (int i = 0; i < R; ++i) next = t.own[i] > t.a ? min(next, t.own[i]) : next;
        t.a = LoraTail::first_of_rows(next);
        if (t.a == kNone) {   // (alike in every wave)
            t.a = -1;
            break;
        }
    }
    return t;
}

// The waves' sums, in LDS as [wave][R][NF][64 lanes][4], added in order, scaled and stored as LoraPlace says. Lane l of a fragment holds row l % 16
// and four ranks from l / 16 * 4 on. A thread takes V of them: all four where a tile has work for every thread, fewer where threads would be idle.
template <int R, int NF>
__device__ __forceinline__ void low_store(const LoraLow& p, const LowOfTile<R>& t, const float* part, int waves, int r0) {
    constexpr int V = R == 1 ? 1 : 4;
    typedef float vec __attribute__((ext_vector_type(V)));
    const float scale = p.scaling != nullptr ? p.scaling[t.a] : 1.0f;
    const bool beside = p.at.beside();
#pragma unroll
    for (int f = 0; f < R; ++f)
        for (int i = threadIdx.x * V; i < NF * 256; i += blockDim.x * V) {
            const int row = (i >> 2) & 15, m = t.row0 + f * 16 + row, r = r0 + (i >> 8) * 16 + ((i & 255) >> 6) * 4 + (i & 3);
            vec sum = {};
            for (int w = 0; w < waves; ++w) sum += *reinterpret_cast<const vec*>(part + (w * R + f) * (NF * 256) + (beside ? i & 255 : i));
            const bool mine = __shfl(t.own[f], row) == t.a;
            if (!mine || m >= p.M || r >= p.at.width) continue;
            const int rank = beside ? r & 15 : r;   // (the first of V)
            vec first, left;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                sum[e] = rank + e < p.at.rank ? sum[e] * scale : 0.0f;
                first[e] = round_bf16(sum[e]);
                left[e] = __builtin_isfinite(first[e]) ? sum[e] - first[e] : 0.0f;   // (nothing is left over of what is infinite or NaN)
            }
            if (p.at.planes == 0) {
                if (r < p.at.pitch()) *reinterpret_cast<vec*>(static_cast<float*>(p.low) + static_cast<int64_t>(m) * p.at.pitch() + r) = sum;
                continue;
            }
            typedef __bf16 halves __attribute__((ext_vector_type(V)));
            const halves one = __builtin_convertvector(first, halves), two = __builtin_convertvector(left, halves);
            bf16_t* const to = static_cast<bf16_t*>(p.low) + p.at.block(m / 16, r) + (((r >> 3) & 3) * 16 + (m & 15)) * 8 + (r & 7);
            *reinterpret_cast<halves*>(to) = beside && r >= 16 ? two : one;
            if (p.at.planes == 2) *reinterpret_cast<halves*>(to + 512) = two;
        }
}

template <int R, int NF, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void lora_low_kernel(LoraLow p) {
    constexpr int BYTES = (R + NF) * 2048;   // of a wave: R * 16 rows of x and NF * 16 of a, 64 of K each
    __shared__ __attribute__((aligned(1024))) char lds[WAVES * BYTES];
    static_assert(R * NF * 1024 <= BYTES, "the sums take the operands' place");
    const LowOfTile<R> t = low_of_tile<R>(p);
    if (t.a < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), frow = lane & 15, fq = lane >> 4;
    const int r0 = blockIdx.z * (NF * 16);
    char* const mine = lds + wave * BYTES;
    // slot (row, position lane % 8) of 8 rows holds chunk position ^ (row / 2 % 8) of its row, so that 16 rows' chunks are read without conflicts
    const int rows_x = min(p.M - t.row0, R * 16), rows_a = min(p.at.rank - r0, NF * 16);
    bf16_t* const x = const_cast<bf16_t*>(p.x + t.row0 * p.lda);
    bf16_t* const a = const_cast<bf16_t*>(p.a + (static_cast<int64_t>(t.a) * p.at.rank + r0) * p.K);
    const int bytes_x = static_cast<int>(((rows_x - 1) * p.lda + p.K) * 2), bytes_a = rows_a * p.K * 2;
    uint32_t off_x[2 * R], off_a[2 * NF];
    int chunk[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) chunk[i] = (lane & 7) ^ (((i * 8 + (lane >> 3)) >> 1) & 7);
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) {
        const int row = i * 8 + (lane >> 3);
        off_x[i] = row < rows_x ? static_cast<uint32_t>((row * p.lda + chunk[i & 1] * 8) * 2) : kOutOfRange;
    }
#pragma unroll
    for (int i = 0; i < 2 * NF; ++i) {
        const int row = i * 8 + (lane >> 3);
        off_a[i] = row < rows_a ? static_cast<uint32_t>((row * p.K + chunk[i & 1] * 8) * 2) : kOutOfRange;
    }
    f32x4 acc[R][NF];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int f = 0; f < NF; ++f) acc[i][f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = wave * 64; k0 < p.K; k0 += WAVES * 64) {   // (what lies past K, M and the rank reads as zeros)
        const uint32_t end[2] = {k0 + chunk[0] * 8 < p.K ? 0u : kOutOfRange, k0 + chunk[1] * 8 < p.K ? 0u : kOutOfRange};
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) load_chunk(__builtin_amdgcn_make_buffer_rsrc(x, 0, bytes_x, kRsrcFlags), mine + i * 1024, off_x[i] | end[i & 1], k0 * 2);
#pragma unroll
        for (int i = 0; i < 2 * NF; ++i) load_chunk(__builtin_amdgcn_make_buffer_rsrc(a, 0, bytes_a, kRsrcFlags), mine + R * 2048 + i * 1024, off_a[i] | end[i & 1], k0 * 2);
        wait_vmem_all();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int at = frow * 128 + (((s * 4 + fq) ^ ((frow >> 1) & 7)) * 16);
            bf16x8 xf[R];
#pragma unroll
            for (int i = 0; i < R; ++i) xf[i] = *reinterpret_cast<const bf16x8*>(mine + i * 2048 + at);
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const bf16x8 af = *reinterpret_cast<const bf16x8*>(mine + (R + f) * 2048 + at);
#pragma unroll
                for (int i = 0; i < R; ++i) acc[i][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, xf[i], acc[i][f], 0, 0, 0);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the operands have been read: their place is free
    }
    __syncthreads();
    float* const part = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int f = 0; f < NF; ++f) *reinterpret_cast<f32x4*>(part + ((wave * R + i) * NF + f) * 256 + lane * 4) = acc[i][f];
    __syncthreads();
    low_store<R, NF>(p, t, part, WAVES, r0);
}

// The same for operands without 16-byte rows: straight from memory, a value at a time.
__global__ __launch_bounds__(256) void lora_low_any_kernel(LoraLow p) {
    constexpr int NF = 2;
    __shared__ float part[4 * NF * 256];
    const LowOfTile<1> t = low_of_tile<1>(p);
    if (t.a < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, frow = lane & 15, fq = lane >> 4;
    const int r0 = blockIdx.z * (NF * 16);
    const bf16_t* const x = p.x + min(t.row0 + frow, p.M - 1) * p.lda;
    f32x4 acc[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto piece = [&](const bf16_t* row, int k, bool ok) {
        Vec16<bf16_t> v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v.v[e] = ok && k + e < p.K ? row[k + e] : static_cast<bf16_t>(0);
        return __builtin_bit_cast(bf16x8, v);
    };
    for (int k0 = wave * 32; k0 < p.K; k0 += 128) {
        const bf16x8 xf = piece(x, k0 + fq * 8, true);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int r = r0 + f * 16 + frow;
            acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(piece(p.a + (static_cast<int64_t>(t.a) * p.at.rank + min(r, p.at.rank - 1)) * p.K, k0 + fq * 8, r < p.at.rank), xf, acc[f], 0, 0, 0);
        }
    }
#pragma unroll
    for (int f = 0; f < NF; ++f) *reinterpret_cast<f32x4*>(part + (wave * NF + f) * 256 + lane * 4) = acc[f];
    __syncthreads();
    low_store<1, NF>(p, t, part, 4, r0);
}

void launch_lora_low(const LoraLow& p, hipStream_t st) {
    // adapters a tile can hold: requests that touch so many rows
    auto grid = [&](int rows, int ranks) {
        const int64_t requests = p.rows_per_request % rows == 0 ? 1 : std::min<int64_t>(rows, (rows - 2) / p.rows_per_request + 2);
        return dim3((unsigned)((p.M + rows - 1) / rows), (unsigned)std::min<int64_t>(requests, p.adapters), (unsigned)((p.at.width + ranks - 1) / ranks));
    };
    if (!p.vec) {
        hipLaunchKernelGGL(lora_low_any_kernel, grid(16, 32), dim3(256), 0, st, p);
        return;
    }
#define CALL(R, NF, W) hipLaunchKernelGGL((lora_low_kernel<R, NF, W>), grid(R * 16, NF * 16), dim3(W * 64), 0, st, p)
    // 32 rows a tile where 256 tiles of 16 would be left, since a comes once a tile. As many waves as the CU's 160 KB hold of one workgroup at
    // a time or two share K, and four where every CU gets several workgroups by itself. us of the whole operator, N = 128, K = 3072, for 16 rows of 8
    // waves, 32 rows of 8 (rank 64: 6) and 32 rows of 4: rank 32: 19.4, 20.4 and 24.3 at 2304 rows, 28.0, 25.5 and 29.1 at 4608, rank 16: 42.8, 42.2 and
    // 41.3 at 13008; rank 64: 23.0, 25.1 and 29.1 at 2304, 33.9, 29.9 and 33.0 at 4608, 57.3, 53.0 and 50.2 at 13008. (16 rows of 16 and 4 waves at
    // 517, rank 16: 18.1 and 21.2, of 8: 18.3.)
    const bool few = (p.M + 15) / 16 < 256;
    const int64_t blocks = static_cast<int64_t>((p.M + 31) / 32) * ((p.at.width + 63) / 64);
    if (p.at.width <= 32) {
        if (few) CALL(1, 2, 8);
        else if (blocks <= 256) CALL(2, 2, 8);
        else CALL(2, 2, 4);
    } else {
        if (few) CALL(1, 4, 8);
        else if (blocks <= 256) CALL(2, 4, 6);
        else CALL(2, 4, 4);
    }
#undef CALL
}

// A product with adapters has one output, no residual and no q/k columns: what serves those is left out of its kernels.
__device__ __forceinline__ GemmParams one_output(const GemmLaunch& L) {
    GemmParams p = L.p[0];
    p.gate = p.resid = nullptr;
    p.Y2 = nullptr;
    p.split_n = p.N;
    p.y2_col0 = p.qk_cols = p.act_begin = p.in_silu = 0;
    p.rows_per_batch = 1;
    p.a_skip = 0;
    p.ldy2 = p.ldresid = 0;
    return p;
}

// The four-wave tiles of gemm_bf16.hip with the adapter's product in front of their epilogue.
template <bool KTAIL>
__global__ __launch_bounds__(kGemmThreads) void lora_ring_kernel(GemmLaunch L, LoraTail tail) {
    constexpr int MI = 4, BM = 64 * MI, BK = 64, NU = 5, UNIT = BM * BK * 2;
    __shared__ __attribute__((aligned(1024))) char lds[NU * UNIT];
    int tm, tn;
    if (!tile_of_block(L, tm, tn)) return;
    const GemmParams p = one_output(L);
    const int m0 = tm * BM, n0 = tn * BM;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm0 = m0 + (wave >> 1) * (32 * MI), wn0 = n0 + (wave & 1) * (32 * MI);
    LoraTail::Ahead<2 * MI, 2 * MI> have;
    tail.begin(have, wm0, p);
    f32x4 acc[2 * MI][2 * MI];
    gemm_tile_slabs<MI, KTAIL>(p, lds, m0, n0, (p.K + BK - 1) / BK, acc, [&]() {
        tail.touch(have, wm0, wn0, p);
        hold(acc);
    });
    hold(acc);
    tail.finish(acc, have, wm0, wn0, p);
    gemm_epilogue<MI, MI>(p, acc, lds, m0, n0, wave, lane);
}

template <int FM, int FN, bool KTAIL>
__global__ __launch_bounds__(kGemmThreads) void lora_rect_kernel(GemmLaunch L, LoraTail tail) {
    constexpr int BM = 32 * FM, BN = 32 * FN, BK = 64;
    __shared__ __attribute__((aligned(1024))) char lds[(3 * BM + 2 * BN) * BK * 2];
    int tm, tn;
    if (!tile_of_block(L, tm, tn)) return;
    const GemmParams p = one_output(L);
    const int m0 = tm * BM, n0 = tn * BN;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm0 = m0 + (wave >> 1) * (16 * FM), wn0 = n0 + (wave & 1) * (16 * FN);
    LoraTail::Ahead<FM, FN> have;
    tail.begin(have, wm0, p);
    f32x4 acc[FM][FN];
    gemm_rect_slabs<FM, FN, KTAIL>(p, lds, m0, n0, (p.K + BK - 1) / BK, acc, [&]() {
        tail.touch(have, wm0, wn0, p);
        hold(acc);
    });
    hold(acc);
    tail.finish(acc, have, wm0, wn0, p);
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

// Row vectors: the loops over K of launch_gemv (gemm_bf16.hip) that fit any K. W always has the non-temporal hint, which leaves the caches to the
// adapters, low and the rows. us of the whole operator at rank 16 with and without it, W from HBM (the same W again at once): 6 x 6144 x 1024 12.9 and 16.4 (10.7,
// 12.5), 1 x 9216 x 3072 17.9 and 21.0 (15.1, 17.4), 4 x 9216 x 3072 25.0 and 28.6 (20.8, 23.2), 1 x 3072 x 12288 33.8 and 40.5 (28.3, 28.7), 6 x 12288 x 12288
// 107 and 195 (105, 195). Where 216 MiB are read again at once beside one or three rows it loses 5 and 6 %, and gains 17 and 10 % from HBM: 1 x 18432 x 6144
// 45.0 and 54.1 (43.9, 41.8), 3 x 36864 x 3072 50.6 and 56.3 (48.4, 45.5).
template <int MM, bool LDS, int U>
__global__ __launch_bounds__(256) void lora_rows_kernel(GemmParams p, LoraTail t) {
    extern __shared__ __attribute__((aligned(16))) char act_lds[];
    LoraRowTail<MM> tail;
    tail.t = t;
    gemv_small_m<MM, LDS, U, false, true>(p, static_cast<int>(blockIdx.x), act_lds, tail);
}

template <int MM>
static void launch_rows_of(const GemmParams& p, const LoraTail& tail, hipStream_t st) {
    const dim3 grid((unsigned)((p.N + 4 * kGemvCols - 1) / (4 * kGemvCols)));
    const size_t act_bytes = static_cast<size_t>(MM) * p.K * 2;
    constexpr int U = MM <= 2 ? 6 : 3;
    if (act_bytes <= kGemvSiluLds) hipLaunchKernelGGL((lora_rows_kernel<MM, true, U>), grid, dim3(256), act_bytes, st, p, tail);
    else hipLaunchKernelGGL((lora_rows_kernel<MM, false, U>), grid, dim3(256), 0, st, p, tail);
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
        const bf16_t* b = t.b + (static_cast<int64_t>(own) * p.N + n) * t.at.rank;
        for (int r = 0; r < t.at.rank; ++r) sum += t.value(m, r) * bf2f(b[r]);
    }
    sum += p.bias ? bf2f(p.bias[n]) : 0.0f;
    if (p.act == FLUX_ACT_GELU_TANH) sum = gelu_tanh_f32(sum);
    p.Y[static_cast<int64_t>(m) * p.ldy + n] = f2bf(sum);
}

void launch_lora_scalar(const GemmParams& p, const LoraTail& tail, hipStream_t st) {
    hipLaunchKernelGGL(lora_scalar_kernel, dim3((unsigned)((static_cast<int64_t>(p.M) * p.N + 255) / 256)), dim3(256), 0, st, p, tail);
}

}  // namespace flux
