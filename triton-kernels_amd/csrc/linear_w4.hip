// Products with weights held in 4 bits, a scale and (or not) a zero point for each group of 32, 64 or 128 columns.
//
//   y[m, n] = act(sum_g s[n, g] sum_{k in g} (q[n, k] - z[n, g]) x[m, k] + b[n])
//
// Half a byte a weight and two operations a row: up to some dozens of rows bound by the bytes of the weights. A multiplication on the VALU would cost more
// than they do: 57 M weights are 28 MB, 5.6 us at a copy's rate, and at three instructions a weight (take it out, convert, multiply) 4.4 us of all VALUs for one
// row. So a weight becomes a bf16 number in one instruction, 16 + q = (q << 3) | 0x4180 for two of them at once, and the matrix cores multiply (16x16x32,
// x the rows and W the columns of the result, whose 16 rows cost one row's time). What is too much, (16 + z) times the sum of x, comes from the matrix cores as well,
// as a product with ones. A group's sum takes its scale behind the product, in fp32: nothing is rounded but y.
//
// us among others of its kind: 1 x 18432 x 3072 8.4, with SiLU 8.8 to 10.3 by the box (floor 5.7), 3 x 9216 x 3072 with SiLU 7.5 to 8.2, 1 x 1000 x 1024 3.1 (a launch), 16 x
// 9216 x 3072 9.0, 24 x 12288 x 3072 12.4 to 12.9, 128 x 9216 x 3072 29, 512 x 9216 x 3072 39.5, 1000 x 9216 x 3072 67 (15 of them for laying the weights out).
#include "common.h"
#include "../../include/flux_hip_serve.h"
#include <algorithm>
#include <math.h>
#include <type_traits>

namespace flux {

typedef __bf16 w4_bf16x8 __attribute__((ext_vector_type(8)));
typedef float w4_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t w4_u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 w4_f16x2 __attribute__((ext_vector_type(2)));
typedef float w4_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 w4_bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kW4Chunk = 128;         // columns of a tile
constexpr int kW4Tile = 16;           // rows of W (outputs) of a tile
constexpr int kW4SiluRows = 8;

struct W4Params {
    const bf16_t* x; const w4_u32x4* q; const bf16_t* s; const uint8_t* z; const bf16_t* bias; bf16_t* y;
    int64_t ldx, ldy;
    int M, N, K, chunks, slab;        // slab: chunks of x in LDS at a time
    int act, silu;
};

// Two times 16 in bf16, in a vector register: v_and_or_b32 takes one scalar constant, and with two of them it was two instructions.
__device__ __forceinline__ uint32_t w4_sixteens() {
    uint32_t one = 0x41804180u;
    asm volatile("" : "+v"(one));
    return one;
}
// Eight weights, 16 + q each.
__device__ __forceinline__ w4_bf16x8 w4_unpack(uint32_t w, uint32_t one) {
    const uint32_t mask = 0x00780078u;
    w4_u32x4 r;
    r.x = ((w << 3) & mask) | one;
    r.y = ((w >> 1) & mask) | one;
    r.z = ((w >> 5) & mask) | one;
    r.w = ((w >> 9) & mask) | one;
    return __builtin_bit_cast(w4_bf16x8, r);
}
// Eight weights, q - z each.
__device__ __forceinline__ w4_bf16x8 w4_unpack_exact(uint32_t w, float z) {
    w4_bf16x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = static_cast<__bf16>(static_cast<float>((w >> (4 * (e / 2) + 16 * (e % 2))) & 15u) - z);
    return r;
}

// The scales (or zero points) of a lane's row in one chunk, as one load.
template <int BYTES> struct W4Word;
template <> struct W4Word<1> { typedef uint8_t type; };
template <> struct W4Word<2> { typedef uint16_t type; };
template <> struct W4Word<4> { typedef uint32_t type; };
template <> struct W4Word<8> { typedef uint64_t type; };

// What a wave holds of 16 outputs x 128 columns.
template <int GPC, bool ZERO> struct W4Piece {
    w4_u32x4 q;
    typename W4Word<2 * GPC>::type s;
    typename W4Word<GPC>::type z;
    __device__ __forceinline__ float scale(int i) const { return bf2f(static_cast<bf16_t>(s >> (16 * i))); }
    __device__ __forceinline__ float zero(int i) const { return ZERO ? static_cast<float>(static_cast<uint8_t>(z >> (8 * i))) : 8.0f; }
};
// A row tile of W: q at the lane's 16 bytes, s and z at its row.
template <int GPC, bool ZERO> struct W4Tile {
    const w4_u32x4* q; const typename W4Word<2 * GPC>::type* s; const typename W4Word<GPC>::type* z;
    __device__ __forceinline__ W4Tile(const W4Params& p, int tile, int lane) {
        const int64_t at = static_cast<int64_t>(tile) * p.chunks;
        q = p.q + at * 64 + lane;
        s = reinterpret_cast<const typename W4Word<2 * GPC>::type*>(p.s) + at * 16 + (lane & 15);
        z = ZERO ? reinterpret_cast<const typename W4Word<GPC>::type*>(p.z) + at * 16 + (lane & 15) : nullptr;
    }
    template <bool ONCE> __device__ __forceinline__ void request(W4Piece<GPC, ZERO>& to, int c) const {
        to.q = ONCE ? __builtin_nontemporal_load(q + static_cast<int64_t>(c) * 64) : q[static_cast<int64_t>(c) * 64];
        to.s = s[c * 16];
        if (ZERO) to.z = z[c * 16];
    }
};

// f(x) = x sigmoid(x) as a bf16 number in x and what it leaves over in lo.
__device__ __forceinline__ void w4_silu(Vec16<bf16_t>& x, Vec16<bf16_t>& lo) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float f = bf2f(x.v[e]);
        f = f * __builtin_amdgcn_rcpf(1.0f + __expf(-f));
        x.v[e] = f2bf(f);
        lo.v[e] = f2bf(fabsf(f) < INFINITY ? f - bf2f(x.v[e]) : 0.0f);
    }
}

// acc += s (q - z) x over one chunk, for MT times 16 rows of x, the lane's `row` bytes behind `a`: the sum of (16 + q) x without (16 + z) times the sum of x, which the
// matrix cores form beside it. Both sums are rounded: some 2^-23 of the sum of (32 + q + z) |x| is lost, however little of it
// is left. `peak` takes the largest sum of x: where x is not finite it leaves a NaN or an infinity.
template <int GPC, bool ZERO, int MT>
__device__ __forceinline__ void w4_chunk(w4_f32x4 (&acc)[MT], const W4Piece<GPC, ZERO>& w, const char* a, const int (&row)[MT], uint32_t sixteens, float& peak) {
    const w4_f32x4 none = {0.f, 0.f, 0.f, 0.f};
    const w4_bf16x8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
    for (int i = 0; i < GPC; ++i) {
        const float zero = w.zero(i), scale = w.scale(i);
        w4_f32x4 t[MT], u[MT];
#pragma unroll
        for (int j = i * 4 / GPC; j < (i + 1) * 4 / GPC; ++j) {
            const bool first = j == i * 4 / GPC;
            const w4_bf16x8 b = w4_unpack(w.q[j], sixteens);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const w4_bf16x8 x = *reinterpret_cast<const w4_bf16x8*>(a + row[m] + j * 64);
                t[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, b, first ? none : t[m], 0, 0, 0);
                u[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, ones, first ? none : u[m], 0, 0, 0);
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            peak = fmaxf(fmaxf(peak, fabsf(u[m][0])), fabsf(u[m][1]));
            peak = fmaxf(fmaxf(peak, fabsf(u[m][2])), fabsf(u[m][3]));
            acc[m] += (t[m] - u[m] * (16.0f + zero)) * scale;
        }
    }
}

// Whether a lane of the wave holds a sum that is not finite, or had one beyond 2^100 on its way.
template <int N, int MT> __device__ __forceinline__ bool w4_lost(const w4_f32x4 (&acc)[N][MT], float peak) {
    bool lost = !(peak < 0x1p100f);
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) lost |= !(fabsf(acc[t][m][i]) < INFINITY);
    return __builtin_amdgcn_ballot_w64(lost) != 0;
}

// The wave's sums once more, with q - z as it is and x from memory: for rows that are not finite.
// part, parts: which chunks of K; a row of x: row(m) of the wave's 16 MT, with SPLIT f(x) as in LDS.
template <bool SPLIT, int GPC, bool ZERO, int MT>
__device__ __forceinline__ void w4_again(w4_f32x4 (&acc)[MT], const W4Params& p, int tile, int m0, int rows, int part, int parts) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
    const W4Tile<GPC, ZERO> w(p, tile, lane);
#pragma unroll 1
    for (int c = part; c < p.chunks; c += parts) {
        W4Piece<GPC, ZERO> piece;
        w.template request<false>(piece, c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = j * GPC / 4, k = c * kW4Chunk + j * 32 + g * 8;
            const w4_bf16x8 b = w4_unpack_exact(piece.q[j], piece.zero(i));
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int row = SPLIT ? l16 & 7 : m * 16 + l16;
                Vec16<bf16_t> x, lo;
#pragma unroll
                for (int e = 0; e < 8; ++e) x.v[e] = 0;
                if (k < p.K && row < rows) x = ld16(p.x + static_cast<int64_t>(m0 + row) * p.ldx + k);
                if (SPLIT) {
                    w4_silu(x, lo);
                    if (l16 >= 8) x = lo;
                }
                const w4_f32x4 t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(w4_bf16x8, x), b, w4_f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                acc[m] += t * piece.scale(i);
            }
        }
    }
}

__device__ __forceinline__ bf16_t w4_result(const W4Params& p, float y, float bias) {
    y += bias;
    return f2bf(p.act == FLUX_ACT_GELU_TANH ? gelu_tanh_f32(y) : y);
}

// A workgroup takes 16 NW outputs of up to 16 rows of x (8 with SPLIT: f(x) as a bf16 number and another one for what that leaves over, in
// rows 8 beneath). KS waves share 16 of them; they take every KS-th chunk of K and add their sums in order. The first vectors of x are asked for in front of the weights: loads
// return in order, and the weights of a wave can wait in registers while x is on its way through LDS.
template <int GPC, bool ZERO, bool SPLIT, int NW, int KS>
__global__ __launch_bounds__(64 * NW * KS, 4) void w4_rows_kernel(W4Params p) {
    constexpr int RB = SPLIT ? 8 : 16, U = 6, PRE = 2, T = 64 * NW * KS;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
    const int tiles = (p.N + kW4Tile - 1) / kW4Tile, part = wave / NW, tile = min(static_cast<int>(blockIdx.x) * NW + wave % NW, tiles - 1), m0 = blockIdx.y * RB, rows = min(RB, p.M - m0), held = SPLIT ? 2 * rows : rows;
    const int stride = p.slab * (kW4Chunk * 2) + 16;                  // bytes of a row of x in LDS, 16 more against conflicts
    // rows of the product without a row of x read the first one; what they sum up is not stored
    const int my_row = l16 < rows ? l16 : (SPLIT && l16 >= 8 && l16 - 8 < rows) ? rows + l16 - 8 : 0;
    const int xrow[1] = {my_row * stride + g * 16};
    const W4Tile<GPC, ZERO> w(p, tile, lane);
    const int out_n = (blockIdx.x * NW + (tid >> 8)) * kW4Tile + (tid & 15);   // (of the thread's result)
    const float bias = p.bias != nullptr ? bf2f(p.bias[min(out_n, p.N - 1)]) : 0.0f;
    w4_f32x4 acc[1][1] = {{{0.f, 0.f, 0.f, 0.f}}};
    float peak = 0.0f;
    const uint32_t sixteens = w4_sixteens();
    W4Piece<GPC, ZERO> piece[U];
    for (int c0 = 0; c0 < p.chunks; c0 += p.slab) {
        const int n = min(p.slab, p.chunks - c0), vectors = rows * n * 16;   // vectors of 8 values of x, 16 a chunk
        auto load = [&](int i) {
            const int m = rows == 1 ? 0 : i / (n * 16), v = i - m * (n * 16), k = (c0 * 16 + v) * 8;
            Vec16<bf16_t> x;
#pragma unroll
            for (int e = 0; e < 8; ++e) x.v[e] = 0;
            if (i < vectors && k < p.K) x = ld16(p.x + (m0 + m) * p.ldx + k);
            return x;
        };
        auto stage = [&](int i, Vec16<bf16_t> hi) {
            const int m = rows == 1 ? 0 : i / (n * 16), v = i - m * (n * 16);
            Vec16<bf16_t> lo;
            if (SPLIT) w4_silu(hi, lo);
            *reinterpret_cast<Vec16<bf16_t>*>(lds + m * stride + v * 16) = hi;
            if (SPLIT) *reinterpret_cast<Vec16<bf16_t>*>(lds + (rows + m) * stride + v * 16) = lo;
        };
        Vec16<bf16_t> x[PRE];
#pragma unroll
        for (int j = 0; j < PRE; ++j) x[j] = load(tid + j * T);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u) w.template request<true>(piece[u], c0 + min(part + KS * u, n - 1));   // (past the end: not used)
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();   // the slab before is read
#pragma unroll
        for (int j = 0; j < PRE; ++j)
            if (tid + j * T < vectors) stage(tid + j * T, x[j]);
        for (int i = tid + PRE * T; i < vectors; i += T) stage(i, load(i));
        __syncthreads();
        for (int base = part; base < n; base += KS * U)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = base + KS * u;
                if (c >= n) break;
                w4_chunk<GPC, ZERO, 1>(acc[0], piece[u], lds + c * (kW4Chunk * 2), xrow, sixteens, peak);
                if (c + KS * U < n) w.template request<true>(piece[u], c0 + c + KS * U);
            }
    }
    if (__builtin_expect(w4_lost(acc, peak), 0)) w4_again<SPLIT, GPC, ZERO, 1>(acc[0], p, tile, m0, rows, part, KS);
    __syncthreads();
    float* const parts = reinterpret_cast<float*>(lds);   // [wave][lane][4]
    *reinterpret_cast<w4_f32x4*>(parts + tid * 4) = acc[0][0];
    __syncthreads();
    const int m = (tid >> 4) & 15;
    if (tid >= NW * 256 || m >= rows || out_n >= p.N) return;
    float y = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
        y += parts[((i * NW + (tid >> 8)) * 64 + (m >> 2) * 16 + (tid & 15)) * 4 + (m & 3)];
        if (SPLIT) y += parts[((i * NW + (tid >> 8)) * 64 + ((m + 8) >> 2) * 16 + (tid & 15)) * 4 + (m & 3)];
    }
    p.y[(m0 + m) * p.ldy + out_n] = w4_result(p, y, bias);
}

// x straight to LDS, 64 x 16 bytes, asked for behind the compiler's back: it would wait for every such load in front of every read of LDS. The kernel waits for
// them itself. What lies past the descriptor's end arrives as zeros.
__device__ __forceinline__ void w4_load_lds(w4_u32x4 rsrc, uint32_t lds_addr, uint32_t voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(lds_addr), "v"(voff), "s"(rsrc) : "memory", "m0");
}

// More rows: up to 16 MT of them a workgroup, whose waves are NW groups of 16 NTW outputs times KS parts of K. A wave keeps CW chunks of weights on
// their way. x goes through LDS, all of K at once where it fits, or in slabs of p.slab chunks, the next one on its way while one is multiplied.
template <int GPC, bool ZERO, int MT, int NTW, int NW, int KS, int CW>
__global__ __launch_bounds__(64 * NW * KS) void w4_tiles_kernel(W4Params p) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    constexpr int RB = 16 * MT, WAVES = NW * KS;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
    const int nw = wave % NW, part = wave / NW, m0 = blockIdx.y * RB, rows = min(RB, p.M - m0);
    const int tiles = (p.N + kW4Tile - 1) / kW4Tile, tile0 = (blockIdx.x * NW + nw) * NTW;
    const int stride = p.slab * (kW4Chunk * 2) + 16, buffer = rows * stride, pieces = p.slab / 4;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)lds));
    auto load_x = [&](int slab) {
        for (int i = wave; i < rows * pieces; i += WAVES) {
            const int m = i / pieces, piece = i - m * pieces;
            const uint64_t at = reinterpret_cast<uint64_t>(p.x + static_cast<int64_t>(m0 + m) * p.ldx);
            w4_u32x4 r;
            r.x = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at));
            r.y = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at >> 32) & 0xffffu);
            r.z = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(p.K) * 2u);
            r.w = 0x00020000u;
            w4_load_lds(r, __builtin_amdgcn_readfirstlane(lds0 + (slab & 1) * buffer + m * stride + piece * 1024), static_cast<uint32_t>(slab * p.slab * (kW4Chunk * 2) + piece * 1024 + lane * 16));
        }
    };
    w4_f32x4 acc[NTW][MT];
#pragma unroll
    for (int t = 0; t < NTW; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
    float peak = 0.0f;
    const uint32_t sixteens = w4_sixteens();
    W4Piece<GPC, ZERO> piece[NTW][CW];
    auto load_w = [&](W4Piece<GPC, ZERO>& to, int t, int chunk) {   // (past the end: not used)
        W4Tile<GPC, ZERO>(p, min(tile0 + t, tiles - 1), lane).template request<false>(to, min(chunk, p.chunks - 1));
    };
    load_x(0);
#pragma unroll
    for (int c = 0; c < CW; ++c)
#pragma unroll
        for (int t = 0; t < NTW; ++t) load_w(piece[t][c], t, c * KS + part);
    // rows of the product without a row of x read the first one; what they sum up is not stored
    int row[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) row[m] = (m * 16 + l16 < rows ? m * 16 + l16 : 0) * stride + g * 16;
    const int per = p.slab / KS, steps = (p.chunks + KS - 1) / KS;   // a wave's chunks of a slab, and of all
    const char* x = lds;
    auto open = [&](int slab) {   // what was asked for has landed, and the slab before is read
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if ((slab + 1) * p.slab < p.chunks) load_x(slab + 1);
        x = lds + (slab & 1) * buffer;
    };
    int next = 0;   // the step at which a slab begins
    for (int base = 0; base < steps; base += CW) {
#pragma unroll
        for (int c = 0; c < CW; ++c) {
            const int step = base + c;
            if (step < steps) {
                if (step == next) {
                    open(step / per);
                    next += per;
                }
                const int chunk = step * KS + part, at = chunk % p.slab;
                if (chunk < p.chunks) {
#pragma unroll
                    for (int t = 0; t < NTW; ++t) w4_chunk<GPC, ZERO, MT>(acc[t], piece[t][c], x + at * (kW4Chunk * 2), row, sixteens, peak);
                }
                if (step + CW < steps)
#pragma unroll
                    for (int t = 0; t < NTW; ++t) load_w(piece[t][c], t, (step + CW) * KS + part);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    if (__builtin_expect(w4_lost(acc, peak), 0))
#pragma unroll
        for (int t = 0; t < NTW; ++t) w4_again<false, GPC, ZERO, MT>(acc[t], p, min(tile0 + t, tiles - 1), m0, rows, part, KS);
    if constexpr (KS > 1) {   // the parts' sums, in order
        __syncthreads();
        float* const parts = reinterpret_cast<float*>(lds);
        auto at = [&](int from, int t, int m) { return reinterpret_cast<w4_f32x4*>(parts + ((((from - 1) * NW + nw) * NTW + t) * MT + m) * 256 + lane * 4); };
        if (part > 0)
#pragma unroll
            for (int t = 0; t < NTW; ++t)
#pragma unroll
                for (int m = 0; m < MT; ++m) *at(part, t, m) = acc[t][m];
        __syncthreads();
        if (part > 0) return;
#pragma unroll
        for (int t = 0; t < NTW; ++t)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 1; i < KS; ++i) acc[t][m] += *at(i, t, m);
    }
#pragma unroll
    for (int t = 0; t < NTW; ++t) {
        const int n = (tile0 + t) * kW4Tile + l16;
        const float bias = p.bias != nullptr && n < p.N ? bf2f(p.bias[n]) : 0.0f;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = m * 16 + g * 4 + i;
                if (r < rows && n < p.N) p.y[static_cast<int64_t>(m0 + r) * p.ldy + n] = w4_result(p, acc[t][m][i], bias);
            }
    }
}
// Hundreds of rows of many outputs: 128 rows a workgroup, all of them each wave's, which takes 16 NT outputs, so that a weight is unpacked once for eight matrix
// instructions, as (q - z) s in bf16. x goes through LDS in four buffers of 128 columns, three of them on their way; weights wait in registers as long. In LDS a row is 256
// bytes, its 16 bytes c at place c ^ (row mod 16): fragments read one place of 16 rows.
// A step is 32 columns, 8 NT matrix instructions in a fixed order. Between them the wave unpacks the next step's weights, two in two slots, and reads 16 rows of the next step's x as soon as
// the last instruction on this step's has them. One wave a SIMD: its slots take some 35 cycles, twice the matrix instruction's 16 (loads of weights 18 % of the time, reads of LDS
// 13 %, loads of x 7 %). 192 or 256 rows (two outputs' tiles a wave) and weights asked for eight slabs ahead made no difference.
template <int GPC, bool ZERO, int NT>
__global__ __launch_bounds__(256, 1) void w4_product_kernel(W4Params p, int row_blocks, int blocks) {
    constexpr int MT = 8, DEEP = 4, SLAB = 128 * 256, NS = MT * NT;
    static_assert(NT <= 4, "a step asks for one tile of weights");
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
    const int per_xcd = gridDim.x / 8, at = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;   // the row blocks of some outputs share an XCD
    if (at >= blocks) return;
    const int m0 = at % row_blocks * 128, rows = min(128, p.M - m0);
    const int tiles = (p.N + kW4Tile - 1) / kW4Tile, tile0 = (at / row_blocks * 4 + wave) * NT;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)lds)) + wave * 1024;
    const int my_row = wave * 4 + g, my_col = (l16 ^ my_row) * 8;   // what the lane fetches: of rows my_row + 16 i
    const uint32_t row2 = static_cast<uint32_t>(p.ldx * 2), voff = my_row * row2 + my_col * 2;
    const uint64_t base = reinterpret_cast<uint64_t>(p.x + m0 * p.ldx);
    const uint32_t bytes = (rows - 1) * row2 + p.K * 2;   // (rows past the end arrive as zeros)
    w4_u32x4 rsrc;
    uint32_t first = 0, more = 0;   // the lane's offset and that of the next load; past the end where its columns are, which would be another row's
    auto open_x = [&](int c) {
        const uint64_t from = base + static_cast<uint64_t>(c) * (kW4Chunk * 2);
        rsrc.x = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(from));
        rsrc.y = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(from >> 32) & 0xffffu);
        rsrc.z = __builtin_amdgcn_readfirstlane(c < p.chunks ? bytes - c * (kW4Chunk * 2) : 0u);
        rsrc.w = 0x00020000u;
        const bool there = c * kW4Chunk + my_col < p.K;
        first = there ? voff : 0x80000000u;
        more = there ? 16 * row2 : 0u;
    };
    auto load_x = [&](int buffer, int i) { w4_load_lds(rsrc, __builtin_amdgcn_readfirstlane(lds0 + buffer * SLAB + i * 4096), first + i * more); };
    W4Piece<GPC, ZERO> piece[DEEP][NT];
    auto load_w = [&](int c, int buffer, int t) {   // (past the end: not used)
        W4Tile<GPC, ZERO>(p, min(tile0 + t, tiles - 1), lane).template request<false>(piece[buffer][t], min(c, p.chunks - 1));
    };
    w4_f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < DEEP; ++c) {   // (of the last one what a step asks for)
#pragma unroll
        for (int t = 0; t < (c < DEEP - 1 ? NT : 1); ++t) load_w(c, c, t);
        open_x(c);
#pragma unroll
        for (int i = 0; i < (c < DEEP - 1 ? MT : 2); ++i) load_x(c, i);
    }
    // Two weights: 1024 + q in fp16, or 1024 + 16 q where that saves a shift; times s (s / 16) less (1024 + z) s ((64 + z) s), exact in fp32, they are rounded once. (Without the
    // product that is taken off, by 1024 + z in fp16 first, 512 x 9216 x 3072 took 45.9 us for 41.4.) `most`: whether that product was a number.
    uint32_t magic = 0x64006400u, upper = 0, two = 0;
    asm volatile("" : "+v"(magic));
    float most = 0.0f;
    w4_f32x2 pair = {0.f, 0.f};
    float scale[2][NT], less[2][NT];
    auto factors = [&](const W4Piece<GPC, ZERO>& of, int t, int i) {
        const float s = of.scale(i), z = of.zero(i);
        scale[0][t] = s;
        less[0][t] = -(1024.0f + z) * s;
        scale[1][t] = s * 0.0625f;
        less[1][t] = -(64.0f + z) * s;
        most = fmaxf(most, fabsf(less[0][t]));
    };
    auto take = [&](uint32_t q, int i) {   // out of a word
        if (i == 0) upper = q >> 8;
        two = ((i < 2 ? q : upper) & (i % 2 == 0 ? 0x000f000fu : 0x00f000f0u)) | magic;
    };
    auto weigh = [&](int t, int i) {
        const w4_f16x2 h = __builtin_bit_cast(w4_f16x2, two);
        pair = w4_f32x2{__builtin_fmaf(static_cast<float>(h.x), scale[i % 2][t], less[i % 2][t]), __builtin_fmaf(static_cast<float>(h.y), scale[i % 2][t], less[i % 2][t])};
    };
    auto packed = [&]() { return __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, w4_bf16x2)); };
    w4_u32x4 w[2][NT];
    w4_bf16x8 a[MT];
    const char* const mine = lds + l16 * 256;
    int place[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) place[j] = ((j * 4 + g) ^ l16) * 16;
    // the first slab is here when no more than what was asked for behind it is missing
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((DEEP - 2) * MT + 2) : "memory");
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        factors(piece[0][t], t, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            take(piece[0][t].q[0], i);
            weigh(t, i);
            w[0][t][i] = packed();
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) a[m] = *reinterpret_cast<const w4_bf16x8*>(mine + m * 4096 + place[0]);
    for (int c0 = 0; c0 < p.chunks; c0 += DEEP) {
#pragma unroll
        for (int b = 0; b < DEEP; ++b) {
            const int c = c0 + b;
            if (c >= p.chunks) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int nj = (j + 1) % 4, nb = j == 3 ? (b + 1) % DEEP : b;   // the next step
                const int to = j == 3 ? b : (b + DEEP - 1) % DEEP, part = nj;   // the buffers of the slab that was read last get a quarter of another one a step
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    const int m = s / NT, t = s % NT;
                    acc[t][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[m], __builtin_bit_cast(w4_bf16x8, w[j & 1][t]), acc[t][m], 0, 0, 0);
                    if (j == 3 && s == NT - 1) {
                        // the next slab is here, as are all but the loads of two behind it, and everyone has read this one
                        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((DEEP - 2) * MT) : "memory");
                        open_x(c + DEEP);
                    }
                    if (t == NT - 1) a[m] = *reinterpret_cast<const w4_bf16x8*>(mine + nb * SLAB + m * 4096 + place[nj]);
                    const int u = s / 8, i = s / 2 % 4;
                    if (s % 2 == 0) {
                        if (s > 0) w[nj & 1][(s - 1) / 8][(s - 1) / 2 % 4] = packed();
                        if (i == 0 && nj * GPC % 4 == 0) factors(piece[nb][u], u, nj * GPC / 4);
                        take(piece[nb][u].q[nj], i);
                    } else {
                        weigh(u, i);
                        if (s == NS - 1) w[nj & 1][u][i] = packed();
                    }
                    if (s == NS / 2 && part < NT) load_w(c + (j == 3 ? DEEP : DEEP - 1), to, part);
                    if (s == NS / 4 || s == 3 * NS / 4) load_x(to, part * 2 + (s > NS / 2));
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(most < INFINITY)) != 0, 0))
#pragma unroll
        for (int t = 0; t < NT; ++t) w4_again<false, GPC, ZERO, MT>(acc[t], p, min(tile0 + t, tiles - 1), m0, rows, 0, 1);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");   // (loads past the end; everyone is done with x)
    // through LDS: rows of 32 NT bytes leave 16 at a time
    constexpr int STRIDE = NT * 32 + 16;
    char* const stage = lds + wave * (128 * STRIDE);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int n = (tile0 + t) * kW4Tile + l16;
        const float bias = p.bias != nullptr && n < p.N ? bf2f(p.bias[n]) : 0.0f;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<bf16_t*>(stage + (m * 16 + g * 4 + i) * STRIDE + t * 32 + l16 * 2) = w4_result(p, acc[t][m][i], bias);
    }
    __builtin_amdgcn_wave_barrier();   // LDS operations of one wave complete in order
    const bool whole = p.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
    for (int i = lane; i < rows * (2 * NT); i += 64) {
        const int m = i / (2 * NT), v = i - m * (2 * NT), n = tile0 * kW4Tile + v * 8;
        const Vec16<bf16_t> y = *reinterpret_cast<const Vec16<bf16_t>*>(stage + m * STRIDE + v * 16);
        bf16_t* const out = p.y + static_cast<int64_t>(m0 + m) * p.ldy + n;
        if (whole && n + 8 <= p.N) st16(out, y);
        else
            for (int e = 0; e < 8; ++e)
                if (n + e < p.N) out[e] = y.v[e];
    }
}

// bytes of LDS: x, one slab or two, or the parts' sums
static int w4_tiles_lds(const W4Params& p, int held, int parts_kb) {
    const int slabs = (p.chunks + p.slab - 1) / p.slab;
    return std::max((slabs > 1 ? 2 : 1) * held * (p.slab * kW4Chunk * 2 + 16), parts_kb * 1024);
}

// W as bf16 [N, K], (q - z) s rounded once. A wave takes a tile, whose rows pass through LDS so that they leave 256 bytes at a time (9216 x 3072: 14.4 us, 17.1 in
// pieces of 64 bytes of 16 rows).
template <int GPC, bool ZERO>
__global__ __launch_bounds__(256) void w4_unpack_kernel(const w4_u32x4* q, const bf16_t* s, const uint8_t* z, bf16_t* out, int N, int K, int chunks, int64_t tiles) {
    constexpr int STRIDE = kW4Chunk * 2 + 16;
    __shared__ __attribute__((aligned(16))) char lds[4][kW4Tile * STRIDE];
    const int wave = threadIdx.x >> 6;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (at >= tiles) return;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const w4_u32x4 w = __builtin_nontemporal_load(q + at * 64 + lane);
    float scale[GPC], zero[GPC];
#pragma unroll
    for (int i = 0; i < GPC; ++i) {
        scale[i] = bf2f(s[(at * 16 + r) * GPC + i]);
        zero[i] = ZERO ? static_cast<float>(z[(at * 16 + r) * GPC + i]) : 8.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        Vec16<bf16_t> o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o.v[e] = f2bf((static_cast<float>((w[j] >> (4 * (e / 2) + 16 * (e % 2))) & 15u) - zero[j * GPC / 4]) * scale[j * GPC / 4]);
        *reinterpret_cast<Vec16<bf16_t>*>(lds[wave] + r * STRIDE + j * 64 + g * 16) = o;
    }
    __builtin_amdgcn_wave_barrier();   // LDS operations of one wave complete in order
    const int64_t n0 = at / chunks * kW4Tile;
    const int k = static_cast<int>(at % chunks) * kW4Chunk + r * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 4 + g;
        if (n0 + row < N && k < K) st16(out + (n0 + row) * K + k, *reinterpret_cast<const Vec16<bf16_t>*>(lds[wave] + row * STRIDE + r * 16));
    }
}

// ------------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------------
static int w4_check(const char* what, const flux_w4& w) {
    if (w.N < 0 || w.K < 0) return fail(FLUX_E_SHAPE, "%s: bad shape [%lld,%lld]", what, (long long)w.N, (long long)w.K);
    if (w.group != 32 && w.group != 64 && w.group != 128) return fail(FLUX_E_UNSUPPORTED, "%s: groups of 32, 64 or 128 columns, not %d", what, w.group);
    if (w.K % w.group != 0) return fail(FLUX_E_SHAPE, "%s: %lld columns are not whole groups of %d", what, (long long)w.K, w.group);
    if (w.N > 0x7fffffff / 64 || w.K > 0x7fffffff / 64) return fail(FLUX_E_SHAPE, "%s: too many rows or columns", what);
    return FLUX_OK;
}
static int w4_pointers(const char* what, const flux_w4& w) {
    if (!w.q || !w.s) return fail(FLUX_E_NULL, "%s: null weights", what);
    if (!aligned16(w.q) || reinterpret_cast<uintptr_t>(w.s) % 8 != 0 || reinterpret_cast<uintptr_t>(w.z) % 4 != 0) return fail(FLUX_E_ALIGN, "%s: weights must be 16-byte aligned, scales 8, zero points 4", what);
    return FLUX_OK;
}

template <int GPC>
static void w4_unpack_launch(const flux_w4& w, void* out, hipStream_t st) {
    const int chunks = static_cast<int>((w.K + kW4Chunk - 1) / kW4Chunk);
    const int64_t tiles = (w.N + kW4Tile - 1) / kW4Tile * chunks;
    const dim3 grid(static_cast<unsigned>((tiles + 3) / 4));
#define CALL(ZERO) hipLaunchKernelGGL((w4_unpack_kernel<GPC, ZERO>), grid, dim3(256), 0, st, static_cast<const w4_u32x4*>(w.q), static_cast<const bf16_t*>(w.s), \
                                      static_cast<const uint8_t*>(w.z), static_cast<bf16_t*>(out), (int)w.N, (int)w.K, chunks, tiles)
    if (w.z) CALL(true); else CALL(false);
#undef CALL
}
static void w4_unpack_any(const flux_w4& w, void* out, hipStream_t st) {
    if (w.group == 32) w4_unpack_launch<4>(w, out, st);
    else if (w.group == 64) w4_unpack_launch<2>(w, out, st);
    else w4_unpack_launch<1>(w, out, st);
}

template <int GPC, bool ZERO>
static void w4_rows_launch(W4Params p, hipStream_t st) {
    const int tiles = (p.N + kW4Tile - 1) / kW4Tile;
    const bool few = tiles <= 256;   // no more than a row tile a CU
    // Up to 4 rows, f(x), and up to 8 rows of few outputs: x through registers. More row tiles a workgroup share the work on x, and leave CUs idle: us for one, two, three and four
    // of them at 3 x 9216 x 3072 with SiLU 10.0, 9.7, 8.1 and 9.2, 4 x 9216 11.8, 10.9, 8.6 and 10.2, 6 x 6144 (two are a workgroup a CU) 8.8 with two and 10.2 with three,
    // 1 x 18432 10.1, 11.8 and 15.9 with four. Eight parts of K pay where there are few outputs and many chunks (2 x 4096 x 8192 10.8 -> 7.7, 8 x 3072 x 3072 6.8 -> 5.6; 1 x
    // 18432 x 3072 10.1 -> 13.7) or many rows.
    if (p.M <= 4 || p.silu || (p.M <= 8 && few)) {
        const int rb = p.silu ? 8 : 16, held = std::min(p.M, rb) * (p.silu ? 2 : 1);
        p.slab = std::min({p.chunks, 64, 48 * 1024 / (held * kW4Chunk * 2) / 4 * 4});   // up to 48 KB of x, so that three workgroups share a CU
        auto call = [&](auto kernel, int nw, int ks) {
            const int bytes = std::max(held * (p.slab * kW4Chunk * 2 + 16), 1024 * nw * ks);
            hipLaunchKernelGGL(kernel, dim3((tiles + nw - 1) / nw, (p.M + rb - 1) / rb), dim3(64 * nw * ks), bytes, st, p);
        };
#define CALL(NW, KS) if (p.silu) call(w4_rows_kernel<GPC, ZERO, true, NW, KS>, NW, KS); else call(w4_rows_kernel<GPC, ZERO, false, NW, KS>, NW, KS)
        if (few && (p.chunks >= 32 || p.M > 4)) { CALL(1, 8); }
        else if (p.silu && p.M >= 3 && tiles > 512) call(w4_rows_kernel<GPC, ZERO, true, 3, 4>, 3, 4);
        else if (p.silu && p.M >= 3 && !few) call(w4_rows_kernel<GPC, ZERO, true, 2, 4>, 2, 4);
        else { CALL(1, 4); }
#undef CALL
        return;
    }
    // More: x fills the LDS of a CU at K = 3072, so workgroups run in rounds of 256. What a round takes there (measured at that K alone; with less of it several workgroups share a CU), us, by the rows and row tiles of a workgroup; the form
    // whose rounds take least: 16 x 9216 9.3 (16 rows, 4 tiles), 24 x 3072 8.5 (32 rows, 2 tiles), 24 x 12288 13.4 (32, 4), 64 x 12288 21.2 (64, 4; 24.8 with
    // 32, 4), 128 x 12288 29.2 (64, 8; 33.9 with 32, 4), 128 x 3072 12.4 (32, 4).
    struct Form { int rows, tiles; float us; };
    static const Form forms[] = {{16, 2, 6.5f}, {16, 4, 9.0f}, {32, 2, 8.5f}, {32, 4, 12.4f}, {64, 4, 19.5f}, {64, 8, 28.5f}};
    int best = 0;
    float best_us = 0.0f;
    for (int i = 0; i < 6; ++i) {
        const int64_t groups = static_cast<int64_t>((tiles + forms[i].tiles - 1) / forms[i].tiles) * ((p.M + forms[i].rows - 1) / forms[i].rows);
        const float us = static_cast<float>((groups + 255) / 256) * forms[i].us;
        if (i == 0 || us < best_us) { best = i; best_us = us; }
    }
    auto call = [&](auto kernel, int mt, int ntw, int nw, int ks) {
        const int held = std::min(p.M, 16 * mt), most = 152 * 1024;
        const int unit = std::max(4, ks);   // chunks: whole loads of 1 KB of a row, and as many for each part
        p.slab = (p.chunks + unit - 1) / unit * unit;
        if (held * (p.slab * kW4Chunk * 2 + 16) > most) p.slab = (most / 2 / held - 16) / (kW4Chunk * 2) / unit * unit;
        hipLaunchKernelGGL(kernel, dim3((tiles + nw * ntw - 1) / (nw * ntw), (p.M + 16 * mt - 1) / (16 * mt)), dim3(64 * nw * ks), w4_tiles_lds(p, held, (ks - 1) * nw * ntw * mt), st, p);
    };
#define CALL(MT, NTW, NW, KS, CW) call(w4_tiles_kernel<GPC, ZERO, MT, NTW, NW, KS, CW>, MT, NTW, NW, KS)
    switch (best) {
        case 0: CALL(1, 1, 2, 4, 6); break;
        case 1: CALL(1, 1, 4, 4, 6); break;
        case 2: CALL(2, 1, 2, 4, 6); break;
        case 3: CALL(2, 1, 4, 4, 6); break;
        case 4: CALL(4, 2, 2, 4, 3); break;
        default: CALL(4, 2, 4, 2, 3); break;
    }
#undef CALL
}

constexpr int kW4MostRows = 128;   // of the kernels that multiply whole numbers

// Beyond them: 16 outputs' tiles a wave of the kernel that unpacks weights between its products, 2 or 3, or 0 where they are laid out first. One round of workgroups, one a CU,
// that leaves less than half of the CUs idle is ahead of a pass that lays thousands of outputs' weights out. us, direct and laid out first: 256 x 9216 x 3072 33.1 and 41.1, 256 x 12288 x
// 3072 34.3 and 49.7, 512 x 9216 x 3072 41.4 and 49.8 (3 tiles), 256 x 18432 x 8192 96 and 171, 384 x 6144 x 8192 71.3 and 70.5 (144 workgroups). Fewer workgroups: 129 x 6144 x 3072 31.5 and
// 31.7 (96), 512 x 3072 x 3072 32.3 and 28.6 (96), 129 x 6144 x 8192 71 and 49; fewer outputs: 1000 x 3072 x 3072 35.2 and 34.0 (192), 640 x 3712 x 8192 72 and 60; two rounds: 1000 x 9216 x
// 3072 80 and 67, 512 x 18432 x 3072 83 and 80.
static int w4_product_tiles(const flux_linear_w4_args& a) {
    if (a.w.N < 4608 || a.ldx < a.w.K || a.ldx >= (int64_t{1} << 23)) return 0;   // (32-bit offsets within 128 rows)
    const int64_t row_blocks = (a.M + 127) / 128, two = row_blocks * ((a.w.N + 127) / 128), three = row_blocks * ((a.w.N + 191) / 192);
    return two < 144 ? 0 : two <= 256 ? 2 : three <= 256 ? 3 : 0;
}
template <int GPC, bool ZERO>
static void w4_product_launch(const W4Params& p, int nt, hipStream_t st) {
    const int row_blocks = (p.M + 127) / 128, blocks = row_blocks * ((p.N + 64 * nt - 1) / (64 * nt));
    const dim3 grid((blocks + 7) / 8 * 8);
    if (nt == 2) hipLaunchKernelGGL((w4_product_kernel<GPC, ZERO, 2>), grid, dim3(256), 4 * 128 * 256, st, p, row_blocks, blocks);
    else hipLaunchKernelGGL((w4_product_kernel<GPC, ZERO, 3>), grid, dim3(256), 4 * 128 * 256, st, p, row_blocks, blocks);
}

static flux_linear_args w4_linear(const flux_linear_w4_args& a, const void* w) {
    flux_linear_args l = {};
    l.A = a.x; l.W = w; l.bias = a.bias; l.Y = a.y;
    l.M = a.M; l.N = a.w.N; l.K = a.w.K;
    l.lda = a.ldx; l.ldw = a.w.K; l.ldy = a.ldy;
    l.split_n = a.w.N; l.act = a.act;
    return l;
}
static int64_t w4_weights_bytes(const flux_w4& w) { return (w.N * w.K * 2 + 255) / 256 * 256; }

}  // namespace flux

using namespace flux;

extern "C" int flux_serve_abi_version(void) { return FLUX_SERVE_ABI_VERSION; }

extern "C" int flux_w4_unpack(const flux_w4* w, void* out, void* stream) {
    if (!w) return fail(FLUX_E_NULL, "flux_w4_unpack: null args");
    int rc = w4_check("flux_w4_unpack", *w);
    if (rc != FLUX_OK || w->N == 0 || w->K == 0) return rc;
    rc = w4_pointers("flux_w4_unpack", *w);
    if (rc != FLUX_OK) return rc;
    if (!out || !aligned16(out)) return fail(FLUX_E_ALIGN, "flux_w4_unpack: out must be 16-byte aligned memory");
    if ((w->N + 15) / 16 * ((w->K + 127) / 128) > int64_t{0x7fffffff} / 64) return fail(FLUX_E_SHAPE, "flux_w4_unpack: too many weights");
    w4_unpack_any(*w, out, static_cast<hipStream_t>(stream));
    return check_launch("flux_w4_unpack");
}

extern "C" int64_t flux_linear_w4_workspace_bytes(const flux_linear_w4_args* a) {
    if (!a || a->M <= kW4MostRows || w4_check("flux_linear_w4_bf16", a->w) != FLUX_OK || a->w.N == 0 || a->w.K == 0 || w4_product_tiles(*a) != 0) return 0;
    const flux_linear_args l = w4_linear(*a, a->w.q);
    return w4_weights_bytes(a->w) + flux_linear_workspace_bytes(&l);
}

extern "C" int flux_linear_w4_bf16(const flux_linear_w4_args* a, void* ws, int64_t ws_bytes, void* stream) {
    const char* const what = "flux_linear_w4_bf16";
    if (!a) return fail(FLUX_E_NULL, "%s: null args", what);
    int rc = w4_check(what, a->w);
    if (rc != FLUX_OK) return rc;
    if (a->M < 0 || a->M > 0x7fffffff / 64) return fail(FLUX_E_SHAPE, "%s: bad number of rows %lld", what, (long long)a->M);
    if (a->act != FLUX_ACT_NONE && a->act != FLUX_ACT_GELU_TANH) return fail(FLUX_E_UNSUPPORTED, "%s: activation %d", what, a->act);
    if (a->in_act != FLUX_ACT_NONE && a->in_act != FLUX_ACT_SILU) return fail(FLUX_E_UNSUPPORTED, "%s: input activation %d", what, a->in_act);
    if (a->in_act != FLUX_ACT_NONE && a->M > kW4SiluRows) return fail(FLUX_E_UNSUPPORTED, "%s: the input activation is for at most %d rows", what, kW4SiluRows);
    if (a->M == 0 || a->w.N == 0) return FLUX_OK;
    if (a->w.K == 0) return fail(FLUX_E_SHAPE, "%s: no columns to sum over", what);
    rc = w4_pointers(what, a->w);
    if (rc != FLUX_OK) return rc;
    if (!a->x || !a->y) return fail(FLUX_E_NULL, "%s: null pointer", what);
    if (a->ldy < a->w.N && a->M > 1) return fail(FLUX_E_SHAPE, "%s: rows of y overlap", what);
    if (!aligned16(a->x) || (a->M > 1 && a->ldx % 8 != 0)) return fail(FLUX_E_ALIGN, "%s: x must be 16-byte aligned, its row stride a multiple of 8", what);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int nt = a->M > kW4MostRows ? w4_product_tiles(*a) : 0;
    if (a->M > kW4MostRows && nt == 0) {
        const int64_t weights = w4_weights_bytes(a->w), need = flux_linear_w4_workspace_bytes(a);
        if (!ws || reinterpret_cast<uintptr_t>(ws) % 256 != 0 || ws_bytes < need) return fail(FLUX_E_SHAPE, "%s: needs %lld bytes of 256-byte aligned workspace", what, (long long)need);
        rc = flux_w4_unpack(&a->w, ws, stream);
        if (rc != FLUX_OK) return rc;
        const flux_linear_args l = w4_linear(*a, ws);
        return flux_linear_bf16_ws(&l, need > weights ? static_cast<char*>(ws) + weights : nullptr, need - weights, stream);
    }
    W4Params p = {static_cast<const bf16_t*>(a->x), static_cast<const w4_u32x4*>(a->w.q), static_cast<const bf16_t*>(a->w.s), static_cast<const uint8_t*>(a->w.z),
                  static_cast<const bf16_t*>(a->bias), static_cast<bf16_t*>(a->y), a->M > 1 ? a->ldx : 0, a->M > 1 ? a->ldy : 0,
                  static_cast<int>(a->M), static_cast<int>(a->w.N), static_cast<int>(a->w.K), static_cast<int>((a->w.K + kW4Chunk - 1) / kW4Chunk), 0, a->act, a->in_act == FLUX_ACT_SILU};
#define CALL(GPC) if (nt != 0 && p.z) w4_product_launch<GPC, true>(p, nt, st); else if (nt != 0) w4_product_launch<GPC, false>(p, nt, st); \
                  else if (p.z) w4_rows_launch<GPC, true>(p, st); else w4_rows_launch<GPC, false>(p, st)
    if (a->w.group == 32) { CALL(4); }
    else if (a->w.group == 64) { CALL(2); }
    else { CALL(1); }
#undef CALL
    return check_launch(what);
}
