// Low-rank adapters beside a shared projection: what the kernels add to the sums of a tile before its epilogue.
//
//   y[m] = act(x[m] W^T + bias + s_i (x[m] a_i^T) b_i^T),  i = the adapter of row m's request
//
// Two launches. The first one (lora_low_kernel) works out low[m] = s_i x[m] a_i^T, a few values a row, and rounds it to bf16, which the matrix
// instructions of the second take: an error of 2^-9 of the adapter's own terms, below what y's rounding to bf16 leaves. The second one is
// the product with W as ever; when a tile's sums are complete, low b_i^T is multiplied onto them from registers, K = 32 of the rank a step. So y
// is written once and rounded once, and the adapter costs rank / K of the product's own time.
//
// Measured, us (the product with W by itself, then the first launch, then the second): 13008 x 12288 x 3072 rank 16 with GELU 738, 15.8 and 738; 4608 x 9216 x
// 3072 rank 64 182, 15.5 and 195; 517 x 2048 x 2048 rank 32, two or three adapters in a tile of rows, 11.7, 4.9 and 14.3; six rows, 6144 x 1024 rank 16, 7.3,
// 3.7 and 8.8. Bound by the matrix instructions, for few rows by W from HBM and two dependent launches. Adapters mixed by row cost a pass
// over x and a step of the tail each: 517 rows of 16 mixed adapters 8.8 and 17.5.
#pragma once

#include "gemm_common.h"
#include "gemm_rows.h"

namespace flux {

struct LoraTail {
    const bf16_t* low;     // [M][width]: zero from the rank on
    const int* owner;      // [M]: the row's adapter, -1: none
    const bf16_t* b;       // [adapters][N][rank]
    int rank, width;       // width: rank rounded up to whole steps of 32
    int vec;               // rows of b may be read so many values at a time: 8, 4 or 1

    // Adds to the fragment rows of a wave: rows m0 .. of the product, columns n0 ... The adapters among the wave's rows are taken one after the
    // other in rising order, each with one read of its columns of b; rows of another adapter count as zeros, and so do values past the rank's end. 0 * inf
    // would still reach them, so what is not finite in b is taken out of the product and reaches its own rows by itself (not_finite_terms). (The sums are
    // touched by matrix instructions only: choosing between old and new sums by row, with vector instructions, spilled 600 registers of the
    // 256-wide tile.)
    // A step's operands: columns of b of one adapter and the rows' low, 32 values each.
    template <int ROWS, int FN>
    struct Step {
        u32x4 b[FN], low[ROWS];
    };
    template <int ROWS, int FN>
    __device__ __forceinline__ void load(Step<ROWS, FN>& to, int a, int k, int m0, int n0, const GemmParams& p) const {
        // Scalar bases and 32-bit offsets: sixteen pointers would not fit the registers. Past the rank's end: values of the same row of b
        // again, which meet zeros of low.
        const int frow = threadIdx.x & 15, at = k + ((threadIdx.x & 63) >> 4) * 8;
        const bf16_t* const col = b + static_cast<int64_t>(a) * p.N * rank;
        const bf16_t* const row = low + static_cast<int64_t>(m0) * width;
        auto column = [&](int j) { return static_cast<uint32_t>(min(n0 + j * 16 + frow, p.N - 1)) * rank; };
        if (vec == 8) {
#pragma unroll
            for (int j = 0; j < FN; ++j) to.b[j] = *reinterpret_cast<const u32x4*>(col + (column(j) + (at < rank ? at : 0)));
        } else if (vec == 4) {
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const u32x2 lo = *reinterpret_cast<const u32x2*>(col + (column(j) + (at < rank ? at : 0)));
                const u32x2 hi = *reinterpret_cast<const u32x2*>(col + (column(j) + (at + 4 < rank ? at + 4 : 0)));
                to.b[j] = u32x4{lo.x, lo.y, hi.x, hi.y};
            }
        } else {
#pragma unroll
            for (int j = 0; j < FN; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) to.b[j][e] = col[column(j) + min(at + 2 * e, rank - 1)] | static_cast<uint32_t>(col[column(j) + min(at + 2 * e + 1, rank - 1)]) << 16;
                asm volatile("" ::: "memory");   // (a column at a time: eight registers of loads)
            }
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) to.low[i] = *reinterpret_cast<const u32x4*>(row + (static_cast<uint32_t>(min(i * 16 + frow, p.M - 1 - m0)) * width + at));
    }

    static constexpr int kNone = 0x7fffffff;
    // The next adapter behind `last` of a wave's rows.
    template <int ROWS>
    static __device__ __forceinline__ int behind(const int (&own)[ROWS], int last) {
        int next = kNone;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) next = own[i] > last ? min(next, own[i]) : next;
        return first_of_rows(next);
    }

    // What a wave asks for before its sums are complete: the adapters of its rows, in front of everything else (begin), and behind its first slabs
    // one value of every row of the first step's operands for the first adapters, so that they are in the L2 when it comes to them (touch).
    // Requested behind the loop over K alone, a tile waits for memory three times in a row with nothing beside it. (The operands themselves do not
    // fit beside the loop's: with them the 256-wide tile moved 450 registers a slab.)
    static constexpr int kTouch = 3;
    // Not for the 192 x 192 tile, whose two groups of waves have no registers to spare beside the loop's.
    template <int ROWS, int FN> static constexpr bool kAhead = !(ROWS == 3 && FN == 6);
    template <int ROWS, int FN>
    struct Ahead {
        int own[ROWS];
        uint32_t low[(ROWS + 3) / 4], b[kTouch][(FN + 3) / 4];
    };
    template <int ROWS, int FN>
    __device__ __forceinline__ void begin(Ahead<ROWS, FN>& to, int m0, const GemmParams& p) const {
        if constexpr (kAhead<ROWS, FN>) owners(to.own, m0, p);
    }
    template <int ROWS>
    __device__ __forceinline__ void owners(int (&own)[ROWS], int m0, const GemmParams& p) const {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) own[i] = owner[min(m0 + i * 16 + static_cast<int>(threadIdx.x & 15), p.M - 1)];
    }
    template <int ROWS, int FN>
    __device__ __forceinline__ void touch(Ahead<ROWS, FN>& to, int m0, int n0, const GemmParams& p) const {
        if constexpr (!kAhead<ROWS, FN>) return;
        const int lane = threadIdx.x & 63;
        int a = behind(to.own, -1), last = 0;
#pragma unroll
        for (int t = 0; t < kTouch; ++t) {   // (fewer adapters than that: the last one again)
            last = a == kNone ? last : a;
#pragma unroll
            for (int i = 0; i < (FN + 3) / 4; ++i) to.b[t][i] = b[(static_cast<int64_t>(last) * p.N + min(n0 + min(i * 64 + lane, FN * 16 - 1), p.N - 1)) * rank];
            if (t + 1 < kTouch) a = a == kNone ? a : behind(to.own, a);
        }
#pragma unroll
        for (int i = 0; i < (ROWS + 3) / 4; ++i) to.low[i] = *reinterpret_cast<const uint32_t*>(low + static_cast<int64_t>(min(m0 + min(i * 64 + lane, ROWS * 16 - 1), p.M - 1)) * width);
    }

    template <int ROWS, int FN>
    __device__ __forceinline__ void finish(f32x4 (&acc)[ROWS][FN], Ahead<ROWS, FN>& have, int m0, int n0, const GemmParams& p) const {
        if constexpr (kAhead<ROWS, FN>) {
#pragma unroll
            for (uint32_t& t : have.low) asm volatile("" ::"v"(t));
#pragma unroll
            for (auto& t : have.b)
#pragma unroll
                for (uint32_t& v : t) asm volatile("" ::"v"(v));
        } else {
            owners(have.own, m0, p);
        }
        if (m0 < p.M && n0 < p.N) finish(acc, have.own, m0, n0, p);
    }
    template <int ROWS, int FN>
    __device__ __forceinline__ void finish(f32x4 (&acc)[ROWS][FN], const int (&own)[ROWS], int m0, int n0, const GemmParams& p) const {
        int a = behind(own, -1);
        if (a == kNone) return;
        bool same = true;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) same = same && own[i] == a;
        const bool all = __ballot(same) == ~uint64_t{0};
        Step<ROWS, FN> s;
        for (int k = 0;;) {
            load(s, a, k, m0, n0, p);
            __builtin_amdgcn_sched_barrier(0);   // the loads stay in front of the products
            if (!all) {
#pragma unroll
                for (int i = 0; i < ROWS; ++i) s.low[i] = own[i] == a ? s.low[i] : u32x4{0, 0, 0, 0};
            }
            uint32_t bad = 0;
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) bad |= not_finite(s.b[j][e]);
            if (__ballot((bad & 0x80008000u) != 0) != 0) not_finite_terms(acc, s, own, a, k);
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, s.b[j]), __builtin_bit_cast(bf16x8, s.low[i]), acc[i][j], 0, 0, 0);
            k += 32;
            if (k >= width) {
                k = 0;
                a = behind(own, a);
                if (a == kNone) break;
            }
        }
    }

    // Of the halves of a word, in their top bits: infinite or NaN, mantissa not zero, value not zero; and all ones where the top bit is set.
    static __device__ __forceinline__ uint32_t not_finite(uint32_t w) { return (w & 0x7f807f80u) + 0x00800080u; }
    static __device__ __forceinline__ uint32_t fraction(uint32_t w) { return ((w & 0x007f007fu) + 0x007f007fu) << 8; }
    static __device__ __forceinline__ uint32_t not_zero(uint32_t w) { return (w & 0x7fff7fffu) + 0x7fff7fffu; }
    static __device__ __forceinline__ uint32_t filled(uint32_t top) {
        top &= 0x80008000u;
        return (top << 1) - (top >> 15);
    }

    // The lane's number, worked out anew: a register that is live across the loop over K is one too many in the 192 x 192 tile.
    static __device__ __forceinline__ int lane_again() { return static_cast<int>(__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u))); }
    static __device__ __forceinline__ int lane(int) { return lane_again(); }

    // What is not finite in a step's columns of b, for the rows of adapter a, as low * b would have it: +inf and -inf by the signs, NaN where b is NaN or
    // low is zero. Both factors become 3.4e38 of their signs, whose product is infinite, and zero everywhere else; one combination of signs at a
    // time, so that terms of one instruction do not cancel before they are rounded, and NaN and zero are of either sign: +inf - inf. b itself is left with 1 of its sign
    // (which keeps an infinite or NaN low what it is).
    template <int ROWS, int FN>
    __device__ __forceinline__ void not_finite_terms(f32x4 (&acc)[ROWS][FN], Step<ROWS, FN>& s, const int (&own)[ROWS], int a, int k) const {
        const int at = k + (lane_again() >> 4) * 8;
#pragma unroll 1
        for (int signs = 0; signs < 4; ++signs) {
            // (the words count as new ones in every turn: what is worked out from them is not kept in registers over the turns)
#pragma unroll
            for (int j = 0; j < FN; ++j) asm volatile("" : "+v"(s.b[j]));
#pragma unroll
            for (int i = 0; i < ROWS; ++i) asm volatile("" : "+v"(s.low[i]));
            const uint32_t sign_b = (signs & 1) ? 0x80008000u : 0u, sign_low = (signs & 2) ? 0x80008000u : 0u;
            u32x4 x[ROWS];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t in = (at + 2 * e < rank ? 0x7f7fu : 0u) | (at + 2 * e + 1 < rank ? 0x7f7f0000u : 0u), with_sign = in | ((in << 1) & sign_low);
#pragma unroll
                for (int i = 0; i < ROWS; ++i) x[i][e] = own[i] == a ? filled((s.low[i][e] ^ ~sign_low) | ~not_zero(s.low[i][e])) & with_sign : 0u;
            }
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                u32x4 huge;
#pragma unroll
                for (int e = 0; e < 4; ++e) huge[e] = filled(not_finite(s.b[j][e]) & ((s.b[j][e] ^ ~sign_b) | fraction(s.b[j][e]))) & (0x7f7f7f7fu | sign_b);
#pragma unroll
                for (int i = 0; i < ROWS; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, huge), __builtin_bit_cast(bf16x8, x[i]), acc[i][j], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);   // (a column at a time)
            }
        }
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = s.b[j][e], n = filled(not_finite(w));
                s.b[j][e] = (w & (~n | 0x80008000u)) | (n & 0x3f803f80u);
            }
    }

    // The smallest value of the wave's 16 rows (lanes 16 apart hold the same row), as a scalar.
    static __device__ __forceinline__ int first_of_rows(int v) {
        v = min(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xf, 0xf, true));    // lane ^ 1
        v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xf, 0xf, true));    // lane ^ 2
        v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xf, 0xf, true));   // mirrored within 8
        v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xf, 0xf, true));   // mirrored within 16
        return __builtin_amdgcn_readfirstlane(v);
    }
};

// The sums are in accumulation registers from here on. Without it the compiler settles the whole kernel's registers by what happens behind the loop
// over K: 360 moves between accumulation and ordinary registers a slab inside it, 1071 us for 814 at 13008 x 12288 x 3072.
template <int ROWS, int FN>
__device__ __forceinline__ void hold(f32x4 (&acc)[ROWS][FN]) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) asm volatile("" : "+a"(acc[i][j]));
}

// The same for row vectors (gemm_rows.h): lane l adds the products of the rank's values l, l + 64, ... to its share of a sum. The adapters' numbers come
// through the scalar cache and the first 64 values behind the first vectors of W, which so wait for nothing.
template <int MM>
struct LoraRowTail {
    LoraTail t;
    int own[MM];
    bf16_t low[MM], b[kGemvCols][MM];
    int64_t row_b[kGemvCols][MM];

    __device__ __forceinline__ void begin() {
        typedef const __attribute__((address_space(4))) int* scalar;
#pragma unroll
        for (int m = 0; m < MM; ++m) own[m] = ((scalar)(reinterpret_cast<uintptr_t>(t.owner)))[m];
    }
    __device__ __forceinline__ void request(int n0, int lane, const GemmParams& p) {
        const int r = lane < t.rank ? lane : 0;
#pragma unroll
        for (int m = 0; m < MM; ++m) {
            low[m] = t.low[static_cast<int64_t>(m) * t.width + r];
#pragma unroll
            for (int c = 0; c < kGemvCols; ++c) {
                row_b[c][m] = (static_cast<int64_t>(max(own[m], 0)) * p.N + min(n0 + c, p.N - 1)) * t.rank;
                b[c][m] = t.b[row_b[c][m] + r];
            }
        }
    }
    __device__ __forceinline__ void add(float (&acc)[kGemvCols][MM], int lane) {
#pragma unroll
        for (int m = 0; m < MM; ++m)
#pragma unroll
            for (int c = 0; c < kGemvCols; ++c) acc[c][m] += own[m] >= 0 && lane < t.rank ? bf2f(low[m]) * bf2f(b[c][m]) : 0.0f;
        for (int r = 64 + lane; r < t.rank; r += 64)
#pragma unroll
            for (int m = 0; m < MM; ++m) {
                const float l = bf2f(t.low[static_cast<int64_t>(m) * t.width + r]);
#pragma unroll
                for (int c = 0; c < kGemvCols; ++c) acc[c][m] += own[m] >= 0 ? l * bf2f(t.b[row_b[c][m] + r]) : 0.0f;
            }
    }
};

// The tail of a launch whose rows begin `rows` further on.
inline LoraTail tail_behind(LoraTail t, int64_t rows) {
    t.low += rows * t.width;
    t.owner += rows;
    return t;
}

void launch_lora_square(const GemmSet& g, const LoraTail& tail, hipStream_t st);
void launch_lora_rect(int fm, int fn, const GemmSet& g, const LoraTail& tail, hipStream_t st);
void launch_lora_pair(int fm, int fn, const GemmSet& g, int splits, float* partial, const LoraTail& tail, hipStream_t st);
void launch_lora_rows(const GemmParams& p, const LoraTail& tail, hipStream_t st);
void launch_lora_scalar(const GemmParams& p, const LoraTail& tail, hipStream_t st);

// The first launch: low and owner.
struct LoraLow {
    const bf16_t* x; const bf16_t* a; const void* adapter; const float* scaling;
    bf16_t* low; int* owner;
    int64_t lda, rows_per_request;
    int M, K, rank, width, adapters;
    int wide_ids;      // 1: adapter is int64
    int vec;           // 1: x and a may be read 16 bytes at a time
};
void launch_lora_low(const LoraLow& p, hipStream_t st);

}  // namespace flux
