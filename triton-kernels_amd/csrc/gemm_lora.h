// Low-rank adapters beside a shared projection: what the kernels add to the sums of a tile before its epilogue.
//
//   y[m] = act(x[m] W^T + bias + s_i (x[m] a_i^T) b_i^T),  i = the adapter of row m's request
//
// Two launches. The first one (lora_low_kernel) works out low[m] = s_i x[m] a_i^T, a few values a row, in fp32 and leaves it as the bf16 numbers that
// the matrix instructions of the second take: the nearest one and the nearest to what that leaves over, 2^-16 of the value off. (One number
// alone is 2^-8 of the adapter's terms off, not of y: where they cancel the rest of y, it is what y's error consists of.) The second one is
// the product with W as ever; when a tile's sums are complete, low b_i^T is multiplied onto them from registers, K = 32 a step: both numbers of 16
// ranks side by side or, beyond rank 16, both of 32 ranks one after the other onto the same columns of b. So y
// is written once and rounded once, and the adapter costs a few times rank / K of the product's own time.
//
// Measured, medians in us (the product with W by itself, then the first launch, then the second): 13008 x 12288 x 3072 rank 16 with GELU 738, 20.6 and 745;
// 4608 x 9216 x 3072 rank 64 182, 16.6 and 207 to 223 by the power limit; 517 x 2048 x 2048 rank 32, two or three adapters in a tile of rows, 12.0, 5.0
// and 14 to 15; six rows, 6144 x 1024 rank 16, 7.3, 4.0 and 9.0. Bound by the matrix instructions, for few rows by W from HBM and two dependent launches.
// Adapters mixed by row cost a pass over x and a step of the tail each: 517 rows of 16 mixed adapters 9.4 and 18.2. Operands without 16-byte rows take a
// kernel for which speed was not sought: 517 x 2048 x 2047 19.0 and 6733 (the product by itself 7671).
#pragma once

#include "gemm_common.h"
#include "gemm_rows.h"

namespace flux {

// How low lies in memory. For the tiles as a wave loads it: of 16 rows and a step of 32, one KB of first numbers, lane l's eight of row l % 16 at l * 16
// bytes, and one of second numbers (planes 2); up to rank 16 the second numbers are the step's other 16 (planes 1), and beyond it, in a
// workspace that has no room for them, there are none (planes 1). (By rows, a load's 64 lanes are 64 requests to the address unit: 4608 x 9216 x 3072, rank
// 64, both numbers: 228 us for 222.) For the kernels without matrix instructions fp32 by rows (planes 0).
struct LoraPlace {
    int rank, width, planes;   // width: rank rounded up to whole steps of 32

    __host__ __device__ bool beside() const { return planes == 1 && rank <= 16; }
    __host__ __device__ int pitch() const { return (rank + 15) / 16 * 16; }   // planes 0: values from row to row
    // Otherwise: where rows 16 n .. and the step of slot k begin.
    __host__ __device__ int64_t block(int64_t n, int k) const { return (n * (width / 32) + k / 32) * planes * 512; }
    __host__ __device__ int64_t bytes(int64_t rows) const { return planes == 0 ? rows * pitch() * 4 : block((rows + 15) / 16, 0) * 2; }
};

struct LoraTail {
    const void* low;       // LoraPlace: zero from the rank on
    const int* owner;      // [M]: the row's adapter, -1: none
    const bf16_t* b;       // [adapters][N][rank]
    LoraPlace at;
    int vec;               // rows of b may be read so many values at a time: 8, 4 or 1

    // planes 0
    __device__ __forceinline__ float value(int64_t m, int r) const { return static_cast<const float*>(low)[m * at.pitch() + r]; }

    // Adds to the fragment rows of a wave: rows m0 .. of the product, columns n0 ... The adapters among the wave's rows are taken one after the
    // other in rising order, each with one read of its columns of b; rows of another adapter count as zeros, and so do values past the rank's end. 0 * inf
    // would still reach them, so what is not finite in b is taken out of the product and reaches its own rows by itself (not_finite_terms). (The sums are
    // touched by matrix instructions only: choosing between old and new sums by row, with vector instructions, spilled 600 registers of the
    // 256-wide tile.)
    // A step's operands: columns of b of one adapter and the rows' low, 32 values each.
    template <int ROWS, int FN>
    struct Step {
        u32x4 b[FN], low[ROWS], rest[ROWS];
    };
    template <int ROWS, int FN>
    __device__ __forceinline__ void load_b(Step<ROWS, FN>& to, int a, int k, int n0, const GemmParams& p) const {
        // Scalar bases and 32-bit offsets: sixteen pointers would not fit the registers. Past the rank's end: values of the same row of b
        // again, which meet zeros of low.
        const int rank = this->at.rank, lane = threadIdx.x & 63, frow = lane & 15, slot = k + (lane >> 4) * 8, at = this->at.beside() ? slot & 15 : slot;
        const bf16_t* const col = b + static_cast<int64_t>(a) * p.N * rank;
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
    }
    // Whether fragment rows without rows of a step's adapter are left out. us with and without: 8192 x 1024 x 1024, rank 64, runs of 12 rows, four
    // fragment rows a wave 63 and 71; 4608 x 9216 x 3072, rank 64, one adapter, nine of them 230 and 226.
    template <int ROWS> static constexpr bool kSkip = ROWS > 1 && ROWS <= 4;
    // of: the fragment rows that are wanted. (Past M: the last rows' block again.)
    template <int ROWS, int FN>
    __device__ __forceinline__ void load_low(Step<ROWS, FN>& to, uint32_t of, int k, int m0, const GemmParams& p) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if (kSkip<ROWS> && !(of >> i & 1u)) continue;
            const u32x4* const from = reinterpret_cast<const u32x4*>(static_cast<const bf16_t*>(low) + at.block(min(m0 / 16 + i, (p.M - 1) / 16), k)) + lane;
            to.low[i] = from[0];
            if (at.planes == 2) to.rest[i] = from[64];
        }
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
    // one value of every line of the first step's operands for the first adapters, so that they are in the L2 when it comes to them (touch).
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
            for (int i = 0; i < (FN + 3) / 4; ++i) to.b[t][i] = b[(static_cast<int64_t>(last) * p.N + min(n0 + min(i * 64 + lane, FN * 16 - 1), p.N - 1)) * at.rank];
            if (t + 1 < kTouch) a = a == kNone ? a : behind(to.own, a);
        }
#pragma unroll
        for (int i = 0; i < (ROWS + 3) / 4; ++i) {   // (eight lines of either plane)
            const int line = min(i * 64 + lane, ROWS * 16 - 1);
            to.low[i] = *reinterpret_cast<const uint32_t*>(static_cast<const bf16_t*>(low) + at.block(min(m0 / 16 + (line >> 4), (p.M - 1) / 16), 0) + (line & (at.planes == 2 ? 15 : 7)) * 64);
        }
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
        Step<ROWS, FN> s;
        uint32_t mine = ~0u;   // fragment rows that hold rows of the adapter: the others have no part in its products
        bool first = true;
        for (int k = 0;;) {
            if (kSkip<ROWS> && k == 0) {
                mine = 0;
#pragma unroll
                for (int i = 0; i < ROWS; ++i) mine |= __ballot(own[i] == a) != 0 ? 1u << i : 0u;
            }
            load_b(s, a, k, n0, p);
            // (low is the same for every adapter: where one step holds the rank it stays in its registers)
            if (first || at.width > 32) load_low(s, at.width > 32 ? mine : ~0u, k, m0, p);
            first = false;
            __builtin_amdgcn_sched_barrier(0);   // the loads stay in front of the products
            uint32_t bad = 0;
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) bad |= not_finite(s.b[j][e]);
            if (__ballot((bad & 0x80008000u) != 0) != 0) not_finite_terms(acc, s, own, a, k);
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
                if (!kSkip<ROWS> || (mine >> i & 1u)) multiply(acc, s.b, s.low[i], i, own[i] == a);
            if (at.planes == 2) {
#pragma unroll
                for (int i = 0; i < ROWS; ++i)
                    if (!kSkip<ROWS> || (mine >> i & 1u)) multiply(acc, s.b, s.rest[i], i, own[i] == a);
            }
            k += 32;
            if (k >= at.width) {
                k = 0;
                a = behind(own, a);
                if (a == kNone) break;
            }
        }
    }

    template <int ROWS, int FN>
    static __device__ __forceinline__ void multiply(f32x4 (&acc)[ROWS][FN], const u32x4 (&w)[FN], const u32x4& row, int i, bool own) {
        const bf16x8 x = __builtin_bit_cast(bf16x8, own ? row : u32x4{0, 0, 0, 0});
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w[j]), x, acc[i][j], 0, 0, 0);
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
    // time, so that terms of one instruction do not cancel before they are rounded, and NaN and zero are of either sign: +inf - inf. b itself is
    // left with 1 of its sign (which keeps an infinite or NaN low what it is, and second numbers without effect beside an infinity).
    template <int ROWS, int FN>
    __device__ __forceinline__ void not_finite_terms(f32x4 (&acc)[ROWS][FN], Step<ROWS, FN>& s, const int (&own)[ROWS], int a, int k) const {
        const int rank = this->at.rank, at = k + (lane_again() >> 4) * 8;
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

// The sums are in accumulation registers from here on: in front of the loop over K and behind it. Without the second the compiler settles the whole
// kernel's registers by what happens behind the loop: 360 moves between accumulation and ordinary registers a slab inside it, 1071 us for 814 at
// 13008 x 12288 x 3072. Without the first the tiles of 7 x 8 and 7 x 9 fragments wait for what they touch and put it aside.
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
    float low[MM];
    bf16_t b[kGemvCols][MM];
    int64_t row_b[kGemvCols][MM];

    __device__ __forceinline__ void begin() {
        typedef const __attribute__((address_space(4))) int* scalar;
#pragma unroll
        for (int m = 0; m < MM; ++m) own[m] = ((scalar)(reinterpret_cast<uintptr_t>(t.owner)))[m];
    }
    __device__ __forceinline__ void request(int n0, int lane, const GemmParams& p) {
        const int r = lane < t.at.rank ? lane : 0;
#pragma unroll
        for (int m = 0; m < MM; ++m) {
            low[m] = t.value(m, r);
#pragma unroll
            for (int c = 0; c < kGemvCols; ++c) {
                row_b[c][m] = (static_cast<int64_t>(max(own[m], 0)) * p.N + min(n0 + c, p.N - 1)) * t.at.rank;
                b[c][m] = t.b[row_b[c][m] + r];
            }
        }
    }
    __device__ __forceinline__ void add(float (&acc)[kGemvCols][MM], int lane) {
#pragma unroll
        for (int m = 0; m < MM; ++m)
#pragma unroll
            for (int c = 0; c < kGemvCols; ++c) acc[c][m] += own[m] >= 0 && lane < t.at.rank ? low[m] * bf2f(b[c][m]) : 0.0f;
        for (int r = 64 + lane; r < t.at.rank; r += 64)
#pragma unroll
            for (int m = 0; m < MM; ++m) {
                const float l = t.value(m, r);
#pragma unroll
                for (int c = 0; c < kGemvCols; ++c) acc[c][m] += own[m] >= 0 ? l * bf2f(t.b[row_b[c][m] + r]) : 0.0f;
            }
    }
};

// The tail of a launch of tiles whose rows begin `rows`, a multiple of 16, further on.
inline LoraTail tail_behind(LoraTail t, int64_t rows) {
    t.low = static_cast<const bf16_t*>(t.low) + t.at.block(rows / 16, 0);
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
    void* low; int* owner;
    LoraPlace at;
    int64_t lda, rows_per_request;
    int M, K, adapters;
    int wide_ids;      // 1: adapter is int64
    int vec;           // 1: x and a may be read 16 bytes at a time
};
void launch_lora_low(const LoraLow& p, hipStream_t st);

}  // namespace flux
