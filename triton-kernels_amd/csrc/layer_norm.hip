// Layer norm with weights and its backward pass.
//
//   h = (x - mean) rstd,  y = h w + b;   g = dy w,  dx = rstd (g - mean(g) - h mean(g h)),  dw = sum_rows dy h,  db = sum_rows dy
//
// About 8 operations a value forward and 15 backward against 4 and 6 bytes (bf16): bound by HBM. So a row crosses it once in each direction:
// it is held in registers by T adjacent lanes (T = 16, 32 or whole waves up to 1024), ITER vectors of 16 bytes a lane, and its two sums are
// a DPP butterfly inside a wave and one exchange through LDS between the waves of a longer row. Rows that are not 16-byte
// addressable are held the same way, an element at a time (VEC = 1). Only rows beyond 1024 lanes are read again, from the caches.
//
// us of the kernels alone (bytes at 5.1 TB/s, a large copy's rate): [4608, 3072] bf16 forward 12.8 (11.1), backward 24.6 (16.6) and 4.0 for the sums of
// the parts; [3, 4336, 3072] bf16 with a weight for each batch element 31.2 (31.2), 55.6 (46.8) and 4.0; [4004, 1024] fp32 8.8 (6.4), 13.2 (9.6)
// and 3.8; 77 rows of 768 3.5, a launch, and 5.2.
#include "common.h"
#include "../../include/flux_hip_tune.h"
#include <algorithm>
#include <initializer_list>
#include <utility>

namespace flux {

constexpr int kLnMost = 1024;     // threads of a workgroup at most

// Sum over T adjacent lanes, T >= 16 uniform over the workgroup: within a wave.
__device__ __forceinline__ float lanes_sum(float v, int T) {
    v = group_sum<16>(v);
    if (T > 16) v += __shfl_xor(v, 16, 64);
    if (T > 32) v += __shfl_xor(v, 32, 64);
    return v;
}

// LDS traffic of the wave is done, then the workgroup's barrier; loads from memory stay in flight across it.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Two sums over T lanes at once. T > 64: the T / 64 waves of the row exchange theirs through `box` (16 waves x 2) and add them in order.
// Calls alternate between two boxes, so that one barrier a call is enough.
__device__ __forceinline__ void row_sums(float& a, float& b, int T, float (*box)[2]) {
    a = lanes_sum(a, T);
    b = lanes_sum(b, T);
    if (T <= 64) return;
    const int wave = threadIdx.x >> 6, waves = T >> 6, first = wave / waves * waves;
    if ((threadIdx.x & 63) == 0) {
        box[wave][0] = a;
        box[wave][1] = b;
    }
    lds_barrier();
    a = b = 0.0f;
    for (int i = 0; i < waves; ++i) {
        a += box[first + i][0];
        b += box[first + i][1];
    }
}

// The packed words are taken to be new ones from here on: what was unpacked from them is worked out again and not kept.
template <typename P> __device__ __forceinline__ void forget(P& p) {
    if constexpr (sizeof(p.w[0]) == 4) {
#pragma unroll
        for (auto& w : p.w) asm volatile("" : "+v"(w));
    }
}

// VEC elements as they lie in memory: whole 16-byte accesses, or one element. bf16 pairs stay packed in their words: element arrays that
// live across a loop take a register each (the backward kernel of 24 columns a lane spilled 143 registers that way).
template <typename T, int VEC> struct Pack;
template <> struct Pack<bf16_t, 8> {
    uint32_t w[4];
    __device__ __forceinline__ float at(int e) const { return __uint_as_float((e & 1) ? (w[e / 2] & 0xffff0000u) : (w[e / 2] << 16)); }
    __device__ __forceinline__ void set2(int e, float a, float b) {
        typedef float f32x2_t __attribute__((ext_vector_type(2)));
        typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
        const f32x2_t v = {a, b};
        w[e / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
    }
};
template <int VEC> struct Pack<float, VEC> {
    float w[VEC];
    __device__ __forceinline__ float at(int e) const { return w[e]; }
    __device__ __forceinline__ void set2(int e, float a, float b) { w[e] = a; w[e + 1] = b; }
};
template <> struct Pack<bf16_t, 1> {
    bf16_t w[1];
    __device__ __forceinline__ float at(int) const { return bf2f(w[0]); }
};
// ONCE: with the non-temporal hint.
template <typename T, int VEC, bool ONCE = false> __device__ __forceinline__ Pack<T, VEC> ld_pack(const T* p) {
    Pack<T, VEC> r;
    if constexpr (VEC == 1) {
        r.w[0] = *p;
    } else {
        typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
        u32x4_t t[sizeof(r) / 16];
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i) t[i] = ONCE ? __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p) + i) : reinterpret_cast<const u32x4_t*>(p)[i];
        r = __builtin_bit_cast(decltype(r), t);
    }
    return r;
}
// f(e) is element e.
template <typename T, int VEC, typename F> __device__ __forceinline__ void st_pack(T* p, F f) {
    if constexpr (VEC == 1) {
        *p = Elem<T>::store(f(0));
    } else {
        Pack<T, VEC> r;
#pragma unroll
        for (int e = 0; e < VEC; e += 2) r.set2(e, f(e), f(e + 1));
        typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
        *reinterpret_cast<u32x4_t*>(p) = __builtin_bit_cast(u32x4_t, r);
    }
}

template <typename T, typename TW>
struct LnFwd {
    const T* x; const TW* w; const TW* b; T* y;
    float* mean; float* rstd;
    int64_t x_sb, x_sl, w_sb, b_sb;
    int rows, seq, n, T_;
    float one, eps;       // one: what is added to w
};

// Offset of row `row` of a [batch, seq] view; `b` its batch element. Views whose rows are evenly strided arrive with seq == rows.
__device__ __forceinline__ int64_t row_offset(int row, int seq, int64_t sb, int64_t sl, int& b) {
    b = seq == 0x7fffffff ? 0 : row / seq;
    return b * sb + static_cast<int64_t>(row - b * seq) * sl;
}

// FULL: the lanes hold exactly a row, so no value is masked (a training step at [3, 4336, 3072] bf16, both kernels with it: 96.0 -> 93.9 us).
template <typename T, typename TW, int VEC, int ITER, bool FULL>
__global__ __launch_bounds__(kLnMost) void ln_fwd_kernel(LnFwd<T, TW> p) {
    __shared__ float box[2][16][2];
    const int G = p.T_, grp = threadIdx.x / G, lane = threadIdx.x - grp * G;
    const int row_raw = blockIdx.x * (blockDim.x / G) + grp;
    const bool ok = row_raw < p.rows;
    const int row = ok ? row_raw : p.rows - 1;
    int b;
    const T* const xr = p.x + row_offset(row, p.seq, p.x_sb, p.x_sl, b);
    Pack<T, VEC> raw[ITER];
    bool in[ITER];
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
        in[it] = FULL || (it * G + lane) * VEC < p.n;
        raw[it] = ld_pack<T, VEC>(xr + (in[it] ? (it * G + lane) * VEC : 0));
    }
    float s = 0.0f, none = 0.0f;
#pragma unroll
    for (int it = 0; it < ITER; ++it)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += in[it] ? raw[it].at(e) : 0.0f;
    row_sums(s, none, G, box[0]);
    const float inv = 1.0f / static_cast<float>(p.n), mean = s * inv;
    float q = 0.0f;
#pragma unroll
    for (int it = 0; it < ITER; ++it)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float d = in[it] ? raw[it].at(e) - mean : 0.0f;
            q += d * d;
        }
    row_sums(q, none, G, box[1]);
    const float rstd = rsqrtf(q * inv + p.eps);
    if (!ok) return;
    if (p.mean != nullptr && lane == 0) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
    }
    const TW* const wr = p.w == nullptr ? nullptr : p.w + b * p.w_sb;
    const TW* const br = p.b == nullptr ? nullptr : p.b + b * p.b_sb;
    T* const yr = p.y + static_cast<int64_t>(row) * p.n;
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
        const int c = (it * G + lane) * VEC;
        if (!in[it]) continue;
        Pack<TW, VEC> w, bb;
        if (wr != nullptr) w = ld_pack<TW, VEC>(wr + c);
        if (br != nullptr) bb = ld_pack<TW, VEC>(br + c);
        st_pack<T, VEC>(yr + c, [&](int e) {
            const float h = (raw[it].at(e) - mean) * rstd;
            return h * (wr != nullptr ? p.one + w.at(e) : 1.0f) + (br != nullptr ? bb.at(e) : 0.0f);
        });
    }
}

// A workgroup per row of any length, read three times (the second and third time from the caches), an element at a time: 512 rows of 32767 bf16 49.3 us
// (13.1 at a copy's rate).
template <typename T, typename TW>
__global__ __launch_bounds__(kLnMost) void ln_fwd_wide_kernel(LnFwd<T, TW> p) {
    __shared__ float box[2][16][2];
    const int row = blockIdx.x;
    int b;
    const T* const xr = p.x + row_offset(row, p.seq, p.x_sb, p.x_sl, b);
    float s = 0.0f, none = 0.0f;
    for (int c = threadIdx.x; c < p.n; c += kLnMost) s += Elem<T>::load(xr[c]);
    row_sums(s, none, kLnMost, box[0]);
    const float inv = 1.0f / static_cast<float>(p.n), mean = s * inv;
    float q = 0.0f;
    for (int c = threadIdx.x; c < p.n; c += kLnMost) {
        const float d = Elem<T>::load(xr[c]) - mean;
        q += d * d;
    }
    row_sums(q, none, kLnMost, box[1]);
    const float rstd = rsqrtf(q * inv + p.eps);
    if (p.mean != nullptr && threadIdx.x == 0) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
    }
    for (int c = threadIdx.x; c < p.n; c += kLnMost) {
        const float h = (Elem<T>::load(xr[c]) - mean) * rstd;
        const float f = p.w != nullptr ? p.one + Elem<TW>::load(p.w[b * p.w_sb + c]) : 1.0f;
        p.y[static_cast<int64_t>(row) * p.n + c] = Elem<T>::store(h * f + (p.b != nullptr ? Elem<TW>::load(p.b[b * p.b_sb + c]) : 0.0f));
    }
}

template <typename T, typename TW>
struct LnBwd {
    const T* dy; const T* x; const TW* w; const float* mean; const float* rstd;
    T* dx;
    float* part;          // [groups][dw, db][blocks][n], null where neither is wanted
    int64_t dy_sb, dy_sl, x_sb, x_sl, w_sb;
    int rows, seq, n, T_; // rows of one weight's group; group = blockIdx.y
    float one;
};

// Backward. T lanes own a row and keep dw and db of their columns in registers over all rows they walk; the rows of a block are folded in LDS
// and leave as one row of `part`, which ln_fold_kernel adds up in order. While a row is worked on the next one's x and dy are on their way.
template <typename T, typename TW, int VEC, int ITER, bool FULL, bool ONCE>
__global__ __launch_bounds__(kLnMost) void ln_bwd_kernel(LnBwd<T, TW> p) {
    __shared__ float box[2][16][2];
    __shared__ float fold[kLnMost * VEC];
    const int G = p.T_, grp = threadIdx.x / G, lane = threadIdx.x - grp * G, groups = blockDim.x / G;
    const int group = blockIdx.y;
    const int step = gridDim.x * groups;
    const TW* const wr = p.w == nullptr ? nullptr : p.w + group * p.w_sb;
    float dw[ITER][VEC], db[ITER][VEC];
    Pack<TW, VEC> w[ITER] = {};
    bool in[ITER];
    int at[ITER];
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
        const int c = (it * G + lane) * VEC;
        in[it] = FULL || c < p.n;
        at[it] = in[it] ? c : 0;
        if (wr != nullptr) w[it] = ld_pack<TW, VEC>(wr + at[it]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[it][e] = db[it][e] = 0.0f;
    }
    struct Row { Pack<T, VEC> x[ITER], dy[ITER]; float mean, rstd; } cur, next;
    auto load = [&](int row_raw, Row& r) {   // past the end: the last row again, not used
        const int row = min(row_raw, p.rows - 1), all = group * p.rows + row;
        int b;
        const T* const xr = p.x + row_offset(all, p.seq, p.x_sb, p.x_sl, b);
        const T* const dr = p.dy + row_offset(all, p.seq, p.dy_sb, p.dy_sl, b);
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
            r.x[it] = ld_pack<T, VEC, ONCE>(xr + at[it]);
            r.dy[it] = ld_pack<T, VEC, ONCE>(dr + at[it]);
        }
        r.mean = p.mean[all];
        r.rstd = p.rstd[all];
    };
    const float inv = 1.0f / static_cast<float>(p.n);
    const int row0 = blockIdx.x * groups + grp;
    int turn = 0;
    load(row0, cur);
    for (int first = blockIdx.x * groups; first < p.rows; first += step, turn ^= 1) {   // (as often for every lane of the workgroup)
        const int row = first + grp;
        const bool ok = row < p.rows;
        if (first + step < p.rows) load(row + step, next);
        if (VEC > 1) {
#pragma unroll
            for (int it = 0; it < ITER; ++it) forget(w[it]);
        }
        float a = 0.0f, c = 0.0f;
#pragma unroll
        for (int it = 0; it < ITER; ++it)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = cur.dy[it].at(e), g = wr != nullptr ? d * (p.one + w[it].at(e)) : d;
                a += in[it] ? g : 0.0f;
                c += in[it] ? g * ((cur.x[it].at(e) - cur.mean) * cur.rstd) : 0.0f;
            }
        row_sums(a, c, G, box[turn]);
        a *= inv;
        c *= inv;
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
            forget(cur.x[it]);
            forget(cur.dy[it]);
            if (VEC > 1) forget(w[it]);
        }
        if (ok) {
            T* const dxr = p.dx == nullptr ? nullptr : p.dx + (static_cast<int64_t>(group) * p.rows + row) * p.n;
#pragma unroll
            for (int it = 0; it < ITER; ++it) {
                if (!in[it]) continue;
                auto one = [&](int e) {
                    const float d = cur.dy[it].at(e), h = (cur.x[it].at(e) - cur.mean) * cur.rstd;
                    const float g = wr != nullptr ? d * (p.one + w[it].at(e)) : d;
                    dw[it][e] += d * h;
                    db[it][e] += d;
                    return cur.rstd * (g - (a + h * c));
                };
                if (dxr != nullptr) {
                    st_pack<T, VEC>(dxr + at[it], one);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) one(e);
                }
            }
        }
        cur = next;
    }
    if (p.part == nullptr) return;
    const int span = G * VEC;   // columns of one `it`
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            lds_barrier();
#pragma unroll
            for (int e = 0; e < VEC; ++e) fold[grp * span + lane * VEC + e] = which == 0 ? dw[it][e] : db[it][e];
            lds_barrier();
            float* const to = p.part + ((static_cast<int64_t>(group) * 2 + which) * gridDim.x + blockIdx.x) * p.n;
            for (int i = threadIdx.x; i < span; i += blockDim.x) {
                float t = 0.0f;
                for (int g = 0; g < groups; ++g) t += fold[g * span + i];
                if (it * span + i < p.n) to[it * span + i] = t;
            }
        }
    }
}

// Few rows: dx by the first `dx_blocks` workgroups, dw and db whole by the others, 64 columns each, which read x and dy once more, from the caches.
// One launch and no workspace.
template <typename T, typename TW, int VEC, int ITER>
__global__ __launch_bounds__(kLnMost) void ln_bwd_few_kernel(LnBwd<T, TW> p, TW* dw_out, TW* db_out, int dx_blocks) {
    __shared__ float box[16][2];
    __shared__ float fold[2][16][64];
    const int group = blockIdx.y;
    if (static_cast<int>(blockIdx.x) < dx_blocks) {
        const int G = p.T_, grp = threadIdx.x / G, lane = threadIdx.x - grp * G;
        const int row_raw = blockIdx.x * (blockDim.x / G) + grp, row = min(row_raw, p.rows - 1), all = group * p.rows + row;
        int b;
        const T* const xr = p.x + row_offset(all, p.seq, p.x_sb, p.x_sl, b);
        const T* const dr = p.dy + row_offset(all, p.seq, p.dy_sb, p.dy_sl, b);
        const TW* const wr = p.w == nullptr ? nullptr : p.w + group * p.w_sb;
        Pack<T, VEC> x[ITER], dy[ITER];
        Pack<TW, VEC> w[ITER] = {};
        int at[ITER];
        bool in[ITER];
#pragma unroll
        for (int it = 0; it < ITER; ++it) {
            const int c = (it * G + lane) * VEC;
            in[it] = c < p.n;
            at[it] = in[it] ? c : 0;
            x[it] = ld_pack<T, VEC>(xr + at[it]);
            dy[it] = ld_pack<T, VEC>(dr + at[it]);
            if (wr != nullptr) w[it] = ld_pack<TW, VEC>(wr + at[it]);
        }
        const float mean = p.mean[all], rstd = p.rstd[all], inv = 1.0f / static_cast<float>(p.n);
        auto scaled = [&](int it, int e) { return wr != nullptr ? dy[it].at(e) * (p.one + w[it].at(e)) : dy[it].at(e); };
        float a = 0.0f, c = 0.0f;
#pragma unroll
        for (int it = 0; it < ITER; ++it)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float g = scaled(it, e);
                a += in[it] ? g : 0.0f;
                c += in[it] ? g * ((x[it].at(e) - mean) * rstd) : 0.0f;
            }
        row_sums(a, c, G, box);
        a *= inv;
        c *= inv;
        if (row_raw >= p.rows) return;
        T* const dxr = p.dx + static_cast<int64_t>(all) * p.n;
#pragma unroll
        for (int it = 0; it < ITER; ++it)
            if (in[it]) st_pack<T, VEC>(dxr + at[it], [&](int e) { return rstd * (scaled(it, e) - (a + (x[it].at(e) - mean) * rstd * c)); });
        return;
    }
    const int lane = threadIdx.x & 63, strip = threadIdx.x >> 6, strips = blockDim.x >> 6;
    const int col = (blockIdx.x - dx_blocks) * 64 + lane, c = min(col, p.n - 1);
    float dw = 0.0f, db = 0.0f;
    for (int row = strip; row < p.rows; row += strips * 8) {
        float d[8], h[8];   // (requested at once, also where fewer are left)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int all = group * p.rows + min(row + i * strips, p.rows - 1);
            int b;
            d[i] = Elem<T>::load(p.dy[row_offset(all, p.seq, p.dy_sb, p.dy_sl, b) + c]);
            h[i] = (Elem<T>::load(p.x[row_offset(all, p.seq, p.x_sb, p.x_sl, b) + c]) - p.mean[all]) * p.rstd[all];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool ok = row + i * strips < p.rows;
            dw += ok ? d[i] * h[i] : 0.0f;
            db += ok ? d[i] : 0.0f;
        }
    }
    fold[0][strip][lane] = dw;
    fold[1][strip][lane] = db;
    __syncthreads();
    TW* const out = strip == 0 ? dw_out : db_out;
    if (strip < 2 && col < p.n && out != nullptr) {
        float t = 0.0f;
        for (int i = 0; i < strips; ++i) t += fold[strip][i][lane];
        out[static_cast<int64_t>(group) * p.n + col] = Elem<TW>::store(t);
    }
}

// Rows of any length: dx, a workgroup per row, an element at a time (512 rows of 32768 bf16: 74.8 us for 19.7 at a copy's rate).
template <typename T, typename TW>
__global__ __launch_bounds__(kLnMost) void ln_bwd_wide_dx_kernel(LnBwd<T, TW> p) {
    __shared__ float box[16][2];
    const int group = blockIdx.y, all = group * p.rows + blockIdx.x;
    int b;
    const T* const xr = p.x + row_offset(all, p.seq, p.x_sb, p.x_sl, b);
    const T* const dr = p.dy + row_offset(all, p.seq, p.dy_sb, p.dy_sl, b);
    const TW* const wr = p.w == nullptr ? nullptr : p.w + group * p.w_sb;
    const float mean = p.mean[all], rstd = p.rstd[all], inv = 1.0f / static_cast<float>(p.n);
    float a = 0.0f, c = 0.0f;
    for (int i = threadIdx.x; i < p.n; i += kLnMost) {
        const float d = Elem<T>::load(dr[i]), g = wr != nullptr ? d * (p.one + Elem<TW>::load(wr[i])) : d;
        a += g;
        c += g * ((Elem<T>::load(xr[i]) - mean) * rstd);
    }
    row_sums(a, c, kLnMost, box);
    a *= inv;
    c *= inv;
    for (int i = threadIdx.x; i < p.n; i += kLnMost) {
        const float d = Elem<T>::load(dr[i]), g = wr != nullptr ? d * (p.one + Elem<TW>::load(wr[i])) : d;
        p.dx[static_cast<int64_t>(all) * p.n + i] = Elem<T>::store(rstd * (g - (a + (Elem<T>::load(xr[i]) - mean) * rstd * c)));
    }
}

// ... and the parts of dw and db: a workgroup takes 64 columns and every gridDim.y-th group of 16 rows of one weight's rows (26.3 us there, and 4.8 for
// their sums).
template <typename T, typename TW>
__global__ __launch_bounds__(kLnMost) void ln_bwd_wide_sums_kernel(LnBwd<T, TW> p) {
    __shared__ float fold[2][16][64];
    const int group = blockIdx.z, lane = threadIdx.x & 63, strip = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    float dw = 0.0f, db = 0.0f;
    if (c < p.n)
        for (int row = blockIdx.y * 16 + strip; row < p.rows; row += gridDim.y * 16) {
            const int all = group * p.rows + row;
            int b;
            const float d = Elem<T>::load(p.dy[row_offset(all, p.seq, p.dy_sb, p.dy_sl, b) + c]);
            dw += d * ((Elem<T>::load(p.x[row_offset(all, p.seq, p.x_sb, p.x_sl, b) + c]) - p.mean[all]) * p.rstd[all]);
            db += d;
        }
    fold[0][strip][lane] = dw;
    fold[1][strip][lane] = db;
    __syncthreads();
    if (strip < 2 && c < p.n) {
        float t = 0.0f;
        for (int i = 0; i < 16; ++i) t += fold[strip][i][lane];
        p.part[((static_cast<int64_t>(group) * 2 + strip) * gridDim.y + blockIdx.y) * p.n + c] = t;
    }
}

// dw[group] and db[group] = the sums of their parts in order, rounded once. A workgroup takes 1024 / strips columns with `strips` threads each.
template <typename TD>
__global__ __launch_bounds__(1024) void ln_fold_kernel(const float* part, TD* dw, TD* db, int parts, int n, int strips) {
    __shared__ float sums[1024 + 32];
    const int cols = 1024 / strips, strip = threadIdx.x / cols, col = threadIdx.x - strip * cols, c = blockIdx.x * cols + col, which = blockIdx.y, group = blockIdx.z;
    TD* const out = which == 0 ? dw : db;
    if (out == nullptr) return;
    const float* const from = part + (static_cast<int64_t>(group) * 2 + which) * parts * n;
    float t = 0.0f;
    if (c < n) {
        for (int i = strip; i < parts; i += strips * 8) {
            float v[8];   // (requested at once, also where fewer are left)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = from[static_cast<int64_t>(min(i + j * strips, parts - 1)) * n + c];
#pragma unroll
            for (int j = 0; j < 8; ++j) t += i + j * strips < parts ? v[j] : 0.0f;
        }
    }
    sums[strip * (cols + 1) + col] = t;
    __syncthreads();
    if (strip == 0 && c < n) {
        float total = 0.0f;
        for (int i = 0; i < strips; ++i) total += sums[i * (cols + 1) + col];
        out[static_cast<int64_t>(group) * n + c] = Elem<TD>::store(total);
    }
}

// ------------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------------
// Lanes per row and units (vectors, or elements) per lane; T == 0: the row takes the kernels for any length.
struct LnPlan { int vec, T, iter; };

static LnPlan ln_plan(int n, int vec, const int* iters, int count) {
    const int units = n / vec;
    LnPlan best = {vec, 0, 0};
    int best_cost = 0x7fffffff;
    for (int i = 0; i < count; ++i) {
        const int need = (units + iters[i] - 1) / iters[i];
        const int T = need <= 16 ? 16 : need <= 32 ? 32 : (need + 63) / 64 * 64;
        if (T > kLnMost) continue;
        // Idle lanes cost in full, waves to be joined through LDS a little: a row in one wave is best as long as its lanes are busy. us forward at
        // 4608 rows of bf16 for 1, 2, 3, 4 and 6 vectors a lane: 20.6, 14.4, 14.1, 14.7 and 12.6 for 384 vectors a row, 10.7, 9.9, 8.4, 9.1 and 9.0
        // for 192; backward 28.7 and 26.6 for one and two vectors, 17.1 and 19.2.
        const int cost = (T * iters[i] - units) * 64 / units * 4 + (T > 64 ? 2 : 0) + T / 256;
        if (cost < best_cost) { best_cost = cost; best = {vec, T, iters[i]}; }
    }
    return best;
}

static bool vector_rows(const void* p, int64_t sb, int64_t sl, int vec) { return aligned16(p) && sb % vec == 0 && sl % vec == 0; }

static LnPlan ln_fwd_plan(const flux_layer_norm_fwd_args& a, int vec) {
    // (4608 x 3072 bf16 an element at a time: 26.7 us for 12.6, backward 38.9 for 26.6)
    const bool wide = a.n % vec == 0 && vector_rows(a.x, a.x_sb, a.x_sl, vec) && aligned16(a.y) && (a.w == nullptr || vector_rows(a.w, a.w_sb, 0, vec)) &&
                      (a.b == nullptr || vector_rows(a.b, a.b_sb, 0, vec));
    static const int iters[] = {1, 2, 3, 4, 6, 8};
    return ln_plan(a.n, wide ? vec : 1, iters, 6);
}

template <typename T, typename TW>
static int ln_fwd_launch(const flux_layer_norm_fwd_args& a, hipStream_t st) {
    const int64_t rows = a.batch * a.seq;
    LnFwd<T, TW> p = {static_cast<const T*>(a.x), static_cast<const TW*>(a.w), static_cast<const TW*>(a.b), static_cast<T*>(a.y), a.mean, a.rstd,
                      a.x_sb, a.x_sl, a.groups > 1 ? a.w_sb : 0, a.groups > 1 ? a.b_sb : 0, static_cast<int>(rows), static_cast<int>(a.seq), a.n, 0,
                      a.plus_one ? 1.0f : 0.0f, a.eps};
    if (a.groups == 1 && (a.batch == 1 || a.x_sb == a.seq * a.x_sl)) p.seq = 0x7fffffff;   // evenly strided rows, one weight
    const LnPlan plan = ln_fwd_plan(a, Elem<T>::VEC);
    if (plan.T == 0) {
        if (rows >= (int64_t{1} << 32) / kLnMost) return fail(FLUX_E_SHAPE, "flux_layer_norm: too many rows of %d", a.n);
        hipLaunchKernelGGL((ln_fwd_wide_kernel<T, TW>), dim3((unsigned)rows), dim3(kLnMost), 0, st, p);
        return check_launch("flux_layer_norm");
    }
    p.T_ = plan.T;
    const int per_block = plan.T >= 256 ? 1 : 256 / plan.T, threads = per_block * plan.T;
    const int64_t blocks = (rows + per_block - 1) / per_block;
    if (blocks >= (int64_t{1} << 32) / threads) return fail(FLUX_E_SHAPE, "flux_layer_norm: too many rows of %d", a.n);   // (threads of a launch)
    const dim3 grid((unsigned)blocks);
#define CALL(V, I)                                                                                                  \
    if (V > 1 && plan.T * I * V == a.n) hipLaunchKernelGGL((ln_fwd_kernel<T, TW, V, I, (V > 1)>), grid, dim3(threads), 0, st, p); \
    else hipLaunchKernelGGL((ln_fwd_kernel<T, TW, V, I, false>), grid, dim3(threads), 0, st, p)
#define BY_ITER(V)                                   \
    switch (plan.iter) {                             \
        case 1: CALL(V, 1); break;                   \
        case 2: CALL(V, 2); break;                   \
        case 3: CALL(V, 3); break;                   \
        case 4: CALL(V, 4); break;                   \
        case 6: CALL(V, 6); break;                   \
        default: CALL(V, 8); break;                  \
    }
    if (plan.vec == 1) { BY_ITER(1) } else { BY_ITER(Elem<T>::VEC) }
#undef BY_ITER
#undef CALL
    return check_launch("flux_layer_norm");
}

// How the backward pass is cut: `blocks` workgroups of `threads` a weight group, each with a part of dw and db.
struct LnBwdPlan { LnPlan row; int threads, blocks; bool few; };

static LnBwdPlan ln_bwd_plan(const flux_layer_norm_bwd_args& a) {
    const int vec = a.x_dtype == FLUX_BF16 ? 8 : 4;
    const int64_t rows = a.groups > 1 ? a.seq : a.batch * a.seq;
    const bool wide = a.n % vec == 0 && vector_rows(a.x, a.x_sb, a.x_sl, vec) && vector_rows(a.dy, a.dy_sb, a.dy_sl, vec) && aligned16(a.dx) &&
                      (a.w == nullptr || vector_rows(a.w, a.w_sb, 0, vec));
    // x and dy of two rows and two sums a column: 16 columns of bf16 or 12 of fp32 a lane are what the 128 registers of 16 waves a CU hold
    static const int iters[] = {1, 2, 3, 4, 8};
    LnBwdPlan p;
    p.few = false;
    p.row = ln_plan(a.n, wide ? vec : 1, iters, wide ? (vec == 8 ? 2 : 3) : 5);
    const int64_t most = std::max<int64_t>(1, 256 / a.groups);   // workgroups a weight group
    if (p.row.T == 0) {
        p.threads = kLnMost;
        p.blocks = static_cast<int>(std::min<int64_t>((rows + 63) / 64, std::max<int64_t>(1, 1024 / ((a.n + 63) / 64) / a.groups)));
        return p;
    }
    // 16 waves a workgroup and one workgroup a CU (us at 4608 x 3072 for one, two and five rows a workgroup: 46.3, 31.5 and 26.7), fewer waves
    // where that leaves CUs without one (512 x 768, four rows and 16: 6.9 and 8.4)
    int per_block = kLnMost / p.row.T;
    while (per_block > 1 && per_block * p.row.T > 256 && (rows + per_block - 1) / per_block < most) per_block /= 2;
    p.threads = per_block * p.row.T;
    p.blocks = static_cast<int>(std::min<int64_t>((rows + per_block - 1) / per_block, most));
    // Up to 128 rows the waves of a workgroup request all of a column's values at once, and with no more such workgroups than CUs that is quicker. us of
    // the kernels, one launch and two: 77 x 768 5.2 and 9.3, 128 x 3072 6.8 and 13.5 (bf16), 256 x 1024 8.2 and 9.6, 512 x 768 13.6 and 9.7; with a
    // weight each 3 x 128 x 3072 7.3 and 17.0, 8 x 128 x 2048 8.9 and 12.6, 32 x 64 x 1024 11.6 and 9.7. And 3 us less of the host's time (27 -> 24, or
    // 49 -> 45 where the engine's thread is slow).
    p.few = (a.dw != nullptr || a.db != nullptr) && rows <= 128 && (a.n + 63) / 64 * a.groups <= 256;
    if (p.few) {
        per_block = kLnMost / p.row.T;
        p.threads = per_block * p.row.T;
        p.blocks = static_cast<int>((rows + per_block - 1) / per_block);
    }
    return p;
}

template <typename T, typename TW>
static int ln_bwd_launch(const flux_layer_norm_bwd_args& a, const LnBwdPlan& plan, float* ws, hipStream_t st) {
    const int64_t rows = a.groups > 1 ? a.seq : a.batch * a.seq;
    const bool sums = a.dw != nullptr || a.db != nullptr;
    LnBwd<T, TW> p = {static_cast<const T*>(a.dy), static_cast<const T*>(a.x), static_cast<const TW*>(a.w), a.mean, a.rstd, static_cast<T*>(a.dx), sums ? ws : nullptr,
                      a.dy_sb, a.dy_sl, a.x_sb, a.x_sl, a.groups > 1 ? a.w_sb : 0, static_cast<int>(rows), static_cast<int>(a.seq), a.n, plan.row.T, a.plus_one ? 1.0f : 0.0f};
    // Nothing reads x and dy again soon. Where they do not fit a third of the 256 MiB cache in front of HBM, they are not put there, which leaves it to
    // dx: a training step at [3, 4336, 3072] bf16 93.9 -> 90.5 us. Smaller ones mostly come from there, and the hint gains nothing: [4608, 3072]
    // 24.8 us and 24.8.
    const bool once = 2 * a.batch * a.seq * a.n * static_cast<int64_t>(sizeof(T)) > (int64_t{256} << 20) / 3;
    if (a.batch == 1 || (a.x_sb == a.seq * a.x_sl && a.dy_sb == a.seq * a.dy_sl)) p.seq = 0x7fffffff;
    if (plan.row.T == 0) {
        if (rows * a.groups >= (int64_t{1} << 32) / kLnMost) return fail(FLUX_E_SHAPE, "flux_layer_norm_bwd: too many rows of %d", a.n);
        if (a.dx != nullptr) hipLaunchKernelGGL((ln_bwd_wide_dx_kernel<T, TW>), dim3((unsigned)rows, (unsigned)a.groups), dim3(kLnMost), 0, st, p);
        if (sums) hipLaunchKernelGGL((ln_bwd_wide_sums_kernel<T, TW>), dim3((unsigned)((a.n + 63) / 64), (unsigned)plan.blocks, (unsigned)a.groups), dim3(kLnMost), 0, st, p);
    } else {
        const dim3 grid((unsigned)plan.blocks, (unsigned)a.groups), threads(plan.threads);
        const int dx_blocks = a.dx != nullptr ? plan.blocks : 0;
        const dim3 both((unsigned)(dx_blocks + (a.n + 63) / 64), (unsigned)a.groups);
#define CALL(V, I)                                                                                                                               \
    if (plan.few) hipLaunchKernelGGL((ln_bwd_few_kernel<T, TW, V, I>), both, threads, 0, st, p, static_cast<TW*>(a.dw), static_cast<TW*>(a.db), dx_blocks); \
    else if (V == 1 || plan.row.T * I * V != a.n) hipLaunchKernelGGL((ln_bwd_kernel<T, TW, V, I, false, false>), grid, threads, 0, st, p);            \
    else if (once) hipLaunchKernelGGL((ln_bwd_kernel<T, TW, V, I, (V > 1), (V > 1)>), grid, threads, 0, st, p);                                  \
    else hipLaunchKernelGGL((ln_bwd_kernel<T, TW, V, I, (V > 1), false>), grid, threads, 0, st, p)
        if (plan.row.vec == 1) {
            switch (plan.row.iter) {
                case 1: CALL(1, 1); break;
                case 2: CALL(1, 2); break;
                case 3: CALL(1, 3); break;
                case 4: CALL(1, 4); break;
                default: CALL(1, 8); break;
            }
        } else {
            constexpr int V = Elem<T>::VEC;
            switch (plan.row.iter) {
                case 1: CALL(V, 1); break;
                case 2: CALL(V, 2); break;
                default:
                    if constexpr (V == 4) { CALL(V, 3); }
                    break;
            }
        }
#undef CALL
    }
    if (sums && !plan.few) {
        int strips = 1;   // eight parts a thread
        while (strips < 32 && strips * 8 < plan.blocks) strips *= 2;
        const int cols = 1024 / strips;
        const dim3 grid((unsigned)((a.n + cols - 1) / cols), 2, (unsigned)a.groups);
        hipLaunchKernelGGL((ln_fold_kernel<TW>), grid, dim3(1024), 0, st, ws, static_cast<TW*>(a.dw), static_cast<TW*>(a.db), plan.blocks, a.n, strips);
    }
    return check_launch("flux_layer_norm_bwd");
}

// One row a batch element and a weight for all rows: the rows are what is evenly strided. Strides that nothing reads become those of contiguous
// rows: plans look at all of them.
static void ln_rows_of(int64_t& batch, int64_t& seq, int64_t groups, int32_t n, std::initializer_list<std::pair<int64_t*, int64_t*>> strides, std::initializer_list<int64_t*> weights) {
    const bool rows = groups == 1 && seq == 1;
    if (rows) std::swap(batch, seq);
    for (const auto& s : strides) {
        if (rows) *s.second = *s.first;
        if (seq == 1) *s.second = n;
        if (batch == 1) *s.first = seq * *s.second;
    }
    for (int64_t* w : weights)
        if (groups == 1) *w = 0;
}

// The backward pass's arguments as its plan and its launch take them, both from here.
static flux_layer_norm_bwd_args ln_bwd_rows(const flux_layer_norm_bwd_args& a) {
    flux_layer_norm_bwd_args r = a;
    ln_rows_of(r.batch, r.seq, r.groups, r.n, {{&r.x_sb, &r.x_sl}, {&r.dy_sb, &r.dy_sl}}, {&r.w_sb});
    return r;
}

static int64_t ln_bwd_bytes(const flux_layer_norm_bwd_args& a, const LnBwdPlan& plan) {
    return plan.few || (!a.dw && !a.db) ? 0 : static_cast<int64_t>(sizeof(float)) * 2 * a.groups * plan.blocks * a.n;
}

static int ln_shape(const char* what, int64_t batch, int64_t seq, int64_t groups, int32_t n) {
    if (batch < 0 || seq < 0 || n <= 0) return fail(FLUX_E_SHAPE, "%s: bad shape [%lld,%lld,%d]", what, (long long)batch, (long long)seq, n);
    if (n > FLUX_MAX_ROW) return fail(FLUX_E_TOO_WIDE, "%s: n = %d exceeds the maximum row length %d", what, n, FLUX_MAX_ROW);
    if (batch != 0 && seq > 0x7fff0000LL / batch) return fail(FLUX_E_SHAPE, "%s: too many rows", what);
    if (groups != 1 && groups != batch) return fail(FLUX_E_SHAPE, "%s: one weight for all rows or one for each batch element, not %lld for %lld", what, (long long)groups, (long long)batch);
    if (groups > 65535) return fail(FLUX_E_SHAPE, "%s: more than 65535 weights", what);
    return FLUX_OK;
}

}  // namespace flux

using namespace flux;

#define BY_TYPES(name, call)                                                                       \
    if (a->x_dtype == FLUX_BF16 && a->w_dtype == FLUX_BF16) return call<bf16_t, bf16_t> ARGS;       \
    if (a->x_dtype == FLUX_BF16 && a->w_dtype == FLUX_F32) return call<bf16_t, float> ARGS;         \
    if (a->x_dtype == FLUX_F32 && a->w_dtype == FLUX_F32) return call<float, float> ARGS;           \
    return fail(FLUX_E_DTYPE, name ": unsupported dtype pair (%d,%d)", a->x_dtype, a->w_dtype)

extern "C" int flux_tune_abi_version(void) { return FLUX_TUNE_ABI_VERSION; }

extern "C" int flux_layer_norm(const flux_layer_norm_fwd_args* a, void* stream) {
    if (!a) return fail(FLUX_E_NULL, "flux_layer_norm: null args");
    const int rc = ln_shape("flux_layer_norm", a->batch, a->seq, a->groups, a->n);
    if (rc != FLUX_OK) return rc;
    if (a->batch * a->seq == 0) return FLUX_OK;
    if (!a->x || !a->y) return fail(FLUX_E_NULL, "flux_layer_norm: null pointer");
    if ((a->mean == nullptr) != (a->rstd == nullptr)) return fail(FLUX_E_NULL, "flux_layer_norm: mean and rstd go together");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    flux_layer_norm_fwd_args rows = *a;
    ln_rows_of(rows.batch, rows.seq, rows.groups, rows.n, {{&rows.x_sb, &rows.x_sl}}, {&rows.w_sb, &rows.b_sb});
#define ARGS (rows, st)
    BY_TYPES("flux_layer_norm", ln_fwd_launch);
#undef ARGS
}

extern "C" int64_t flux_layer_norm_bwd_workspace_bytes(const flux_layer_norm_bwd_args* a) {
    if (!a || (!a->dw && !a->db) || ln_shape("flux_layer_norm_bwd", a->batch, a->seq, a->groups, a->n) != FLUX_OK || a->batch * a->seq == 0) return 0;
    const flux_layer_norm_bwd_args by_row = ln_bwd_rows(*a);
    return ln_bwd_bytes(by_row, ln_bwd_plan(by_row));
}

extern "C" int flux_layer_norm_bwd(const flux_layer_norm_bwd_args* a, void* ws, int64_t ws_bytes, void* stream) {
    if (!a) return fail(FLUX_E_NULL, "flux_layer_norm_bwd: null args");
    const int rc = ln_shape("flux_layer_norm_bwd", a->batch, a->seq, a->groups, a->n);
    if (rc != FLUX_OK) return rc;
    if (!a->dx && !a->dw && !a->db) return FLUX_OK;
    if (a->batch * a->seq == 0) return a->dw || a->db ? fail(FLUX_E_SHAPE, "flux_layer_norm_bwd: no rows to sum over") : FLUX_OK;
    if (!a->x || !a->dy || !a->mean || !a->rstd) return fail(FLUX_E_NULL, "flux_layer_norm_bwd: null pointer");
    const flux_layer_norm_bwd_args by_row = ln_bwd_rows(*a);
    const LnBwdPlan plan = ln_bwd_plan(by_row);
    const int64_t need = ln_bwd_bytes(by_row, plan);
    if (need > 0 && (!ws || reinterpret_cast<uintptr_t>(ws) % 4 != 0)) return fail(FLUX_E_NULL, "flux_layer_norm_bwd: the workspace must be 4-byte aligned memory");
    if (ws_bytes < need) return fail(FLUX_E_SHAPE, "flux_layer_norm_bwd: workspace of %lld bytes is too small", (long long)ws_bytes);
    const hipStream_t st = static_cast<hipStream_t>(stream);
#define ARGS (by_row, plan, static_cast<float*>(ws), st)
    BY_TYPES("flux_layer_norm_bwd", ln_bwd_launch);
#undef ARGS
}
