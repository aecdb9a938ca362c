// Rotation of q and k by positions of several axes, without a table, and the table itself.
//
//   (x0, x1) -> (x0 c - x1 s, x0 s + x1 c),  angle = ids[b, l, axis(pair)] theta^(-2j/d)
//
// Two reads and two writes of q and k and 3 operations a value: bound by HBM, if the angles are not worked out once for every head. A
// thread owns one 16-byte vector of a row (4 pairs of bf16, 2 of fp32) and walks eight heads of its position, so an angle is worked out once for
// all of them and a row needs no exchange between lanes. In turns (angle / 2 pi, as the frequencies arrive here) an angle of any
// size loses its whole turns exactly in 64 bits; what is left of a quarter turn goes through the Taylor series of sine and cosine in fp32.
//
// 24 + 24 heads of 128 at 32760 positions, bf16: 158 us, 5.1 TB/s, which a large copy reaches too; 16 + 4 heads of 128 at 2 x 1133 positions, fp32: 10.2 us
// (9.1 at that rate); one position of 24 + 8 heads for four requests 4.4 us and a table of 4608 positions 4.2, launches both.
#include "common.h"
#include "../../include/flux_hip_tune.h"
#include <cmath>

namespace flux {

constexpr int kRopeBlock = 256;
constexpr int kRopePairs = FLUX_ROPE_MOST_DIM / 2;
constexpr int kFewPairs = 64;    // of heads of up to 128

// P: pairs that a launch's arguments have room for.
template <int P>
struct RopeIds {
    const void* ids;
    int64_t sb, sl, sa;
    int dtype;
    double turns[P];      // theta^(-2j/d) / 2 pi of every pair
    unsigned char axis[P];
};

template <int P>
__device__ __forceinline__ double position(const RopeIds<P>& r, int64_t at) {
    switch (r.dtype) {   // (uniform)
        case FLUX_IDS_F32: return static_cast<const float*>(r.ids)[at];
        case FLUX_IDS_F64: return static_cast<const double*>(r.ids)[at];
        case FLUX_IDS_I32: return static_cast<const int32_t*>(r.ids)[at];
        default: return static_cast<double>(static_cast<const int64_t*>(r.ids)[at]);
    }
}

// Sine and cosine of 2 pi t. t - rint(4 t) / 4 is exact; |x| <= pi / 4 is left, where the series' first terms left out are below
// x^11 / 11! = 1.8e-9 and x^12 / 12! = 1.2e-10.
__device__ __forceinline__ void sincos_turns(double t, float& s, float& c) {
    const double whole = rint(t), quarters = rint((t - whole) * 4.0);
    const float x = static_cast<float>(((t - whole) - quarters * 0.25) * 6.283185307179586476925);
    const float z = x * x;
    const float sn = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
    const float cs = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
    const int q = static_cast<int>(quarters);
    const float a = (q & 1) ? cs : sn, b = (q & 1) ? sn : cs;
    s = (q & 2) ? -a : a;
    c = ((q + 1) & 2) ? -b : b;
}

struct RopeSide {
    const void* x; void* y;
    int64_t sb, sh, sl;
};
template <int P>
struct RopeNd {
    RopeSide q, k;
    int64_t L;
    int Hq, H;            // heads of q; of both, k's behind q's
    int D, lanes;         // lanes: threads of a row
    float sign;
    RopeIds<P> at;
};

// HEADS: heads that a thread walks with the same angles.
template <typename T, int VEC, int HEADS, int P>
__global__ __launch_bounds__(kRopeBlock) void rope_nd_kernel(RopeNd<P> p) {
    const int rows = kRopeBlock / p.lanes;                 // positions of a workgroup
    const int row = threadIdx.x / p.lanes, lane = threadIdx.x - row * p.lanes;
    // Consecutive workgroups go round the eight XCDs; each of them takes one eighth of the sequence in which the head groups of a
    // stretch of positions follow one another, so that a row of a fused projection is fetched into one L2.
    const int64_t head_groups = (p.H + HEADS - 1) / HEADS;
    const int64_t vb = static_cast<int64_t>(blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
    const int64_t stretch = vb / head_groups, pos_raw = stretch * rows + row;
    if (row >= rows || pos_raw >= p.L) return;
    const int h0 = static_cast<int>(vb - stretch * head_groups) * HEADS;
    const int64_t b = blockIdx.y, pos = pos_raw;
    const int c0 = lane * VEC;

    // a head's address is one of two affine functions; heads past the last are the last one again, loaded and not stored
    T in[HEADS][VEC];
    auto side = [&](int h, int64_t& at_x, int64_t& at_y, const T*& x, T*& y) {
        const bool is_k = h >= p.Hq;
        const RopeSide& s = is_k ? p.k : p.q;
        const int hs = is_k ? h - p.Hq : h, heads = is_k ? p.H - p.Hq : p.Hq;
        x = static_cast<const T*>(s.x);
        y = static_cast<T*>(s.y);
        at_x = b * s.sb + hs * s.sh + pos * s.sl + c0;
        at_y = ((b * heads + hs) * p.L + pos) * p.D + c0;
    };
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        int64_t ax, ay;
        const T* x;
        T* y;
        side(min(h0 + i, p.H - 1), ax, ay, x, y);
        if constexpr (VEC == 2) {
            in[i][0] = x[ax];
            in[i][1] = x[ax + 1];
        } else {
            const Vec16<T> v = ld16(x + ax);
#pragma unroll
            for (int e = 0; e < VEC; ++e) in[i][e] = v.v[e];
        }
    }
    float c[VEC / 2], s[VEC / 2];
    const int64_t id0 = b * p.at.sb + pos * p.at.sl;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
        const int pair = c0 / 2 + i;
        sincos_turns(position(p.at, id0 + p.at.axis[pair] * p.at.sa) * p.at.turns[pair], s[i], c[i]);
        s[i] *= p.sign;
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        if (h0 + i >= p.H) break;
        int64_t ax, ay;
        const T* x;
        T* y;
        side(h0 + i, ax, ay, x, y);
        T out[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
            const float x0 = Elem<T>::load(in[i][e]), x1 = Elem<T>::load(in[i][e + 1]);
            // (which of two products is rounded is not left to the compiler: a token's result does not go with the number of heads a thread walks)
            out[e] = Elem<T>::store(fmaf(x0, c[e / 2], -(x1 * s[e / 2])));
            out[e + 1] = Elem<T>::store(fmaf(x0, s[e / 2], x1 * c[e / 2]));
        }
        if constexpr (VEC == 2) {
            y[ay] = out[0];
            y[ay + 1] = out[1];
        } else {
            Vec16<T> v;
#pragma unroll
            for (int e = 0; e < VEC; ++e) v.v[e] = out[e];
            st16(y + ay, v);
        }
    }
}

// A thread a matrix.
template <int P>
__global__ __launch_bounds__(kRopeBlock) void rope_table_kernel(RopeIds<P> at, float* out, int64_t L, int pairs, int64_t total) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kRopeBlock + threadIdx.x;
    if (i >= total) return;
    const int64_t row = i / pairs, b = row / L, pos = row - b * L;
    const int pair = static_cast<int>(i - row * pairs);
    float s, c;
    sincos_turns(position(at, b * at.sb + pos * at.sl + at.axis[pair] * at.sa) * at.turns[pair], s, c);
    const Vec16<float> v = {{c, -s, s, c}};
    st16(out + i * 4, v);
}

// The frequencies of every pair, in turns: r^j with r = theta^(-2/d), eight apart from one another by one multiplication, so that pair j
// carries j / 8 roundings of 2^-53 and the angle as many of the rounding that its product with the position has anyway.
template <int P>
static void read_ids(const flux_rope_ids& a, RopeIds<P>& r) {
    r.ids = a.ids;
    r.sb = a.sb;
    r.sl = a.sl;
    r.sa = a.sa;
    r.dtype = a.dtype;
    int pairs = 0;
    for (int i = 0; i < a.n_axes; ++i) {
        const int d = a.axes_dim[i];
        const double step = std::log2(a.theta) * -2.0 / d, r8 = std::exp2(8 * step);
        for (int j = 0; j < d / 2; ++j) {
            r.turns[pairs + j] = j < 8 ? std::exp2(j * step) * 0.15915494309189533577 : r.turns[pairs + j - 8] * r8;
            r.axis[pairs + j] = static_cast<unsigned char>(i);
        }
        pairs += d / 2;
    }
}
static int check_ids(const flux_rope_ids& a, int& pairs, const char* what) {
    if (!a.ids) return fail(FLUX_E_NULL, "%s: null ids", what);
    if (a.dtype < FLUX_IDS_F32 || a.dtype > FLUX_IDS_I64) return fail(FLUX_E_DTYPE, "%s: unsupported type of ids %d", what, a.dtype);
    if (a.n_axes < 1 || a.n_axes > FLUX_ROPE_MOST_AXES) return fail(FLUX_E_SHAPE, "%s: %d axes, 1 to %d are taken", what, a.n_axes, FLUX_ROPE_MOST_AXES);
    if (!(a.theta > 0.0) || !std::isfinite(a.theta)) return fail(FLUX_E_SHAPE, "%s: theta must be a positive number", what);
    pairs = 0;
    for (int i = 0; i < a.n_axes; ++i) {
        const int d = a.axes_dim[i];
        if (d <= 0 || d % 2 != 0 || d > FLUX_ROPE_MOST_DIM || pairs + d / 2 > kRopePairs) return fail(FLUX_E_SHAPE, "%s: axes of an even number of values, %d in all at most", what, FLUX_ROPE_MOST_DIM);
        pairs += d / 2;
    }
    return FLUX_OK;
}

template <typename T>
static bool vectors(const flux_src4& s, const void* out) {
    return s.ptr == nullptr || (aligned16(s.ptr) && aligned16(out) && s.sb % Elem<T>::VEC == 0 && s.sh % Elem<T>::VEC == 0 && s.sl % Elem<T>::VEC == 0);
}

template <typename T, int P>
static int rope_launch(const flux_rope_nd_args& a, hipStream_t st) {
    RopeNd<P> p;
    read_ids(a.at, p.at);
    p.q = {a.q.ptr, a.q_out, a.q.sb, a.q.sh, a.q.sl};
    p.k = {a.k.ptr, a.k_out, a.k.sb, a.k.sh, a.k.sl};
    p.L = a.L;
    p.Hq = static_cast<int>(a.Hq);
    p.H = static_cast<int>(a.Hq + a.Hk);
    p.D = a.D;
    p.sign = a.inverse ? -1.0f : 1.0f;
    const bool wide = a.D % Elem<T>::VEC == 0 && vectors<T>(a.q, a.q_out) && vectors<T>(a.k, a.k_out);
    p.lanes = a.D / (wide ? Elem<T>::VEC : 2);
    const int rows = kRopeBlock / p.lanes;
    const int64_t stretches = (a.L + rows - 1) / rows;
    // Angles for eight heads at once where that leaves a workgroup for every CU, for two otherwise: with 256 of them and more the angles cost, with
    // fewer the chain of a thread's loads and stores. us for eight, four, two and one (24 + 24 heads of 128, bf16): 155, 156, 178 and 264 at L = 32760,
    // 21.9, 25.3, 31.3 and 39.7 at 4608, 8.8, 8.9, 9.5 and 11.5 at 1107, 5.2, 4.3, 4.3 and 4.4 at 256, 4.9, 3.9, 3.5 and 3.3 at 1.
    const int heads = a.B * stretches * ((p.H + 7) / 8) >= 256 ? 8 : 2;
    const int64_t blocks = stretches * ((p.H + heads - 1) / heads);
    if (a.B > 65535 || blocks > (int64_t{1} << 32) / kRopeBlock - 8) return fail(FLUX_E_SHAPE, "flux_rope_nd: grid too large (B=%lld, L=%lld, %d heads)", (long long)a.B, (long long)a.L, p.H);
    const dim3 grid((unsigned)((blocks + 7) / 8 * 8), (unsigned)a.B);
#define CALL(V, HEADS) hipLaunchKernelGGL((rope_nd_kernel<T, V, HEADS, P>), grid, dim3(kRopeBlock), 0, st, p)
    if (wide) {
        if (heads == 8) CALL(Elem<T>::VEC, 8);
        else CALL(Elem<T>::VEC, 2);
    } else {
        if (heads == 8) CALL(2, 8);
        else CALL(2, 2);
    }
#undef CALL
    return check_launch("flux_rope_nd");
}

template <int P>
static void table_launch(const flux_rope_ids& at, float* out, int64_t L, int pairs, int64_t total, hipStream_t st) {
    RopeIds<P> r;
    read_ids(at, r);
    hipLaunchKernelGGL((rope_table_kernel<P>), dim3((unsigned)((total + kRopeBlock - 1) / kRopeBlock)), dim3(kRopeBlock), 0, st, r, out, L, pairs, total);
}

}  // namespace flux

using namespace flux;

extern "C" int flux_rope_nd(const flux_rope_nd_args* a, void* stream) {
    if (!a) return fail(FLUX_E_NULL, "flux_rope_nd: null args");
    if (a->B < 0 || a->L < 0 || a->Hq < 0 || a->Hk < 0 || a->Hq + a->Hk > 0x7ffffff || a->L > 0x7fffffffLL) return fail(FLUX_E_SHAPE, "flux_rope_nd: bad shape B=%lld Hq=%lld Hk=%lld L=%lld", (long long)a->B, (long long)a->Hq, (long long)a->Hk, (long long)a->L);
    if (a->B == 0 || a->L == 0 || a->Hq + a->Hk == 0) return FLUX_OK;
    if ((a->Hq > 0 && (!a->q.ptr || !a->q_out)) || (a->Hk > 0 && (!a->k.ptr || !a->k_out))) return fail(FLUX_E_NULL, "flux_rope_nd: null pointer");
    int pairs;
    const int rc = check_ids(a->at, pairs, "flux_rope_nd");
    if (rc != FLUX_OK) return rc;
    if (a->D != 2 * pairs) return fail(FLUX_E_SHAPE, "flux_rope_nd: axes of %d values in all for rows of %d", 2 * pairs, a->D);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == FLUX_BF16) return pairs <= kFewPairs ? rope_launch<bf16_t, kFewPairs>(*a, st) : rope_launch<bf16_t, kRopePairs>(*a, st);
    if (a->dtype == FLUX_F32) return pairs <= kFewPairs ? rope_launch<float, kFewPairs>(*a, st) : rope_launch<float, kRopePairs>(*a, st);
    return fail(FLUX_E_DTYPE, "flux_rope_nd: unsupported dtype %d", a->dtype);
}

extern "C" int flux_rope_table(const flux_rope_ids* at, float* out, int64_t B, int64_t L, void* stream) {
    if (!at) return fail(FLUX_E_NULL, "flux_rope_table: null args");
    if (B < 0 || L < 0 || B > 0x7fffffffLL || L > 0x7fffffffLL) return fail(FLUX_E_SHAPE, "flux_rope_table: bad shape B=%lld L=%lld", (long long)B, (long long)L);
    if (B == 0 || L == 0) return FLUX_OK;
    int pairs;
    const int rc = check_ids(*at, pairs, "flux_rope_table");
    if (rc != FLUX_OK) return rc;
    if (!out) return fail(FLUX_E_NULL, "flux_rope_table: null pointer");
    if (!aligned16(out)) return fail(FLUX_E_ALIGN, "flux_rope_table: the table is not 16-byte aligned");
    if (B * L > ((int64_t{1} << 32) - kRopeBlock) / pairs) return fail(FLUX_E_SHAPE, "flux_rope_table: too many positions");
    const int64_t total = B * L * pairs;
    if (pairs <= kFewPairs) table_launch<kFewPairs>(*at, out, L, pairs, total, static_cast<hipStream_t>(stream));
    else table_launch<kRopePairs>(*at, out, L, pairs, total, static_cast<hipStream_t>(stream));
    return check_launch("flux_rope_table");
}
