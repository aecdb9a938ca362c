// Products with weights held in 4 bits, a scale and (or not) a zero point for each group of 32, 64 or 128 columns.
//
//   y[m, n] = act(sum_g s[n, g] sum_{k in g} (q[n, k] - z[n, g]) x[m, k] + b[n])
//
// Half a byte a weight and two operations a row: up to some dozens of rows bound by the bytes of the weights. A multiplication on the VALU would cost more
// than they do: 57 M weights are 28 MB, 5.6 us at a copy's rate, and at three instructions a weight (take it out, convert, multiply) 4.4 us of all VALUs for one
// row. So a weight becomes a bf16 number in one instruction, 16 + q = (q << 3) | 0x4180 for two of them at once, and the matrix cores multiply (16x16x32,
// x the rows and W the columns of the result, whose 16 rows cost one row's time): the sum that is too much, (16 + z) sum x, is where a group's sum
// starts. Sums of x by group are formed once, as x goes to LDS. A group's sum takes its scale behind the product, in fp32: nothing is rounded but y.
#include "common.h"
#include "../../include/flux_hip_serve.h"
#include <algorithm>
#include <math.h>

namespace flux {

typedef __bf16 w4_bf16x8 __attribute__((ext_vector_type(8)));
typedef float w4_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t w4_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kW4Chunk = 128;         // columns of a tile
constexpr int kW4Tile = 16;           // rows of W (outputs) of a tile
constexpr int kW4SiluRows = 8;

struct W4Params {
    const bf16_t* x; const w4_u32x4* q; const bf16_t* s; const uint8_t* z; const bf16_t* bias; bf16_t* y;
    int64_t ldx, ldy;
    int M, N, K, chunks, slab;        // slab: chunks of x in LDS at a time
    int act, silu;
};

// Eight weights, 16 + q each.
__device__ __forceinline__ w4_bf16x8 w4_unpack(uint32_t w) {
    const uint32_t mask = 0x00780078u, one = 0x41804180u;
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

// A workgroup of four waves takes 16 outputs of up to 16 rows of x (8 with SPLIT: f(x) as a bf16 number and another one for what that leaves over, in
// rows 8 beneath). The waves take every fourth chunk of K and add their sums in order.
// GPC: groups of a chunk.
template <int GPC, bool ZERO, bool SPLIT>
__global__ __launch_bounds__(256) void w4_rows_kernel(W4Params p) {
    constexpr int RB = SPLIT ? 8 : 16, U = 6;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
    const int tile = blockIdx.x, m0 = blockIdx.y * RB, rows = min(RB, p.M - m0), held = SPLIT ? 2 * rows : rows;
    const int stride = p.slab * (kW4Chunk * 2) + 16;                  // bytes of a row of x in LDS, 16 more against conflicts
    float* const sums = reinterpret_cast<float*>(lds + held * stride);  // [group of the slab][16]: -sum x
    int* const odd = reinterpret_cast<int*>(sums + p.slab * GPC * 16);
    // rows of the product without a row of x read the first one; what they sum up is not stored
    const int my_row = l16 < rows ? l16 : (SPLIT && l16 >= 8 && l16 - 8 < rows) ? rows + l16 - 8 : 0;
    const char* const xrow = lds + my_row * stride + g * 16;
    const w4_u32x4* const q = p.q + static_cast<int64_t>(tile) * p.chunks * 64 + lane;
    const bf16_t* const s = p.s + (static_cast<int64_t>(tile) * p.chunks * 16 + l16) * GPC;
    const uint8_t* const z = ZERO ? p.z + (static_cast<int64_t>(tile) * p.chunks * 16 + l16) * GPC : nullptr;
    if (tid == 0) *odd = 0;
    w4_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    w4_u32x4 wq[U];
    bf16_t ws[U][GPC];
    uint8_t wz[U][GPC];
    for (int c0 = 0; c0 < p.chunks; c0 += p.slab) {
        const int n = min(p.slab, p.chunks - c0);
        auto request = [&](int u, int c) {   // (past the end: the slab's first chunk again, not used)
            const int64_t at = c0 + (c < n ? c : 0);
            wq[u] = __builtin_nontemporal_load(q + at * 64);
#pragma unroll
            for (int i = 0; i < GPC; ++i) {
                ws[u][i] = s[at * 16 * GPC + i];
                if (ZERO) wz[u][i] = z[at * 16 * GPC + i];
            }
        };
#pragma unroll
        for (int u = 0; u < U; ++u) request(u, wave + 4 * u);
        __syncthreads();   // the slab before is read
        for (int i = tid; i < rows * n * 16; i += 256) {   // 8 values each; 16 threads a chunk
            const int m = i / (n * 16), v = i - m * (n * 16), k = (c0 * 16 + v) * 8;
            Vec16<bf16_t> hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) hi.v[e] = 0;
            if (k < p.K) hi = ld16(p.x + (m0 + m) * p.ldx + k);
            float sh = 0.0f, sl = 0.0f;
            bool far = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float f = bf2f(hi.v[e]);
                if (SPLIT) {
                    f = f * __builtin_amdgcn_rcpf(1.0f + __expf(-f));
                    hi.v[e] = f2bf(f);
                    lo.v[e] = f2bf(fabsf(f) < INFINITY ? f - bf2f(hi.v[e]) : 0.0f);
                    sl += bf2f(lo.v[e]);
                }
                sh += bf2f(hi.v[e]);
                far |= !(fabsf(f) < 0x1p100f);   // (16 + z) x would leave fp32's range, or is not a number
            }
            if (far) *odd = 1;
            sh = group_sum<16 / GPC>(sh);
            *reinterpret_cast<Vec16<bf16_t>*>(lds + m * stride + v * 16) = hi;
            if (v % (16 / GPC) == 0) sums[v / (16 / GPC) * 16 + m] = -sh;
            if (SPLIT) {
                sl = group_sum<16 / GPC>(sl);
                *reinterpret_cast<Vec16<bf16_t>*>(lds + (rows + m) * stride + v * 16) = lo;
                if (v % (16 / GPC) == 0) sums[v / (16 / GPC) * 16 + 8 + m] = -sl;
            }
        }
        __syncthreads();
        const bool exact = *odd != 0;
        for (int base = wave; base < n; base += 4 * U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = base + 4 * u;
                if (c < n) {
#pragma unroll
                    for (int i = 0; i < GPC; ++i) {
                        const float zero = ZERO ? static_cast<float>(wz[u][i]) : 8.0f;
                        w4_f32x4 t = *reinterpret_cast<const w4_f32x4*>(sums + (c * GPC + i) * 16 + g * 4) * (16.0f + zero);
                        if (exact) t = w4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = i * 4 / GPC; j < (i + 1) * 4 / GPC; ++j) {
                            const w4_bf16x8 a = *reinterpret_cast<const w4_bf16x8*>(xrow + c * (kW4Chunk * 2) + j * 64);
                            const w4_bf16x8 b = exact ? w4_unpack_exact(wq[u][j], zero) : w4_unpack(wq[u][j]);
                            t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, t, 0, 0, 0);
                        }
                        acc += t * bf2f(ws[u][i]);
                    }
                }
                request(u, c + 4 * U);
            }
        }
    }
    __syncthreads();
    float* const parts = reinterpret_cast<float*>(lds);   // [wave][lane][4]
    *reinterpret_cast<w4_f32x4*>(parts + tid * 4) = acc;
    __syncthreads();
    const int m = tid >> 4, col = tid & 15, nn = tile * kW4Tile + col;
    if (m >= rows || nn >= p.N) return;
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        y += parts[(w * 64 + (m >> 2) * 16 + col) * 4 + (m & 3)];
        if (SPLIT) y += parts[(w * 64 + ((m + 8) >> 2) * 16 + col) * 4 + (m & 3)];
    }
    if (p.bias != nullptr) y += bf2f(p.bias[nn]);
    if (p.act == FLUX_ACT_GELU_TANH) y = gelu_tanh_f32(y);
    p.y[(m0 + m) * p.ldy + nn] = f2bf(y);
}

// W as bf16 [N, K], (q - z) s rounded once. A wave takes a tile; a lane's row is written as four pieces of 16 bytes.
template <int GPC, bool ZERO>
__global__ __launch_bounds__(256) void w4_unpack_kernel(const w4_u32x4* q, const bf16_t* s, const uint8_t* z, bf16_t* out, int N, int K, int chunks, int64_t tiles) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (at >= tiles) return;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int64_t n = at / chunks * kW4Tile + r;
    const int k0 = static_cast<int>(at % chunks) * kW4Chunk + g * 8;
    const w4_u32x4 w = q[at * 64 + lane];
    float scale[GPC], zero[GPC];
#pragma unroll
    for (int i = 0; i < GPC; ++i) {
        scale[i] = bf2f(s[(at * 16 + r) * GPC + i]);
        zero[i] = ZERO ? static_cast<float>(z[(at * 16 + r) * GPC + i]) : 8.0f;
    }
    if (n >= N) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = k0 + j * 32;
        if (k >= K) break;
        Vec16<bf16_t> o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o.v[e] = f2bf((static_cast<float>((w[j] >> (4 * (e / 2) + 16 * (e % 2))) & 15u) - zero[j * GPC / 4]) * scale[j * GPC / 4]);
        st16(out + n * K + k, o);
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

template <int GPC>
static void w4_rows_launch(W4Params p, hipStream_t st) {
    const int rb = p.silu ? 8 : 16, held = std::min(p.M, rb) * (p.silu ? 2 : 1);
    // up to 48 KB of x, so that three workgroups share a CU
    p.slab = std::min({p.chunks, 64, 48 * 1024 / (held * kW4Chunk * 2) / 4 * 4});
    const int bytes = std::max(held * (p.slab * kW4Chunk * 2 + 16) + p.slab * GPC * 64 + 16, 4096);
    const dim3 grid(static_cast<unsigned>((p.N + kW4Tile - 1) / kW4Tile), static_cast<unsigned>((p.M + rb - 1) / rb));
#define CALL(ZERO, SPLIT) hipLaunchKernelGGL((w4_rows_kernel<GPC, ZERO, SPLIT>), grid, dim3(256), bytes, st, p)
    if (p.z) { if (p.silu) CALL(true, true); else CALL(true, false); }
    else { if (p.silu) CALL(false, true); else CALL(false, false); }
#undef CALL
}

constexpr int kW4MostRows = 64;   // beyond them the weights are laid out first

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
    if (!a || a->M <= kW4MostRows || w4_check("flux_linear_w4_bf16", a->w) != FLUX_OK || a->w.N == 0 || a->w.K == 0) return 0;
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
    if (a->M > kW4MostRows) {
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
    if (a->w.group == 32) w4_rows_launch<4>(p, st);
    else if (a->w.group == 64) w4_rows_launch<2>(p, st);
    else w4_rows_launch<1>(p, st);
    return check_launch(what);
}
