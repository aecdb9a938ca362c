// The main loops of the four-wave tiles and the epilogue of the square one (gemm_bf16.hip says what they are made for), for the kernels that
// multiply and for those that add an adapter's product to the same tile (gemm_lora.hip).
#pragma once

#include "gemm_common.h"

namespace flux {

// Branch-free epilogue for interior tiles whose outputs (and residual operands) are 16-byte
// addressable and whose columns all go to one destination. GELU is all-or-nothing for the wave.
// Everything lane-dependent is computed once; per store only a wave-uniform row offset changes, so
// the stores use a scalar base plus a 32-bit lane offset.
template <int MI, int NJ, bool GELU, bool GATE>
__device__ __forceinline__ void gemm_epilogue_fast(const GemmParams& p, f32x4 (&acc)[2 * MI][2 * NJ], char* lds, int m0, int n0,
                                                   int wave, int lane) {
    constexpr int WROWS = 32 * MI, WCOLS = 32 * NJ;
    constexpr int C_PITCH = WCOLS * 2, C_CH = WCOLS / 8;
    constexpr int RPI = 64 / C_CH;      // rows per wave-wide 16-byte access
    constexpr int NIT = 32 / RPI;       // accesses per 32-row block
    constexpr int NQ = 2 * NJ;          // column quads of a lane: one per 16-column fragment
    const int wm = wave >> 1, wn = wave & 1;
    const int frow = lane & 15, fq = lane >> 4;
    char* cw = lds + wave * (WROWS * C_PITCH);
    const int wave_n0 = n0 + wn * WCOLS;
    const int wave_m0 = m0 + wm * WROWS;

    float bv[NQ][4];
    if (p.bias != nullptr) {
        const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(p.bias), 0, p.N * 2, kRsrcFlags);
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const u32x2 raw = __builtin_amdgcn_raw_buffer_load_b64(rb, (wave_n0 + q * 16 + fq * 4) * 2, 0, 0);
            bv[q][0] = __uint_as_float(raw.x << 16);
            bv[q][1] = __uint_as_float(raw.x & 0xffff0000u);
            bv[q][2] = __uint_as_float(raw.y << 16);
            bv[q][3] = __uint_as_float(raw.y & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) bv[q][e] = 0.0f;
    }

    int waddr[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) waddr[q] = frow * C_PITCH + (((q * 2 + (fq >> 1)) ^ (frow & (C_CH - 1))) * 16) + (fq & 1) * 8;
    const int rrow = lane / C_CH, rch = lane % C_CH;
    // read address for access `it` of a block: row = it*RPI + rrow; the swizzle term repeats every 16 rows
    constexpr int NSW = (16 / RPI) < NIT ? (16 / RPI) : NIT;
    int raddr[NSW];
#pragma unroll
    for (int t = 0; t < NSW; ++t) {
        const int row = t * RPI + rrow;
        raddr[t] = row * C_PITCH + ((rch ^ (row & (C_CH - 1))) * 16);
    }

    const bool to_y = wave_n0 < p.split_n;
    char* dst_u = reinterpret_cast<char*>(to_y ? p.Y + wave_n0 : p.Y2 + (wave_n0 - p.split_n + p.y2_col0));
    const int64_t dst_ld = (to_y ? p.ldy : p.ldy2) * 2;            // bytes
    const uint32_t dst_lane = static_cast<uint32_t>(rrow * dst_ld + rch * 16);
    // Gated residual: the rows of resid this lane adds to are requested a whole 32-row block ahead,
    // into the other half of rs, so that they land while the block in front is converted and stored.
    // (Requested where they are used, every 16-byte store waited for a load round trip of its own,
    // and, the memory counter being in-order, for the store in front of it: 32 round trips in a row
    // per wave.) The tile lies inside one batch element (the caller checks), so the gate vector of
    // this lane's eight columns is loaded once.
    const char* res_u = nullptr;
    uint32_t res_lane = 0;
    Vec16<bf16_t> gt;
    Vec16<bf16_t> rs[2][NIT];
    auto request_resid = [&](int i) {
#pragma unroll
        for (int it = 0; it < NIT; ++it)
            rs[i & 1][it] = *reinterpret_cast<const Vec16<bf16_t>*>(res_u + static_cast<int64_t>(wave_m0 + i * 32 + it * RPI) * p.ldresid * 2 + res_lane);
    };
    if (GATE) {
        res_u = reinterpret_cast<const char*>(p.resid + wave_n0);
        res_lane = static_cast<uint32_t>(rrow * p.ldresid * 2 + rch * 16);
        gt = ld16(p.gate + static_cast<int64_t>(m0 / p.rows_per_batch) * p.gate_stride + wave_n0 + rch * 8);
        request_resid(0);
    }

#pragma unroll
    for (int i = 0; i < MI; ++i) {
        if (GATE) {
            if (i + 1 < MI) request_resid(i + 1);
            __builtin_amdgcn_sched_barrier(0);   // the loads stay in front of the conversion below
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = acc[2 * i + t][q][e] + bv[q][e];
                    if (GELU) v[e] = tanh_gelu_fast(v[e]);
                }
                *reinterpret_cast<u32x2*>(cw + (i * 32 + t * 16) * C_PITCH + waddr[q]) = pack4_bf16(v[0], v[1], v[2], v[3]);
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int it = 0; it < NIT; ++it) {
            const int row_u = i * 32 + it * RPI;                 // wave-uniform part of the row
            Vec16<bf16_t> y = *reinterpret_cast<const Vec16<bf16_t>*>(cw + (i * 32 + (it / NSW) * NSW * RPI) * C_PITCH + raddr[it % NSW]);
            const int64_t m_u = wave_m0 + row_u;
            if (GATE) {
                const Vec16<bf16_t> r = rs[i & 1][it];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float y0 = bf2f(r.v[e]) + bf2f(f2bf(bf2f(gt.v[e]) * bf2f(y.v[e])));
                    const float y1 = bf2f(r.v[e + 1]) + bf2f(f2bf(bf2f(gt.v[e + 1]) * bf2f(y.v[e + 1])));
                    const uint32_t w = pack2_bf16(y0, y1);
                    y.v[e] = static_cast<bf16_t>(w & 0xffffu);
                    y.v[e + 1] = static_cast<bf16_t>(w >> 16);
                }
            }
            *reinterpret_cast<Vec16<bf16_t>*>(dst_u + m_u * dst_ld + dst_lane) = y;
        }
    }
}

template <int MI, int NJ>
__device__ __forceinline__ void gemm_epilogue(const GemmParams& p, f32x4 (&acc)[2 * MI][2 * NJ], char* lds, int m0, int n0,
                                              int wave, int lane) {
    constexpr int BM = 64 * MI, BN = 64 * NJ, WCOLS = 32 * NJ;
    const int wave_n0 = n0 + (wave & 1) * WCOLS;
    const bool gelu_all = p.act == FLUX_ACT_GELU_TANH && wave_n0 >= p.act_begin;
    const bool gelu_none = p.act != FLUX_ACT_GELU_TANH || wave_n0 + WCOLS <= p.act_begin;
    if constexpr (NJ == 4) {
        if (wave_n0 < p.qk_cols) {   // the host admits the fusion only when the q/k columns are whole tiles
            const bool ragged = m0 + BM > p.M || m0 / p.qk_seq_len != (m0 + BM - 1) / p.qk_seq_len;
            if (ragged) gemm_epilogue_qk<2 * MI, NJ, 2 * MI, true>(p, acc, lds, m0, n0, 0, wave, lane);
            else gemm_epilogue_qk<2 * MI, NJ, 2 * MI, false>(p, acc, lds, m0, n0, 0, wave, lane);
            return;
        }
    }
    // (with a gate: the fast path loads one gate vector per tile, so the tile must not span batch elements)
    const bool fast = p.vec_io && m0 + BM <= p.M && n0 + BN <= p.N && (gelu_all || gelu_none) &&
                      (p.gate == nullptr || m0 / p.rows_per_batch == (m0 + BM - 1) / p.rows_per_batch) &&
                      (wave_n0 + WCOLS <= p.split_n || wave_n0 >= p.split_n) && (p.bias == nullptr || p.bias_vec) &&
                      static_cast<int64_t>(BM) * p.ldy * 2 < 0x7fffffffLL && static_cast<int64_t>(BM) * p.ldy2 * 2 < 0x7fffffffLL &&
                      static_cast<int64_t>(BM) * p.ldresid * 2 < 0x7fffffffLL;
    if (fast) {
        if (p.gate != nullptr) {
            if (gelu_all) gemm_epilogue_fast<MI, NJ, true, true>(p, acc, lds, m0, n0, wave, lane);
            else gemm_epilogue_fast<MI, NJ, false, true>(p, acc, lds, m0, n0, wave, lane);
        } else {
            if (gelu_all) gemm_epilogue_fast<MI, NJ, true, false>(p, acc, lds, m0, n0, wave, lane);
            else gemm_epilogue_fast<MI, NJ, false, false>(p, acc, lds, m0, n0, wave, lane);
        }
    } else {
        gemm_epilogue_checked<2 * MI, 2 * NJ, 2 * MI>(p, acc, lds, m0, n0, 0, wave, lane);
    }
}

// ------------------------------------------------------------------------------------------------
// Tiled kernel: 64*MI x 64*MI output tile per workgroup of four waves (2 x 2, a wave owns
// 32*MI x 32*MI as (2*MI)^2 accumulators of v_mfma_f32_16x16x32_bf16), K in slabs of 64 = two MFMA
// steps of K = 32. With two whole-slab LDS stages the memory pipeline would drain at every barrier
// (the wait in front of it is for ALL outstanding loads). Here LDS is a ring of five units, a unit
// holding one operand's share of a slab (BM rows x 128 bytes): A(kt) lives in unit 2kt % 5 and
// W(kt) in unit (2kt+1) % 5. While slab kt is computed, slab kt+1 and A(kt+2) occupy the other
// three units. The barrier of slab kt sits a quarter into its last step; right behind it the unit
// of A(kt) is free and takes the loads of W(kt+2), one per slot, and the loads of A(kt+3) follow at
// an even pace in front of the next barrier. The wait in front of a barrier only covers W of the
// next slab: the loads of A two slabs ahead stay in flight across it. Every load has more than
// three quarters of a slab of MFMA time to land and the memory pipeline never runs empty.
//
//   slab kt :  step 0            step 1 = [MFMA x PER*BS] wait+barrier [rest, reads step 0 of kt+1]
//   loads   :  ...... A(kt+2) ......................      |  W(kt+2) x PU, one per slot
//
// Ring offsets are wave-uniform scalars that advance by two units per slab.
// ------------------------------------------------------------------------------------------------
// Multiplies the first ke K slabs of the tile at (m0, n0) into acc (cleared first). On return every
// buffer load of the wave has landed and all waves have passed a barrier, so the ring may be
// reused (the epilogue parks its bf16 blocks there).
// ahead(): loads of the caller's own, requested behind those of the first slabs; they have landed on return.
struct NothingAhead {
    __device__ __forceinline__ void operator()() const {}
};
template <int MI, bool KTAIL, typename Ahead = NothingAhead>
__device__ __forceinline__ void gemm_tile_slabs(const GemmParams& p, char* lds, int m0, int n0, int ke,
                                                f32x4 (&acc)[2 * MI][2 * MI], Ahead ahead = Ahead()) {
    constexpr int NJ = MI;
    constexpr int FM = 2 * MI, FN = 2 * NJ;      // 16-row fragments per wave and side
    constexpr int BM = 64 * MI, BN = BM, BK = 64;
    constexpr int ROWB = BK * 2, KSUB = BK / 32;
    constexpr int UNIT = BM * ROWB, NU = 5;
    constexpr int PU = BM / 32;                  // buffer loads per thread per unit
    constexpr int NL = 2 * PU;                   // loads per group G(kt) = W(kt+1), A(kt+2)
    constexpr int WROWS = 32 * MI, WCOLS = 32 * NJ;
    constexpr int READS = FM + FN, MFMAS = FM * FN, PER = MFMAS / READS;
    constexpr int BS = READS / 4;                // slots of the last step in front of the barrier
    constexpr int NSLOT = KSUB * READS;          // issue slots per slab
    constexpr int GB = (KSUB - 1) * READS + BS;  // first slot behind the barrier
    constexpr int EARLY = PU;                    // W loads of a group, all issued right behind the previous slab's barrier
    static_assert(MFMAS % READS == 0 && KSUB == 2 && NSLOT == 2 * NL && NSLOT - GB >= PU, "schedule shape");
    static_assert(2 * (NSLOT - GB) >= READS, "the next slab's first fragments are read two per slot behind the barrier");
    static_assert(4 * WROWS * WCOLS * 2 <= NU * UNIT, "epilogue tile must fit the ring");
    (void)BN; (void)WCOLS;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;

    // loader mapping: LDS slot (row = pass*32 + tid/8, position tid%8) holds logical chunk
    // position ^ ((row>>1)&7) of that row
    const int lrow = tid >> 3;
    const int lchunk = (tid & 7) ^ ((lrow >> 1) & 7);
    const int rows_a = min(p.M - m0, BM), rows_b = min(p.N - n0, BN);
    const int64_t a0 = row_of_a(p, m0);
    bf16_t* const base_a = const_cast<bf16_t*>(p.A + a0);
    bf16_t* const base_b = const_cast<bf16_t*>(p.W + static_cast<int64_t>(n0) * p.ldw);
    const int bytes_a = static_cast<int>((row_of_a(p, m0 + rows_a - 1) - a0 + p.K) * 2);
    const int bytes_b = static_cast<int>(((rows_b - 1) * p.ldw + p.K) * 2);
    uint32_t voff_a[PU], voff_b[PU];
#pragma unroll
    for (int i = 0; i < PU; ++i) {
        const int r = i * 32 + lrow;
        voff_a[i] = r < rows_a ? static_cast<uint32_t>((row_of_a(p, m0 + r) - a0 + lchunk * 8) * 2) : kOutOfRange;
        voff_b[i] = r < rows_b ? static_cast<uint32_t>((r * p.ldw + lchunk * 8) * 2) : kOutOfRange;
    }
    // the slab range ends at ke: everything from there on reads as zeros, like the K tail
    const int k_end = min(p.K, ke * BK);
    // Slabs past the end and the part of the last slab past K read as zeros. With a K tail (KTAIL)
    // that is "this thread's chunk starts at or past K" (K is a multiple of 8, so a chunk is all in
    // or all out) and the mask is a per-lane offset bit. Without one a slab is all in or all out,
    // the mask is wave-uniform and selects a buffer resource of zero records instead, which keeps
    // the vector ALU out of the loop.
    auto slab_mask = [&](int kt) -> uint32_t {
        if constexpr (KTAIL) return kt * BK + lchunk * 8 >= k_end ? kOutOfRange : 0u;
        else return kt * BK >= k_end ? kOutOfRange : 0u;
    };
    // ring offsets are wave-uniform byte offsets of a unit inside the ring
    auto load_a = [&](int uoff, int pass, int kt, uint32_t mask) {
        if constexpr (KTAIL) {
            load_chunk(__builtin_amdgcn_make_buffer_rsrc(base_a, 0, bytes_a, kRsrcFlags), lds + uoff + pass * 4096 + wave * 1024,
                       voff_a[pass] | mask, kt * ROWB);
        } else {
            load_chunk(__builtin_amdgcn_make_buffer_rsrc(base_a, 0, mask ? 0 : bytes_a, kRsrcFlags),
                       lds + uoff + pass * 4096 + wave * 1024, voff_a[pass], kt * ROWB);
        }
    };
    auto load_w = [&](int uoff, int pass, int kt, uint32_t mask) {
        if constexpr (KTAIL) {
            load_chunk(__builtin_amdgcn_make_buffer_rsrc(base_b, 0, bytes_b, kRsrcFlags), lds + uoff + pass * 4096 + wave * 1024,
                       voff_b[pass] | mask, kt * ROWB);
        } else {
            load_chunk(__builtin_amdgcn_make_buffer_rsrc(base_b, 0, mask ? 0 : bytes_b, kRsrcFlags),
                       lds + uoff + pass * 4096 + wave * 1024, voff_b[pass], kt * ROWB);
        }
    };

    // fragment addressing
    // v_mfma_f32_16x16x32_bf16 operand: lane holds row lane % 16, k = (lane / 16) * 8 .. +8 of a K=32 step
    const int frow = lane & 15, fq = lane >> 4;
    int koff_a[KSUB], koff_w[KSUB];
#pragma unroll
    for (int kk = 0; kk < KSUB; ++kk) {
        const int ko = ((kk * 4 + fq) ^ ((frow >> 1) & 7)) * 16;
        koff_a[kk] = (wm * WROWS + frow) * ROWB + ko;
        koff_w[kk] = (wn * WCOLS + frow) * ROWB + ko;
    }

#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = 0.0f;

    bf16x8 xa[2][FM], wb[2][FN];
    // r-th fragment of K-step kk of the slab whose units start at ua / uw, in the order the MFMAs
    // first need them: x0, w0..w(FN-1), x1..x(FM-1)
    auto read_frag = [&](int buf, int ua, int uw, int kk, int r) {
        const char* pa = lds + (ua + koff_a[kk]);
        const char* pw = lds + (uw + koff_w[kk]);
        if (r == 0) xa[buf][0] = *reinterpret_cast<const bf16x8*>(pa);
        else if (r <= FN) wb[buf][r - 1] = *reinterpret_cast<const bf16x8*>(pw + (r - 1) * 16 * ROWB);
        else xa[buf][r - FN] = *reinterpret_cast<const bf16x8*>(pa + (r - FN) * 16 * ROWB);
    };
    auto mfma_one = [&](int buf, int idx) {
        // boustrophedon over the accumulator grid: from one MFMA to the next only one of the two
        // operands changes, also at the end of a row (about 1 % less time at the power limit)
        const int i = idx / FN, j = (i & 1) ? FN - 1 - idx % FN : idx % FN;
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[buf][j], xa[buf][i], acc[i][j], 0, 0, 0);
    };

    // ua/uw: units of slab kt, ua1/uw1: of slab kt+1, ua2: of A(kt+2); W(kt+2) takes over ua once
    // the barrier has retired it. m2: load mask of slab kt+2; the mask of slab kt+3 is
    // worked out in the shadow of an MFMA so that the loop back-edge carries register moves only.
    auto slab = [&](int kt, int ua, int uw, int ua1, int uw1, int ua2, uint32_t m2, uint32_t& m3) {
        const int uw2 = ua;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < NSLOT; ++s) {
            const int stp = s / READS, r = s % READS;
            if (s == GB) {
                wait_loads_and_barrier<PU>();  // slab kt+1 is complete in LDS; this slab's units are free
                __builtin_amdgcn_sched_barrier(0);
            }
            auto slot_reads = [&]() {
                if (stp < KSUB - 1) {
                    read_frag((stp & 1) ^ 1, ua, uw, stp + 1, r);
                } else if (r >= BS) {
                    // two per slot: the last one is requested a few MFMAs before the slab ends, so the
                    // wait at the top of the next slab finds it done
                    const int lo = 2 * (r - BS);
                    for (int f = lo; f < lo + 2 && f < READS; ++f) read_frag(0, ua1, uw1, 0, f);
                }
            };
            // one memory instruction per MFMA interval: the fragment read goes in front of the slot's
            // first MFMA, the buffer load behind it. The slab's first MFMA waits for the fragments
            // requested at the end of the previous slab, and that wait is for every outstanding LDS
            // read: the first read of this slab is therefore issued behind it, not in front.
            if (s != 0) slot_reads();
            mfma_one(stp & 1, r * PER);
            if (s == 0) {
                __builtin_amdgcn_sched_barrier(0);
                slot_reads();
            }
            if (s == 1) m3 = slab_mask(kt + 3);
            __builtin_amdgcn_sched_barrier(0);
            if (s < GB) {
                // A(kt+2): PU loads spread evenly over the slots in front of the barrier
#pragma unroll
                for (int i = 0; i < PU; ++i)
                    if ((i * GB) / PU == s) load_a(ua2, i, kt + 2, m2);
            } else if (s - GB < PU) {
                load_w(uw2, s - GB, kt + 2, m2);   // W(kt+2): one per slot right behind the barrier
            }
#pragma unroll
            for (int m = 1; m < PER; ++m) mfma_one(stp & 1, r * PER + m);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // Prologue: slab 0, A(1) and the first loads of G(0); slab 0 must have landed, the rest flies on.
    {
        const uint32_t k0 = slab_mask(0), k1 = slab_mask(1);
#pragma unroll
        for (int i = 0; i < PU; ++i) load_a(0, i, 0, k0);
#pragma unroll
        for (int i = 0; i < PU; ++i) load_w(UNIT, i, 0, k0);
#pragma unroll
        for (int i = 0; i < PU; ++i) load_a(2 * UNIT, i, 1, k1);
#pragma unroll
        for (int i = 0; i < EARLY; ++i) load_w(3 * UNIT, i, 1, k1);
        ahead();
        wait_loads_and_barrier<PU + EARLY>();
#pragma unroll
        for (int r = 0; r < READS; ++r) read_frag(0, 0, UNIT, 0, r);
        __builtin_amdgcn_sched_barrier(0);
    }
    static_assert(EARLY <= PU, "loads behind the barrier must all belong to W");

    {
        int ua = 0, uw = UNIT, ua1 = 2 * UNIT, uw1 = 3 * UNIT, ua2 = 4 * UNIT;
        uint32_t m2 = slab_mask(2);
        for (int kt = 0; kt < ke; ++kt) {
            uint32_t m3;
            slab(kt, ua, uw, ua1, uw1, ua2, m2, m3);
            // the ring advances by two units
            const int t0 = ua, t1 = uw;
            ua = ua1; uw = uw1; ua1 = ua2; uw1 = t0; ua2 = t1;
            m2 = m3;
        }
    }
    // The last slab's trailing loads were masked (they move no data but still write zeros to LDS):
    // retire them before the epilogue reuses the ring.
    wait_vmem_all();
    __syncthreads();
}

// ------------------------------------------------------------------------------------------------
// Rectangular tiles: (32*FM) x (32*FN) per workgroup, a wave owns (16*FM) x (16*FN) as FM x FN
// accumulators. One workgroup per CU means a launch costs whole rounds of 256 tiles; 4608 x 3072
// (linear2 of the Flux block) is 216 tiles of 256 x 256, 0.84 of a round with 40 CUs idle, but
// exactly 256 tiles of 288 x 192 (FM = 9, FN = 6: 216 accumulation registers). The main loop is the
// one above with the two operands' slabs in rings of their own, because their units now differ in
// size: three units of A (BM rows x 128 bytes) and two of W (BN rows), 156 KB. While slab kt is
// multiplied, A(kt+1), W(kt+1) and A(kt+2) occupy the other units; behind the barrier of slab kt the
// unit of W(kt) takes W(kt+2), and the loads of A(kt+3) go into the unit of A(kt) in front of the
// next barrier. A step has FM + FN fragment reads for FM * FN MFMAs, which no longer divide: slot r
// issues MFMAs [r * MFMAS / READS, (r + 1) * MFMAS / READS).
// Rows past M or N read as zeros and are not stored.
// ------------------------------------------------------------------------------------------------
template <int FM, int FN, bool KTAIL, typename Ahead = NothingAhead>
__device__ __forceinline__ void gemm_rect_slabs(const GemmParams& p, char* lds, int m0, int n0, int ke, f32x4 (&acc)[FM][FN], Ahead ahead = Ahead()) {
    constexpr int BM = 32 * FM, BN = 32 * FN, BK = 64;
    constexpr int ROWB = BK * 2, KSUB = BK / 32;
    constexpr int UNIT_A = BM * ROWB, UNIT_W = BN * ROWB, W0 = 3 * UNIT_A;   // W ring behind the A ring
    constexpr int PA = BM / 32, PW = BN / 32;    // buffer loads per thread per unit of A / W
    constexpr int WROWS = 16 * FM, WCOLS = 16 * FN;
    constexpr int READS = FM + FN, MFMAS = FM * FN;
    constexpr int BS = READS / 4;                // slots of the last step in front of the barrier
    constexpr int NSLOT = KSUB * READS;          // issue slots per slab
    constexpr int GB = (KSUB - 1) * READS + BS;  // first slot behind the barrier
    static_assert(KSUB == 2 && GB >= PA && NSLOT - GB >= PW && MFMAS >= READS, "schedule shape");
    static_assert(2 * (NSLOT - GB) >= READS, "the next slab's first fragments are read two per slot behind the barrier");
    static_assert(BM % 32 == 0 && BN % 32 == 0 && (WROWS / 2) % 8 == 0 && (WCOLS / 2) % 8 == 0, "row swizzle must not see the wave offset");
    static_assert(3 * UNIT_A + 2 * UNIT_W <= 160 * 1024, "rings must fit the LDS");
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;

    // loader mapping as in the square kernel: LDS slot (row = pass*32 + tid/8, position tid%8) holds
    // logical chunk position ^ ((row>>1)&7) of that row
    const int lrow = tid >> 3;
    const int lchunk = (tid & 7) ^ ((lrow >> 1) & 7);
    const int rows_a = min(p.M - m0, BM), rows_b = min(p.N - n0, BN);
    const int64_t a0 = row_of_a(p, m0);
    bf16_t* const base_a = const_cast<bf16_t*>(p.A + a0);
    bf16_t* const base_b = const_cast<bf16_t*>(p.W + static_cast<int64_t>(n0) * p.ldw);
    const int bytes_a = static_cast<int>((row_of_a(p, m0 + rows_a - 1) - a0 + p.K) * 2);
    const int bytes_b = static_cast<int>(((rows_b - 1) * p.ldw + p.K) * 2);
    uint32_t voff_a[PA], voff_b[PW];
#pragma unroll
    for (int i = 0; i < PA; ++i) voff_a[i] = i * 32 + lrow < rows_a ? static_cast<uint32_t>((row_of_a(p, m0 + i * 32 + lrow) - a0 + lchunk * 8) * 2) : kOutOfRange;
#pragma unroll
    for (int i = 0; i < PW; ++i) voff_b[i] = i * 32 + lrow >= rows_b ? kOutOfRange : static_cast<uint32_t>(((i * 32 + lrow) * p.ldw + lchunk * 8) * 2);
    const int k_end = min(p.K, ke * BK);
    auto slab_mask = [&](int kt) -> uint32_t {
        if constexpr (KTAIL) return kt * BK + lchunk * 8 >= k_end ? kOutOfRange : 0u;
        else return kt * BK >= k_end ? kOutOfRange : 0u;
    };
    auto load_a = [&](int uoff, int pass, int kt, uint32_t mask) {
        if constexpr (KTAIL) {
            load_chunk(__builtin_amdgcn_make_buffer_rsrc(base_a, 0, bytes_a, kRsrcFlags), lds + uoff + pass * 4096 + wave * 1024,
                       voff_a[pass] | mask, kt * ROWB);
        } else {
            load_chunk(__builtin_amdgcn_make_buffer_rsrc(base_a, 0, mask ? 0 : bytes_a, kRsrcFlags),
                       lds + uoff + pass * 4096 + wave * 1024, voff_a[pass], kt * ROWB);
        }
    };
    auto load_w = [&](int uoff, int pass, int kt, uint32_t mask) {
        if constexpr (KTAIL) {
            load_chunk(__builtin_amdgcn_make_buffer_rsrc(base_b, 0, bytes_b, kRsrcFlags), lds + W0 + uoff + pass * 4096 + wave * 1024,
                       voff_b[pass] | mask, kt * ROWB);
        } else {
            load_chunk(__builtin_amdgcn_make_buffer_rsrc(base_b, 0, mask ? 0 : bytes_b, kRsrcFlags),
                       lds + W0 + uoff + pass * 4096 + wave * 1024, voff_b[pass], kt * ROWB);
        }
    };

    const int frow = lane & 15, fq = lane >> 4;
    int koff_a[KSUB], koff_w[KSUB];
#pragma unroll
    for (int kk = 0; kk < KSUB; ++kk) {
        const int ko = ((kk * 4 + fq) ^ ((frow >> 1) & 7)) * 16;
        koff_a[kk] = (wm * WROWS + frow) * ROWB + ko;
        koff_w[kk] = W0 + (wn * WCOLS + frow) * ROWB + ko;
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = 0.0f;

    bf16x8 xa[2][FM], wb[2][FN];
    auto read_frag = [&](int buf, int ua, int uw, int kk, int r) {
        const char* pa = lds + (ua + koff_a[kk]);
        const char* pw = lds + (uw + koff_w[kk]);
        if (r == 0) xa[buf][0] = *reinterpret_cast<const bf16x8*>(pa);
        else if (r <= FN) wb[buf][r - 1] = *reinterpret_cast<const bf16x8*>(pw + (r - 1) * 16 * ROWB);
        else xa[buf][r - FN] = *reinterpret_cast<const bf16x8*>(pa + (r - FN) * 16 * ROWB);
    };
    auto mfma_one = [&](int buf, int idx) {
        const int i = idx / FN, j = (i & 1) ? FN - 1 - idx % FN : idx % FN;   // boustrophedon, as above
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[buf][j], xa[buf][i], acc[i][j], 0, 0, 0);
    };

    // ua, ua1, ua2: units of A(kt), A(kt+1), A(kt+2); uw, uw1: of W(kt), W(kt+1); W(kt+2) takes over uw
    // behind the barrier
    auto slab = [&](int kt, int ua, int ua1, int ua2, int uw, int uw1, uint32_t m2, uint32_t& m3) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < NSLOT; ++s) {
            const int stp = s / READS, r = s % READS;
            const int lo = r * MFMAS / READS, hi = (r + 1) * MFMAS / READS;
            if (s == GB) {
                wait_loads_and_barrier<PA>();  // W(kt+1) has landed (A(kt+1) before it); this slab's units are free
                __builtin_amdgcn_sched_barrier(0);
            }
            auto slot_reads = [&]() {
                if (stp < KSUB - 1) {
                    read_frag((stp & 1) ^ 1, ua, uw, stp + 1, r);
                } else if (r >= BS) {
                    const int f0 = 2 * (r - BS);
                    for (int f = f0; f < f0 + 2 && f < READS; ++f) read_frag(0, ua1, uw1, 0, f);
                }
            };
            if (s != 0) slot_reads();
            mfma_one(stp & 1, lo);
            if (s == 0) {
                __builtin_amdgcn_sched_barrier(0);
                slot_reads();
            }
            if (s == 1) m3 = slab_mask(kt + 3);
            __builtin_amdgcn_sched_barrier(0);
            if (s < GB) {
#pragma unroll
                for (int i = 0; i < PA; ++i)
                    if ((i * GB) / PA == s) load_a(ua2, i, kt + 2, m2);
            } else if (s - GB < PW) {
                load_w(uw, s - GB, kt + 2, m2);
            }
#pragma unroll
            for (int m = lo + 1; m < hi; ++m) mfma_one(stp & 1, m);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    {
        const uint32_t k0 = slab_mask(0), k1 = slab_mask(1);
#pragma unroll
        for (int i = 0; i < PA; ++i) load_a(0, i, 0, k0);
#pragma unroll
        for (int i = 0; i < PW; ++i) load_w(0, i, 0, k0);
#pragma unroll
        for (int i = 0; i < PA; ++i) load_a(UNIT_A, i, 1, k1);
#pragma unroll
        for (int i = 0; i < PW; ++i) load_w(UNIT_W, i, 1, k1);
        ahead();
        wait_loads_and_barrier<PA + PW>();
#pragma unroll
        for (int r = 0; r < READS; ++r) read_frag(0, 0, 0, 0, r);
        __builtin_amdgcn_sched_barrier(0);
    }
    {
        int ua = 0, ua1 = UNIT_A, ua2 = 2 * UNIT_A, uw = 0, uw1 = UNIT_W;
        uint32_t m2 = slab_mask(2);
        for (int kt = 0; kt < ke; ++kt) {
            uint32_t m3;
            slab(kt, ua, ua1, ua2, uw, uw1, m2, m3);
            const int t0 = ua, t1 = uw;
            ua = ua1; ua1 = ua2; ua2 = t0;
            uw = uw1; uw1 = t1;
            m2 = m3;
        }
    }
    wait_vmem_all();
    __syncthreads();
}

}  // namespace flux
