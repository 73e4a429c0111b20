// kernels_delta_bwd.h -- backward pass of the gated delta rule (kernels_delta.h has the forward formulas and the layouts)
//
// With dO, dS1 the gradients of a chunk's outputs and of the state behind it:
//     dU = scale P^T dO + e^{c} K dS1,   Z = T^T (beta dU) = dV,
//     dS0 = e^{b_C} dS1 + Q^T (scale e^{b} dO) - K^T (e^{b} Z)                                (the reverse chain)
//     dA = -tril(Z E^T, -1),  dP = scale tril(dO U^T),  G = dA e^{D} beta (of the column),  H = dP e^{D}
//     dQ = scale e^{b} dO S0^T + H K,   dK = -e^{b} Z S0^T + e^{c} U dS1^T + (G + G^T) K + H^T Q
//     dbeta_j = dU_j . E_j + sum_i dA_ij (k_i . k_j) e^{D_ij} = Z_j . E_j / beta_j      (since Z + A^T Z = beta dU)
//     dg_m = sum_{j < m <= i} (dA A + dP P)_ij + sum_{i >= m} (q_i . dQ1_i + k_i . dK1_i) + sum_{i < m} k_i . dK2_i
//            + e^{b_C} <S0, dS1>,   dQ1, dK1 = the S0 terms of dQ, dK;  dK2 = the dS1 term of dK
// The reverse chain is the forward one with other operands; everything else of all chunks follows at once.  dg is summed over the positions it reaches, not as a difference of running sums.
#pragma once
#include "kernels_delta.h"

namespace helen {

// The reverse chain, built like delta_forward_kernel: wave w owns token tile w of dO, dU and Z and its quarter of dS's rows.  Bound
// as that one is, and it writes dS and Z: 32 sequences of 1000 tokens, 8 heads of 128, bf16: 231 us, 0.46 GB of them.
template <typename In, int DK>
__global__ __launch_bounds__(256, In::kTerms == 1 ? 2 : 1) void delta_backward_kernel(const DeltaArgs a) {
    constexpr int NC = kColumnTiles, NI = In::kTerms, KS = DK / 32, MW = DK / 64;
    typedef typename In::raw raw;
    __shared__ bf16x8 sbuf[KS * 3 * NC * 64], ybuf[2 * NI * NC * 64], wbuf[2 * 3 * NC * 64], dbuf[2 * 3 * NC * 64], zbuf[2 * 3 * NC * 64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = lane & 15, q = lane >> 4;
    const int groups = a.dv_width / (16 * NC);
    const unsigned item = xcd_order(blockIdx.x, gridDim.x);
    if (item >= (unsigned)a.nseq * a.hv * groups) return;
    const int hv = item / groups % a.hv, s = item / groups / a.hv, h = hv / a.group;
    const int col = NC * (16 * (item % groups) + j);
    const Span sp = span_of(a, s);
    const int chunks = (sp.len + kDeltaChunk - 1) / kDeltaChunk;
    const size_t st = (((size_t)s * a.hv + hv) * DK + state_row(MW * w) + 8 * q) * a.dv_width + col;

    f32x4 S[MW][NC];
    load_state<MW, NC>(a.ds1, a.zeros, st, a.dv_width, S);

    bf16x8 kf[KS][NI], kt[MW][2][NI], qt[MW][2][NI], tt[2][3], pt[2][3];
    f32x4 beta, eb, ec;
    float whole;
    Columns<In, NC> y[4];
    const int row = 16 * w + 4 * q;
    const ChainAddress<In, DK> at(a, sp, h, hv, w, lane);
    RowOffsets yrow(a.do_t, row, col);
    unsigned tile_at[4], state_at[4], dv_at[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        state_at[r] = (8 * q + r) * a.dv_width + col;
        tile_at[r] = (4 * q + r) * a.dv_width + col;
        dv_at[r] = (row + r) * a.hv * a.dv_width + col;
    }
    auto load_rows = [&](int c) { at.rows(0, a.kf, c, kf); };
    auto load_columns = [&](int c) {
        at.columns(a.ktf, c, kt);
        at.columns(a.qtf, c, qt);
    };
    auto load_tri = [&](int c, const bf16x8* from, bf16x8 (&to)[2][3]) { at.transposed(from, c, to); };
    auto load_scales = [&](int c) {
        const float* sc = a.sc + (at.vslot + (size_t)c * a.hv) * 256;
        beta = *(const f32x4*)(sc + row);
        eb = *(const f32x4*)(sc + 64 + row);
        ec = *(const f32x4*)(sc + 128 + row);
        whole = (sc + 64)[63];
    };
    // (no conditional loads, see delta_forward_kernel; rows behind the end meet q = k = 0)
    auto load_dout = [&](int c) {
        yrow.clamp(sp.len - c * kDeltaChunk);
        const raw* p = (const raw*)a.dout + (sp.begin + c * kDeltaChunk) * a.do_t + hv * a.do_h;
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = Columns<In, NC>::load(p + yrow.at[r]);
    };
    auto dout = [&](int nc, int r) { return y[r].get(nc); };
    // dS (behind chunk c) and dO (of chunk c) for all waves
    auto share = [&](int c) {
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            if constexpr (MW == 2) {
                bf16x8 t[3];
                split8<3>(S[0][nc], S[1][nc], t);
#pragma unroll
                for (int k = 0; k < 3; ++k) sbuf[((w * 3 + k) * NC + nc) * 64 + lane] = t[k];
            } else {
                share_tile<3, NC>(sbuf, w, nc, lane, S[0][nc]);
            }
            share_tile<NI, NC>(ybuf, w, nc, lane,
                               (f32x4){dout(nc, 0), dout(nc, 1), dout(nc, 2), dout(nc, 3)});
        }
        float* to = a.dstates + ((at.vslot + (size_t)c * a.hv) * DK + state_row(MW * w)) * a.dv_width;
#pragma unroll
        for (int i = 0; i < MW; ++i) store_tile<NC>(to + (size_t)4 * i * a.dv_width, state_at, S[i]);
    };
    if (chunks > 0) {
        const int c = chunks - 1;
        load_dout(c);
        load_rows(c);
        load_scales(c);
        load_tri(c, a.ptf, pt);
        load_tri(c, a.ttf, tt);
        load_columns(c);
        share(c);
    }
    lds_barrier();
    for (int c = chunks - 1; c >= 0; --c) {
        const int next = max(c - 1, 0), n = sp.len - c * kDeltaChunk;
        f32x4 D[NC], P[2][NC];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) D[nc] = P[0][nc] = P[1][nc] = splat4(0.f);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) {
                bf16x8 b[3];
                shared_frag<3, NC>(sbuf, ks, nc, lane, b);
                D[nc] = mm(kf[ks], b, D[nc]);
            }
#pragma unroll
        for (int nc = 0; nc < NC; ++nc)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                bf16x8 b[NI];
                shared_frag<NI, NC>(ybuf, ks, nc, lane, b);
                P[ks][nc] = mm(pt[ks], b, P[ks][nc]);
            }
        const f32x4 head = eb;
        const float hold = whole;
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            f32x4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                D[nc][r] = beta_of(beta[r]) * (ec[r] * D[nc][r] + a.scale * (P[0][nc][r] + P[1][nc][r]));
                x[r] = a.scale * eb[r] * dout(nc, r);
            }
            share_tile<3, NC>(dbuf, w, nc, lane, D[nc]);
            share_tile<3, NC>(wbuf, w, nc, lane, x);
        }
        load_rows(next);
        load_scales(next);
        load_dout(next);
        load_tri(next, a.ptf, pt);
        issue_loads();
        lds_barrier();
        f32x4 Z[NC];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            f32x4 z0 = splat4(0.f), z1 = splat4(0.f);
            bf16x8 b[2][3];
            shared_frag<3, NC>(dbuf, 0, nc, lane, b[0]);
            shared_frag<3, NC>(dbuf, 1, nc, lane, b[1]);
            z0 = mm(tt[0], b[0], z0);
            z1 = mm(tt[1], b[1], z1);
            Z[nc] = z0 + z1;
        }
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            f32x4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = -head[r] * Z[nc][r];
            share_tile<3, NC>(zbuf, w, nc, lane, x);
        }
        store_tile<NC>(a.z + ((at.vslot + (size_t)c * a.hv) * kDeltaChunk + 16 * w) * a.dv_width, tile_at, Z);
        raw* const dv = (raw*)a.dv + ((size_t)(sp.begin + c * kDeltaChunk) * a.hv + hv) * a.dv_width;
        auto put = [&](int r) {
            float x[NC];
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) x[nc] = Z[nc][r];
            Columns<In, NC>::store(dv + dv_at[r], x);
        };
        if (n >= kDeltaChunk) {
#pragma unroll
            for (int r = 0; r < 4; ++r) put(r);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (row + r < n) put(r);
        }
        load_tri(next, a.ttf, tt);
        issue_loads();
        lds_barrier();
#pragma unroll
        for (int i = 0; i < MW; ++i)
#pragma unroll
            for (int nc = 0; nc < NC; ++nc)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[i][nc][r] *= hold;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) {
                bf16x8 b[3], e[3];
                shared_frag<3, NC>(zbuf, ks, nc, lane, b);
                shared_frag<3, NC>(wbuf, ks, nc, lane, e);
#pragma unroll
                for (int i = 0; i < MW; ++i) {
                    S[i][nc] = mm(kt[i][ks], b, S[i][nc]);
                    S[i][nc] = mm(qt[i][ks], e, S[i][nc]);
                }
            }
        load_columns(next);
        issue_loads();
        if (c > 0) share(next);
        lds_barrier();
    }
    if (a.ds0) {
        float* const to = a.ds0 + (((size_t)s * a.hv + hv) * DK + state_row(MW * w)) * a.dv_width;
#pragma unroll
        for (int i = 0; i < MW; ++i) store_tile<NC>(to + (size_t)4 * i * a.dv_width, state_at, S[i]);
    }
}

// The reverse chain for few long ones, as delta_forward_long_kernel: waves 0 .. 3 do what the next chunk waits for, waves 4 .. 7
// what comes from dO alone, one chunk ahead (P^T dO and Q^T (scale e^b dO), handed over as fp32 tiles), and the stores.  8191
// tokens in two sequences, 16 heads of 128, bf16: 182 us, 2.3 us a chunk of the longer one.  fp32 at width 128 spills 7 registers.
template <typename In, int DK>
__global__ __launch_bounds__(512) void delta_backward_long_kernel(const DeltaArgs a) {
    constexpr int NI = In::kTerms, KS = DK / 32, MW = DK / 64;
    constexpr bool OWN = MW == 2;
    typedef typename In::raw raw;
    __shared__ bf16x8 sbuf[KS * 3 * 64], ybuf[2 * NI * 64], wbuf[2 * 3 * 64], dbuf[2 * 3 * 64], zbuf[2 * 3 * 64];
    __shared__ f32x4 pfull[4 * 64], wfull[4 * MW * 64], zfull[4 * 64], sfull[4 * MW * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
    const int j = lane & 15, q = lane >> 4;
    const int groups = a.dv_width / 16;
    const unsigned item = xcd_order(blockIdx.x, gridDim.x);
    if (item >= (unsigned)a.nseq * a.hv * groups) return;
    const int hv = item / groups % a.hv, s = item / groups / a.hv, h = hv / a.group;
    const int col = 16 * (item % groups) + j;
    const Span sp = span_of(a, s);
    const int chunks = (sp.len + kDeltaChunk - 1) / kDeltaChunk;
    const int row = 16 * w + 4 * q;
    const ChainAddress<In, DK> at(a, sp, h, hv, w, lane);
    unsigned tile_at[4], state_at[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        tile_at[r] = (4 * q + r) * a.dv_width + col;
        state_at[r] = (8 * q + r) * a.dv_width + col;
    }

    auto chain = [&](auto two_) {
        constexpr bool TWO = decltype(two_)::value;
        f32x4 S[MW][1];
        load_state<MW, 1>(a.ds1, a.zeros, (((size_t)s * a.hv + hv) * DK + state_row(MW * w) + 8 * q) * a.dv_width + col, a.dv_width, S);
        struct Operands {
            bf16x8 kf[KS][NI], kt[MW][2][NI], tt[TWO ? 2 : 1][3];
            f32x4 beta, eb, ec;
            float whole;
        } first, second;
        bf16x8 own[3];
        auto load_k = [&](int c, Operands& to) {
            const float* sc = a.sc + (at.vslot + (size_t)c * a.hv) * 256;
            at.rows(OWN ? w : 0, a.kf, c, to.kf);
            to.beta = *(const f32x4*)(sc + row);
            to.ec = *(const f32x4*)(sc + 128 + row);
        };
        auto load_scales = [&](int c, Operands& to) {
            const float* sc = a.sc + (at.vslot + (size_t)c * a.hv) * 256;
            to.eb = *(const f32x4*)(sc + 64 + row);
            to.whole = (sc + 64)[63];
        };
        auto share_state = [&]() {
            if constexpr (OWN) {
                split8<3>(S[0][0], S[1][0], own);
#pragma unroll
                for (int k = 0; k < 3; ++k) sbuf[(w * 3 + k) * 64 + lane] = own[k];
            } else {
                share_tile<3, 1>(sbuf, w, 0, lane, S[0][0]);
            }
#pragma unroll
            for (int i = 0; i < MW; ++i) sfull[(MW * w + i) * 64 + lane] = S[i][0];
        };
        auto step = [&](int c, Operands& now, Operands& then) {
            const int next = max(c - 1, 0);
            f32x4 sum[2] = {splat4(0.f), splat4(0.f)}, D;
            const f32x4 p = pfull[w * 64 + lane];
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                bf16x8 b[3];
                if (OWN && i == 0) {
#pragma unroll
                    for (int t = 0; t < 3; ++t) b[t] = own[t];
                } else {
                    shared_frag<3, 1>(sbuf, OWN ? (w + i) & 3 : i, 0, lane, b);
                }
                sum[i & 1] = mm(now.kf[i], b, sum[i & 1]);
            }
            load_k(next, then);
            between_products<KS * 3>();
#pragma unroll
            for (int r = 0; r < 4; ++r) D[r] = beta_of(now.beta[r]) * (now.ec[r] * (sum[0][r] + sum[1][r]) + a.scale * p[r]);
            share_tile<3, 1>(dbuf, w, 0, lane, D);
            issue_loads();
            lds_barrier();
            bf16x8 x[2][3];
            shared_frag<3, 1>(dbuf, 1, 0, lane, x[1]);
            if constexpr (TWO) shared_frag<3, 1>(dbuf, 0, 0, lane, x[0]);
            f32x4 z0 = splat4(0.f), z1 = splat4(0.f);
            if constexpr (TWO) z0 = mm(now.tt[0], x[0], z0);
            z1 = mm(now.tt[TWO], x[1], z1);
            at.transposed(a.ttf, next, then.tt);
            load_scales(next, then);
            between_products<TWO ? 12 : 6>();
            f32x4 Z = z0 + z1;
            zfull[w * 64 + lane] = Z;
#pragma unroll
            for (int r = 0; r < 4; ++r) Z[r] *= -now.eb[r];
            share_tile<3, 1>(zbuf, w, 0, lane, Z);
            issue_loads();
            lds_barrier();
            shared_frag<3, 1>(zbuf, 0, 0, lane, x[0]);
            shared_frag<3, 1>(zbuf, 1, 0, lane, x[1]);
#pragma unroll
            for (int i = 0; i < MW; ++i) {
                const f32x4 y = wfull[(MW * w + i) * 64 + lane];
#pragma unroll
                for (int r = 0; r < 4; ++r) S[i][0][r] = now.whole * S[i][0][r] + y[r];
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int i = 0; i < MW; ++i) S[i][0] = mm(now.kt[i][ks], x[ks], S[i][0]);
            at.columns(a.ktf, next, then.kt);
            between_products<2 * MW * 3>();
            share_state();
            issue_loads();
            lds_barrier();
        };
        if (chunks > 0) {
            load_k(chunks - 1, first);
            load_scales(chunks - 1, first);
            at.transposed(a.ttf, chunks - 1, first.tt);
            at.columns(a.ktf, chunks - 1, first.kt);
            share_state();
        }
        lds_barrier();
        lds_barrier();
        if (chunks & 1) {
            step(chunks - 1, first, second);
            first = second;
        }
        loads_done();
        for (int c = (chunks & ~1) - 1; c >= 0; c -= 2) {
            step(c, first, second);
            step(c - 1, second, first);
        }
        if (a.ds0) {
            float* const to = a.ds0 + (((size_t)s * a.hv + hv) * DK + state_row(MW * w)) * a.dv_width;
#pragma unroll
            for (int i = 0; i < MW; ++i) store_tile<1>(to + (size_t)4 * i * a.dv_width, state_at, S[i]);
        }
    };
    auto output = [&](auto two_) {
        constexpr bool TWO = decltype(two_)::value;
        bf16x8 qt[MW][2][NI], pt[TWO ? 2 : 1][3];
        f32x4 eb, W[MW];
        Columns<In, 1> y[4];
        RowOffsets yrow(a.do_t, row, col);
        unsigned dv_at[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) dv_at[r] = (row + r) * a.hv * a.dv_width + col;
        auto load = [&](int c) {
            eb = *(const f32x4*)(a.sc + (at.vslot + (size_t)c * a.hv) * 256 + 64 + row);
            yrow.clamp(sp.len - c * kDeltaChunk);
            const raw* p = (const raw*)a.dout + (sp.begin + c * kDeltaChunk) * a.do_t + hv * a.do_h;
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = Columns<In, 1>::load(p + yrow.at[r]);
        };
        auto share = [&]() {
            f32x4 x = {y[0].get(0), y[1].get(0), y[2].get(0), y[3].get(0)};
            share_tile<NI, 1>(ybuf, w, 0, lane, x);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] *= a.scale * eb[r];
            share_tile<3, 1>(wbuf, w, 0, lane, x);
        };
        auto from_p = [&]() {
            bf16x8 b[2][NI];
            if constexpr (TWO) shared_frag<NI, 1>(ybuf, 0, 0, lane, b[0]);
            shared_frag<NI, 1>(ybuf, 1, 0, lane, b[1]);
            f32x4 p0 = splat4(0.f), p1 = splat4(0.f);
            if constexpr (TWO) p0 = mm(pt[0], b[0], p0);
            p1 = mm(pt[TWO], b[1], p1);
            pfull[w * 64 + lane] = p0 + p1;
        };
        auto from_q = [&]() {
            bf16x8 b[2][3];
            shared_frag<3, 1>(wbuf, 0, 0, lane, b[0]);
            shared_frag<3, 1>(wbuf, 1, 0, lane, b[1]);
#pragma unroll
            for (int i = 0; i < MW; ++i) {
                W[i] = splat4(0.f);
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) W[i] = mm(qt[i][ks], b[ks], W[i]);
            }
        };
        if (chunks > 0) {
            load(chunks - 1);
            at.transposed(a.ptf, chunks - 1, pt);
            at.columns(a.qtf, chunks - 1, qt);
            share();
        }
        lds_barrier();
        if (chunks > 0) {
            const int next = max(chunks - 2, 0);
            from_p();
            from_q();
            load(next);
            at.transposed(a.ptf, next, pt);
            at.columns(a.qtf, next, qt);
        }
        issue_loads();
        lds_barrier();
        const int part = 4 * (item % groups) + w;
        unsigned fetched = 0;
        for (int c = chunks - 1; c >= 0; --c) {
            const int after = max(c - 2, 0);
            settle(fetched);
            {
                const int ahead = max(c - kFetchAhead - 1, 0);
                const size_t t0 = (at.vslot + (size_t)ahead * a.hv) * kTriFrags * 3 * 64, k0 = (at.kslot + (size_t)ahead * a.hk) * at.kSlot;
                const Piece piece[5] = {{a.kf + k0, DK / 8 * NI}, {a.ttf + t0, kTriFrags * 3}, {a.ktf + k0, DK / 8 * NI}, {a.qtf + k0, DK / 8 * NI}, {a.ptf + t0, kTriFrags * 3}};
                fetched = fetch(piece, part, lane);
            }
#pragma unroll
            for (int i = 0; i < MW; ++i) wfull[(MW * w + i) * 64 + lane] = W[i];
            share();                        // dO of chunk c - 1
            load(after);
            issue_loads();
            lds_barrier();
            from_p();
            at.transposed(a.ptf, after, pt);
            {
                float* const to = a.dstates + ((at.vslot + (size_t)c * a.hv) * DK + state_row(MW * w)) * a.dv_width;
#pragma unroll
                for (int i = 0; i < MW; ++i) {
                    const f32x4 x[1] = {sfull[(MW * w + i) * 64 + lane]};
                    store_tile<1>(to + (size_t)4 * i * a.dv_width, state_at, x);
                }
            }
            issue_loads();
            lds_barrier();
            from_q();
            at.columns(a.qtf, after, qt);
            {
                const f32x4 Z[1] = {zfull[w * 64 + lane]};
                store_tile<1>(a.z + ((at.vslot + (size_t)c * a.hv) * kDeltaChunk + 16 * w) * a.dv_width, tile_at, Z);
                const int n = sp.len - c * kDeltaChunk;
                raw* const dv = (raw*)a.dv + ((size_t)(sp.begin + c * kDeltaChunk) * a.hv + hv) * a.dv_width;
                if (n >= kDeltaChunk) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) dv[dv_at[r]] = In::from_f32(Z[0][r]);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (row + r < n) dv[dv_at[r]] = In::from_f32(Z[0][r]);
                }
            }
            issue_loads();
            lds_barrier();
        }
    };
    if (wave < 4) w < 2 ? chain(Is<true>()) : chain(Is<false>());
    else w < 2 ? output(Is<true>()) : output(Is<false>());
}

// sum over the 16 lanes of a quarter, over a wave, and running sums
__device__ __forceinline__ float sum16(float x) { return dpp_add<0x121>(dpp_add<0x122>(dpp_add<0x124>(dpp_add<0x128>(x)))); }
__device__ __forceinline__ float sum64(float x) {
    x = sum16(x);
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}
__device__ __forceinline__ float sum_before(float x, int lane) {      // over the lanes below
    float sum = x;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const float y = __shfl_up(sum, m);
        sum += lane >= m ? y : 0.f;
    }
    const float y = __shfl_up(sum, 1);
    return lane ? y : 0.f;
}
__device__ __forceinline__ float sum_from(float x, int lane) {        // over this lane and those above
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const float y = __shfl_down(x, m);
        x += lane + m < 64 ? y : 0.f;
    }
    return x;
}

// ------------------------------------------------------------------------------------------------
// dQ, dK, dbeta and dg of one chunk: a workgroup of DK / 16 waves per (slot, key head).  The value heads of the key head follow
// one another and are summed in registers: no atomics, one order.
//   64 x DK results: wave w has dk tile w (column j is state_row(w) + 8 (j / 4) + j % 4) of all four token tiles
//   64 x 64 results: the ten tiles on and below the diagonal go round the waves
// dv is walked 32 columns a step: Z, E and dO of the step as fragments in LDS (two buffers, one barrier a step), the rows of
// S0 and dS1 straight into the registers of the one wave that needs them.  What it waits for is memory, so loads run two
// steps ahead, over the ends of the heads too, and every wave stages as much as the others.
// What bounds it: one workgroup a CU (128 KB of LDS, 256 registers; with shared key heads 9 of them spilled at width 128, 7 for fp16
// and 12 for fp32) has nothing to hide its start and its 64 x 64 part behind: its waves wait for half of the time, the matrix pipe is
// busy for 20 % of it.  32 x 1000 tokens, 4 key and 8 value heads of 128, bf16: 377 us for 0.56 GB read and 0.12 written, 1.8 TB/s
// (500 us with loads one step ahead).
// ------------------------------------------------------------------------------------------------
template <typename In, int DK, bool SHARED>
__global__ __launch_bounds__(DK * 4) void delta_grads_kernel(const DeltaArgs a) {
    constexpr int NI = In::kTerms, W = DK / 16, TPW = (10 + W - 1) / W, RB = 64 / W;
    typedef typename In::raw raw;
    constexpr int kStage = 4 * (6 + NI);
    __shared__ bf16x8 stage[2 * kStage * 64];
    __shared__ bf16x8 fr[3 * (8 + 2 * kTriFrags) * 64];
    __shared__ __attribute__((aligned(16))) Decays dec;
    __shared__ float bs[64], scl[192], sums[2][W][64], dbeta[64], gamma[W], part[W][64];
    static_assert(sizeof(stage) >= 3 * 64 * kTriStride * 4, "the 64 x 64 gradients take the stage's place");
    float* const gmat = (float*)stage;
    float* const hmat = gmat + 64 * kTriStride;
    float* const dmat = hmat + 64 * kTriStride;
    const int lane0 = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slot = blockIdx.x / a.hk, h = blockIdx.x % a.hk;
    Span sp;
    const int s = sequence_of(a, slot, lane0, &sp);
    const int c = slot - sp.slot;
    const int start = sp.begin + c * kDeltaChunk;
    const int n = min(kDeltaChunk, sp.begin + sp.len - start);
    if (c < 0 || n <= 0) {
        if (s == a.nseq - 1) {      // rows behind the last sequence: their gradients are zero
            const int end = sp.begin + sp.len;
            const int lo = max(end, (slot - a.nseq) * kDeltaChunk), hi = min(a.tokens, (slot - a.nseq + 1) * kDeltaChunk);
            for (int t = lo; t < hi; ++t) {
                for (int d = threadIdx.x; d < DK; d += DK * 4)
                    ((raw*)a.dq)[((size_t)t * a.hk + h) * DK + d] = ((raw*)a.dk)[((size_t)t * a.hk + h) * DK + d] = raw(0);
                for (int hv = h * a.group; hv < (h + 1) * a.group; ++hv) {
                    for (int d = threadIdx.x; d < a.dv_width; d += DK * 4)
                        ((raw*)a.dv)[((size_t)t * a.hv + hv) * a.dv_width + d] = raw(0);
                    if (threadIdx.x == 0) a.dg[(size_t)t * a.hv + hv] = a.dbeta[(size_t)t * a.hv + hv] = 0.f;
                }
            }
        }
        return;
    }
    const size_t kslot = (size_t)slot * a.hk + h;
    int tm[TPW], tn[TPW];          // this wave's 64 x 64 tiles
    bool own[TPW];
#pragma unroll
    for (int t = 0; t < TPW; ++t) {
        own[t] = w + W * t < 10;
        const int id = own[t] ? w + W * t : w;
        tm[t] = id < 1 ? 0 : (id < 3 ? 1 : (id < 6 ? 2 : 3));
        tn[t] = id - tm[t] * (tm[t] + 1) / 2;
    }
    f32x4 dQ[4], dK[4];            // by token tile, summed over the value heads
    if constexpr (SHARED) {
#pragma unroll
        for (int m = 0; m < 4; ++m) dQ[m] = dK[m] = splat4(0.f);
    }
    // Who stages what of token tile w & 3: with four waves everything; with eight waves 0 .. 3 Z and the first half of dO's columns,
    // 4 .. 7 E and the second half.  No load is conditional (behind one the compiler's counts of what is in flight are too low).
    constexpr int YH = W == 4 ? 2 : 1;
    const int second = W == 4 ? 0 : w >> 2;
    const int steps = a.dv_width / 32, last = a.group * steps - 1;
    struct Rows {                  // of the states: dk row j of the wave's tile, columns 4 q and 16 + 4 q of the step
        f32x4 s[2], d[2];
    } rows[2];
    struct Tokens {                // of the stage
        f32x4 x[2], e[2], y[YH];
    } toks[2];
    auto load_rows = [&](int at, Rows& to, unsigned lane) {      // step `at` of all heads' steps
        const int step = min(at, last), head = step / steps, d0 = 32 * (step - head * steps);
        const size_t base = (((size_t)slot * a.hv + h * a.group + head) * DK + state_row(w)) * a.dv_width + d0;
        const unsigned off = (8 * (lane >> 2 & 3) + (lane & 3)) * a.dv_width + 4 * (lane >> 4);
        to.s[0] = *(const f32x4*)(a.states + base + off);
        to.s[1] = *(const f32x4*)(a.states + base + 16 + off);
        to.d[0] = *(const f32x4*)(a.dstates + base + off);
        to.d[1] = *(const f32x4*)(a.dstates + base + 16 + off);
    };
    auto load_tokens = [&](int at, Tokens& to, unsigned lane) {
        const int step = min(at, last), head = step / steps, d0 = 32 * (step - head * steps), hv = h * a.group + head;
        const size_t base = (((size_t)slot * a.hv + hv) * kDeltaChunk + 16 * (w & 3)) * a.dv_width + d0;
        const unsigned off = (lane & 15) * a.dv_width + 4 * (lane >> 4);
        const float* const x = (second ? a.e : a.z) + base;
        to.x[0] = *(const f32x4*)(x + off);
        to.x[1] = *(const f32x4*)(x + 16 + off);
        if constexpr (W == 4) {
            to.e[0] = *(const f32x4*)(a.e + base + off);
            to.e[1] = *(const f32x4*)(a.e + base + 16 + off);
        }
        const int row = min(16 * (w & 3) + (int)(lane & 15), n - 1);
        const raw* const y = (const raw*)a.dout + (start + row) * a.do_t + hv * a.do_h + d0 + 16 * second + 4 * (lane >> 4);
#pragma unroll
        for (int i = 0; i < YH; ++i) to.y[i] = load4<In>(y + 16 * i);
    };
    auto put = [&](bf16x8* to, const Tokens& from, unsigned lane) {
        bf16x8 t[3];
        split8<3>(from.x[0], from.x[1], t);
#pragma unroll
        for (int k = 0; k < 3; ++k) to[(12 * second + (w & 3) * 3 + k) * 64 + lane] = t[k];
        const bool live = 16 * (w & 3) + (int)(lane & 15) < n;
#pragma unroll
        for (int i = 0; i < YH; ++i) {
            u32x2 y[NI];
            split4<NI>(live ? from.y[i] : splat4(0.f), y);
#pragma unroll
            for (int k = 0; k < NI; ++k) ((u32x2*)(to + (24 + (w & 3) * NI + k) * 64 + lane))[second + i] = y[k];
        }
        if constexpr (W == 4) {
            split8<3>(from.e[0], from.e[1], t);
#pragma unroll
            for (int k = 0; k < 3; ++k) to[(12 + (w & 3) * 3 + k) * 64 + lane] = t[k];
        }
    };
    // gates of a head: g and beta by wave 0, the scales by waves 1 .. 3, a value a thread
    float gate[2] = {0.f, 0.f};
    auto load_gates = [&](int hv) {
        if (w == 0) {
            const int row = min(lane0, n - 1);
            gate[0] = a.g[(start + row) * a.g_t + hv * a.g_h];
            gate[1] = a.beta[(start + row) * a.b_t + hv * a.b_h];
        } else if (w < 4) {
            gate[0] = (a.sc + ((size_t)slot * a.hv + hv) * 256 + 64 * (w - 1))[lane0];
        }
    };
    load_gates(h * a.group);
    load_rows(0, rows[0], lane0);
    load_tokens(0, toks[0], lane0);
    load_rows(1, rows[1], lane0);
    load_tokens(1, toks[1], lane0);

    int at = 0;
    for (int hv = h * a.group; hv < (h + 1) * a.group; ++hv) {
        const unsigned lane = in_block(lane0);      // (nothing of a head's addresses is kept over the loop)
        const int j = lane & 15, q = lane >> 4;
        lds_barrier();
        if (w == 0) {
            dec.set(lane, (int)lane < n ? gate[0] : 0.f);
            bs[lane] = (int)lane < n ? gate[1] : 0.f;
        } else if (w < 4) {
            scl[64 * (w - 1) + lane] = gate[0];
        }
        load_gates(min(hv + 1, (h + 1) * a.group - 1));
        f32x4 q1[4], k1[4], k2[4], da[TPW], dp[TPW];
#pragma unroll
        for (int m = 0; m < 4; ++m) q1[m] = k1[m] = k2[m] = splat4(0.f);
#pragma unroll
        for (int t = 0; t < TPW; ++t) da[t] = dp[t] = splat4(0.f);
        float dots = 0.f;
        put(stage, toks[0], lane);
        load_tokens(at + 2, toks[0], lane);
        auto step = [&](int k, bool more, Rows& rw, Tokens& tk) {        // tk: the next step's tokens
            const bf16x8* const from = stage + (k & 1) * kStage * 64;
            bf16x8 st[3], dt[3];
#pragma unroll
            for (int r = 0; r < 4; ++r) dots += rw.s[0][r] * rw.d[0][r] + rw.s[1][r] * rw.d[1][r];
            split8<3>(rw.s[0], rw.s[1], st);
            split8<3>(rw.d[0], rw.d[1], dt);
            load_rows(at + k + 2, rw, lane);
            lds_barrier();
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                bf16x8 x[3], y[NI];
#pragma unroll
                for (int t = 0; t < 3; ++t) x[t] = from[(m * 3 + t) * 64 + lane];
                k1[m] = mm(x, st, k1[m]);
#pragma unroll
                for (int t = 0; t < NI; ++t) y[t] = from[(24 + m * NI + t) * 64 + lane];
                q1[m] = mm(y, st, q1[m]);
#pragma unroll
                for (int t = 0; t < 3; ++t) x[t] = from[(12 + m * 3 + t) * 64 + lane];
                k2[m] = mm(x, dt, k2[m]);
            }
#pragma unroll
            for (int t = 0; t < TPW; ++t) {
                if (!own[t]) continue;
                bf16x8 x[3], e[3], y[NI];
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    x[i] = from[(tm[t] * 3 + i) * 64 + lane];
                    e[i] = from[(12 + tn[t] * 3 + i) * 64 + lane];
                }
#pragma unroll
                for (int i = 0; i < NI; ++i) y[i] = from[(24 + tm[t] * NI + i) * 64 + lane];
                da[t] = mm(x, e, da[t]);
                dp[t] = mm(y, e, dp[t]);
            }
            if (more) {
                put(stage + ((k & 1) ^ 1) * kStage * 64, tk, lane);
                load_tokens(at + k + 3, tk, lane);
            }
        };
        for (int k = 0; k < steps; k += 2) {             // (steps is even)
            step(k, true, rows[0], toks[1]);
            step(k + 1, k + 2 < steps, rows[1], toks[0]);
        }
        // (the last step leaves toks[0] as it was: the next head's first)
        at += steps;
        // K^T and Q^T of this wave's dk tile: B operands below, and -- element r of half m of step ks -- the values of token
        // 16 (2 ks + m) + 4 q + r that the dots need
        bf16x8 kt[2][NI], qt[2][NI];
        f32x4 kk[TPW], qk[TPW];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int t = 0; t < NI; ++t) {
                const size_t f = ((kslot * (DK / 16) * 2 + 2 * w + ks) * NI + t) * 64;
                kt[ks][t] = (a.ktf + f)[lane];
                qt[ks][t] = (a.qtf + f)[lane];
            }
#pragma unroll
        for (int t = 0; t < TPW; ++t) {
            const f32x4* const x = a.dots + (kslot * 10 + tm[t] * (tm[t] + 1) / 2 + tn[t]) * 128;
            kk[t] = x[lane];
            qk[t] = (x + 64)[lane];
        }
        dots = sum64(dots);
        if (lane == 0) gamma[w] = dots;
        // the 64 x 64 gradients, in the stage's place
        lds_barrier();
#pragma unroll
        for (int t = 0; t < TPW; ++t) {
            if (!own[t]) continue;
            const f32x4 decay = dec.rows(tm[t], tn[t], j, q);
            const int col = 16 * tn[t] + j;
            const float beta = bs[col], beta1 = beta_of(beta);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * tm[t] + 4 * q + r;
                if (col == i) dbeta[i] = da[t][r] / beta1;
                const float e = col <= i ? decay[r] : 0.f;
                const float A = col < i ? -da[t][r] * (beta1 * e) : 0.f, P = col <= i ? a.scale * beta * dp[t][r] : 0.f;
                if (col <= i) gmat[i * kTriStride + col] = gmat[col * kTriStride + i] = A;
                hmat[i * kTriStride + col] = P * e;
                dmat[i * kTriStride + col] = col < i ? A * kk[t][r] + P * (qk[t][r] * e) : 0.f;
            }
        }
        // rows' scales, and the dots with q and k that dg needs
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const int t0 = 16 * m + 4 * q;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float beta = scl[t0 + r], eb = scl[64 + t0 + r], ec = scl[128 + t0 + r];
                float kv = 0.f, qv = 0.f;
#pragma unroll
                for (int t = NI - 1; t >= 0; --t) {
                    kv += (float)kt[m >> 1][t][4 * (m & 1) + r];
                    qv += (float)qt[m >> 1][t][4 * (m & 1) + r];
                }
                q1[m][r] *= a.scale * eb;
                k1[m][r] *= -eb;
                k2[m][r] *= ec * beta;
                const float from = sum16(qv * q1[m][r] + kv * k1[m][r]), to = sum16(kv * k2[m][r]);
                k1[m][r] += k2[m][r];
                if (j == 0) {
                    sums[0][w][t0 + r] = from;
                    sums[1][w][t0 + r] = to;
                }
            }
        }
        lds_barrier();
        // A operands of the products with K and Q: G + G^T (8 fragments), H, H^T
        for (int f = w; f < 8 + 2 * kTriFrags; f += W) {
            f32x4 lo, hi;
            if (f < 8) {
                const f32x4* m4 = (const f32x4*)(gmat + (16 * (f >> 1) + j) * kTriStride + 32 * (f & 1) + 4 * q);
                lo = m4[0];
                hi = m4[4];
            } else if (f < 8 + kTriFrags) {
                const int mt = tri_row(f - 8), ks = tri_step(f - 8);
                const f32x4* m4 = (const f32x4*)(hmat + (16 * mt + j) * kTriStride + 32 * ks + 4 * q);
                lo = m4[0];
                hi = (mt & 1) || ks < (mt >> 1) ? m4[4] : splat4(0.f);
            } else {
                const int mt = trt_row(f - 8 - kTriFrags), ks = trt_step(f - 8 - kTriFrags);
                const bool half = (mt & 1) && ks == (mt >> 1);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    lo[e] = half ? 0.f : hmat[(32 * ks + 4 * q + e) * kTriStride + 16 * mt + j];
                    hi[e] = hmat[(32 * ks + 16 + 4 * q + e) * kTriStride + 16 * mt + j];
                }
            }
            bf16x8 t[3];
            split8<3>(lo, hi, t);
#pragma unroll
            for (int k = 0; k < 3; ++k) fr[(f * 3 + k) * 64 + lane] = t[k];
        }
        // dg: sums of column `lane` over rows i >= m, for m in this wave's rows; what the rows below this wave's give follows
        float run[RB];
        {
            float below = 0.f;
#pragma unroll
            for (int m = RB - 1; m >= 0; --m) {
                const int i = RB * w + m;
                below += (int)lane < i ? dmat[i * kTriStride + lane] : 0.f;
                run[m] = below;
            }
            part[w][lane] = below;
        }
        lds_barrier();
        // dQ += H K,  dK += (G + G^T) K + H^T Q
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                bf16x8 x[3];
#pragma unroll
                for (int t = 0; t < 3; ++t) x[t] = fr[((2 * m + ks) * 3 + t) * 64 + lane];
                k1[m] = mm(x, kt[ks], k1[m]);
                if (ks <= m / 2) {
#pragma unroll
                    for (int t = 0; t < 3; ++t) x[t] = fr[((8 + tri_index(m, ks)) * 3 + t) * 64 + lane];
                    q1[m] = mm(x, kt[ks], q1[m]);
                }
                if (ks >= m / 2) {
#pragma unroll
                    for (int t = 0; t < 3; ++t) x[t] = fr[((8 + kTriFrags + trt_index(m, ks)) * 3 + t) * 64 + lane];
                    k1[m] = mm(x, qt[ks], k1[m]);
                }
            }
        // dg_m of this wave's rows: the rectangle, what leaves before m and arrives from m on, what the state carries over
        {
            float below = 0.f, f = 0.f, g = 0.f, hold = 0.f;
#pragma unroll
            for (int k = 1; k < W; ++k) below += k > w ? part[k][lane] : 0.f;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                f += sums[0][k][lane];
                g += sums[1][k][lane];
                hold += gamma[k];
            }
            const float whole = dec.block(0) * dec.block(1) * dec.block(2) * dec.block(3);
            float mine = sum_from(f, lane) + sum_before(g, lane) + whole * hold;
#pragma unroll
            for (int m = 0; m < RB; ++m) {
                const float x = sum64((int)lane < RB * w + m ? run[m] + below : 0.f);
                mine += (int)lane == RB * w + m ? x : 0.f;
            }
            if ((int)lane / RB == w && (int)lane < n) {
                a.dg[(size_t)(start + lane) * a.hv + hv] = mine;
                a.dbeta[(size_t)(start + lane) * a.hv + hv] = dbeta[lane];
            }
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            if constexpr (SHARED) {
                dQ[m] += q1[m];
                dK[m] += k1[m];
            } else {
                dQ[m] = q1[m];
                dK[m] = k1[m];
            }
        }
    }
    const int j = lane0 & 15, q = lane0 >> 4;
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int t = 16 * m + 4 * q + r;
            if (t >= n) continue;
            const size_t to = ((size_t)(start + t) * a.hk + h) * DK + state_row(w) + 8 * (j >> 2) + (j & 3);
            ((raw*)a.dq)[to] = In::from_f32(dQ[m][r]);
            ((raw*)a.dk)[to] = In::from_f32(dK[m][r]);
        }
}

}  // namespace helen
