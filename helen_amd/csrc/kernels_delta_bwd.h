// kernels_delta_bwd.h -- backward pass of the gated delta rule (kernels_delta.h has the forward formulas and the layouts)
//
// With dO, dS1 the gradients of a chunk's outputs and of the state behind it:
//     dU = scale P^T dO + e^{c} K dS1,   Z = T^T dU,   dV = beta Z,
//     dS0 = e^{b_C} dS1 + Q^T (scale e^{b} dO) - K^T (e^{b} beta Z)                        (the reverse chain)
//     dA = -tril(Z U^T, -1),  dP = scale tril(dO U^T),  G = beta dA e^{D},  H = dP e^{D}
//     dQ = scale e^{b} dO S0^T + H K,   dK = -e^{b} beta Z S0^T + e^{c} U dS1^T + (G + G^T) K + H^T Q
//     dbeta_i = Z_i . R_i + sum_j dA_ij (k_i . k_j) e^{D_ij}
//     dg_m = sum_{j < m <= i} (dA A + dP P)_ij + sum_{i >= m} (q_i . dQ1_i + k_i . dK1_i) + sum_{i < m} k_i . dK2_i
//            + e^{b_C} <S0, dS1>,   dQ1, dK1 = the S0 terms of dQ, dK;  dK2 = the dS1 term of dK
// The reverse chain is the forward one with other operands; everything else of all chunks follows at once.  dg is summed over the positions it reaches, not as a difference of running sums.
#pragma once
#include "kernels_delta.h"

namespace helen {

// The reverse chain, built like delta_forward_kernel: wave w owns token tile w of dO, dU and Z and its quarter of dS's rows.
template <typename In, int DK, int NC>
__global__ __launch_bounds__(256) void delta_backward_kernel(const DeltaArgs a) {
    constexpr int NI = In::kTerms, KS = DK / 32, MW = DK / 64;
    typedef typename In::raw raw;
    __shared__ bf16x8 sbuf[KS * 3 * NC * 64], ybuf[2 * NI * NC * 64], wbuf[2 * 3 * NC * 64], dbuf[2 * 3 * NC * 64], zbuf[2 * 3 * NC * 64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = lane & 15, q = lane >> 4;
    const int groups = a.dv_width / (16 * NC);
    const unsigned item = xcd_order(blockIdx.x, gridDim.x);
    if (item >= (unsigned)a.nseq * a.hv * groups) return;
    const int hv = item / groups % a.hv, s = item / groups / a.hv, h = hv / a.group;
    const int col = 16 * NC * (item % groups) + j;
    const Span sp = span_of(a, s);
    const int chunks = (sp.len + kDeltaChunk - 1) / kDeltaChunk;
    const size_t st = (((size_t)s * a.hv + hv) * DK + 16 * MW * w + 4 * q) * a.dv_width + col;

    f32x4 S[MW][NC];
#pragma unroll
    for (int i = 0; i < MW; ++i)
#pragma unroll
        for (int nc = 0; nc < NC; ++nc)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[i][nc][r] = a.ds1 ? a.ds1[st + (size_t)(16 * i + r) * a.dv_width + 16 * nc] : 0.f;

    bf16x8 kf[KS][NI], kt[MW][2][NI], qt[MW][2][NI], tt[2][3], pt[2][3];
    f32x4 beta, eb, ec;
    float whole;
    raw y[NC][4];
    const bf16x8* const kf0 = a.kf + (size_t)sp.slot * a.hk * (DK / 8 * NI * 64) + (size_t)h * (DK / 8 * NI * 64) + lane;
    const bf16x8* const kt0 = a.ktf + (kf0 - a.kf);
    const bf16x8* const qt0 = a.qtf + (kf0 - a.kf);
    const size_t vslot0 = (size_t)sp.slot * a.hv + hv;
    const int row = 16 * w + 4 * q;
    auto load_rows = [&](int c) {
        const size_t at = (size_t)c * a.hk * (DK / 8 * NI * 64) + w * KS * NI * 64;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int t = 0; t < NI; ++t) kf[ks][t] = kf0[at + (ks * NI + t) * 64];
    };
    auto load_scales = [&](int c) {
        const float* sc = a.sc + (vslot0 + (size_t)c * a.hv) * 256;
        beta = *(const f32x4*)(sc + row);
        eb = *(const f32x4*)(sc + 64 + row);
        ec = *(const f32x4*)(sc + 128 + row);
        whole = sc[64 + 63];
    };
    auto load_dout = [&](int c) {
        const int n = sp.len - c * kDeltaChunk;
        const raw* p = (const raw*)a.dout + (sp.begin + c * kDeltaChunk + row) * a.do_t + hv * a.do_h + col;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) y[nc][r] = row + r < n ? p[r * a.do_t + 16 * nc] : raw(0);
    };
    auto load_tri = [&](int c, const bf16x8* from, bf16x8 (&to)[2][3]) {
        const size_t at = (vslot0 + (size_t)c * a.hv) * kTriFrags * 3 * 64 + lane;
#pragma unroll
        for (int t = 0; t < 3; ++t) {
            if (w < 2) to[0][t] = from[at + (trt_index(w, 0) * 3 + t) * 64];
            to[1][t] = from[at + (trt_index(w, 1) * 3 + t) * 64];
        }
    };
    auto load_columns = [&](int c) {
        const size_t at = (size_t)c * a.hk * (DK / 8 * NI * 64) + w * MW * 2 * NI * 64;
#pragma unroll
        for (int i = 0; i < MW; ++i)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int t = 0; t < NI; ++t) {
                    kt[i][ks][t] = kt0[at + ((2 * i + ks) * NI + t) * 64];
                    qt[i][ks][t] = qt0[at + ((2 * i + ks) * NI + t) * 64];
                }
    };
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
                               (f32x4){In::to_f32(y[nc][0]), In::to_f32(y[nc][1]), In::to_f32(y[nc][2]), In::to_f32(y[nc][3])});
        }
        float* to = a.dstates + ((vslot0 + (size_t)c * a.hv) * DK + 16 * MW * w + 4 * q) * a.dv_width + col;
#pragma unroll
        for (int i = 0; i < MW; ++i)
#pragma unroll
            for (int nc = 0; nc < NC; ++nc)
#pragma unroll
                for (int r = 0; r < 4; ++r) to[(size_t)(16 * i + r) * a.dv_width + 16 * nc] = S[i][nc][r];
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
        f32x4 E[NC], P[NC];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) E[nc] = P[nc] = splat4(0.f);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) {
                bf16x8 b[3];
                shared_frag<3, NC>(sbuf, ks, nc, lane, b);
                E[nc] = mm(kf[ks], b, E[nc]);
            }
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            bf16x8 b[NI];
            if (w < 2) {
                shared_frag<NI, NC>(ybuf, 0, nc, lane, b);
                P[nc] = mm(pt[0], b, P[nc]);
            }
            shared_frag<NI, NC>(ybuf, 1, nc, lane, b);
            P[nc] = mm(pt[1], b, P[nc]);
        }
        const f32x4 step = beta, head = eb;
        const float hold = whole;
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            f32x4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                E[nc][r] = ec[r] * E[nc][r] + a.scale * P[nc][r];
                x[r] = a.scale * eb[r] * In::to_f32(y[nc][r]);
            }
            share_tile<3, NC>(dbuf, w, nc, lane, E[nc]);
            share_tile<3, NC>(wbuf, w, nc, lane, x);
        }
        if (c > 0) {
            load_dout(c - 1);
            load_rows(c - 1);
            load_scales(c - 1);
            load_tri(c - 1, a.ptf, pt);
        }
        lds_barrier();
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            f32x4 Z = splat4(0.f);
            bf16x8 b[3];
            if (w < 2) {
                shared_frag<3, NC>(dbuf, 0, nc, lane, b);
                Z = mm(tt[0], b, Z);
            }
            shared_frag<3, NC>(dbuf, 1, nc, lane, b);
            Z = mm(tt[1], b, Z);
            const int n = sp.len - c * kDeltaChunk;
            float* to = a.z + ((vslot0 + (size_t)c * a.hv) * kDeltaChunk + row) * a.dv_width + col + 16 * nc;
            raw* dv = (raw*)a.dv + ((size_t)(sp.begin + c * kDeltaChunk + row) * a.hv + hv) * a.dv_width + col + 16 * nc;
            f32x4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                to[r * a.dv_width] = Z[r];
                const float d = step[r] * Z[r];
                if (row + r < n) dv[(size_t)r * a.hv * a.dv_width] = In::from_f32(d);
                x[r] = -head[r] * d;
            }
            share_tile<3, NC>(zbuf, w, nc, lane, x);
        }
        if (c > 0) load_tri(c - 1, a.ttf, tt);
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
        if (c > 0) {
            load_columns(c - 1);
            share(c - 1);
        }
        lds_barrier();
    }
    if (a.ds0) {
#pragma unroll
        for (int i = 0; i < MW; ++i)
#pragma unroll
            for (int nc = 0; nc < NC; ++nc)
#pragma unroll
                for (int r = 0; r < 4; ++r) a.ds0[st + (size_t)(16 * i + r) * a.dv_width + 16 * nc] = S[i][nc][r];
    }
}

// sum over the 16 lanes of a quarter
__device__ __forceinline__ float sum16(float x) {
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) x += __shfl_xor(x, m);
    return x;
}

// ------------------------------------------------------------------------------------------------
// dQ, dK, dbeta and dg of one chunk: a workgroup per (slot, key head).  The value heads of the key head follow one another
// and are summed in registers: no atomics, one order.  Wave w: token tile w of everything that is 64 x 64 and of the staging,
// columns dk = w DK/4 .. of everything that is 64 x DK.
// ------------------------------------------------------------------------------------------------
template <typename In, int DK>
__global__ __launch_bounds__(256) void delta_grads_kernel(const DeltaArgs a) {
    constexpr int NI = In::kTerms, KS = DK / 32, NT = DK / 64;
    typedef typename In::raw raw;
    constexpr int kStage = 4 * (6 + NI), kTail = 3 * (8 + 2 * kTriFrags), kKeys = 4 * KS * NI;
    constexpr int kFrags = kTail > kKeys ? (kTail > kStage ? kTail : kStage) : (kKeys > kStage ? kKeys : kStage);
    __shared__ bf16x8 fr[kFrags * 64];
    __shared__ f32x4 gmat4[64 * kTriStride / 4], hmat4[64 * kTriStride / 4], dmat4[64 * kTriStride / 4];
    __shared__ float gs[64], bs[64], sums[2][4][64], zr[64], da_row[64], gamma[4], part[4][64];
    float* const gmat = (float*)gmat4;
    float* const hmat = (float*)hmat4;
    float* const dmat = (float*)dmat4;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = lane & 15, q = lane >> 4;
    const int slot = blockIdx.x / a.hk, h = blockIdx.x % a.hk;
    const int s = sequence_of(a, slot, lane);
    const Span sp = span_of(a, s);
    const int c = slot - sp.slot;
    const int start = sp.begin + c * kDeltaChunk;
    const int n = min(kDeltaChunk, sp.begin + sp.len - start);
    if (c < 0 || n <= 0) {
        if (s == a.nseq - 1) {      // rows behind the last sequence: their gradients are zero
            const int end = sp.begin + sp.len;
            const int lo = max(end, (slot - a.nseq) * kDeltaChunk), hi = min(a.tokens, (slot - a.nseq + 1) * kDeltaChunk);
            for (int t = lo; t < hi; ++t) {
                for (int d = threadIdx.x; d < DK; d += 256)
                    ((raw*)a.dq)[((size_t)t * a.hk + h) * DK + d] = ((raw*)a.dk)[((size_t)t * a.hk + h) * DK + d] = raw(0);
                for (int hv = h * a.group; hv < (h + 1) * a.group; ++hv) {
                    for (int d = threadIdx.x; d < a.dv_width; d += 256)
                        ((raw*)a.dv)[((size_t)t * a.hv + hv) * a.dv_width + d] = raw(0);
                    if (threadIdx.x == 0) a.dg[(size_t)t * a.hv + hv] = a.dbeta[(size_t)t * a.hv + hv] = 0.f;
                }
            }
        }
        return;
    }
    const size_t kslot = (size_t)slot * a.hk + h;

    // K K^T and Q K^T, row tile w
    f32x4 kk[4], qk[4];
    for (int f = w; f < kKeys; f += 4) fr[f * 64 + lane] = a.kf[(kslot * kKeys + f) * 64 + lane];
    __syncthreads();
    {
        bf16x8 qf[KS][NI];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int t = 0; t < NI; ++t) qf[ks][t] = a.qf[(((kslot * 4 + w) * KS + ks) * NI + t) * 64 + lane];
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            kk[nt] = qk[nt] = splat4(0.f);
            if (nt <= w) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    bf16x8 b[NI], kf[NI];
#pragma unroll
                    for (int t = 0; t < NI; ++t) {
                        b[t] = fr[((nt * KS + ks) * NI + t) * 64 + lane];
                        kf[t] = fr[((w * KS + ks) * NI + t) * 64 + lane];
                    }
                    kk[nt] = mm(kf, b, kk[nt]);
                    qk[nt] = mm(qf[ks], b, qk[nt]);
                }
            }
        }
    }

    f32x4 dQ[NT][4], dK[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) dQ[i][mt] = dK[i][mt] = splat4(0.f);

    for (int hv = h * a.group; hv < (h + 1) * a.group; ++hv) {
        const size_t vslot = (size_t)slot * a.hv + hv;
        const float* sc = a.sc + vslot * 256;
        __syncthreads();
        if (w == 0) {
            const bool in = lane < n;
            gs[lane] = in ? a.g[(start + lane) * a.g_t + hv * a.g_h] : 0.f;
            bs[lane] = in ? a.beta[(start + lane) * a.b_t + hv * a.b_h] : 0.f;
        }
        // products over dv, 32 columns a step
        f32x4 q1[NT][4], k1[NT][4], k2[NT][4], da[4], dp[4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) q1[i][mt] = k1[i][mt] = k2[i][mt] = splat4(0.f);
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) da[nt] = dp[nt] = splat4(0.f);
        float dots = 0.f, zrow = 0.f;
        for (int d0 = 0; d0 < a.dv_width; d0 += 32) {
            const int row = 16 * w + j;
            const size_t at = (vslot * kDeltaChunk + row) * a.dv_width + d0 + 4 * q;
            const f32x4 z0 = *(const f32x4*)(a.z + at), z1 = *(const f32x4*)(a.z + at + 16);
            const f32x4 u0 = *(const f32x4*)(a.u + at), u1 = *(const f32x4*)(a.u + at + 16);
            const f32x4 r0 = *(const f32x4*)(a.r + at), r1 = *(const f32x4*)(a.r + at + 16);
            f32x4 y0 = splat4(0.f), y1 = splat4(0.f);
            if (row < n) {
                const raw* yp = (const raw*)a.dout + (start + row) * a.do_t + hv * a.do_h + d0 + 4 * q;
                y0 = load4<In>(yp);
                y1 = load4<In>(yp + 16);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) zrow += z0[r] * r0[r] + z1[r] * r1[r];
            bf16x8 zt[3], ut[3], yt[NI];
            split8<3>(z0, z1, zt);
            split8<3>(u0, u1, ut);
            split8<NI>(y0, y1, yt);
            __syncthreads();
#pragma unroll
            for (int t = 0; t < 3; ++t) {
                fr[(w * 3 + t) * 64 + lane] = zt[t];
                fr[(12 + w * 3 + t) * 64 + lane] = ut[t];
            }
#pragma unroll
            for (int t = 0; t < NI; ++t) fr[(24 + w * NI + t) * 64 + lane] = yt[t];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const size_t sat = (vslot * DK + 16 * (w * NT + i) + j) * a.dv_width + d0 + 4 * q;
                const f32x4 a0 = *(const f32x4*)(a.states + sat), a1 = *(const f32x4*)(a.states + sat + 16);
                const f32x4 b0 = *(const f32x4*)(a.dstates + sat), b1 = *(const f32x4*)(a.dstates + sat + 16);
#pragma unroll
                for (int r = 0; r < 4; ++r) dots += a0[r] * b0[r] + a1[r] * b1[r];
                bf16x8 st[3], dt[3];
                split8<3>(a0, a1, st);
                split8<3>(b0, b1, dt);
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) {
                    bf16x8 zf[3], uf[3], yf[NI];
#pragma unroll
                    for (int t = 0; t < 3; ++t) {
                        zf[t] = fr[(mt * 3 + t) * 64 + lane];
                        uf[t] = fr[(12 + mt * 3 + t) * 64 + lane];
                    }
#pragma unroll
                    for (int t = 0; t < NI; ++t) yf[t] = fr[(24 + mt * NI + t) * 64 + lane];
                    q1[i][mt] = mm(yf, st, q1[i][mt]);
                    k1[i][mt] = mm(zf, st, k1[i][mt]);
                    k2[i][mt] = mm(uf, dt, k2[i][mt]);
                }
            }
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
                if (nt <= w) {
                    bf16x8 uf[3];
#pragma unroll
                    for (int t = 0; t < 3; ++t) uf[t] = fr[(12 + nt * 3 + t) * 64 + lane];
                    da[nt] = mm(zt, uf, da[nt]);
                    dp[nt] = mm(yt, uf, dp[nt]);
                }
        }
        // Z_i . R_i, <S0, dS1>
        zrow += __shfl_xor(zrow, 16);
        zrow += __shfl_xor(zrow, 32);
        if (q == 0) zr[16 * w + j] = zrow;
        dots = sum16(dots);
        dots += __shfl_xor(dots, 16);
        dots += __shfl_xor(dots, 32);
        if (lane == 0) gamma[w] = dots;
        // rows' scales, and the dots with q and k that dg needs
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            const f32x4 beta = *(const f32x4*)(sc + 16 * mt + 4 * q), eb = *(const f32x4*)(sc + 64 + 16 * mt + 4 * q),
                        ec = *(const f32x4*)(sc + 128 + 16 * mt + 4 * q);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * mt + 4 * q + r;
                float from = 0.f, to = 0.f;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const int d = 16 * (w * NT + i) + j;
                    q1[i][mt][r] *= a.scale * eb[r];
                    k1[i][mt][r] *= -(eb[r] * beta[r]);
                    k2[i][mt][r] *= ec[r];
                    if (t < n) {
                        const float qv = In::to_f32(((const raw*)a.q)[(start + t) * a.q_t + h * a.q_h + d]);
                        const float kv = In::to_f32(((const raw*)a.k)[(start + t) * a.k_t + h * a.k_h + d]);
                        from += qv * q1[i][mt][r] + kv * k1[i][mt][r];
                        to += kv * k2[i][mt][r];
                    }
                    dQ[i][mt][r] += q1[i][mt][r];
                    dK[i][mt][r] += k1[i][mt][r] + k2[i][mt][r];
                }
                from = sum16(from);
                to = sum16(to);
                if (j == 0) {
                    sums[0][w][t] = from;
                    sums[1][w][t] = to;
                }
            }
        }
        // the 64 x 64 gradients
        float block[4];
        f32x4 decay[4];
        block_sums(gs, block);
        decays(gs, block, w, j, q, decay);
        f32x4 row_sum = splat4(0.f);
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            if (nt > w) continue;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * w + 4 * q + r, col = 16 * nt + j;
                const float e = col <= i ? decay[nt][r] : 0.f;
                const float A = col < i ? -da[nt][r] : 0.f, P = col <= i ? a.scale * dp[nt][r] : 0.f;
                const float ke = col < i ? kk[nt][r] * e : 0.f;
                row_sum[r] += A * ke;
                const float g = A * (bs[i] * e);
                if (col <= i) gmat[i * kTriStride + col] = gmat[col * kTriStride + i] = g;
                hmat[i * kTriStride + col] = P * e;
                dmat[i * kTriStride + col] = A * (bs[i] * ke) + (col < i ? P * (qk[nt][r] * e) : 0.f);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float x = sum16(row_sum[r]);
            if (j == 0) da_row[16 * w + 4 * q + r] = x;
        }
        __syncthreads();
        // A operands of the products with K and Q: G + G^T (8 fragments), H, H^T
        for (int f = w; f < 8 + 2 * kTriFrags; f += 4) {
            f32x4 lo, hi;
            if (f < 8) {
                const f32x4* m4 = gmat4 + ((16 * (f >> 1) + j) * kTriStride + 32 * (f & 1) + 4 * q) / 4;
                lo = m4[0];
                hi = m4[4];
            } else if (f < 8 + kTriFrags) {
                const int mt = tri_row(f - 8), ks = tri_step(f - 8);
                const f32x4* m4 = hmat4 + ((16 * mt + j) * kTriStride + 32 * ks + 4 * q) / 4;
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
        // dg, first half: sums of column `lane` over rows i >= m, for m in this wave's 16 rows (in place, below)
        {
            float below = 0.f;
            for (int i = 16 * (w + 1); i < 64; ++i) below += lane < i ? dmat[i * kTriStride + lane] : 0.f;
            float run[16];
#pragma unroll
            for (int m = 15; m >= 0; --m) {
                const int i = 16 * w + m;
                below += lane < i ? dmat[i * kTriStride + lane] : 0.f;
                run[m] = below;
            }
            __syncthreads();
#pragma unroll
            for (int m = 0; m < 16; ++m)
                if (lane < 16 * w + m) dmat[(16 * w + m) * kTriStride + lane] = run[m];
        }
        __syncthreads();
        {
            float x = 0.f;
#pragma unroll
            for (int m = 0; m < 16; ++m) x += 16 * w + m < lane ? dmat[lane * kTriStride + 16 * w + m] : 0.f;
            part[w][lane] = x;
        }
        __syncthreads();
        if (w == 0) {
            float x = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
            float from = 0.f, to = 0.f;
            for (int i = 0; i < 64; ++i) {
                from += i >= lane ? (sums[0][0][i] + sums[0][1][i]) + (sums[0][2][i] + sums[0][3][i]) : 0.f;
                to += i < lane ? (sums[1][0][i] + sums[1][1][i]) + (sums[1][2][i] + sums[1][3][i]) : 0.f;
            }
            x += from + to + sc[64 + 63] * ((gamma[0] + gamma[1]) + (gamma[2] + gamma[3]));
            if (lane < n) {
                a.dg[(size_t)(start + lane) * a.hv + hv] = x;
                a.dbeta[(size_t)(start + lane) * a.hv + hv] = zr[lane] + da_row[lane];
            }
        }
        // dQ += H K,  dK += (G + G^T) K + H^T Q
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                bf16x8 kt[NI], qt[NI];
#pragma unroll
                for (int t = 0; t < NI; ++t) {
                    const size_t at = ((kslot * (DK / 16) * 2 + 2 * (w * NT + i) + ks) * NI + t) * 64 + lane;
                    kt[t] = a.ktf[at];
                    qt[t] = a.qtf[at];
                }
#pragma unroll
                for (int mt = 0; mt < 4; ++mt) {
                    bf16x8 m[3];
#pragma unroll
                    for (int t = 0; t < 3; ++t) m[t] = fr[((2 * mt + ks) * 3 + t) * 64 + lane];
                    dK[i][mt] = mm(m, kt, dK[i][mt]);
                    if (ks <= mt / 2) {
#pragma unroll
                        for (int t = 0; t < 3; ++t) m[t] = fr[((8 + tri_index(mt, ks)) * 3 + t) * 64 + lane];
                        dQ[i][mt] = mm(m, kt, dQ[i][mt]);
                    }
                    if (ks >= mt / 2) {
#pragma unroll
                        for (int t = 0; t < 3; ++t) m[t] = fr[((8 + kTriFrags + trt_index(mt, ks)) * 3 + t) * 64 + lane];
                        dK[i][mt] = mm(m, qt, dK[i][mt]);
                    }
                }
            }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * mt + 4 * q + r;
                if (t >= n) continue;
                const size_t at = ((size_t)(start + t) * a.hk + h) * DK + 16 * (w * NT + i) + j;
                ((raw*)a.dq)[at] = In::from_f32(dQ[i][mt][r]);
                ((raw*)a.dk)[at] = In::from_f32(dK[i][mt][r]);
            }
}

}  // namespace helen
