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
// The reverse chain is the forward one with other operands (a wave owns 16 columns of dS); everything else of all chunks
// follows at once.  dg is summed over the positions it reaches, not as a difference of running sums.
#pragma once
#include "kernels_delta.h"

namespace helen {

template <typename In, int DK>
__global__ __launch_bounds__(256) void delta_backward_kernel(const DeltaArgs a) {
    constexpr int NI = In::kTerms, KS = DK / 32, MT = DK / 16;
    typedef typename In::raw raw;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = lane & 15, q = lane >> 4;
    const int groups = (a.dv_width + 63) >> 6;
    const int tile = 4 * (blockIdx.x % groups) + w, col = tile * 16 + j;
    if (tile * 16 >= a.dv_width) return;
    const int hv = blockIdx.x / groups % a.hv, s = blockIdx.x / groups / a.hv, h = hv / a.group;
    const Span sp = span_of(a, s);
    const size_t st = ((size_t)s * a.hv + hv) * DK * a.dv_width;
    f32x4 S[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[m][r] = a.ds1 ? a.ds1[st + (size_t)(16 * m + 4 * q + r) * a.dv_width + col] : 0.f;

    for (int c = (sp.len + kDeltaChunk - 1) / kDeltaChunk - 1; c >= 0; --c) {
        const int start = sp.begin + c * kDeltaChunk, n = min(kDeltaChunk, sp.len - c * kDeltaChunk);
        const size_t slot = (size_t)sp.slot + c, kslot = slot * a.hk + h, vslot = slot * a.hv + hv;
        const float* sc = a.sc + vslot * 256;
        {
            float* to = a.dstates + vslot * DK * a.dv_width + col;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r) to[(size_t)(16 * m + 4 * q + r) * a.dv_width] = S[m][r];
        }
        bf16x8 sb[KS][3];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) split8<3>(S[2 * ks], S[2 * ks + 1], sb[ks]);
        f32x4 Y[4];      // dO
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * mt + 4 * q + r;
                Y[mt][r] = t < n ? In::to_f32(((const raw*)a.dout)[(start + t) * a.do_t + hv * a.do_h + col]) : 0.f;
            }
        bf16x8 yb[2][NI];
        split8<NI>(Y[0], Y[1], yb[0]);
        split8<NI>(Y[2], Y[3], yb[1]);
        f32x4 U[4];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            U[mt] = splat4(0.f);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8 kf[NI];
#pragma unroll
                for (int t = 0; t < NI; ++t) kf[t] = a.kf[(((kslot * 4 + mt) * KS + ks) * NI + t) * 64 + lane];
                U[mt] = mm(kf, sb[ks], U[mt]);
            }
            f32x4 p = splat4(0.f);
#pragma unroll
            for (int ks = mt / 2; ks < 2; ++ks) {
                bf16x8 pt[3];
#pragma unroll
                for (int t = 0; t < 3; ++t) pt[t] = a.ptf[((vslot * kTriFrags + trt_index(mt, ks)) * 3 + t) * 64 + lane];
                p = mm(pt, yb[ks], p);
            }
            const f32x4 ec = *(const f32x4*)(sc + 128 + 16 * mt + 4 * q);
#pragma unroll
            for (int r = 0; r < 4; ++r) U[mt][r] = ec[r] * U[mt][r] + a.scale * p[r];
        }
        bf16x8 ub[2][3];
        split8<3>(U[0], U[1], ub[0]);
        split8<3>(U[2], U[3], ub[1]);
        f32x4 Z[4];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            Z[mt] = splat4(0.f);
#pragma unroll
            for (int ks = mt / 2; ks < 2; ++ks) {
                bf16x8 tt[3];
#pragma unroll
                for (int t = 0; t < 3; ++t) tt[t] = a.ttf[((vslot * kTriFrags + trt_index(mt, ks)) * 3 + t) * 64 + lane];
                Z[mt] = mm(tt, ub[ks], Z[mt]);
            }
            const f32x4 beta = *(const f32x4*)(sc + 16 * mt + 4 * q), eb = *(const f32x4*)(sc + 64 + 16 * mt + 4 * q);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * mt + 4 * q + r;
                a.z[(vslot * kDeltaChunk + t) * a.dv_width + col] = Z[mt][r];
                const float dv = beta[r] * Z[mt][r];
                if (t < n) ((raw*)a.dv)[((size_t)(start + t) * a.hv + hv) * a.dv_width + col] = In::from_f32(dv);
                Z[mt][r] = -eb[r] * dv;
                Y[mt][r] *= a.scale * eb[r];
            }
        }
        bf16x8 zb[2][3], wb[2][3];
        split8<3>(Z[0], Z[1], zb[0]);
        split8<3>(Z[2], Z[3], zb[1]);
        split8<3>(Y[0], Y[1], wb[0]);
        split8<3>(Y[2], Y[3], wb[1]);
        const float whole = sc[64 + 63];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int r = 0; r < 4; ++r) S[m][r] *= whole;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                bf16x8 kt[NI], qt[NI];
#pragma unroll
                for (int t = 0; t < NI; ++t) {
                    const size_t at = ((kslot * MT * 2 + 2 * m + ks) * NI + t) * 64 + lane;
                    kt[t] = a.ktf[at];
                    qt[t] = a.qtf[at];
                }
                S[m] = mm(kt, zb[ks], S[m]);
                S[m] = mm(qt, wb[ks], S[m]);
            }
        }
    }
    if (a.ds0) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) a.ds0[st + (size_t)(16 * m + 4 * q + r) * a.dv_width + col] = S[m][r];
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
