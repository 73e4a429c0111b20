// kernels_delta.h -- the gated delta rule over whole sequences, in chunks of 64 tokens: preparation and forward chain
//
// Per sequence and value head, with a state S [Dk, Dv] and e^{g} the decay of a token:
//     u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t),   S_t = e^{g_t} S_{t-1} + k_t u_t^T,   o_t = scale S_t^T q_t
// In a chunk of C = 64 tokens, with D_ij = sum of g over (j, i], b_i the sum from the chunk's start and c_i the sum after i
// to its end, all C tokens are products (S0 = the state before the chunk):
//     A_ij = beta_i (k_i . k_j) e^{D_ij} (j < i),  T = (I + A)^-1,   R = V - e^{b} K S0,   U = T beta R,
//     O = scale (e^{b} Q S0 + P U),  P_ij = (q_i . k_j) e^{D_ij} (j <= i),   S1 = e^{b_C} S0 + K^T (e^{c} U)
// A, T and P do not depend on the state: delta_prep_kernel makes them for every chunk at once.  What is left, one chunk after
// another, is delta_forward_kernel: a wave owns 16 columns of S in registers (a column of S needs no other column), so a
// chain has no exchange between waves at all.
//
// Arithmetic: as in the fp32x3 recurrence, an fp32 value is the sum of three bf16 terms and a product of two such values the
// six leading products of terms on v_mfma_f32_16x16x32_bf16 with fp32 accumulation.  bf16 inputs are ONE term (their products
// with S are exact), fp16 inputs two, fp32 inputs three; S, U, R, T and P keep three, so states and everything that feeds
// them stay fp32-class whatever the inputs' type.  Decays between two positions are sums of the g between them, never a
// difference of two running sums: a strong decay (or g = -inf, a reset) costs the other positions no digits.
//
// Fragments.  lane l: j = l & 15, q = l >> 4.  The k index of an MFMA may be permuted if both operands agree; here element
// e = 0..7 of lane quarter q is k = 32 s + (e < 4 ? 4 q + e : 16 + 4 q + e - 4), which is exactly how two stacked D tiles of
// 16 rows lie in the accumulators.  A result (S, U, R) thus becomes the next product's B operand without any exchange.
#pragma once
#include "kernels_common.h"

namespace helen {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kDeltaChunk = 64;
constexpr int kTriFrags = 6;      // 16 x 32 fragments of a 64 x 64 triangle that are not all zero

// ---- element types: how many bf16 terms hold one value exactly, and loads ----
struct InBf16 {
    typedef unsigned short raw;
    static constexpr int kTerms = 1;
    static __device__ __forceinline__ float to_f32(raw x) { return __builtin_bit_cast(float, (unsigned)x << 16); }
    static __device__ __forceinline__ raw from_f32(float f) {
        return (raw)(__builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){f, 0.f}, bf16x2_t)) & 0xffffu);
    }
};
struct InF16 {
    typedef unsigned short raw;
    static constexpr int kTerms = 2;
    static __device__ __forceinline__ float to_f32(raw x) { return (float)__builtin_bit_cast(_Float16, x); }
    static __device__ __forceinline__ raw from_f32(float f) { return __builtin_bit_cast(raw, (_Float16)f); }
};
struct InF32 {
    typedef float raw;
    static constexpr int kTerms = 3;
    static __device__ __forceinline__ float to_f32(raw x) { return x; }
    static __device__ __forceinline__ raw from_f32(float f) { return f; }
};

// N bf16 terms of eight fp32 values (x = t[0] + t[1] + t[2] exactly: 3 x 8 significand bits)
template <int N>
__device__ __forceinline__ void split8(const f32x4 lo, const f32x4 hi, bf16x8 (&t)[N]) {
    u32x4 out[N];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        f32x2 x = p < 2 ? (f32x2){lo[2 * p], lo[2 * p + 1]} : (f32x2){hi[2 * p - 4], hi[2 * p - 3]};
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const unsigned b = __builtin_bit_cast(unsigned, __builtin_convertvector(x, bf16x2_t));
            out[n][p] = b;
            if (n + 1 < N) {
                x.x -= __builtin_bit_cast(float, b << 16);
                x.y -= __builtin_bit_cast(float, b & 0xffff0000u);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) t[n] = __builtin_bit_cast(bf16x8, out[n]);
}

// c += A B over 32 k, of operands in NA and NB terms: the products of terms whose orders add up to 2 at most, small ones first
template <int NA, int NB, int ORDER = 2>
__device__ __forceinline__ f32x4 mm(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], f32x4 c) {
#pragma unroll
    for (int s = ORDER; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], c, 0, 0, 0);
    return c;
}

// four elements -> fp32 (the pointer is aligned to four elements)
template <typename In>
__device__ __forceinline__ f32x4 load4(const typename In::raw* p) {
    if constexpr (sizeof(typename In::raw) == 4) {
        return *(const f32x4*)p;
    } else {
        const u32x2 w = *(const u32x2*)p;
        return (f32x4){In::to_f32((unsigned short)w.x), In::to_f32((unsigned short)(w.x >> 16)),
                       In::to_f32((unsigned short)w.y), In::to_f32((unsigned short)(w.y >> 16))};
    }
}

// ---- arguments of the launches (built by ops_delta.hip) ----
struct DeltaArgs {
    const void *q, *k, *v, *dout;
    const float *g, *beta;
    const int* offsets;         // [nseq + 1] or null: nseq sequences of seq_len tokens each
    const float* s0;            // [nseq, Hv, Dk, Dv] or null
    float* s1;                  // same, or null
    void* o;
    const float* ds1;           // backward: gradient of the final state, or null
    float* ds0;                 // backward: gradient of the initial state, or null
    void *dq, *dk, *dv;
    float *dg, *dbeta;
    long q_t, q_h, k_t, k_h, v_t, v_h, o_t, o_h, do_t, do_h, g_t, g_h, b_t, b_h;   // strides in elements: token, head
    int tokens, nseq, seq_len, hk, hv, group, dv_width, slots;
    float scale;
    int zero_tail;              // rows behind the last sequence: 1 = zero them, 0 = leave them
    // workspace: fragments per (slot, key head) and per (slot, value head)
    bf16x8 *kf, *ktf, *qf, *qtf;
    bf16x8 *tf, *ttf, *pf, *ptf;
    float* sc;                  // [slot, hv][4][64]: beta, e^b, e^c, -
    float *states, *u, *r;      // kept for the backward pass: [slot, hv, Dk, Dv], [slot, hv, 64, Dv] twice
    float *dstates, *z;         // backward: [slot, hv, Dk, Dv], [slot, hv, 64, Dv]
};

// Sequences and their chunks.  Chunk c of sequence s has slot begin / 64 + s + c: slots of different sequences never meet
// (ceil(n / 64) <= floor((begin + n) / 64) + 1 - floor(begin / 64)) and no table has to be built.  Offsets that do not
// ascend within [0, tokens] give wrong values, never an access out of range.
struct Span {
    int begin, len, slot;
};
__device__ __forceinline__ Span span_of(const DeltaArgs& a, int s) {
    int b, e;
    if (a.offsets) {
        b = min(max(a.offsets[s], 0), a.tokens);
        e = min(max(a.offsets[s + 1], b), a.tokens);
    } else {
        b = s * a.seq_len;
        e = b + a.seq_len;
    }
    return {b, e - b, b / kDeltaChunk + s};
}
// The sequence that holds a slot: 64 probes a round.
__device__ __forceinline__ int sequence_of(const DeltaArgs& a, int slot, int lane) {
    int lo = 0, n = a.nseq;
    while (n > 1) {
        const int step = (n + 63) >> 6;
        const int s = lo + lane * step;
        bool below = false;
        if (lane * step < n) {
            const int b = a.offsets ? min(max(a.offsets[s], 0), a.tokens) : s * a.seq_len;
            below = b / kDeltaChunk + s <= slot;
        }
        const int hits = __popcll(__ballot(below));
        const int at = max(hits - 1, 0) * step;
        lo += at;
        n = min(step, n - at);
    }
    return lo;
}

// lower triangle (tf, pf): fragment f = row tile mt, k step ks of mt's; the last step of an even row tile ends in a zero half
__device__ __forceinline__ int tri_row(int f) { return f < 2 ? f : (f < 4 ? 2 : 3); }
__device__ __forceinline__ int tri_step(int f) { return f < 2 ? 0 : (f & 1); }
__device__ __forceinline__ constexpr int tri_index(int mt, int ks) { return mt < 2 ? mt : 2 * mt - 2 + ks; }
// its transpose (ttf, ptf): rows are tokens j, k steps the tokens i >= j: (0,0) (0,1) (1,0) (1,1) (2,1) (3,1)
__device__ __forceinline__ int trt_row(int f) { return f < 4 ? f >> 1 : f - 2; }
__device__ __forceinline__ int trt_step(int f) { return f < 4 ? f & 1 : 1; }
__device__ __forceinline__ constexpr int trt_index(int mt, int ks) { return mt < 2 ? 2 * mt + ks : mt + 2; }

// sums of the chunk's g (64 values in LDS) over its four blocks of 16
__device__ __forceinline__ void block_sums(const float* gs, float (&block)[4]) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        block[b] = 0.f;
#pragma unroll
        for (int m = 0; m < 16; ++m) block[b] += gs[16 * b + m];
    }
}
// sums of g from the chunk's start up to and with token `lane`, and of those after it
__device__ __forceinline__ void head_tail(const float* gs, const float (&block)[4], int lane, float* head_out, float* tail_out) {
    const int j = lane & 15, b = lane >> 4;
    float head = 0.f, tail = 0.f;
#pragma unroll
    for (int m = 0; m < 16; ++m) {
        head += m <= j ? gs[16 * b + m] : 0.f;
        tail += m > j ? gs[16 * b + m] : 0.f;
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        head += m < b ? block[m] : 0.f;
        tail += m > b ? block[m] : 0.f;
    }
    *head_out = head;
    *tail_out = tail;
}
// e^{D_ij} of rows i = 16 w + 4 q + r, columns 16 nt + j, nt <= w (on and below the diagonal; what lies above is not used)
__device__ __forceinline__ void decays(const float* gs, const float (&block)[4], int w, int j, int q, f32x4 (&out)[4]) {
    f32x4 head = splat4(0.f), within = splat4(0.f);
#pragma unroll
    for (int m = 0; m < 16; ++m) {
        const float gm = gs[16 * w + m];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            head[r] += m <= 4 * q + r ? gm : 0.f;
            within[r] += (m > j && m <= 4 * q + r) ? gm : 0.f;
        }
    }
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
        if (nt > w) continue;
        float tail = 0.f;
        if (nt < w) {
#pragma unroll
            for (int m = 0; m < 16; ++m) tail += m > j ? gs[16 * nt + m] : 0.f;
#pragma unroll
            for (int m = 0; m < 4; ++m) tail += (m > nt && m < w) ? block[m] : 0.f;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) out[nt][r] = expf(nt < w ? tail + head[r] : within[r]);
    }
}

constexpr int kTriStride = 68;    // floats per row of a 64 x 64 matrix in LDS: rows 16-byte aligned, four banks apart

// ------------------------------------------------------------------------------------------------
// Everything of a chunk that does not depend on the state.  One workgroup per (slot, key head); the value heads that share
// the key head follow one another (K K^T and Q K^T are theirs together).
// ------------------------------------------------------------------------------------------------
template <typename In, int DK, int PT, bool BWD>
__global__ __launch_bounds__(256) void delta_prep_kernel(const DeltaArgs a) {
    constexpr int NI = In::kTerms, KS = DK / 32;
    typedef typename In::raw raw;
    __shared__ bf16x8 kfr[4 * KS * NI * 64];
    __shared__ f32x4 amat4[64 * kTriStride / 4], pmat4[64 * kTriStride / 4], tmat4[64 * kTriStride / 4];
    __shared__ float gs[64], bs[64];
    float* const amat = (float*)amat4;
    float* const pmat = (float*)pmat4;
    float* const tmat = (float*)tmat4;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = lane & 15, q = lane >> 4;
    const int slot = blockIdx.x / a.hk, h = blockIdx.x % a.hk;
    const int s = sequence_of(a, slot, lane);
    const Span sp = span_of(a, s);
    const int c = slot - sp.slot;
    const int start = sp.begin + c * kDeltaChunk;
    const int n = min(kDeltaChunk, sp.begin + sp.len - start);
    if (c < 0 || n <= 0) {
        // a slot of no chunk; those behind the last sequence's zero the rows behind it where that is asked for
        if (a.zero_tail && s == a.nseq - 1) {
            const int end = sp.begin + sp.len;
            const int lo = max(end, (slot - a.nseq) * kDeltaChunk), hi = min(a.tokens, (slot - a.nseq + 1) * kDeltaChunk);
            if (a.o)
                for (int t = lo; t < hi; ++t)
                    for (int hv = h * a.group; hv < (h + 1) * a.group; ++hv)
                        for (int d = threadIdx.x; d < a.dv_width; d += 256) ((raw*)a.o)[t * a.o_t + hv * a.o_h + d] = raw(0);
        }
        return;
    }

    // K and Q rows of this wave's 16 tokens as fragments; rows behind the sequence's end are zero
    bf16x8 kf[KS][NI], qf[KS][NI];
    const int row = 16 * w + j;
    const bool live = row < n;
    {
        const raw* kp = (const raw*)a.k + (start + (live ? row : 0)) * a.k_t + h * a.k_h;
        const raw* qp = (const raw*)a.q + (start + (live ? row : 0)) * a.q_t + h * a.q_h;
        const size_t at = ((size_t)(slot * (size_t)a.hk + h) * 4 + w) * KS * NI * 64 + lane;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = 32 * ks + 4 * q;
            const f32x4 zero = splat4(0.f);
            split8<NI>(live ? load4<In>(kp + d) : zero, live ? load4<In>(kp + d + 16) : zero, kf[ks]);
            split8<NI>(live ? load4<In>(qp + d) : zero, live ? load4<In>(qp + d + 16) : zero, qf[ks]);
#pragma unroll
            for (int t = 0; t < NI; ++t) {
                a.kf[at + (ks * NI + t) * 64] = kf[ks][t];
                a.qf[at + (ks * NI + t) * 64] = qf[ks][t];
                kfr[((w * KS + ks) * NI + t) * 64 + lane] = kf[ks][t];
            }
        }
    }
    __syncthreads();
    // K K^T and Q K^T, tiles (w, nt <= w): lane holds rows 16 w + 4 q + r, column 16 nt + j
    f32x4 kk[4], qk[4];
#pragma unroll
    for (int nt = 0; nt < 4; ++nt) {
        kk[nt] = qk[nt] = splat4(0.f);
        if (nt <= w) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8 b[NI];
#pragma unroll
                for (int t = 0; t < NI; ++t) b[t] = kfr[((nt * KS + ks) * NI + t) * 64 + lane];
                kk[nt] = mm(kf[ks], b, kk[nt]);
                qk[nt] = mm(qf[ks], b, qk[nt]);
            }
        }
    }
    // K^T (and Q^T): rows dk, k = tokens.  Element (token t, d) lies in fragment (t / 16, d / 32) at lane t % 16 + 16 ((d % 16) / 4)
    auto transposed = [&](bf16x8* to) {
        const unsigned short* src = (const unsigned short*)kfr;
        for (int f = w; f < (DK / 16) * 2; f += 4) {
            const int d = 16 * (f >> 1) + j;
            const int ks = d >> 5, half = (d >> 4) & 1, dq = (d & 15) >> 2, e = d & 3;
#pragma unroll
            for (int t = 0; t < NI; ++t) {
                u32x4 out;
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    unsigned x[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int el = 2 * p + i;
                        const int tok = 32 * (f & 1) + (el < 4 ? 4 * q + el : 16 + 4 * q + el - 4);
                        x[i] = src[((((tok >> 4) * KS + ks) * NI + t) * 64 + (tok & 15) + 16 * dq) * 8 + 4 * half + e];
                    }
                    out[p] = x[0] | x[1] << 16;
                }
                to[(((size_t)(slot * (size_t)a.hk + h) * (DK / 16) * 2 + f) * NI + t) * 64 + lane] = __builtin_bit_cast(bf16x8, out);
            }
        }
    };
    transposed(a.ktf);
    if constexpr (BWD) {
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int t = 0; t < NI; ++t) kfr[((w * KS + ks) * NI + t) * 64 + lane] = qf[ks][t];
        __syncthreads();
        transposed(a.qtf);
    }

    for (int hv = h * a.group; hv < (h + 1) * a.group; ++hv) {
        __syncthreads();
        if (w == 0) {
            const bool in = lane < n;
            gs[lane] = in ? a.g[(start + lane) * a.g_t + hv * a.g_h] : 0.f;
            bs[lane] = in ? a.beta[(start + lane) * a.b_t + hv * a.b_h] : 0.f;
        }
        __syncthreads();
        float block[4];
        block_sums(gs, block);
        if (w == 0) {
            float head, tail;
            head_tail(gs, block, lane, &head, &tail);
            float* sc = a.sc + (size_t)(slot * (size_t)a.hv + hv) * 256;
            sc[lane] = bs[lane];
            sc[64 + lane] = expf(head);
            sc[128 + lane] = expf(tail);
        }
        f32x4 decay[4];
        decays(gs, block, w, j, q, decay);
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            if (nt > w) continue;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * w + 4 * q + r, col = 16 * nt + j;
                amat[i * kTriStride + col] = col < i ? bs[i] * (kk[nt][r] * decay[nt][r]) : 0.f;
                pmat[i * kTriStride + col] = col <= i ? qk[nt][r] * decay[nt][r] : 0.f;
            }
        }
        __syncthreads();
        // T = (I + A)^-1: the 16 x 16 diagonal blocks by forward substitution, column j of block w in every lane quarter
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float v = i == j ? 1.f : 0.f;
#pragma unroll
            for (int m4 = 0; m4 < 4; ++m4) {
                if (4 * m4 < i) {
                    const f32x4 arow = amat4[((16 * w + i) * kTriStride + 16 * w) / 4 + m4];
#pragma unroll
                    for (int m = 0; m < 4; ++m)
                        if (4 * m4 + m < i) v -= arow[m] * x[4 * m4 + m];
                }
            }
            x[i] = v;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if ((i >> 2) == q) tmat[(16 * w + i) * kTriStride + 16 * w + j] = x[i];
        __syncthreads();
        // below the diagonal: T_iw = -T_ii sum_m A_im T_mw, wave w its block column, on the exact fp32 MFMA
        f32x4 tcol[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) tcol[0][r] = tmat[(16 * w + 4 * q + r) * kTriStride + 16 * w + j];
#pragma unroll
        for (int di = 1; di < 4; ++di) {
            if (w + di > 3) continue;
            const int i = w + di;
            f32x4 acc = splat4(0.f);
#pragma unroll
            for (int m = 0; m < di; ++m) {
                const f32x4 arow = amat4[((16 * i + j) * kTriStride + 16 * (w + m) + 4 * q) / 4];
#pragma unroll
                for (int r = 0; r < 4; ++r) acc = mfma4(arow[r], tcol[m][r], acc);
            }
            const f32x4 trow = tmat4[((16 * i + j) * kTriStride + 16 * i + 4 * q) / 4];
            f32x4 res = splat4(0.f);
#pragma unroll
            for (int r = 0; r < 4; ++r) res = mfma4(trow[r], acc[r], res);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                tcol[di][r] = -res[r];
                tmat[(16 * i + 4 * q + r) * kTriStride + 16 * w + j] = -res[r];
            }
        }
        __syncthreads();
        // T and P as A operands of the chain
        const size_t at = (size_t)(slot * (size_t)a.hv + hv) * kTriFrags;
        for (int f = w; f < 2 * kTriFrags; f += 4) {
            const bool isp = f >= kTriFrags;
            const int ff = isp ? f - kTriFrags : f;
            const int mt = tri_row(ff), ks = tri_step(ff);
            const f32x4* m4 = (isp ? pmat4 : tmat4) + ((16 * mt + j) * kTriStride + 32 * ks + 4 * q) / 4;
            const f32x4 lo = m4[0], hi = (mt & 1) || ks < (mt >> 1) ? m4[4] : splat4(0.f);
            bf16x8 t[3];
            split8<3>(lo, hi, t);
            if (isp) {
#pragma unroll
                for (int k = 0; k < PT; ++k) a.pf[((at + ff) * PT + k) * 64 + lane] = t[k];
            } else {
#pragma unroll
                for (int k = 0; k < 3; ++k) a.tf[((at + ff) * 3 + k) * 64 + lane] = t[k];
            }
        }
        if constexpr (BWD) {
            for (int f = w; f < 2 * kTriFrags; f += 4) {
                const bool isp = f >= kTriFrags;
                const int ff = isp ? f - kTriFrags : f;
                const int mt = trt_row(ff), ks = trt_step(ff);
                const float* src = isp ? pmat : tmat;
                f32x4 lo, hi;
                const bool half = (mt & 1) && ks == (mt >> 1);      // the first half lies above the diagonal's block
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    lo[e] = half ? 0.f : src[(32 * ks + 4 * q + e) * kTriStride + 16 * mt + j];
                    hi[e] = src[(32 * ks + 16 + 4 * q + e) * kTriStride + 16 * mt + j];
                }
                bf16x8 t[3];
                split8<3>(lo, hi, t);
#pragma unroll
                for (int k = 0; k < 3; ++k) (isp ? a.ptf : a.ttf)[((at + ff) * 3 + k) * 64 + lane] = t[k];
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// The chain: one wave per (sequence, value head, 16 columns of the state).
// ------------------------------------------------------------------------------------------------
template <typename In, int DK, int PT, bool KEEP>
__global__ __launch_bounds__(256) void delta_forward_kernel(const DeltaArgs a) {
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
        for (int r = 0; r < 4; ++r) S[m][r] = a.s0 ? a.s0[st + (size_t)(16 * m + 4 * q + r) * a.dv_width + col] : 0.f;

    for (int c = 0; c * kDeltaChunk < sp.len; ++c) {
        const int start = sp.begin + c * kDeltaChunk, n = min(kDeltaChunk, sp.len - c * kDeltaChunk);
        const size_t slot = (size_t)sp.slot + c, kslot = slot * a.hk + h, vslot = slot * a.hv + hv;
        const float* sc = a.sc + vslot * 256;
        if constexpr (KEEP) {
            float* to = a.states + vslot * DK * a.dv_width + col;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r) to[(size_t)(16 * m + 4 * q + r) * a.dv_width] = S[m][r];
        }
        bf16x8 sb[KS][3];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) split8<3>(S[2 * ks], S[2 * ks + 1], sb[ks]);
        f32x4 R[4], O[4];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            R[mt] = O[mt] = splat4(0.f);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8 kf[NI], qf[NI];
#pragma unroll
                for (int t = 0; t < NI; ++t) {
                    const size_t at = (((kslot * 4 + mt) * KS + ks) * NI + t) * 64 + lane;
                    kf[t] = a.kf[at];
                    qf[t] = a.qf[at];
                }
                R[mt] = mm(kf, sb[ks], R[mt]);
                O[mt] = mm(qf, sb[ks], O[mt]);
            }
        }
        f32x4 X[4];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            const f32x4 beta = *(const f32x4*)(sc + 16 * mt + 4 * q), eb = *(const f32x4*)(sc + 64 + 16 * mt + 4 * q);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * mt + 4 * q + r;
                const float v = t < n ? In::to_f32(((const raw*)a.v)[(start + t) * a.v_t + hv * a.v_h + col]) : 0.f;
                R[mt][r] = v - eb[r] * R[mt][r];
                O[mt][r] *= eb[r];
                X[mt][r] = beta[r] * R[mt][r];
                if constexpr (KEEP) a.r[(vslot * kDeltaChunk + t) * a.dv_width + col] = R[mt][r];
            }
        }
        bf16x8 xb[2][3];
        split8<3>(X[0], X[1], xb[0]);
        split8<3>(X[2], X[3], xb[1]);
        f32x4 U[4];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            U[mt] = splat4(0.f);
#pragma unroll
            for (int ks = 0; ks <= mt / 2; ++ks) {
                bf16x8 tf[3];
#pragma unroll
                for (int t = 0; t < 3; ++t) tf[t] = a.tf[((vslot * kTriFrags + tri_index(mt, ks)) * 3 + t) * 64 + lane];
                U[mt] = mm(tf, xb[ks], U[mt]);
            }
            if constexpr (KEEP) {
#pragma unroll
                for (int r = 0; r < 4; ++r) a.u[(vslot * kDeltaChunk + 16 * mt + 4 * q + r) * a.dv_width + col] = U[mt][r];
            }
        }
        bf16x8 ub[2][PT];
        split8<PT>(U[0], U[1], ub[0]);
        split8<PT>(U[2], U[3], ub[1]);
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
            for (int ks = 0; ks <= mt / 2; ++ks) {
                bf16x8 pf[PT];
#pragma unroll
                for (int t = 0; t < PT; ++t) pf[t] = a.pf[((vslot * kTriFrags + tri_index(mt, ks)) * PT + t) * 64 + lane];
                O[mt] = mm<PT, PT, PT - 1>(pf, ub[ks], O[mt]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * mt + 4 * q + r;
                if (a.o && t < n) ((raw*)a.o)[(start + t) * a.o_t + hv * a.o_h + col] = In::from_f32(a.scale * O[mt][r]);
            }
        }
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            const f32x4 ec = *(const f32x4*)(sc + 128 + 16 * mt + 4 * q);
#pragma unroll
            for (int r = 0; r < 4; ++r) U[mt][r] *= ec[r];
        }
        const float whole = sc[64 + 63];
        bf16x8 uc[2][3];
        split8<3>(U[0], U[1], uc[0]);
        split8<3>(U[2], U[3], uc[1]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int r = 0; r < 4; ++r) S[m][r] *= whole;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                bf16x8 kt[NI];
#pragma unroll
                for (int t = 0; t < NI; ++t) kt[t] = a.ktf[((kslot * MT * 2 + 2 * m + ks) * NI + t) * 64 + lane];
                S[m] = mm(kt, uc[ks], S[m]);
            }
        }
    }
    if (a.s1) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) a.s1[st + (size_t)(16 * m + 4 * q + r) * a.dv_width + col] = S[m][r];
    }
}

}  // namespace helen
