// kernels_delta.h -- the gated delta rule over whole sequences, in chunks of 64 tokens: preparation and forward chain
//
// Per sequence and value head, with a state S [Dk, Dv] and e^{g} the decay of a token:
//     u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t),   S_t = e^{g_t} S_{t-1} + k_t u_t^T,   o_t = scale S_t^T q_t
// In a chunk of C = 64 tokens, with D_ij = sum of g over (j, i], b_i the sum from the chunk's start and c_i the sum after i
// to its end, all C tokens are products (S0 = the state before the chunk):
//     A_ij = (k_i . k_j) e^{D_ij} beta_j (j < i),  T = (I + A)^-1,   R = V - e^{b} K S0,   E = T R,   U = beta E,
//     O = scale (e^{b} Q S0 + P U),  P_ij = (q_i . k_j) e^{D_ij} (j <= i),   S1 = e^{b_C} S0 + K^T (e^{c} U)
// (E_t = v_t - e^{g_t} S_{t-1}^T k_t, what the state got wrong.  With beta on the columns of A the backward pass needs E alone:
// d beta = Z . E / beta, see kernels_delta_bwd.h.  A beta below 2^-64 counts as 2^-64 in A, far below a rounding, so that this
// quotient exists where beta is zero; U takes beta as it is.)
// A, T and P do not depend on the state: delta_prep_kernel makes them for every chunk at once.  What is left, one chunk after
// another, is delta_forward_kernel: a column of S needs no other column, so a chain is split over its columns.
//
// Arithmetic: as in the fp32x3 recurrence, an fp32 value is the sum of three bf16 terms and a product of two such values the
// six leading products of terms on v_mfma_f32_16x16x32_bf16 with fp32 accumulation.  bf16 inputs are ONE term (their products
// with S are exact), fp16 inputs two, fp32 inputs three; whatever is computed (S, E, U, R, T, P, the gradients' G and H) has
// three in every product, so a call with 16-bit inputs gives the float32 call's results, rounded once.  Decays between two
// positions are sums of the g between them, never a difference of two running sums: a strong decay (or g = -inf, a reset) costs
// the other positions no digits.
//
// Fragments.  lane l: j = l & 15, q = l >> 4.  The k index of an MFMA may be permuted if both operands agree, so that a result (S,
// U, R) becomes the next product's B operand without any exchange: two stacked D tiles lie in the accumulators as element
// e = 0 .. 7 of lane quarter q.  Over tokens that is k = 32 s + (e < 4 ? 4 q + e : 16 + 4 q + e - 4); over dk the rows of S go to the
// tiles in such an order (state_row) that it is k = 32 s + 8 q + e, eight neighbours of a row of K or Q.
//
// Times of kernels here and in kernels_delta_bwd.h are the fastest of six launches under a kernel trace (the first ones, on cold
// caches and clocks, are up to a fifth longer); shares of the matrix pipe, waits and bytes come from its counters.
#pragma once
#include "kernels_common.h"

namespace helen {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

template <bool B>
struct Is {
    static constexpr bool value = B;
};

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

// VALU instructions stay on their side of this, all others may cross
__device__ __forceinline__ void valu_fence() { __builtin_amdgcn_sched_barrier(0x4 | 0x8 | 0x10 | 0x80); }

// N bf16 terms of 2 P fp32 values: x = t[0] + t[1] + t[2] exactly (3 x 8 significand bits).  One level of all values after the
// other: a VALU instruction that needs the result of the one right before it costs 9 cycles here instead of 4 to 5, and left
// alone the compiler puts each value's chain in one piece.
template <int N, int P>
__device__ __forceinline__ void split_pairs(f32x2 (&x)[P], unsigned (&t)[N][P]) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int p = 0; p < P; ++p) t[n][p] = __builtin_bit_cast(unsigned, __builtin_convertvector(x[p], bf16x2_t));
        if (n + 1 < N) {
            f32x2 hi[P];
            valu_fence();
#pragma unroll
            for (int p = 0; p < P; ++p) hi[p] = (f32x2){__builtin_bit_cast(float, t[n][p] << 16), __builtin_bit_cast(float, t[n][p] & 0xffff0000u)};
            valu_fence();
#pragma unroll
            for (int p = 0; p < P; ++p) {
                x[p].x -= hi[p].x;
                x[p].y -= hi[p].y;
            }
            valu_fence();
        }
    }
}
template <int N>
__device__ __forceinline__ void split8(const f32x4 lo, const f32x4 hi, bf16x8 (&t)[N]) {
    f32x2 x[4] = {{lo[0], lo[1]}, {lo[2], lo[3]}, {hi[0], hi[1]}, {hi[2], hi[3]}};
    unsigned w[N][4];
    split_pairs<N, 4>(x, w);
#pragma unroll
    for (int n = 0; n < N; ++n) t[n] = __builtin_bit_cast(bf16x8, (u32x4){w[n][0], w[n][1], w[n][2], w[n][3]});
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

// NC neighbouring elements of a row
template <typename In, int NC>
struct Columns {
    typedef typename In::raw raw;
    typedef raw vec __attribute__((ext_vector_type(NC)));
    typedef vec vec_any __attribute__((aligned(sizeof(raw))));      // rows may begin anywhere
    vec v;
    static __device__ __forceinline__ Columns load(const raw* p) { return {*(const vec_any*)p}; }
    __device__ __forceinline__ float get(int nc) const { return In::to_f32(v[nc]); }
    static __device__ __forceinline__ void store(raw* p, const float (&x)[NC]) {
        vec t;
        if constexpr (In::kTerms == 1) {      // (two a conversion)
            typedef unsigned pairs __attribute__((ext_vector_type(NC / 2)));
            pairs y;
#pragma unroll
            for (int p = 0; p < NC / 2; ++p) y[p] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){x[2 * p], x[2 * p + 1]}, bf16x2_t));
            t = __builtin_bit_cast(vec, y);
        } else {
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) t[nc] = In::from_f32(x[nc]);
        }
        *(vec_any*)p = t;
    }
};
template <typename In>
struct Columns<In, 1> {
    typedef typename In::raw raw;
    raw v;
    static __device__ __forceinline__ Columns load(const raw* p) { return {*p}; }
    __device__ __forceinline__ float get(int) const { return In::to_f32(v); }
    static __device__ __forceinline__ void store(raw* p, const float (&x)[1]) { *p = In::from_f32(x[0]); }
};

// LDS writes of every wave are visible behind this; loads and stores to memory stay in flight over it
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
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
    void* sink;                 // where rows behind a sequence's end are stored
    bf16x8* zeros;              // three fragments of zeros: the k step of a triangle's row tile that lies above the diagonal
    int zero_tail;              // rows behind the last sequence: 1 = zero them, 0 = leave them
    // workspace: fragments per (slot, key head) and per (slot, value head)
    bf16x8 *kf, *ktf, *qf, *qtf;           // (kf, qf null where the chain takes the inputs' rows)
    bf16x8 *tf, *ttf, *pf, *ptf;
    f32x4* dots;                // kept: [slot, hk][10 tiles][K K^T | Q K^T][lane]
    float* sc;                  // [slot, hv][4][64]: beta, e^b (its last one is e^{b_C}), e^c, beta e^c
    float *states, *e;          // kept for the backward pass: [slot, hv, Dk, Dv], [slot, hv, 64, Dv]
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
// The sequence that holds a slot, 64 probes a round, and its span (read in the last round: one trip to memory less)
__device__ __forceinline__ int sequence_of(const DeltaArgs& a, int slot, int lane, Span* span) {
    int lo = 0, n = a.nseq;
    while (true) {
        const int step = (n + 63) >> 6;
        const int s = min(lo + lane * step, a.nseq - 1);
        int b, e;
        if (a.offsets) {
            b = min(max(a.offsets[s], 0), a.tokens);
            e = min(max(a.offsets[s + 1], b), a.tokens);
        } else {
            b = s * a.seq_len;
            e = b + a.seq_len;
        }
        const int hits = __popcll(__ballot(lane * step < n && b / kDeltaChunk + s <= slot));
        const int at = max(hits - 1, 0);
        if (step == 1) {
            b = __builtin_amdgcn_readlane(b, at);
            e = __builtin_amdgcn_readlane(e, at);
            lo += at;
            *span = {b, e - b, b / kDeltaChunk + lo};
            return lo;
        }
        lo += at * step;
        n = min(step, n - at * step);
    }
}

// lower triangle (tf, pf): fragment f = row tile mt, k step ks of mt's; the last step of an even row tile ends in a zero half
__device__ __forceinline__ int tri_row(int f) { return f < 2 ? f : (f < 4 ? 2 : 3); }
__device__ __forceinline__ int tri_step(int f) { return f < 2 ? 0 : (f & 1); }
__device__ __forceinline__ constexpr int tri_index(int mt, int ks) { return mt < 2 ? mt : 2 * mt - 2 + ks; }
// its transpose (ttf, ptf): rows are tokens j, k steps the tokens i >= j: (0,0) (0,1) (1,0) (1,1) (2,1) (3,1)
__device__ __forceinline__ int trt_row(int f) { return f < 4 ? f >> 1 : f - 2; }
__device__ __forceinline__ int trt_step(int f) { return f < 4 ? f & 1 : 1; }
__device__ __forceinline__ constexpr int trt_index(int mt, int ks) { return mt < 2 ? 2 * mt + ks : mt + 2; }

__device__ __forceinline__ float beta_of(float beta) { return fabsf(beta) < 0x1p-64f ? 0x1p-64f : beta; }

// e^x of a decay: 2^(x log2 e) with the product's rounding error put back (v_exp_f32 alone would be off by |x| 2^-24); 0 from
// -150 down, -inf included; a NaN stays one
__device__ __forceinline__ float exp_decay(float x) {
    x = x < -150.f ? -150.f : x;
    const float t = x * 1.44269504f;
    const float low = __builtin_fmaf(x, 1.44269504f, -t) + x * 1.9259630e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, low * 0.693147181f, e);
}

// the lane's own value plus others of its row of 16 lanes (rotations and shifts on the VALU; shifts bring in zeros)
template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
    return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// What a chunk's decays are made of, in LDS.  e^{D_ij} is a product: from j to the end of its block of 16 tokens, over the blocks
// between, from the start of i's block to i -- and inside a block the same over groups of four.  Each factor is e to a sum of
// the g it covers.  (All are at most one where g <= 0: a product that underflows stands for a decay that does.)
struct Decays {
    float g[64];
    float head[64], tail[64];      // e^(sum of g): from the block's start up to and with the token; after it to the block's end
    float head4[64], tail4[64];    // the same in groups of four
    // the 64 lanes of one wave
    __device__ __forceinline__ void set(int lane, float x) {
        const int e = lane & 3;
        g[lane] = x;
        const float h = dpp_add<0x118>(dpp_add<0x114>(dpp_add<0x112>(dpp_add<0x111>(x))));
        const float t = dpp_add<0x108>(dpp_add<0x104>(dpp_add<0x102>(dpp_add<0x101>(dpp<0x101>(x)))));
        // (neighbours are read by all lanes, and then chosen: a lane that is switched off gives nothing)
        const float b1 = dpp<0x111>(x), n1 = dpp<0x101>(x);
        float h4 = x + (e >= 1 ? b1 : 0.f), t4 = x + (e <= 2 ? n1 : 0.f);
        const float b2 = dpp<0x112>(h4), n2 = dpp<0x102>(t4);
        h4 += e >= 2 ? b2 : 0.f;
        t4 += e <= 1 ? n2 : 0.f;
        t4 = dpp<0x101>(t4);
        head[lane] = exp_decay(h);
        tail[lane] = exp_decay(t);
        head4[lane] = exp_decay(h4);
        tail4[lane] = exp_decay(e <= 2 ? t4 : 0.f);
    }
    __device__ __forceinline__ float block(int b) const { return head[16 * b + 15]; }
    // e^b and e^c of token `lane`
    __device__ __forceinline__ void ends(int lane, float* from_start, float* to_end) const {
        float a = head[lane], b = tail[lane];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const float x = block(m);
            a *= m < (lane >> 4) ? x : 1.f;
            b *= m > (lane >> 4) ? x : 1.f;
        }
        *from_start = a;
        *to_end = b;
    }
    __device__ __forceinline__ float between(int mt, int nt) const {
        float x = 1.f;
        if (nt + 1 < mt) x *= block(nt + 1);
        if (nt + 2 < mt) x *= block(nt + 2);
        return x;
    }
    __device__ __forceinline__ float between4(int mt, int iq, int jq) const {      // groups of four jq < k < iq of block mt
        float x = jq < 1 && iq > 1 ? head4[16 * mt + 7] : 1.f;
        return jq < 2 && iq > 2 ? x * head4[16 * mt + 11] : x;
    }
    // e^{D_ij} of tile (mt, nt <= mt); what lies above the diagonal is not used.
    // rows: i = 16 mt + 4 q + r, column 16 nt + j (as results lie)
    __device__ __forceinline__ f32x4 rows(int mt, int nt, int j, int q) const {
        f32x4 d;
        if (nt < mt) {
            const float t = tail[16 * nt + j] * between(mt, nt);
            const f32x4 h = *(const f32x4*)&head[16 * mt + 4 * q];
#pragma unroll
            for (int r = 0; r < 4; ++r) d[r] = h[r] * t;
        } else {
            const f32x4 x = *(const f32x4*)&g[16 * mt + 4 * q], h = *(const f32x4*)&head4[16 * mt + 4 * q];
            const int jq = j >> 2, je = j & 3;
            const float t = tail4[16 * mt + j] * between4(mt, q, jq);
            const float d1 = je < 1 ? x[1] : 0.f, d2 = d1 + (je < 2 ? x[2] : 0.f), d3 = d2 + (je < 3 ? x[3] : 0.f);
            const bool same = q == jq;
            d[0] = same ? 1.f : h[0] * t;
            d[1] = same ? exp_decay(d1) : h[1] * t;
            d[2] = same ? exp_decay(d2) : h[2] * t;
            d[3] = same ? exp_decay(d3) : h[3] * t;
        }
        return d;
    }
    // columns: row 16 mt + j, column 16 nt + 4 q + r (as left-hand operands lie)
    __device__ __forceinline__ f32x4 columns(int mt, int nt, int j, int q) const {
        f32x4 d;
        if (nt < mt) {
            const float h = head[16 * mt + j] * between(mt, nt);
            const f32x4 t = *(const f32x4*)&tail[16 * nt + 4 * q];
#pragma unroll
            for (int r = 0; r < 4; ++r) d[r] = h * t[r];
        } else {
            const f32x4 x = *(const f32x4*)&g[16 * mt + 4 * q], t = *(const f32x4*)&tail4[16 * mt + 4 * q];
            const int iq = j >> 2, ie = j & 3;
            const float h = head4[16 * mt + j] * between4(mt, iq, q);
            const float d2 = ie > 2 ? x[3] : 0.f, d1 = d2 + (ie > 1 ? x[2] : 0.f), d0 = d1 + (ie > 0 ? x[1] : 0.f);
            const bool same = q == iq;
            d[0] = same ? exp_decay(d0) : h * t[0];
            d[1] = same ? exp_decay(d1) : h * t[1];
            d[2] = same ? exp_decay(d2) : h * t[2];
            d[3] = same ? 1.f : h * t[3];
        }
        return d;
    }
};

constexpr int kTriStride = 68;    // floats per row of a 64 x 64 matrix in LDS: rows 16-byte aligned, four banks apart

// ------------------------------------------------------------------------------------------------
// Everything of a chunk that does not depend on the state.  One workgroup per (slot, key head); the value heads that share
// the key head follow one another (K K^T and Q K^T are theirs together).
//
// What becomes a left-hand operand is computed transposed, (Q K^T)^T = K Q^T: a result tile then already lies as that operand
// (lane = row, four neighbouring columns), so P goes from the accumulators to memory, and A to LDS and back in whole
// fragments.  K^T comes from the matrix pipe too: K times a selection of 16 columns is K's tile with lane = dk.
// What bounds it: bandwidth, mostly its own writing.  16,384 tokens, 16 key and 32 value heads of 128, bf16: 0.10 GB read and 0.52
// written in 117 us, 5.3 TB/s, what a large copy reaches; the four workgroups a CU (35 KB of LDS, 128 registers) took it there
// (from 140 us to 109, then with P in two terms).
// ------------------------------------------------------------------------------------------------
template <typename In, int DK, bool BWD>
__global__ __launch_bounds__(256, In::kTerms == 1 ? (BWD ? 3 : 4) : 1) void delta_prep_kernel(const DeltaArgs a) {
    constexpr int NI = In::kTerms, KS = DK / 32;
    constexpr int kTile = 64 + 4;               // an operand tile in LDS: [column / 4][row] x 4, column groups 17 apart
    typedef typename In::raw raw;
    // K and Q of all rows; later, in their place, A and T (three or four workgroups fit a CU)
    constexpr int kRows = 4 * KS * NI * 64, kTiles = 10 * 64 + 10 * kTile;
    __shared__ f32x4 pool[2 * kRows > kTiles ? 2 * kRows : kTiles];
    bf16x8* const kfr = (bf16x8*)pool;
    bf16x8* const qfr = kfr + kRows;
    f32x4* const atile = pool;
    f32x4* const ttile = pool + 10 * 64;
    __shared__ __attribute__((aligned(16))) Decays dec;
    __shared__ __attribute__((aligned(16))) float bs[64];
    const int lane0 = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slot = blockIdx.x / a.hk, h = blockIdx.x % a.hk;
    if (blockIdx.x == 0 && threadIdx.x < 192) ((u32x4*)a.zeros)[threadIdx.x] = (u32x4){0, 0, 0, 0};
    Span sp;
    const int s = sequence_of(a, slot, lane0, &sp);
    const int c = slot - sp.slot;
    const int start = sp.begin + c * kDeltaChunk;
    const int n = min(kDeltaChunk, sp.begin + sp.len - start);
    if (c < 0 || n <= 0) {
        // a slot of no chunk; those behind the last sequence's zero the rows behind it where that is asked for
        if (a.zero_tail && s == a.nseq - 1) {
            const int end = sp.begin + sp.len;
            const int lo = max(end, (slot - a.nseq) * kDeltaChunk), hi = min(a.tokens, (slot - a.nseq + 1) * kDeltaChunk);
            for (int t = lo; t < hi; ++t)
                for (int hv = h * a.group; hv < (h + 1) * a.group; ++hv)
                    for (int d = threadIdx.x; d < a.dv_width; d += 256) ((raw*)a.o)[t * a.o_t + hv * a.o_h + d] = raw(0);
        }
        return;
    }
    // g and beta of the value head that is next, a token a lane of wave 3
    float gx = 0.f, bx = 0.f;
    auto load_gates = [&](int hv) {
        if (w == 3 && lane0 < n) {
            gx = a.g[(start + lane0) * a.g_t + hv * a.g_h];
            bx = a.beta[(start + lane0) * a.b_t + hv * a.b_h];
        }
    };
    load_gates(h * a.group);

    // tiles (row tile, column tile) of this wave: those of its fragments of T, P ({0,1}, {2,3}, {4}, {5}) ...
    const int count = w < 2 ? 3 : 2;
    const int tm[3] = {w == 0 ? 0 : (w == 1 ? 2 : 3), w == 0 ? 1 : (w == 1 ? 2 : 3), w == 0 ? 1 : 2};
    const int tn[3] = {w == 3 ? 2 : 0, w == 0 ? 0 : (w == 3 ? 3 : 1), w == 0 ? 1 : 2};
    // ... and of T^T, P^T ({(0,0), (1,0)}, {(1,1), (3,1)}, {(0,1)}, {(2,1)})
    const int um[3] = {w == 0 ? 0 : 2, w == 0 ? 1 : 3, w == 0 ? 1 : 3};
    const int un[3] = {w == 0 ? 0 : (w == 1 ? 1 : (w == 2 ? 0 : 2)), w == 0 ? 0 : (w == 1 ? 1 : (w == 2 ? 0 : 2)), w == 0 ? 1 : 3};
    f32x4 kkt[3], qkt[3], kk[3], qk[3];
    {
        const int lane = lane0, j = lane & 15, q = lane >> 4;
        // K and Q rows of this wave's 16 tokens as fragments; rows behind the sequence's end are zero
        bf16x8 kf[KS][NI], qf[KS][NI];
        const int row = 16 * w + j;
        const bool live = row < n;
        const raw* kp = (const raw*)a.k + (start + (live ? row : 0)) * a.k_t + h * a.k_h + 8 * q;
        const raw* qp = (const raw*)a.q + (start + (live ? row : 0)) * a.q_t + h * a.q_h + 8 * q;
        if constexpr (NI == 1) {
            const bf16x8 none = __builtin_bit_cast(bf16x8, (u32x4){0u, 0u, 0u, 0u});
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                kf[ks][0] = *(const bf16x8*)(kp + 32 * ks);
                qf[ks][0] = *(const bf16x8*)(qp + 32 * ks);
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                kf[ks][0] = live ? kf[ks][0] : none;
                qf[ks][0] = live ? qf[ks][0] : none;
            }
        } else {
            f32x4 kx[KS][2], qx[KS][2];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    kx[ks][i] = load4<In>(kp + 32 * ks + 4 * i);
                    qx[ks][i] = load4<In>(qp + 32 * ks + 4 * i);
                }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const f32x4 zero = splat4(0.f);
                split8<NI>(live ? kx[ks][0] : zero, live ? kx[ks][1] : zero, kf[ks]);
                split8<NI>(live ? qx[ks][0] : zero, live ? qx[ks][1] : zero, qf[ks]);
            }
        }
        const size_t rows_at = (((size_t)slot * a.hk + h) * 4 + w) * KS * NI * 64;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int t = 0; t < NI; ++t) {
                kfr[((w * KS + ks) * NI + t) * 64 + lane] = kf[ks][t];
                qfr[((w * KS + ks) * NI + t) * 64 + lane] = qf[ks][t];
                if (NI > 1 || BWD || a.kf) {
                    (a.kf + rows_at + (ks * NI + t) * 64)[lane] = kf[ks][t];
                    (a.qf + rows_at + (ks * NI + t) * 64)[lane] = qf[ks][t];
                }
            }
        // K^T, Q^T: half (w & 1) of the fragments of token step w >> 1, dk tiles 2 ks + i
        const unsigned one = q == (j >> 2) ? 0x3f80u << (16 * (j & 1)) : 0u;
        const unsigned lo = j & 2 ? 0u : one, hi = j & 2 ? one : 0u;
        const bf16x8 pick[2] = {__builtin_bit_cast(bf16x8, (u32x4){lo, hi, 0u, 0u}), __builtin_bit_cast(bf16x8, (u32x4){0u, 0u, lo, hi})};
        auto turn = [&](const bf16x8 (&from)[KS][NI], bf16x8* to) {
            to += ((size_t)slot * a.hk + h) * (DK / 8) * NI * 64 + (w >> 1) * NI * 64;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int t = 0; t < NI; ++t) {
                        const f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(from[ks][t], pick[i], splat4(0.f), 0, 0, 0);
                        const u32x2 y = {__builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){x[0], x[1]}, bf16x2_t)),
                                         __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){x[2], x[3]}, bf16x2_t))};
                        ((u32x2*)(to + ((2 * ks + i) * 2 * NI + t) * 64))[2 * (unsigned)lane + (w & 1)] = y;
                    }
        };
        turn(kf, a.ktf);
        if constexpr (BWD) turn(qf, a.qtf);
        lds_barrier();
        auto product = [&](const bf16x8* x, int xt, const bf16x8* y, int yt) {
            f32x4 sum = splat4(0.f);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8 xf[NI], yf[NI];
#pragma unroll
                for (int t = 0; t < NI; ++t) {
                    xf[t] = x[((xt * KS + ks) * NI + t) * 64 + lane];
                    yf[t] = y[((yt * KS + ks) * NI + t) * 64 + lane];
                }
                sum = mm(xf, yf, sum);
            }
            return sum;
        };
#pragma unroll
        for (int t = 0; t < 3; ++t) {
            if (t >= count) continue;
            kkt[t] = product(kfr, tn[t], kfr, tm[t]);
            qkt[t] = product(kfr, tn[t], qfr, tm[t]);
        }
        if constexpr (BWD) {
#pragma unroll
            for (int t = 0; t < 3; ++t) {
                if (t >= count) continue;
                kk[t] = product(kfr, um[t], kfr, un[t]);
                qk[t] = product(qfr, um[t], kfr, un[t]);
                f32x4* to = a.dots + (((size_t)slot * a.hk + h) * 10 + um[t] * (um[t] + 1) / 2 + un[t]) * 128 + lane;
                to[0] = kk[t];
                to[64] = qk[t];
            }
        }
    }

    for (int hv = h * a.group; hv < (h + 1) * a.group; ++hv) {
        const unsigned lane = in_block(lane0);      // (nothing of a head's addresses is kept over the loop)
        const int j = lane & 15, q = lane >> 4;
        const size_t vslot = (size_t)slot * a.hv + hv;
        if (w == 3) {
            dec.set(lane, gx);
            bs[lane] = bx;
            if (hv + 1 < (h + 1) * a.group) load_gates(hv + 1);
        }
        lds_barrier();
        if (w == 2) {
            float from_start, to_end;
            dec.ends(lane, &from_start, &to_end);
            float* sc = a.sc + vslot * 256;
            sc[lane] = bs[lane];
            (sc + 64)[lane] = from_start;
            (sc + 128)[lane] = to_end;
            (sc + 192)[lane] = bs[lane] * to_end;
        }
        // A to LDS, P to memory: row 16 tm + j, columns 16 tn + 4 q + r
        f32x4 P[3];
#pragma unroll
        for (int t = 0; t < 3; ++t) {
            P[t] = splat4(0.f);
            if (t >= count) continue;
            const f32x4 e = dec.columns(tm[t], tn[t], j, q), b = *(const f32x4*)&bs[16 * tn[t] + 4 * q];
            const bool diagonal = tm[t] == tn[t];
            f32x4 A;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                A[r] = diagonal && 4 * q + r >= j ? 0.f : beta_of(b[r]) * (kkt[t][r] * e[r]);
                P[t][r] = diagonal && 4 * q + r > j ? 0.f : qkt[t][r] * e[r];
            }
            atile[(tm[t] * (tm[t] + 1) / 2 + tn[t]) * 64 + lane] = A;
        }
        auto put_p = [&](int f, const f32x4 lo, const f32x4 hi) {
            bf16x8 t[3];
            split8<3>(lo, hi, t);
            bf16x8* const to = a.pf + (vslot * kTriFrags + f) * 3 * 64;
#pragma unroll
            for (int k = 0; k < 3; ++k) (to + k * 64)[lane] = t[k];
        };
        if (w == 0) {
            put_p(0, P[0], splat4(0.f));
            put_p(1, P[1], P[2]);
        } else if (w == 1) {
            put_p(2, P[0], P[1]);
            put_p(3, P[2], splat4(0.f));
        } else {
            put_p(w + 2, P[0], P[1]);
        }
        if constexpr (BWD) {       // P^T: row = token 16 un + j, elements tokens 16 um + 4 q + r
#pragma unroll
            for (int t = 0; t < 3; ++t) {
                P[t] = splat4(0.f);
                if (t >= count) continue;
                const f32x4 e = dec.rows(um[t], un[t], j, q);
#pragma unroll
                for (int r = 0; r < 4; ++r) P[t][r] = um[t] == un[t] && j > 4 * q + r ? 0.f : qk[t][r] * e[r];
            }
            auto put_pt = [&](int f, const f32x4 lo, const f32x4 hi) {
                bf16x8 t[3];
                split8<3>(lo, hi, t);
                bf16x8* const to = a.ptf + (vslot * kTriFrags + f) * 3 * 64;
#pragma unroll
                for (int k = 0; k < 3; ++k) (to + k * 64)[lane] = t[k];
            };
            const f32x4 none = splat4(0.f);
            if (w == 0) {
                put_pt(trt_index(0, 0), P[0], P[1]);
                put_pt(trt_index(1, 0), none, P[2]);
            } else if (w == 1) {
                put_pt(trt_index(1, 1), P[0], P[1]);
                put_pt(trt_index(3, 1), none, P[2]);
            } else {
                put_pt(w == 2 ? trt_index(0, 1) : trt_index(2, 1), P[0], P[1]);
            }
        }
        lds_barrier();
        // T = (I + A)^-1: the 16 x 16 diagonal blocks by forward substitution, column j of block w in every lane quarter.  Four
        // rows at a time: solved one after the other, then taken out of all rows below.
        f32x4 tcol[4];
        {
            const f32x4* const from = atile + (w * (w + 1) / 2 + w) * 64;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = i == j ? 1.f : 0.f;
#pragma unroll
            for (int m4 = 0; m4 < 4; ++m4) {
                f32x4 row[16];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i > 4 * m4) row[i] = from[16 * m4 + i];
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (i > 4 * m4 + m) x[i] -= row[i][m] * x[4 * m4 + m];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float x0 = x[r], x1 = x[4 + r], x2 = x[8 + r], x3 = x[12 + r];
                asm("" : "+v"(x0), "+v"(x1), "+v"(x2), "+v"(x3));      // (values: a choice of addresses would put x in memory)
                tcol[0][r] = q < 2 ? (q == 0 ? x0 : x1) : (q == 2 ? x2 : x3);
            }
        }
        // a tile of T (lane = column, rows 4 q + r) as a left-hand operand
        auto put_t = [&](int id, const f32x4 x) {
            float* const to = (float*)(ttile + id * kTile + (j >> 2) * 17 + 4 * q) + (j & 3);
#pragma unroll
            for (int r = 0; r < 4; ++r) to[4 * r] = x[r];
        };
        put_t(w * (w + 1) / 2 + w, tcol[0]);
        lds_barrier();
        // below the diagonal: T_iw = -T_ii sum_m A_im T_mw, wave w its block column, on the exact fp32 MFMA
#pragma unroll
        for (int di = 1; di < 4; ++di) {
            if (w + di > 3) continue;
            const int i = w + di, row = i * (i + 1) / 2;
            f32x4 acc = splat4(0.f);
#pragma unroll
            for (int m = 0; m < di; ++m) {
                const f32x4 arow = atile[(row + w + m) * 64 + lane];
#pragma unroll
                for (int r = 0; r < 4; ++r) acc = mfma4(arow[r], tcol[m][r], acc);
            }
            const f32x4 trow = ttile[(row + i) * kTile + 17 * q + j];
            f32x4 res = splat4(0.f);
#pragma unroll
            for (int r = 0; r < 4; ++r) res = mfma4(trow[r], acc[r], res);
#pragma unroll
            for (int r = 0; r < 4; ++r) tcol[di][r] = -res[r];
            put_t(row + w, tcol[di]);
        }
        if constexpr (BWD) {
            auto put_tt = [&](int ks, const f32x4 lo, const f32x4 hi) {
                bf16x8 t[3];
                split8<3>(lo, hi, t);
                bf16x8* const to = a.ttf + (vslot * kTriFrags + trt_index(w, ks)) * 3 * 64;
#pragma unroll
                for (int k = 0; k < 3; ++k) (to + k * 64)[lane] = t[k];
            };
            const f32x4 none = splat4(0.f);
            if (w == 0) {
                put_tt(0, tcol[0], tcol[1]);
                put_tt(1, tcol[2], tcol[3]);
            } else if (w == 1) {
                put_tt(0, none, tcol[0]);
                put_tt(1, tcol[1], tcol[2]);
            } else if (w == 2) {
                put_tt(1, tcol[0], tcol[1]);
            } else {
                put_tt(1, none, tcol[0]);
            }
        }
        lds_barrier();
        for (int f = w; f < kTriFrags; f += 4) {
            const int mt = tri_row(f), nt = 2 * tri_step(f), id = mt * (mt + 1) / 2 + nt;
            const f32x4 x0 = ttile[id * kTile + 17 * q + j], x1 = nt + 1 <= mt ? ttile[(id + 1) * kTile + 17 * q + j] : splat4(0.f);
            bf16x8 t[3];
            split8<3>(x0, x1, t);
            bf16x8* const to = a.tf + (vslot * kTriFrags + f) * 3 * 64;
#pragma unroll
            for (int k = 0; k < 3; ++k) (to + k * 64)[lane] = t[k];
        }
    }
}

// four values in N terms: the half of a fragment that one row tile is
template <int N>
__device__ __forceinline__ void split4(const f32x4 v, u32x2 (&t)[N]) {
    f32x2 x[2] = {{v[0], v[1]}, {v[2], v[3]}};
    unsigned w[N][2];
    split_pairs<N, 2>(x, w);
#pragma unroll
    for (int n = 0; n < N; ++n) t[n] = (u32x2){w[n][0], w[n][1]};
}
// row tile mt of a [64 or DK x 16 NC] operand that the workgroup shares: fragments [k step][term][column tile][lane]
template <int N, int NC>
__device__ __forceinline__ void share_tile(bf16x8* buf, int mt, int nc, int lane, const f32x4 v) {
    u32x2 t[N];
    split4<N>(v, t);
#pragma unroll
    for (int n = 0; n < N; ++n)
        ((u32x2*)(buf + (((mt >> 1) * N + n) * NC + nc) * 64 + lane))[mt & 1] = t[n];
}
template <int N, int NC>
__device__ __forceinline__ void shared_frag(const bf16x8* buf, int ks, int nc, int lane, bf16x8 (&b)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) b[n] = buf[((ks * N + n) * NC + nc) * 64 + lane];
}
// loads stay above this (they are issued here, and not where their values are first needed)
__device__ __forceinline__ void issue_loads() { asm volatile("" ::: "memory"); }
// workgroups go round the eight XCDs: neighbours in `logical` order (the column groups of one head, which read the same
// fragments) stay on one of them.  The grid is padded to a multiple of eight.
__device__ __forceinline__ unsigned xcd_order(unsigned block, unsigned grid) { return (block & 7) * (grid >> 3) + (block >> 3); }

constexpr int kColumnTiles = 2;    // of a four-wave chain

// Where a wave of a chain finds its left-hand fragments: uniform bases plus the lane
template <typename In, int DK>
struct ChainAddress {
    static constexpr int NI = In::kTerms, kSlot = DK / 8 * NI * 64;    // fragments of a (slot, key head), times 64 lanes
    const bf16x8* zeros;
    size_t kslot, vslot;
    int hk, hv, w;
    unsigned lane;
    __device__ __forceinline__ ChainAddress(const DeltaArgs& a, const Span& sp, int h, int head, int wave, int l)
        : zeros(a.zeros), kslot((size_t)sp.slot * a.hk + h), vslot((size_t)sp.slot * a.hv + head), hk(a.hk), hv(a.hv), w(wave), lane(l) {}
    // row tile w of K or Q with the k steps in the order first, first + 1, ..: to[i] is step (first + i) % (DK / 32)
    __device__ __forceinline__ void rows(int first, const bf16x8* from, int c, bf16x8 (&to)[DK / 32][NI]) const {
        from += (kslot + (size_t)c * hk) * kSlot + w * (DK / 32) * NI * 64;
#pragma unroll
        for (int i = 0; i < DK / 32; ++i)
#pragma unroll
            for (int t = 0; t < NI; ++t) to[i][t] = (from + (((first + i) & (DK / 32 - 1)) * NI + t) * 64)[lane];
    }
    // the wave's dk tiles of K^T or Q^T
    __device__ __forceinline__ void columns(const bf16x8* from, int c, bf16x8 (&to)[DK / 64][2][NI]) const {
        from += (kslot + (size_t)c * hk) * kSlot + w * (DK / 64) * 2 * NI * 64;
#pragma unroll
        for (int i = 0; i < DK / 64; ++i)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int t = 0; t < NI; ++t) to[i][ks][t] = (from + ((2 * i + ks) * NI + t) * 64)[lane];
    }
    // Row tile w of T or P; row tiles 0 and 1 have one k step.  A kernel that does not tell the waves apart takes the other one from
    // the zeros.
    template <int N>
    __device__ __forceinline__ void triangle(const bf16x8* from, int c, bf16x8 (&to)[1][N]) const {
        from += ((vslot + (size_t)c * hv) * kTriFrags + w) * N * 64;
#pragma unroll
        for (int t = 0; t < N; ++t) to[0][t] = (from + t * 64)[lane];
    }
    template <int N>
    __device__ __forceinline__ void triangle(const bf16x8* from, int c, bf16x8 (&to)[2][N]) const {
        from += ((vslot + (size_t)c * hv) * kTriFrags + tri_index(w, 0)) * N * 64;
        const bf16x8* const second = w < 2 ? zeros : from + N * 64;
#pragma unroll
        for (int t = 0; t < N; ++t) {
            to[0][t] = (from + t * 64)[lane];
            to[1][t] = (second + t * 64)[lane];
        }
    }
    // row tile w of T^T or P^T; row tiles 2 and 3 have only the second k step
    __device__ __forceinline__ void transposed(const bf16x8* from, int c, bf16x8 (&to)[1][3]) const {
        from += ((vslot + (size_t)c * hv) * kTriFrags + trt_index(w, 1)) * 3 * 64;
#pragma unroll
        for (int t = 0; t < 3; ++t) to[0][t] = (from + t * 64)[lane];
    }
    __device__ __forceinline__ void transposed(const bf16x8* from, int c, bf16x8 (&to)[2][3]) const {
        from += ((vslot + (size_t)c * hv) * kTriFrags + trt_index(w, 1)) * 3 * 64;
        const bf16x8* const first = w < 2 ? from - 3 * 64 : zeros;
#pragma unroll
        for (int t = 0; t < 3; ++t) {
            to[0][t] = (first + t * 64)[lane];
            to[1][t] = (from + t * 64)[lane];
        }
    }
};
// Row tile w of K or Q straight from the inputs: in bf16 the rows are the fragments; dead rows stand for the last live one (what
// comes of them meets zeros).  The preparation then writes 32 KB less a key head and chunk, and the loads are of 64 bytes a row.
// 64 sequences of 1000 tokens, 4 heads of 128: preparation 88 -> 60 us, chain 169 -> 176 (here and below with P and U in two terms;
// it is 66 and 188 with three).  Chains that also write their states lose more than that (32 x 1000 tokens: 97 -> 84, 230 ->
// 247, reverse 235 -> 243), and so do the eight-wave ones (16,384 tokens: 116 -> 91, 473 -> 555): they take the fragments.
template <typename In, int DK>
struct InputRows {
    typedef typename In::raw raw;
    const raw* from;
    long stride;
    unsigned col;
    int row, len;
    __device__ __forceinline__ InputRows(const void* rows, long t, long head_at, const Span& sp, int w, int lane)
        : from((const raw*)rows + sp.begin * t + head_at), stride(t), col(8 * (lane >> 4)), row(16 * w + (lane & 15)), len(sp.len) {}
    __device__ __forceinline__ void load(int c, bf16x8 (&to)[DK / 32][1]) const {
        const raw* const p = from + c * kDeltaChunk * stride;
        const unsigned off = min(row, len - c * kDeltaChunk - 1) * (unsigned)stride + col;
#pragma unroll
        for (int i = 0; i < DK / 32; ++i) to[i][0] = *(const bf16x8*)(p + 32 * i + off);
    }
};
// Dk of row 4 q + r of tile t of the states as the chains hold them: state_row(t) + 8 q + r
__device__ __forceinline__ constexpr int state_row(int tile) { return 32 * (tile >> 1) + 4 * (tile & 1); }

// Element offsets of a lane's four rows of a chunk in a [tokens, ..] tensor (the host has checked that they fit 32 bits); rows
// from n on stand for row n - 1.
struct RowOffsets {
    unsigned at[4], stride;
    int row, col, full;
    __device__ __forceinline__ RowOffsets(long stride_, int row_, int col_) : stride((unsigned)stride_), row(row_), col(col_), full(1) {
#pragma unroll
        for (int r = 0; r < 4; ++r) at[r] = (row + r) * stride + col;
    }
    __device__ __forceinline__ void clamp(int n) {
        if (n < kDeltaChunk || !full) {
            full = n >= kDeltaChunk;
#pragma unroll
            for (int r = 0; r < 4; ++r) at[r] = min(row + r, n - 1) * stride + col;
        }
    }
};

// NC neighbouring D tiles to a [.., dv] fp32 matrix; at[r]: the lane's offset in row r of its four
template <int NC>
__device__ __forceinline__ void store_tile(float* to, const unsigned (&at)[4], const f32x4 (&x)[NC]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float row[NC];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) row[nc] = x[nc][r];
        Columns<InF32, NC>::store(to + at[r], row);
    }
}

// A wave's rows of a state [DK, dv]: MW row tiles; zero where there is no state.  The loads are not
// conditional (they read some zeros then): behind a skipped load the compiler waits for everything that is in flight.
template <int MW, int NC>
__device__ __forceinline__ void load_state(const float* state, const void* zeros, size_t at, int dv, f32x4 (&S)[MW][NC]) {
    typedef Columns<InF32, NC> Cols;
    const float* const from = state ? state + at : (const float*)zeros;
    const size_t stride = state ? dv : 0;
#pragma unroll
    for (int i = 0; i < MW; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const Cols x = Cols::load(from + (4 * i + r) * stride);
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) S[i][nc][r] = state ? x.get(nc) : 0.f;
        }
}

// ------------------------------------------------------------------------------------------------
// The chain: a workgroup per (sequence, value head, 32 columns of the state).  Each of its four waves owns a quarter of
// the ROWS of everything: token tile w of R, U and O, the dk tiles of S from w DK/64 on.  The other waves' rows of a right-hand
// operand (S, R, U) come through LDS as bf16 terms, three barriers a chunk; every left-hand fragment is read by
// one wave only, straight into registers, and the next chunk's are loaded into the registers the present chunk is done with.
// What bounds it: the way through a chunk.  Two workgroups fit a CU (registers), so a SIMD has two waves to hide behind each other
// 120 products of 16 cycles, some 400 VALU instructions (the splits), 85 LDS accesses and 45 loads a wave and chunk: the matrix
// pipe is busy for 30 % of the time, and a wave waits for a quarter of it.  fp16 and fp32 at width 128 have one workgroup a CU
// (280 and more registers).  64 sequences of 1000 tokens, 4 heads of 128, bf16: 188 us, 134 TFLOP/s of the recurrence's own 6 Dk Dv a
// token (176 us with P and U in two terms, when bf16 results were 1.1e-4 of their norm from a float32 evaluation's, not 3.5e-5).
// Two column tiles share every left-hand fragment; with one it was 244 us instead of 169, and keeping the states 370 instead of
// 232 (32 x 1000, 8 heads; both with fragments of K and Q, and two terms).
// ------------------------------------------------------------------------------------------------
template <typename In, int DK, bool KEEP>
__global__ __launch_bounds__(256, In::kTerms == 1 ? 2 : 1) void delta_forward_kernel(const DeltaArgs a) {
    constexpr int NC = kColumnTiles, NI = In::kTerms, KS = DK / 32, MW = DK / 64;
    typedef typename In::raw raw;
    __shared__ bf16x8 sbuf[KS * 3 * NC * 64], xbuf[2 * 3 * NC * 64], ubuf[2 * 3 * NC * 64], cbuf[2 * 3 * NC * 64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = lane & 15, q = lane >> 4;
    const int groups = a.dv_width / (16 * NC);
    const unsigned item = xcd_order(blockIdx.x, gridDim.x);
    if (item >= (unsigned)a.nseq * a.hv * groups) return;
    const int hv = item / groups % a.hv, s = item / groups / a.hv, h = hv / a.group;
    const int col = NC * (16 * (item % groups) + j);    // column tile nc has columns 16 NC g + NC j + nc: a lane's are neighbours
    const Span sp = span_of(a, s);
    const int chunks = (sp.len + kDeltaChunk - 1) / kDeltaChunk;
    const size_t st = (((size_t)s * a.hv + hv) * DK + state_row(MW * w) + 8 * q) * a.dv_width + col;

    f32x4 S[MW][NC];
    load_state<MW, NC>(a.s0, a.zeros, st, a.dv_width, S);

    bf16x8 kf[KS][NI], qf[KS][NI], kt[MW][2][NI], tf[2][3], pf[2][3];
    f32x4 beta, eb, ec;
    float whole;
    Columns<In, NC> v[4];
    const int row = 16 * w + 4 * q;                 // this lane's tokens: row .. row + 3
    const ChainAddress<In, DK> at(a, sp, h, hv, w, lane);
    // (No load of the loop is conditional: the compiler counts what is in flight, and a skipped load would make it wait for
    // everything.  Rows behind the sequence's end read its last row: their k and beta are zero.)
    RowOffsets vrow(a.v_t, row, col), orow(a.o_t, row, col);
    auto load_tokens = [&](int c) {
        const float* sc = a.sc + (at.vslot + (size_t)c * a.hv) * 256;
        beta = *(const f32x4*)(sc + row);
        eb = *(const f32x4*)(sc + 64 + row);
        ec = *(const f32x4*)(sc + 128 + row);
        whole = (sc + 64)[63];
        vrow.clamp(sp.len - c * kDeltaChunk);
        const raw* p = (const raw*)a.v + (sp.begin + c * kDeltaChunk) * a.v_t + hv * a.v_h;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = Columns<In, NC>::load(p + vrow.at[r]);
    };
    const InputRows<In, DK> krows(a.k, a.k_t, h * a.k_h, sp, w, lane), qrows(a.q, a.q_t, h * a.q_h, sp, w, lane);
    auto load_k = [&](int c) {
        if constexpr (NI == 1 && !KEEP) krows.load(c, kf);
        else at.rows(0, a.kf, c, kf);
    };
    auto load_q = [&](int c) {
        if constexpr (NI == 1 && !KEEP) qrows.load(c, qf);
        else at.rows(0, a.qf, c, qf);
    };
    auto load_kt = [&](int c) { at.columns(a.ktf, c, kt); };
    auto load_t = [&](int c) { at.template triangle<3>(a.tf, c, tf); };
    auto load_p = [&](int c) { at.template triangle<3>(a.pf, c, pf); };
    unsigned tile_at[4], state_at[4];               // D tile of a [.., dv] matrix, of a state: this lane's four elements
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        tile_at[r] = (4 * q + r) * a.dv_width + col;
        state_at[r] = (8 * q + r) * a.dv_width + col;
    }
    auto share_state = [&](int c) {
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
        }
        if constexpr (KEEP) {
            float* to = a.states + ((at.vslot + (size_t)c * a.hv) * DK + state_row(MW * w)) * a.dv_width;
#pragma unroll
            for (int i = 0; i < MW; ++i) store_tile<NC>(to + (size_t)4 * i * a.dv_width, state_at, S[i]);
        }
    };
    if (chunks > 0) {
        load_k(0);
        load_tokens(0);
        load_q(0);
        load_t(0);
        load_p(0);
        load_kt(0);
        share_state(0);
    }
    lds_barrier();
    for (int c = 0; c < chunks; ++c) {
        const int next = min(c + 1, chunks - 1), n = sp.len - c * kDeltaChunk;
        f32x4 R[NC], O[NC], U[NC];
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) R[nc] = O[nc] = splat4(0.f);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) {
                bf16x8 b[3];
                shared_frag<3, NC>(sbuf, ks, nc, lane, b);
                R[nc] = mm(kf[ks], b, R[nc]);
                O[nc] = mm(qf[ks], b, O[nc]);
            }
        const f32x4 after = ec, step = beta, head = eb;
        const float hold = whole;
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
#pragma unroll
            for (int r = 0; r < 4; ++r) R[nc][r] = v[r].get(nc) - eb[r] * R[nc][r];
            share_tile<3, NC>(xbuf, w, nc, lane, R[nc]);
        }
        load_k(next);
        load_tokens(next);
        issue_loads();
        lds_barrier();
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            bf16x8 x[2][3];
            shared_frag<3, NC>(xbuf, 0, nc, lane, x[0]);
            shared_frag<3, NC>(xbuf, 1, nc, lane, x[1]);
            f32x4 u0 = splat4(0.f), u1 = splat4(0.f);
            u0 = mm(tf[0], x[0], u0);
            u1 = mm(tf[1], x[1], u1);
            U[nc] = u0 + u1;
        }
        if constexpr (KEEP) store_tile<NC>(a.e + ((at.vslot + (size_t)c * a.hv) * kDeltaChunk + 16 * w) * a.dv_width, tile_at, U);
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
#pragma unroll
            for (int r = 0; r < 4; ++r) U[nc][r] *= step[r];
            share_tile<3, NC>(ubuf, w, nc, lane, U[nc]);
#pragma unroll
            for (int r = 0; r < 4; ++r) U[nc][r] *= after[r];
            share_tile<3, NC>(cbuf, w, nc, lane, U[nc]);
        }
        load_q(next);
        load_t(next);
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
                bf16x8 x[3];
                shared_frag<3, NC>(cbuf, ks, nc, lane, x);
#pragma unroll
                for (int i = 0; i < MW; ++i) S[i][nc] = mm(kt[i][ks], x, S[i][nc]);
            }
        load_kt(next);
        issue_loads();
        if (c + 1 < chunks) share_state(next);
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
            bf16x8 x[2][3];
            shared_frag<3, NC>(ubuf, 0, nc, lane, x[0]);
            shared_frag<3, NC>(ubuf, 1, nc, lane, x[1]);
            f32x4 p0 = splat4(0.f);
#pragma unroll
            for (int r = 0; r < 4; ++r) O[nc][r] *= head[r];
            p0 = mm(pf[0], x[0], p0);
            O[nc] = mm(pf[1], x[1], O[nc]) + p0;
        }
        load_p(next);
        issue_loads();
        raw* const to = (raw*)a.o + (sp.begin + c * kDeltaChunk) * a.o_t + hv * a.o_h;
        auto put = [&](int r) {
            float x[NC];
#pragma unroll
            for (int nc = 0; nc < NC; ++nc) x[nc] = a.scale * O[nc][r];
            Columns<In, NC>::store(to + orow.at[r], x);
        };
        if (n >= kDeltaChunk) {
#pragma unroll
            for (int r = 0; r < 4; ++r) put(r);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (row + r < n) put(r);
        }
        lds_barrier();
    }
    if (a.s1) {
        float* const to = a.s1 + (((size_t)s * a.hv + hv) * DK + state_row(MW * w)) * a.dv_width;
#pragma unroll
        for (int i = 0; i < MW; ++i) store_tile<NC>(to + (size_t)4 * i * a.dv_width, state_at, S[i]);
    }
}

// ------------------------------------------------------------------------------------------------
// The same for few long chains: 16 columns of the state, and eight waves.  A wave alone on its SIMD issues an instruction
// every 5 to 9 cycles, and the chain is as long as what its waves have to issue; so waves 0 .. 3 do only what the next chunk
// waits for (R, E and S), and waves 4 .. 7, one on each SIMD beside them, the output and every store: from S, E and U as they
// pass by in LDS, a phase later.  Waves whose row tile of T and P has one k step run code of their own (without: 510 us, not 473).
// What bounds it: a chunk is 4,100 cycles, of which the matrix pipe works for 870 and the waves wait for half.  The CU's loads, 89 KB
// of fragments and rows a chunk, take 1,400 at the 64 bytes a cycle of its L1, and three barriers keep them and the products from
// each other.  16,384 tokens, 32 heads of 128, bf16: 498 us, 103 TFLOP/s (473 with P, U and S in two terms for the output); the
// four-wave kernel on 256 chains takes 1.4 times as long (one sequence of 2048 tokens, 32 heads: 118 us a call against 84).
// fp32 at width 128 spills 8 registers, 10 where it keeps the states.
// ------------------------------------------------------------------------------------------------
// Fetches a chunk's fragments into the XCD's L2 before the workgroups of its head need them.  They all come by at the same time,
// and what misses there comes at a lower rate.  Each of the head's waves takes another part: one load, a lane a line of 128 bytes.
// The value is handed to `settle` a chunk later.  8191 tokens in two sequences, 16 heads of 128: forward chain 215 us without, 194
// with, reverse chain 226 and 182; 16,384 tokens x 32 heads: no difference.
struct Piece {
    const bf16x8* at;
    int kib;
};
template <int N>
__device__ __forceinline__ unsigned fetch(const Piece (&piece)[N], int part, int lane) {
    int line = part * 64 + lane;
    const char* from = (const char*)piece[N - 1].at + 1024 * (piece[N - 1].kib - 1);     // (parts behind the end: a line again)
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (line >= 0 && line < 8 * piece[i].kib) from = (const char*)piece[i].at + 128 * line;
        line -= 8 * piece[i].kib;
    }
    return *(const unsigned*)from;
}
__device__ __forceinline__ void settle(unsigned x) { asm volatile("" ::"v"(x)); }
constexpr int kFetchAhead = 3;

// loads and matrix products by turns: a load is issued while the pipe works on the product before it
template <int N>
__device__ __forceinline__ void between_products() {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
    }
}

// Before a loop whose loads are a turn ahead: nothing is in flight here, so that the compiler's counts inside it are those of the
// loop alone (it waits for what any path into the loop might have left).
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }

template <typename In, int DK, bool KEEP>
__global__ __launch_bounds__(512) void delta_forward_long_kernel(const DeltaArgs a) {
    constexpr int NI = In::kTerms, KS = DK / 32, MW = DK / 64;
    constexpr bool OWN = MW == 2;        // a wave's rows of S are a whole k step: it takes that one from its registers
    typedef typename In::raw raw;
    __shared__ bf16x8 sbuf[KS * 3 * 64], xbuf[2 * 3 * 64], ubuf[2 * 3 * 64], cbuf[2 * 3 * 64];
    __shared__ f32x4 ebuf[4 * 64], sfull[KEEP ? 4 * MW * 64 : 1];
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
        load_state<MW, 1>(a.s0, a.zeros, (((size_t)s * a.hv + hv) * DK + state_row(MW * w) + 8 * q) * a.dv_width + col, a.dv_width, S);
        struct Operands {        // of one chunk; the next one's are loaded into a second set meanwhile
            bf16x8 kf[KS][NI], kt[MW][2][NI], tf[TWO ? 2 : 1][3];
            f32x4 eb, weight;     // weight: beta e^c
            float whole;
            Columns<In, 1> v[4];
        } first, second;
        bf16x8 own[3];
        RowOffsets vrow(a.v_t, row, col);
        auto load_k = [&](int c, Operands& to) { at.rows(OWN ? w : 0, a.kf, c, to.kf); };
        auto load_tokens = [&](int c, Operands& to) {
            const float* sc = a.sc + (at.vslot + (size_t)c * a.hv) * 256;
            to.eb = *(const f32x4*)(sc + 64 + row);
            vrow.clamp(sp.len - c * kDeltaChunk);
            const raw* p = (const raw*)a.v + (sp.begin + c * kDeltaChunk) * a.v_t + hv * a.v_h;
#pragma unroll
            for (int r = 0; r < 4; ++r) to.v[r] = Columns<In, 1>::load(p + vrow.at[r]);
        };
        auto load_scales = [&](int c, Operands& to) {
            const float* sc = a.sc + (at.vslot + (size_t)c * a.hv) * 256;
            to.weight = *(const f32x4*)(sc + 192 + row);
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
            if constexpr (KEEP) {
#pragma unroll
                for (int i = 0; i < MW; ++i) sfull[(MW * w + i) * 64 + lane] = S[i][0];
            }
        };
        auto step = [&](int c, Operands& now, Operands& then) {
            const int next = min(c + 1, chunks - 1);
            f32x4 sum[2] = {splat4(0.f), splat4(0.f)}, R;
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
            load_tokens(next, then);
            between_products<KS * 3>();
#pragma unroll
            for (int r = 0; r < 4; ++r) R[r] = now.v[r].get(0) - now.eb[r] * (sum[0][r] + sum[1][r]);
            share_tile<3, 1>(xbuf, w, 0, lane, R);
            issue_loads();
            lds_barrier();
            bf16x8 x[2][3];
            shared_frag<3, 1>(xbuf, 0, 0, lane, x[0]);
            if constexpr (TWO) shared_frag<3, 1>(xbuf, 1, 0, lane, x[1]);
            f32x4 e0 = splat4(0.f), e1 = splat4(0.f);
            e0 = mm(now.tf[0], x[0], e0);
            if constexpr (TWO) e1 = mm(now.tf[1], x[1], e1);
            at.template triangle<3>(a.tf, next, then.tf);
            load_scales(next, then);
            between_products<TWO ? 12 : 6>();
            f32x4 E = e0 + e1;
            ebuf[w * 64 + lane] = E;
#pragma unroll
            for (int r = 0; r < 4; ++r) E[r] *= now.weight[r];
            share_tile<3, 1>(cbuf, w, 0, lane, E);
            issue_loads();
            lds_barrier();
            shared_frag<3, 1>(cbuf, 0, 0, lane, x[0]);
            shared_frag<3, 1>(cbuf, 1, 0, lane, x[1]);
#pragma unroll
            for (int i = 0; i < MW; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[i][0][r] *= now.whole;
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
            load_k(0, first);
            load_tokens(0, first);
            load_scales(0, first);
            at.template triangle<3>(a.tf, 0, first.tf);
            at.columns(a.ktf, 0, first.kt);
            share_state();
        }
        lds_barrier();
        if (chunks & 1) {
            step(0, first, second);
            first = second;
        }
        loads_done();
        for (int c = chunks & 1; c < chunks; c += 2) {
            step(c, first, second);
            step(c + 1, second, first);
        }
        if (a.s1) {
            float* const to = a.s1 + (((size_t)s * a.hv + hv) * DK + state_row(MW * w)) * a.dv_width;
#pragma unroll
            for (int i = 0; i < MW; ++i) store_tile<1>(to + (size_t)4 * i * a.dv_width, state_at, S[i]);
        }
    };
    auto output = [&](auto two_) {
        constexpr bool TWO = decltype(two_)::value;
        // The output transposed, S^T Q^T and U^T P^T (the operands change places, the fragments are the same): a lane then has
        // four neighbouring columns of one token, one store of a chunk
        bf16x8 qf[KS][NI], pf[TWO ? 2 : 1][3];
        f32x4 beta, O = splat4(0.f);
        float eb = 0.f;
        const int token = 16 * w + j;
        const unsigned o_at = token * (unsigned)a.o_t + col - j + 4 * q;
        auto load_scales = [&](int c) {
            const float* sc = a.sc + (at.vslot + (size_t)c * a.hv) * 256;
            beta = *(const f32x4*)(sc + row);
            eb = (sc + 64)[token];
        };
        // o of chunk c: O + P U, and its store
        auto finish = [&](int c) {
            bf16x8 x[2][3];
            shared_frag<3, 1>(ubuf, 0, 0, lane, x[0]);
            if constexpr (TWO) {
                shared_frag<3, 1>(ubuf, 1, 0, lane, x[1]);
                f32x4 p0 = splat4(0.f);
                p0 = mm(x[0], pf[0], p0);
                O = mm(x[1], pf[1], O) + p0;
            } else {
                O = mm(x[0], pf[0], O);
            }
            raw* const to = (raw*)a.o + (sp.begin + c * kDeltaChunk) * a.o_t + hv * a.o_h;
            const float y[4] = {a.scale * O[0], a.scale * O[1], a.scale * O[2], a.scale * O[3]};
            if (token < sp.len - c * kDeltaChunk) Columns<In, 4>::store(to + o_at, y);
        };
        const int part = 4 * (item % groups) + w;
        auto fetch_chunk = [&](int c) {
            const bf16x8* const tri = a.tf + (at.vslot + (size_t)c * a.hv) * kTriFrags * 3 * 64;
            const bf16x8* const pri = a.pf + (at.vslot + (size_t)c * a.hv) * kTriFrags * 3 * 64;
            const size_t k0 = (at.kslot + (size_t)c * a.hk) * at.kSlot;
            const Piece piece[5] = {{a.kf + k0, DK / 8 * NI}, {tri, kTriFrags * 3}, {a.ktf + k0, DK / 8 * NI}, {a.qf + k0, DK / 8 * NI}, {pri, kTriFrags * 3}};
            return fetch(piece, part, lane);
        };
        unsigned fetched = 0;
        if (chunks > 0) {
            at.rows(0, a.qf, 0, qf);
            load_scales(0);
            settle(fetch_chunk(min(1, chunks - 1)));
            settle(fetch_chunk(min(2, chunks - 1)));
        }
        lds_barrier();
        for (int c = 0; c < chunks; ++c) {
            const int next = min(c + 1, chunks - 1);
            settle(fetched);
            fetched = fetch_chunk(min(c + kFetchAhead, chunks - 1));
            if (c > 0) finish(c - 1);
            at.template triangle<3>(a.pf, c, pf);
            issue_loads();
            lds_barrier();
            f32x4 sum[2] = {splat4(0.f), splat4(0.f)};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                bf16x8 b[3];
#pragma unroll
                for (int t = 0; t < 3; ++t) b[t] = sbuf[(ks * 3 + t) * 64 + lane];
                sum[ks & 1] = mm(b, qf[ks], sum[ks & 1]);
            }
            if constexpr (KEEP) {
                float* const to = a.states + ((at.vslot + (size_t)c * a.hv) * DK + state_row(MW * w)) * a.dv_width;
#pragma unroll
                for (int i = 0; i < MW; ++i) {
                    const f32x4 x[1] = {sfull[(MW * w + i) * 64 + lane]};
                    store_tile<1>(to + (size_t)4 * i * a.dv_width, state_at, x);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) O[r] = eb * (sum[0][r] + sum[1][r]);
            const f32x4 step = beta;
            at.rows(0, a.qf, next, qf);
            load_scales(next);
            issue_loads();
            lds_barrier();
            f32x4 U = ebuf[w * 64 + lane];
            if constexpr (KEEP) {
                const f32x4 x[1] = {U};
                store_tile<1>(a.e + ((at.vslot + (size_t)c * a.hv) * kDeltaChunk + 16 * w) * a.dv_width, tile_at, x);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) U[r] *= step[r];
            share_tile<3, 1>(ubuf, w, 0, lane, U);
            lds_barrier();
        }
        if (chunks > 0) finish(chunks - 1);
    };
    if (wave < 4) w < 2 ? chain(Is<false>()) : chain(Is<true>());
    else w < 2 ? output(Is<false>()) : output(Is<true>());
}

// Which of the two: the eight-wave kernel while each of its workgroups has a CU to itself.  One sequence of 2048 tokens, bf16, widths
// 128, forward / forward + keep / backward calls in us, four waves against eight: 256 chains 118, 147, 211 against 84, 119, 176;
// 288 chains 124, 154, 236 against 120, 177, 242; 512 chains 134, 205, 324 against 164, 271, 348 (fp16, fp32 and width_k 64 cross
// over at the same place, with the forward call of bf16 at 288 chains alone on the other side).  Chains are counted, not their
// lengths: many short sequences beside a few long ones go to the kernel for many.
constexpr int kComputeUnits = 256;
inline bool chains_are_few(const DeltaArgs& a) { return (long)a.nseq * a.hv * (a.dv_width / 16) <= kComputeUnits; }
inline unsigned chain_grid(const DeltaArgs& a, int columns) {      // columns of the state a workgroup takes
    return (unsigned)(((long)a.nseq * a.hv * (a.dv_width / columns) + 7) / 8 * 8);
}

}  // namespace helen
