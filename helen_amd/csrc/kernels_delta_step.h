// kernels_delta_step.h -- the gated delta rule for single tokens over a pool of states
//
//     u = beta (v - e^g S^T k),   S <- e^g S + k u^T,   o = scale S^T q = scale (e^g S^T q + (q . k) u)
// The right-hand form of o needs only the OLD state, so S^T k and S^T q are one pass over a state that stays in registers
// between its load and its store: a state is read once and written once, and that is the whole cost.
// Bound by bandwidth: 252 streams, 32 heads of 128 x 128: 1.06 GB in 211 us, 5.0 TB/s.  One stream is a launch and its host side:
// 10.2 us a call, where a fill of one line costs 3.8.
// A workgroup takes 64 columns of one row's head; rows of the call that name the same slot are successive tokens of one stream and
// are taken in order by the workgroup of the first of them.  To find them each workgroup reads all of `slots`: nothing beside its
// state up to some thousand rows, but at 4,000 rows of 64 x 64 states as many bytes (from the caches), and growing with their square.
#pragma once
#include "kernels_delta.h"

namespace helen {

struct DeltaStepArgs {
    const void *q, *k, *v;
    const float *g, *beta;
    const int* slots;           // [rows] or null: row i is slot i
    float* state;               // [pool, Hv, Dk, Dv]
    void* o;
    long q_t, q_h, k_t, k_h, v_t, v_h, o_t, o_h, g_t, g_h, b_t, b_h, s_t;
    int rows, pool, hk, hv, group, dv_width;
    float scale;
};

template <typename In, int DK>
__global__ __launch_bounds__(256) void delta_step_kernel(const DeltaStepArgs a) {
    constexpr int NR = DK / 16;
    typedef typename In::raw raw;
    __shared__ __attribute__((aligned(16))) float red[4][16][12];
    __shared__ float ks[DK], qs[DK];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int c4 = tid & 15, rg = tid >> 4;             // columns 4 c4 .., rows rg + 16 i
    const int blocks = a.dv_width >> 6;
    const int hv = blockIdx.x / blocks % a.hv, row = blockIdx.x / blocks / a.hv, h = hv / a.group;
    const int col = 64 * (blockIdx.x % blocks) + 4 * c4;
    const int slot = a.slots ? a.slots[row] : row;
    if (slot < 0 || slot >= a.pool) {
        // -1 is a padded row: its output is zero; any other number outside the pool is an error that must show
        if (rg == 0) {
            raw* to = (raw*)a.o + row * a.o_t + hv * a.o_h + col;
            for (int r = 0; r < 4; ++r) to[r] = In::from_f32(slot == -1 ? 0.f : __builtin_nanf(""));
        }
        return;
    }
    float* const st = a.state + slot * a.s_t + (long)hv * DK * a.dv_width + (long)rg * a.dv_width + col;
    f32x4 S[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) S[i] = *(const f32x4*)(st + (long)(16 * i) * a.dv_width);
    bool later = false;
    if (a.slots) {
        bool earlier = false;
        for (int b = tid; b < a.rows; b += 256) {
            const bool same = a.slots[b] == slot;
            earlier |= same && b < row;
            later |= same && b > row;
        }
        if (__syncthreads_or(earlier)) return;
        later = __syncthreads_or(later);
    }
    int at = row;
    while (true) {
        __syncthreads();
        for (int d = tid; d < DK; d += 256) {
            ks[d] = In::to_f32(((const raw*)a.k)[at * a.k_t + h * a.k_h + d]);
            qs[d] = In::to_f32(((const raw*)a.q)[at * a.q_t + h * a.q_h + d]);
        }
        const f32x4 v = load4<In>((const raw*)a.v + at * a.v_t + hv * a.v_h + col);
        const float alpha = expf(a.g[at * a.g_t + hv * a.g_h]), beta = a.beta[at * a.b_t + hv * a.b_h];
        __syncthreads();
        f32x4 pk = splat4(0.f), pq = splat4(0.f);
        float qk = 0.f;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const float kv = ks[rg + 16 * i], qv = qs[rg + 16 * i];
            qk += kv * qv;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pk[r] += kv * S[i][r];
                pq[r] += qv * S[i][r];
            }
        }
#pragma unroll
        for (int m = 16; m < 64; m <<= 1) {
            qk += __shfl_xor(qk, m);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pk[r] += __shfl_xor(pk[r], m);
                pq[r] += __shfl_xor(pq[r], m);
            }
        }
        if (lane < 16) {
            *(f32x4*)&red[w][c4][0] = pk;
            *(f32x4*)&red[w][c4][4] = pq;
            red[w][c4][8] = qk;
        }
        __syncthreads();
        pk = pq = splat4(0.f);
        qk = 0.f;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            pk += *(const f32x4*)&red[m][c4][0];
            pq += *(const f32x4*)&red[m][c4][4];
            qk += red[m][c4][8];
        }
        f32x4 u;
#pragma unroll
        for (int r = 0; r < 4; ++r) u[r] = beta * (v[r] - alpha * pk[r]);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const float kv = ks[rg + 16 * i];
#pragma unroll
            for (int r = 0; r < 4; ++r) S[i][r] = alpha * S[i][r] + kv * u[r];
        }
        if (rg == 0) {
            raw* to = (raw*)a.o + at * a.o_t + hv * a.o_h + col;
#pragma unroll
            for (int r = 0; r < 4; ++r) to[r] = In::from_f32(a.scale * (alpha * pq[r] + qk * u[r]));
        }
        if (!later) break;
        do ++at;
        while (at < a.rows && a.slots[at] != slot);
        if (at >= a.rows) break;
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) *(f32x4*)(st + (long)(16 * i) * a.dv_width) = S[i];
}

}  // namespace helen
