// kernels_norm.h -- layer norm over the last dimension and its gradients
//
//     y = (x - mean) rstd w + b,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//     dx = rstd (e - mean(e) - h mean(e h)),  e = dy w,  h = (x - mean) rstd;   dw = sum over rows of dy h,  db = sum of dy
// A row is read once into registers and both moments are taken from there (the second one around the mean: no cancellation).
// L lanes share a row: 16 for narrow rows (four rows a wave), 64, or a whole workgroup for wide ones.  Rows of any alignment
// are read in 16-byte pieces (gfx950 takes unaligned wide loads), only a row's last piece element by element.
// The weight's gradient is a sum over all rows: a workgroup keeps its columns' sums in registers over all the rows it takes,
// writes them once, and a second small kernel adds the workgroups' sums in their order -- no atomics, the same bits each time.
#pragma once
#include "kernels_delta.h"

namespace helen {

struct NormArgs {
    const void *x, *w, *b, *dy;
    void *y, *dx, *dw, *db;
    float *mean, *rstd, *partial, *sums;
    long rows, x_t, y_t, dy_t, dx_t;
    int width, groups;
    float eps;
};

template <typename In>
struct Pieces {
    typedef typename In::raw raw;
    static constexpr int V = 16 / (int)sizeof(raw);
    typedef raw vec __attribute__((ext_vector_type(16 / sizeof(raw))));
    typedef vec vec_any __attribute__((aligned(sizeof(raw))));
    // as they lie in memory, zero behind the row's end (`left` elements)
    static __device__ __forceinline__ vec read(const raw* p, int left) {
        vec t;
        if (left >= V) {
            t = *(const vec_any*)p;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) t[i] = i < left ? p[i] : raw(0);
        }
        return t;
    }
    static __device__ __forceinline__ void widen(const vec t, float (&to)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) to[i] = In::to_f32(t[i]);
    }
    static __device__ __forceinline__ void load(const raw* p, int left, float (&to)[V]) { widen(read(p, left), to); }
    static __device__ __forceinline__ void store(raw* p, int left, const float (&from)[V]) {
        if (left >= V) {
            Columns<In, V>::store(p, from);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < left) p[i] = In::from_f32(from[i]);
        }
    }
};
// V elements of a weight (its own type) from column `at`
template <typename W, int V>
__device__ __forceinline__ void load_weight(const void* w, int at, int left, float (&to)[V], float otherwise) {
    const typename W::raw* p = (const typename W::raw*)w + at;
    if (w && left >= V) {
        constexpr int PV = Pieces<W>::V < V ? Pieces<W>::V : V;
        typedef typename W::raw vec __attribute__((ext_vector_type(PV), aligned(sizeof(typename W::raw))));
#pragma unroll
        for (int c = 0; c < V / PV; ++c) {
            const vec t = *(const vec*)(p + c * PV);
#pragma unroll
            for (int i = 0; i < PV; ++i) to[c * PV + i] = W::to_f32(t[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) to[i] = w && i < left ? W::to_f32(p[i]) : otherwise;
    }
}

// sum over the L lanes of a row; L = 256: over the workgroup (`red` is free again after the call)
template <int L, int N>
__device__ __forceinline__ void row_sum(float (&x)[N], float (*red)[N]) {
    static_assert(L >= 16, "a row of 16 lanes is summed by rotations");
#pragma unroll
    for (int n = 0; n < N; ++n) {
        x[n] = dpp_add<0x121>(dpp_add<0x122>(dpp_add<0x124>(dpp_add<0x128>(x[n]))));
        if constexpr (L > 16) {
            x[n] += __shfl_xor(x[n], 16);
            x[n] += __shfl_xor(x[n], 32);
        }
    }
    if constexpr (L == 256) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) red[w][n] = x[n];
        lds_barrier();
#pragma unroll
        for (int n = 0; n < N; ++n) x[n] = (red[0][n] + red[1][n]) + (red[2][n] + red[3][n]);
        lds_barrier();
    }
}

// Bandwidth is what bounds both directions.  A workgroup takes rows `groups` apart and has the next one's loads in flight while it
// works on a row; the weights of its columns stay in registers.
template <typename In, typename W, int L, int NV>
__global__ __launch_bounds__(256) void norm_forward_kernel(const NormArgs a) {
    typedef typename In::raw raw;
    typedef Pieces<In> P;
    constexpr int V = P::V;
    __shared__ float red[4][1];
    const int t = threadIdx.x % L;
    const long step = (long)a.groups * (256 / L);
    long row = blockIdx.x * (long)(256 / L) + threadIdx.x / L;
    if (row >= a.rows) return;          // (L = 256: the whole workgroup)
    typename P::vec next[NV];
    float w[NV][V], b[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (t + i * L) * V;
        next[i] = P::read((const raw*)a.x + row * a.x_t + at, a.width - at);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (t + i * L) * V;
        load_weight<W, V>(a.w, at, a.width - at, w[i], 1.f);
        load_weight<W, V>(a.b, at, a.width - at, b[i], 0.f);
    }
    while (true) {
        float v[NV][V], s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) P::widen(next[i], v[i]);
        const long after = row + step;
        if (after < a.rows) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int at = (t + i * L) * V;
                next[i] = P::read((const raw*)a.x + after * a.x_t + at, a.width - at);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) s[0] += v[i][e];
        row_sum<L, 1>(s, red);
        const float mean = s[0] / a.width;
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[i][e] -= mean;
                s[0] += (t + i * L) * V + e < a.width ? v[i][e] * v[i][e] : 0.f;
            }
        row_sum<L, 1>(s, red);
        const float rstd = 1.f / sqrtf(s[0] / a.width + a.eps);
        if (t == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = (t + i * L) * V, left = a.width - at;
            if (left <= 0) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) v[i][e] = v[i][e] * rstd * w[i][e] + b[i][e];
            P::store((raw*)a.y + row * a.y_t + at, left, v[i]);
        }
        if (after >= a.rows) break;
        row = after;
    }
}

template <typename In, typename W, int L, int NV>
__global__ __launch_bounds__(256) void norm_backward_kernel(const NormArgs a) {
    typedef typename In::raw raw;
    typedef Pieces<In> P;
    constexpr int V = P::V, R = 256 / L;
    __shared__ float red[4][2];
    __shared__ float cols[R > 1 ? 256 * V : 1];
    const int t = threadIdx.x % L;
    const long step = (long)a.groups * R;
    float w[NV][V], dw[NV][V], db[NV][V];
    typename P::vec nx[NV], ny[NV];
    float nmean = 0.f, nrstd = 0.f;
    long row = blockIdx.x * (long)R + threadIdx.x / L;
    auto read = [&](long r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = (t + i * L) * V;
            nx[i] = P::read((const raw*)a.x + r * a.x_t + at, a.width - at);
            ny[i] = P::read((const raw*)a.dy + r * a.dy_t + at, a.width - at);
        }
        nmean = a.mean[r];
        nrstd = a.rstd[r];
    };
    if (row < a.rows) read(row);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (t + i * L) * V;
        load_weight<W, V>(a.w, at, a.width - at, w[i], 1.f);
#pragma unroll
        for (int e = 0; e < V; ++e) dw[i][e] = db[i][e] = 0.f;
    }
    for (; row < a.rows; row += step) {
        float h[NV][V], g[NV][V], s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            P::widen(nx[i], h[i]);
            P::widen(ny[i], g[i]);
        }
        const float mean = nmean, rstd = nrstd;
        if (row + step < a.rows) read(row + step);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[i][e] = (h[i][e] - mean) * rstd;
                dw[i][e] += g[i][e] * h[i][e];
                db[i][e] += g[i][e];
                g[i][e] *= w[i][e];
                s[0] += g[i][e];
                s[1] += g[i][e] * h[i][e];
            }
        row_sum<L, 2>(s, red);
        const float c0 = s[0] / a.width, c1 = s[1] / a.width;
        raw* dx = (raw*)a.dx + row * a.dx_t;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = (t + i * L) * V, left = a.width - at;
            if (left <= 0) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) h[i][e] = rstd * (g[i][e] - c0 - h[i][e] * c1);
            P::store(dx + at, left, h[i]);
        }
    }
    // the workgroup's sums of its columns: [group][dw | db][width]
    float* const out = a.partial + (long)blockIdx.x * 2 * a.width;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float x[V];
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = k ? db[i][e] : dw[i][e];
            if constexpr (R > 1) {
                lds_barrier();
#pragma unroll
                for (int e = 0; e < V; ++e) cols[e * 256 + threadIdx.x] = x[e];
                lds_barrier();
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x[e] = 0.f;
#pragma unroll
                    for (int r = 0; r < R; ++r) x[e] += cols[e * 256 + r * L + t];
                }
            }
            if ((int)threadIdx.x < L) {
                const int at = (t + i * L) * V;
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (at + e < a.width) out[(long)k * a.width + at + e] = x[e];
            }
        }
}

// rows wider than the registers hold: the row is read again for each of its sums (it stays in the caches)
template <typename In, typename W>
__global__ __launch_bounds__(256) void norm_forward_wide_kernel(const NormArgs a) {
    typedef typename In::raw raw;
    constexpr int V = Pieces<In>::V;
    __shared__ float red[4][1];
    const long row = blockIdx.x;
    const raw* x = (const raw*)a.x + row * a.x_t;
    float v[V], s[1] = {0.f};
    for (int at = threadIdx.x * V; at < a.width; at += 256 * V) {
        Pieces<In>::load(x + at, a.width - at, v);
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] += v[e];
    }
    row_sum<256, 1>(s, red);
    const float mean = s[0] / a.width;
    s[0] = 0.f;
    for (int at = threadIdx.x * V; at < a.width; at += 256 * V) {
        Pieces<In>::load(x + at, a.width - at, v);
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] += at + e < a.width ? (v[e] - mean) * (v[e] - mean) : 0.f;
    }
    row_sum<256, 1>(s, red);
    const float rstd = 1.f / sqrtf(s[0] / a.width + a.eps);
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
    raw* y = (raw*)a.y + row * a.y_t;
    for (int at = threadIdx.x * V; at < a.width; at += 256 * V) {
        const int left = a.width - at;
        float w[V], b[V];
        Pieces<In>::load(x + at, left, v);
        load_weight<W, V>(a.w, at, left, w, 1.f);
        load_weight<W, V>(a.b, at, left, b, 0.f);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (v[e] - mean) * rstd * w[e] + b[e];
        Pieces<In>::store(y + at, left, v);
    }
}
// Their gradients in two passes: a row's two sums, then strips of 256 pieces of columns over rows `groups` apart, with the strip's
// sums of the weight's gradient in registers.  (x and dy are read twice.  With a row to a workgroup, its sums of columns in memory,
// 4096 x 16384 float32 took 523 us; this takes 274.)
template <typename In, typename W>
__global__ __launch_bounds__(256) void norm_backward_sums_kernel(const NormArgs a) {
    typedef typename In::raw raw;
    constexpr int V = Pieces<In>::V;
    __shared__ float red[4][2];
    const long row = blockIdx.x;
    const raw* x = (const raw*)a.x + row * a.x_t;
    const raw* dy = (const raw*)a.dy + row * a.dy_t;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float h[V], g[V], w[V], s[2] = {0.f, 0.f};
    for (int at = threadIdx.x * V; at < a.width; at += 256 * V) {
        Pieces<In>::load(x + at, a.width - at, h);
        Pieces<In>::load(dy + at, a.width - at, g);
        load_weight<W, V>(a.w, at, a.width - at, w, 1.f);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            s[0] += g[e] * w[e];
            s[1] += g[e] * w[e] * ((h[e] - mean) * rstd);
        }
    }
    row_sum<256, 2>(s, red);
    if (threadIdx.x < 2) a.sums[2 * row + threadIdx.x] = (threadIdx.x ? s[1] : s[0]) / a.width;
}
template <typename In, typename W>
__global__ __launch_bounds__(256) void norm_backward_strip_kernel(const NormArgs a) {
    typedef typename In::raw raw;
    typedef Pieces<In> P;
    constexpr int V = P::V;
    const int at = (blockIdx.x * 256 + threadIdx.x) * V, left = a.width - at;
    if (left <= 0) return;
    float w[V], dw[V], db[V];
    load_weight<W, V>(a.w, at, left, w, 1.f);
#pragma unroll
    for (int e = 0; e < V; ++e) dw[e] = db[e] = 0.f;
    long row = blockIdx.y;
    typename P::vec nx, ny;
    if (row < a.rows) {
        nx = P::read((const raw*)a.x + row * a.x_t + at, left);
        ny = P::read((const raw*)a.dy + row * a.dy_t + at, left);
    }
    for (; row < a.rows; row += a.groups) {
        float h[V], g[V];
        P::widen(nx, h);
        P::widen(ny, g);
        const long next = row + a.groups;
        if (next < a.rows) {
            nx = P::read((const raw*)a.x + next * a.x_t + at, left);
            ny = P::read((const raw*)a.dy + next * a.dy_t + at, left);
        }
        const float mean = a.mean[row], rstd = a.rstd[row], c0 = a.sums[2 * row], c1 = a.sums[2 * row + 1];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            h[e] = (h[e] - mean) * rstd;
            dw[e] += g[e] * h[e];
            db[e] += g[e];
            h[e] = rstd * (g[e] * w[e] - c0 - h[e] * c1);
        }
        P::store((raw*)a.dx + row * a.dx_t + at, left, h);
    }
    float* const out = a.partial + (long)blockIdx.y * 2 * a.width + at;
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (e < left) {
            out[e] = dw[e];
            out[(long)a.width + e] = db[e];
        }
}

// the workgroups' sums, added in a fixed order: 32 columns and 32 runs of groups a workgroup, which goes on with the columns
// gridDim.x strips further where the grid is smaller than the row
template <typename W>
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const NormArgs a) {
    __shared__ float part[32][33];
    const int c = threadIdx.x & 31, run = threadIdx.x >> 5;
    for (long first = blockIdx.x * 32l; first < 2l * a.width; first += gridDim.x * 32l) {
        const long at = first + c;
        float x = 0.f;
        if (at < 2l * a.width) {
            const float* p = a.partial + at;
            for (int g = run; g < a.groups; g += 32 * 16) {
                float y[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = g + 32 * i < a.groups ? p[(long)(g + 32 * i) * 2 * a.width] : 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) x += y[i];
            }
        }
        part[run][c] = x;
        lds_barrier();
        if (run == 0 && at < 2l * a.width) {
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 32; ++r) sum += part[r][c];
            void* to = at < a.width ? a.dw : a.db;
            if (to) ((typename W::raw*)to)[at < a.width ? at : at - a.width] = W::from_f32(sum);
        }
        lds_barrier();
    }
}

}  // namespace helen
