// Layer norm, forward and backward.
#pragma once
#include "jq_memory.h"

namespace jq {

// Rows are walked in vectors of 16 bytes by groups of G lanes: lane i of a group has
// vectors i, i + G, ... (NV of them), so a row stays in registers between its
// statistics and its result and is read once. Up to a wave's 64 lanes a group is
// part of a wave and a block has several; G = 256 and 1024 are a block each. Bound by
// the rows' traffic: 262,144 rows of 256 in bfloat16 forward (268 MB) 49 us, 5.5 TB/s,
// backward (403 MB) 80 us, 5.0 TB/s, where a plain copy reaches 6.0. A wave per row that
// reads it three times and a column's sums apart took 722 us in all, 136 now; sums by
// shuffles through LDS, and rows turned to float32 as they come, 62 and 93. Widths that
// leave lanes idle, or have a block a row, are slower: 134 MB of bfloat16 rows forward 44 us
// at widths of 256 and 1,000, 71 at 300, 66 at 1,500; backward 104 and 172 at 256 and 8,000
// (256 registers: one wave a SIMD), 423 at 12,000 (87 registers spilled).
constexpr int norm_block(int group) { return group > 256 ? group : 256; }

template <class T, int G, int NV>
struct NormRow {
    static constexpr int N = Vec<T>::N, BLOCK = norm_block(G), GROUPS = BLOCK / G;
    float x[NV * N];

    __device__ __forceinline__ static int lane() { return threadIdx.x % G; }

    // f(first element, index in x, count) for this lane's vectors
    template <class F>
    __device__ __forceinline__ static void each(int width, F &&f)
    {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int c = (lane() + u * G) * N;
            if (c < width) f(c, u * N, min(N, width - c));
        }
    }

    // this lane's vectors of a row as they lie in memory, and x from them: a row on its
    // way is not waited for before it is taken
    typedef typename Vec<T>::type Raw;
    __device__ __forceinline__ static void fetch(const T *row, int width, Raw (&raw)[NV])
    {
        typedef Raw At __attribute__((aligned(sizeof(T))));   // any element alignment
#pragma unroll
        for (int u = 0; u < NV; ++u) raw[u] = Raw{};
        each(width, [&](int c, int i, int n) {
            const T *p = row + c;
            if (n == N) raw[i / N] = *reinterpret_cast<const At *>(p);
            else
#pragma unroll
                for (int e = 0; e < N; ++e) {   // without a branch for each element: their loads go out together
                    const T y = p[e < n ? e : n - 1];
                    raw[i / N][e] = e < n ? y : T(0.f);
                }
        });
    }
    __device__ __forceinline__ void take(const Raw (&raw)[NV])
    {
#pragma unroll
        for (int i = 0; i < NV * N; ++i) x[i] = (float)raw[i / N][i % N];
    }

    // x = this lane's columns of p (weights), or `other` without p and past the row's end
    template <class W>
    __device__ __forceinline__ static void columns(const W *p, int width, float other, float (&x)[NV * N])
    {
#pragma unroll
        for (int i = 0; i < NV * N; ++i) x[i] = other;
        if (p) each(width, [&](int c, int i, int n) { load_vec(p + c, n, x + i, other); });
    }

    // n elements (all of a vector but at the row's end) at any element alignment
    template <class U>
    __device__ __forceinline__ static void load_vec(const U *p, int n, float *x, float other)
    {
        constexpr int M = Vec<U>::N < N ? Vec<U>::N : N;
        typedef U V __attribute__((ext_vector_type(M), aligned(sizeof(U))));
        if (n == N) {
#pragma unroll
            for (int i = 0; i < N; i += M) {
                const V v = *reinterpret_cast<const V *>(p + i);
#pragma unroll
                for (int e = 0; e < M; ++e) x[i + e] = (float)v[e];
            }
        } else {   // without a branch for each element: their loads go out together
            U v[N];
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = p[e < n ? e : n - 1];
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = e < n ? (float)v[e] : other;
        }
    }
    __device__ __forceinline__ static void store_vec(T *p, int n, const float *x)
    {
        if (n == N) {
            typedef typename Vec<T>::type V __attribute__((aligned(sizeof(T))));
            V v;
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = from_float<T>(x[e]);
            *reinterpret_cast<V *>(p) = v;
        } else
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (e < n) p[e] = from_float<T>(x[e]);
    }

    // the group's sums of a and b, in every lane; red: 2 * BLOCK / 64 floats of LDS
    __device__ __forceinline__ static void sum(float &a, float &b, float *red)
    {
        a = group_total<(G < 64 ? G : 64)>(a);
        b = group_total<(G < 64 ? G : 64)>(b);
        if constexpr (G > 64) {
            constexpr int W = G / 64;
            __syncthreads();
            if (threadIdx.x % 64 == 0) {
                red[threadIdx.x / 64] = a;
                red[W + threadIdx.x / 64] = b;
            }
            __syncthreads();
            a = b = 0.f;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                a += red[i];
                b += red[W + i];
            }
        }
    }
};

struct NormArgs {
    const void *x, *w, *bias, *d;   // d: gradient of the result (backward)
    void *o;                        // result, or gradient of x
    int64_t x_stride, o_stride, d_stride, rows;
    int width;
    float eps, *mean, *rstd, *part;
};

// out = (x - mean) rstd w + bias. The variance is that of the differences, so an
// offset far from 0 costs no digits. Groups go over rows a grid's stride apart, with
// weight and bias in registers and the next row on its way.
template <class T, class W, int G, int NV>
__global__ __launch_bounds__(norm_block(G)) void k_norm_forward(NormArgs a)
{
    using R = NormRow<T, G, NV>;
    constexpr int N = R::N;
    __shared__ float red[2 * R::BLOCK / 64];
    const int64_t step = (int64_t)gridDim.x * R::GROUPS;
    int64_t r = (int64_t)blockIdx.x * R::GROUPS + threadIdx.x / G;
    if (r >= a.rows) return;   // groups of more than a wave are blocks: none waits for it
    R row;
    typename R::Raw next[NV];
    R::fetch(static_cast<const T *>(a.x) + r * a.x_stride, a.width, next);
    const W *w = static_cast<const W *>(a.w), *bias = static_cast<const W *>(a.bias);
    float weight[NV * N], offset[NV * N];
    R::columns(w, a.width, 1.f, weight);
    R::columns(bias, a.width, 0.f, offset);
    for (;;) {
        const int64_t then = r + step;
        row.take(next);
        if (then < a.rows) R::fetch(static_cast<const T *>(a.x) + then * a.x_stride, a.width, next);
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < NV * N; ++i) s += row.x[i];
        R::sum(s, q, red);
        const float mean = s / a.width;
        q = 0.f;
        R::each(a.width, [&](int, int i, int n) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                row.x[i + e] -= mean;
                if (e < n) q = fmaf(row.x[i + e], row.x[i + e], q);
            }
        });
        R::sum(q, s, red);
        const float rstd = 1.f / sqrtf(q / a.width + a.eps);
        T *o = static_cast<T *>(a.o) + r * a.o_stride;
        R::each(a.width, [&](int c, int i, int n) {
            float y[N];
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = row.x[i + e] * rstd * weight[i + e] + offset[i + e];
            R::store_vec(o + c, n, y);
        });
        if (R::lane() == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
        if (then >= a.rows) break;
        r = then;
    }
}

// dx = rstd (g - mean(g) - xhat mean(g xhat)), g = d w, and this block's part of
// dw = sum d xhat and db = sum d: its groups go over rows a grid's stride apart with
// the sums of their columns in registers, and join them in order at the end.
// part[block][0][c]: dw, [1]: db.
template <class T, class W, int G, int NV>
__global__ __launch_bounds__(norm_block(G)) void k_norm_backward(NormArgs a)
{
    using R = NormRow<T, G, NV>;
    constexpr int N = R::N;
    __shared__ float red[2 * R::BLOCK / 64];
    __shared__ float join[R::GROUPS > 1 ? R::BLOCK * N : 1];
    const W *w = static_cast<const W *>(a.w);
    float dw[NV * N] = {}, db[NV * N] = {}, weight[NV * N];
    R::columns(w, a.width, 1.f, weight);
    constexpr int JOIN = R::GROUPS > 8 ? 8 : 1;   // groups joined at once: all would take the registers of waves that the rows need
    constexpr bool AHEAD = NV == 1;   // the next row is on its way: wider rows have no registers left for it
    const int64_t step = (int64_t)gridDim.x * R::GROUPS;
    R row, d;
    typename R::Raw next[NV], next_d[NV];
    float next_mean, next_rstd;
    const auto fetch = [&](int64_t r) {
        R::fetch(static_cast<const T *>(a.x) + r * a.x_stride, a.width, next);
        R::fetch(static_cast<const T *>(a.d) + r * a.d_stride, a.width, next_d);
        next_mean = a.mean[r];
        next_rstd = a.rstd[r];
    };
    const int64_t first = (int64_t)blockIdx.x * R::GROUPS + threadIdx.x / G;
    if (AHEAD && first < a.rows) fetch(first);
    for (int64_t r = first; r < a.rows; r += step) {
        if (!AHEAD) fetch(r);
        row.take(next);
        d.take(next_d);
        const float mean = next_mean, rstd = next_rstd;
        if (AHEAD && r + step < a.rows) fetch(r + step);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV * N; ++i) {   // past the row's end d is 0
            row.x[i] = (row.x[i] - mean) * rstd;
            db[i] += d.x[i];
            dw[i] = fmaf(d.x[i], row.x[i], dw[i]);
            d.x[i] *= weight[i];
            s1 += d.x[i];
            s2 = fmaf(d.x[i], row.x[i], s2);
        }
        if (a.o) {
            R::sum(s1, s2, red);
            s1 /= a.width;
            s2 /= a.width;
            T *o = static_cast<T *>(a.o) + r * a.o_stride;
            R::each(a.width, [&](int c, int i, int n) {
                float y[N];
#pragma unroll
                for (int e = 0; e < N; ++e) y[e] = rstd * (d.x[i + e] - s1 - row.x[i + e] * s2);
                R::store_vec(o + c, n, y);
            });
        }
    }
    if (!a.part) return;
    float *part = a.part + (int64_t)blockIdx.x * 2 * a.width;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            float y[N];
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = which ? db[u * N + e] : dw[u * N + e];
            if constexpr (R::GROUPS > 1) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < N; ++e) join[threadIdx.x * N + e] = y[e];
                __syncthreads();
                if (threadIdx.x >= G) continue;
#pragma unroll JOIN
                for (int g = 1; g < R::GROUPS; ++g)
#pragma unroll
                    for (int e = 0; e < N; ++e) y[e] += join[(g * G + threadIdx.x) * N + e];
            }
            const int c = (R::lane() + u * G) * N;
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (c + e < a.width) part[which * a.width + c + e] = y[e];
        }
}

// Rows wider than a block's registers: read again for each step of the same sums.
template <class T, class W>
__global__ __launch_bounds__(1024) void k_norm_forward_wide(NormArgs a)
{
    using R = NormRow<T, 1024, 1>;
    __shared__ float red[32];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
        const W *w = static_cast<const W *>(a.w), *bias = static_cast<const W *>(a.bias);
        float s = 0.f, q = 0.f;
        for (int c = threadIdx.x; c < a.width; c += 1024) s += (float)x[c];
        R::sum(s, q, red);
        const float mean = s / a.width;
        q = 0.f;
        for (int c = threadIdx.x; c < a.width; c += 1024) q = fmaf((float)x[c] - mean, (float)x[c] - mean, q);
        R::sum(q, s, red);
        const float rstd = 1.f / sqrtf(q / a.width + a.eps);
        T *o = static_cast<T *>(a.o) + r * a.o_stride;
        for (int c = threadIdx.x; c < a.width; c += 1024)
            o[c] = from_float<T>(((float)x[c] - mean) * rstd * (w ? (float)w[c] : 1.f) + (bias ? (float)bias[c] : 0.f));
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

template <class T, class W>
__global__ __launch_bounds__(1024) void k_norm_dx_wide(NormArgs a)
{
    using R = NormRow<T, 1024, 1>;
    __shared__ float red[32];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.x_stride, *d = static_cast<const T *>(a.d) + r * a.d_stride;
        const W *w = static_cast<const W *>(a.w);
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (int c = threadIdx.x; c < a.width; c += 1024) {
            const float g = (float)d[c] * (w ? (float)w[c] : 1.f);
            s1 += g;
            s2 = fmaf(g, ((float)x[c] - mean) * rstd, s2);
        }
        R::sum(s1, s2, red);
        s1 /= a.width;
        s2 /= a.width;
        T *o = static_cast<T *>(a.o) + r * a.o_stride;
        for (int c = threadIdx.x; c < a.width; c += 1024)
            o[c] = from_float<T>(rstd * ((float)d[c] * (w ? (float)w[c] : 1.f) - s1 - ((float)x[c] - mean) * rstd * s2));
    }
}

// part as in k_norm_backward: blockIdx.y's range of rows, 256 columns a block.
template <class T>
__global__ __launch_bounds__(256) void k_norm_dw_wide(NormArgs a)
{
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.width) return;
    const T *x = static_cast<const T *>(a.x) + c, *d = static_cast<const T *>(a.d) + c;
    float sw = 0.f, sb = 0.f;
    for (int64_t r = a.rows * blockIdx.y / gridDim.y; r < a.rows * (blockIdx.y + 1) / gridDim.y; ++r) {
        const float g = (float)d[r * a.d_stride];
        sw = fmaf(g, ((float)x[r * a.x_stride] - a.mean[r]) * a.rstd[r], sw);
        sb += g;
    }
    a.part[(int64_t)(2 * blockIdx.y) * a.width + c] = sw;
    a.part[(int64_t)(2 * blockIdx.y + 1) * a.width + c] = sb;
}

// The blocks' sums joined: 16 columns of dw (blockIdx.y 0) or db a block, each by 16
// threads that take every 16th part and are joined in order.
template <class W>
__global__ __launch_bounds__(256) void k_norm_join(const float *__restrict__ part, int parts, int width,
                                                   W *__restrict__ dw, W *__restrict__ db)
{
    W *out = blockIdx.y ? db : dw;
    if (!out) return;
    __shared__ float sum[16][16];
    const int i = threadIdx.x % 16, j = threadIdx.x / 16, c = blockIdx.x * 16 + i;
    float s = 0.f;
    if (c < width)
#pragma unroll 8
        for (int y = j; y < parts; y += 16) s += part[(2 * (int64_t)y + blockIdx.y) * width + c];
    sum[j][i] = s;
    __syncthreads();
    if (j || c >= width) return;
    for (int y = 1; y < 16; ++y) s += sum[y][i];
    out[c] = from_float<W>(s);
}

}  // namespace jq
