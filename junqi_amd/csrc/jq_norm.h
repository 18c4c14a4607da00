// Layer norm, forward and backward.
#pragma once
#include "jq_memory.h"

namespace jq {

// One wave per row: the mean, then the squares of what is off it, then the result.
template <class T, class W>
__global__ __launch_bounds__(64) void k_norm_forward(const T *__restrict__ x, int64_t x_stride, int width,
                                                     const W *__restrict__ w, const W *__restrict__ bias, float eps,
                                                     T *__restrict__ o, int64_t o_stride, float *mean_out,
                                                     float *rstd_out)
{
    const int64_t r = blockIdx.x;
    x += r * x_stride;
    o += r * o_stride;
    float sum = 0.f, sq = 0.f;
    for (int c = threadIdx.x; c < width; c += 64) sum += (float)x[c];
    const float mean = wave_total(sum) / width;
    for (int c = threadIdx.x; c < width; c += 64) sq += ((float)x[c] - mean) * ((float)x[c] - mean);
    const float rstd = rsqrtf(wave_total(sq) / width + eps);
    for (int c = threadIdx.x; c < width; c += 64)
        o[c] = from_float<T>(((float)x[c] - mean) * rstd * (w ? (float)w[c] : 1.f) + (bias ? (float)bias[c] : 0.f));
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[r] = mean;
        if (rstd_out) rstd_out[r] = rstd;
    }
}

// dx = rstd (g - mean(g) - xhat mean(g xhat)), g = d_out w. One wave per row.
template <class T, class W>
__global__ __launch_bounds__(64) void k_norm_dx(const T *__restrict__ x, int64_t x_stride, int width,
                                                const W *__restrict__ w, const float *__restrict__ mean,
                                                const float *__restrict__ rstd, const T *__restrict__ d,
                                                int64_t d_stride, T *__restrict__ dx, int64_t dx_stride)
{
    const int64_t r = blockIdx.x;
    x += r * x_stride;
    d += r * d_stride;
    dx += r * dx_stride;
    const float m = mean[r], rs = rstd[r];
    float g1 = 0.f, g2 = 0.f;
    for (int c = threadIdx.x; c < width; c += 64) {
        const float g = (float)d[c] * (w ? (float)w[c] : 1.f);
        g1 += g;
        g2 += g * (((float)x[c] - m) * rs);
    }
    g1 = wave_total(g1) / width;
    g2 = wave_total(g2) / width;
    for (int c = threadIdx.x; c < width; c += 64) {
        const float g = (float)d[c] * (w ? (float)w[c] : 1.f);
        dx[c] = from_float<T>(rs * (g - g1 - ((float)x[c] - m) * rs * g2));
    }
}

constexpr int NORM_PARTS = 512;   // row ranges that are summed apart

// Sums of one range of rows for 64 columns: part[y][0][c] of d_out xhat, [1] of d_out.
template <class T>
__global__ __launch_bounds__(64) void k_norm_dw(const T *__restrict__ x, int64_t x_stride, int64_t rows, int width,
                                                const float *__restrict__ mean, const float *__restrict__ rstd,
                                                const T *__restrict__ d, int64_t d_stride, float *__restrict__ part)
{
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (c >= width) return;
    float sw = 0.f, sb = 0.f;
    for (int64_t r = rows * blockIdx.y / gridDim.y; r < rows * (blockIdx.y + 1) / gridDim.y; ++r) {
        const float g = (float)d[r * d_stride + c];
        sw += g * (((float)x[r * x_stride + c] - mean[r]) * rstd[r]);
        sb += g;
    }
    part[(int64_t)(2 * blockIdx.y) * width + c] = sw;
    part[(int64_t)(2 * blockIdx.y + 1) * width + c] = sb;
}

// The ranges' sums joined in order.
template <class W>
__global__ __launch_bounds__(64) void k_norm_join(const float *__restrict__ part, int parts, int width,
                                                  W *__restrict__ dw, W *__restrict__ db)
{
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (c >= width) return;
    float sw = 0.f, sb = 0.f;
    for (int y = 0; y < parts; ++y) {
        sw += part[(int64_t)(2 * y) * width + c];
        sb += part[(int64_t)(2 * y + 1) * width + c];
    }
    if (dw) dw[c] = from_float<W>(sw);
    if (db) db[c] = from_float<W>(sb);
}

}  // namespace jq
