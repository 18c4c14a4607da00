// Rotary positions with several axes.
#pragma once
#include "jq_memory.h"

namespace jq {

struct RotaryArgs {
    jq_rows x, o;
    int64_t n1;
    int heads, dim, pairs, axes;
    const void *positions;
    int64_t p0, p1;
    int ends[JQ_ROTARY_MAX_AXES];
    const float *frequencies;
    bool positions64, interleaved, inverse;
};

// cos and sin of position * frequency: the product and its whole turns in 64 bits,
// so that the angle of a far ply keeps float32's precision.
__device__ __forceinline__ void turn_of(int64_t position, float frequency, float &c, float &s)
{
    const double half = (double)position * (double)frequency * 0.31830988618379067154;   // half turns
    sincospif((float)(half - 2.0 * rint(0.5 * half)), &s, &c);
}

// One block per token: a pair's angle is computed once for all heads.
template <class T>
__global__ __launch_bounds__(64) void k_rotary(RotaryArgs a)
{
    const int64_t b = blockIdx.x / a.n1, t = blockIdx.x % a.n1;
    const int64_t at = b * a.p0 + t * a.p1;
    for (int p = threadIdx.x; p < a.pairs; p += 64) {
        int axis = 0;
        while (p >= a.ends[axis]) ++axis;
        const int64_t pos = a.positions64 ? static_cast<const int64_t *>(a.positions)[at + axis]
                                          : static_cast<const int32_t *>(a.positions)[at + axis];
        float c, s;
        turn_of(pos, a.frequencies[p], c, s);
        if (a.inverse) s = -s;
        const int i = a.interleaved ? 2 * p : p, j = a.interleaved ? 2 * p + 1 : a.pairs + p;
        for (int h = 0; h < a.heads; ++h) {
            const T *x = row_at<const T>(a.x, b, t, h);
            T *o = row_at<T>(a.o, b, t, h);
            const float u = (float)x[i], v = (float)x[j];
            o[i] = from_float<T>(u * c - v * s);
            o[j] = from_float<T>(v * c + u * s);
        }
    }
    for (int h = 0; h < a.heads; ++h)
        for (int i = 2 * a.pairs + threadIdx.x; i < a.dim; i += 64)
            row_at<T>(a.o, b, t, h)[i] = row_at<const T>(a.x, b, t, h)[i];
}

}  // namespace jq
