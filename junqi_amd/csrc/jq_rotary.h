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

// A block takes `tokens` tokens at a time: first the cosines and sines of their
// pairs, once for all heads, into LDS; then the heads' elements, N at a time at any
// element alignment. Work item (token, head, i): i below `turns` turns N elements
// (two parts of N where pairs are apart), the others copy. Bound by the rows'
// traffic: 262,144 tokens of 8 heads of 64 in bfloat16 (537 MB) in 94 us, 5.7 TB/s;
// with two heads a token the angles count, 528,771 tokens of 2 heads of 56 in float32
// (478 MB) in 118 us, 4.0 TB/s. A block per token, an angle per pair and thread: 237
// and 301 us. Pairs apart that are no whole vectors go one at a time: 8 heads of 12 or 20
// pairs in bfloat16 (537 MB) in 290 us, of 16 or 24 in 97.
constexpr int ROTARY_TABLE = 2048;   // pairs of a block's tokens at most (unless one token has more)
template <class T, int N, bool INTERLEAVED>
__global__ __launch_bounds__(256) void k_rotary(RotaryArgs a, int64_t all, int tokens)
{
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    extern __shared__ __align__(8) char lds[];   // offsets of each token's rows; cos of (token, pair), then sin
    int64_t *in_at = reinterpret_cast<int64_t *>(lds), *out_at = in_at + tokens;
    float *cs = reinterpret_cast<float *>(out_at + tokens), *sn = cs + tokens * a.pairs;
    const int turns = INTERLEAVED ? 2 * a.pairs / N : a.pairs / N, rest = a.dim - 2 * a.pairs;
    const bool whole = rest % N == 0;   // the rest is copied in vectors too, or by element
    const int items = turns + (whole ? rest / N : rest);
    // this thread's first item, and the way to its next, 256 on
    const unsigned per = items, heads = a.heads, x0 = threadIdx.x;
    const unsigned i0 = x0 % per, h0 = x0 / per % heads, k0 = x0 / per / heads;
    const unsigned di = 256 % per, dh = 256 / per % heads, dk = 256 / per / heads;
    for (int64_t t0 = (int64_t)blockIdx.x * tokens; t0 < all; t0 += (int64_t)gridDim.x * tokens) {
        const int n = (int)min((int64_t)tokens, all - t0);
        __syncthreads();
        for (int token = threadIdx.x; token < n; token += 256) {
            const int64_t b = (t0 + token) / a.n1, t = (t0 + token) % a.n1;
            in_at[token] = b * a.x.batch + t * a.x.ply;
            out_at[token] = b * a.o.batch + t * a.o.ply;
        }
        for (int x = threadIdx.x; x < n * a.pairs; x += 256) {
            const int token = (unsigned)x / (unsigned)a.pairs, p = x - token * a.pairs;
            const int64_t b = a.n1 == all ? 0 : (t0 + token) / a.n1, at = b * a.p0 + (t0 + token - b * a.n1) * a.p1;
            int axis = 0;
            while (p >= a.ends[axis]) ++axis;
            const int64_t pos = a.positions64 ? static_cast<const int64_t *>(a.positions)[at + axis]
                                              : static_cast<const int32_t *>(a.positions)[at + axis];
            float c, s;
            turn_of(pos, a.frequencies[p], c, s);
            cs[x] = c;
            sn[x] = a.inverse ? -s : s;
        }
        __syncthreads();
        for (unsigned at = i0, head = h0, token = k0; token < (unsigned)n;) {
            const int i = at;
            const T *in = static_cast<const T *>(a.x.data) + in_at[token] + head * a.x.head;
            T *out = static_cast<T *>(a.o.data) + out_at[token] + head * a.o.head;
            const float *c0 = cs + token * a.pairs, *s0 = sn + token * a.pairs;
            at += di;
            const bool over = at >= per;
            at -= over ? per : 0;
            head += dh + over;
            const bool past = head >= heads;
            head -= past ? heads : 0;
            token += dk + past;
            if (i >= turns) {
                const int c = 2 * a.pairs + (i - turns) * (whole ? N : 1);
                if (whole) *reinterpret_cast<V *>(out + c) = *reinterpret_cast<const V *>(in + c);
                else out[c] = in[c];
            } else if constexpr (INTERLEAVED) {
                const V u = *reinterpret_cast<const V *>(in + i * N);
                V y;
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const int p = (i * N + e) / 2;
                    const float c = c0[p], s = s0[p], u0 = (float)u[e], u1 = (float)u[e + 1];
                    y[e] = from_float<T>(u0 * c - u1 * s);
                    y[e + 1] = from_float<T>(u1 * c + u0 * s);
                }
                *reinterpret_cast<V *>(out + i * N) = y;
            } else {
                const V u = *reinterpret_cast<const V *>(in + i * N), v = *reinterpret_cast<const V *>(in + a.pairs + i * N);
                V y, z;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const int p = i * N + e;
                    const float c = c0[p], s = s0[p], u0 = (float)u[e], u1 = (float)v[e];
                    y[e] = from_float<T>(u0 * c - u1 * s);
                    z[e] = from_float<T>(u1 * c + u0 * s);
                }
                *reinterpret_cast<V *>(out + i * N) = y;
                *reinterpret_cast<V *>(out + a.pairs + i * N) = z;
            }
        }
    }
}

}  // namespace jq
