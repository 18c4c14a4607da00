// The causal convolution over a few plies, forward and backward, and its step of one ply.
#pragma once
#include "jq_memory.h"
#include "jq_scan.h"

namespace jq {

// out_t = bias + sum over j of weight[j] x_{t - taps + 1 + j}, then x sigmoid(x) where
// `silu`; inputs before a game's start are not there. A thread has V channels of 16 bytes
// together and walks a run of plies with the last inputs in registers, so a row is read
// once but for the taps - 1 before a run.
constexpr int CONV_TAPS = 8;   // largest taps
constexpr int CONV_AHEAD = 4;  // plies whose rows are on their way

// Channels of a thread: 16 bytes, 8 where 8 taps of 8 channels would not fit the registers.
template <class T, int TAPS> constexpr int conv_vec() { return TAPS > 4 ? 4 : 16 / (int)sizeof(T); }

struct ConvArgs {
    jq_rows x, out;
    int batch, plies, channels, taps;
    bool silu;
    const void *weight, *bias;   // (channels, taps), (channels)
    const uint8_t *starts;
    int64_t starts_batch, starts_ply;
    const int32_t *lengths;
    const void *s_in;   // (batch, taps - 1, channels): the inputs before
    void *s_out;
    int run, runs, parts, tx;   // plies of a run, runs of a game, blocks that share the items (game, run), threads across channels
    // backward
    jq_rows d_out, dx;
    const void *d_final;
    void *d_initial;
    float *part;   // (parts, taps + 1, channels): each block's share of dweight and dbias
};

// The weights of a thread's channels, those of the last `taps` of TAPS.
template <class W, int V, int TAPS>
__device__ __forceinline__ void load_weights(const ConvArgs &a, int c, int n, float (&w)[TAPS][V], float (&bias)[V])
{
    const W *weight = static_cast<const W *>(a.weight), *b = static_cast<const W *>(a.bias);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int64_t ch = c + min(e, n - 1);
        bias[e] = b ? (float)b[ch] : 0.f;
#pragma unroll
        for (int j = 0; j < TAPS; ++j) w[j][e] = j >= TAPS - a.taps ? (float)weight[ch * a.taps + j - (TAPS - a.taps)] : 0.f;
    }
}

// The input at ply t, before the first one the state's.
template <class T, int V>
__device__ __forceinline__ typename Pack<T, V>::type conv_input(const ConvArgs &a, int64_t b, int t, int c, int n)
{
    if (t >= 0) return load_some<T, V>(row_at<const T>(a.x, b, t, 0) + c, n);
    if (!a.s_in) return typename Pack<T, V>::type{};
    return load_some<T, V>(static_cast<const T *>(a.s_in) + (b * (a.taps - 1) + a.taps - 1 + t) * a.channels + c, n);
}

__device__ __forceinline__ bool conv_start(const ConvArgs &a, int64_t b, int t)
{
    return t >= 0 && a.starts && a.starts[b * a.starts_batch + t * a.starts_ply];
}

// x with the taps that reach back further than `reach` plies left out.
template <int V, int TAPS>
__device__ __forceinline__ void conv_sum(const float (&x)[TAPS][V], const float (&w)[TAPS][V], int reach, float (&o)[V])
{
#pragma unroll
    for (int j = 0; j < TAPS; ++j) {
        if (TAPS - 1 - j > reach) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf(w[j][e], x[j][e], o[e]);
    }
}

template <class T, class W, int TAPS>
__global__ __launch_bounds__(256) void k_conv_forward(ConvArgs a)
{
    constexpr int V = conv_vec<T, TAPS>();
    typedef typename Pack<T, V>::type Raw;
    const int blocks_x = ((a.channels + V - 1) / V + a.tx - 1) / a.tx;
    const int c = (blockIdx.x % blocks_x * a.tx + threadIdx.x % a.tx) * V, n = a.channels - c;
    if (n <= 0) return;
    const int ty = 256 / a.tx, part = blockIdx.x / blocks_x;
    float w[TAPS][V], bias[V], x[TAPS][V];
    load_weights<W, V, TAPS>(a, c, n, w, bias);
    const int64_t items = (int64_t)a.batch * a.runs;
    for (int64_t item = (int64_t)part * ty + threadIdx.x / a.tx; item < items; item += (int64_t)a.parts * ty) {
        const int64_t b = item / a.runs;
        const int i = item % a.runs, t0 = i * a.run, t1 = min(t0 + a.run, a.plies);
        const int len = a.lengths ? min(max(a.lengths[b], 0), a.plies) : a.plies, end = min(t1, len);
        const bool last = i == max(len - 1, 0) / a.run;
        if (end > t0 || last) {
#pragma unroll
            for (int j = 0; j < TAPS; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) x[j][e] = 0.f;
            int reach = a.taps - 1;
            for (int at = t0 - (a.taps - 1); at < end; at += CONV_AHEAD) {
                Raw raw[CONV_AHEAD];
                bool start[CONV_AHEAD];
#pragma unroll
                for (int k = 0; k < CONV_AHEAD; ++k) {
                    const int t = min(at + k, end - 1);
                    raw[k] = conv_input<T, V>(a, b, t, c, n);
                    start[k] = conv_start(a, b, t);
                }
#pragma unroll
                for (int k = 0; k < CONV_AHEAD; ++k) {
                    const int t = at + k;
                    if (t >= end) continue;
                    if (start[k]) {
                        reach = -1;
#pragma unroll
                        for (int j = 0; j < TAPS; ++j)
#pragma unroll
                            for (int e = 0; e < V; ++e) x[j][e] = 0.f;
                    }
                    reach = min(reach + 1, a.taps - 1);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
#pragma unroll
                        for (int j = 0; j + 1 < TAPS; ++j) x[j][e] = x[j + 1][e];
                        x[TAPS - 1][e] = (float)raw[k][e];
                    }
                    if (t < t0) continue;
                    float o[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) o[e] = bias[e];
                    if (reach >= TAPS - 1) conv_sum<V, TAPS>(x, w, TAPS - 1, o);
                    else conv_sum<V, TAPS>(x, w, reach, o);
                    if (a.silu)
#pragma unroll
                        for (int e = 0; e < V; ++e) o[e] *= sigmoid(o[e]);
                    store_floats<T, V>(row_at<T>(a.out, b, t, 0) + c, n, o);
                }
            }
            if (last && a.s_out)
#pragma unroll
                for (int j = 1; j < TAPS; ++j) {
                    const int e = j - 1 - (TAPS - a.taps);
                    if (e >= 0) store_floats<T, V>(static_cast<T *>(a.s_out) + (b * (a.taps - 1) + e) * a.channels + c, n, x[j]);
                }
        }
        const Raw zero{};
        for (int t = max(t0, end); t < t1; ++t) store_some<T, V>(row_at<T>(a.out, b, t, 0) + c, n, zero);
    }
}

// Backward over a run: with g the gradient of the sum at ply t (from the inputs again),
// the plies that it reaches back to gain weight g, their gradients given out once the last
// ply that sees them is done; dweight and dbias stay in registers over a block's runs.
template <class T, class W, int TAPS>
__global__ __launch_bounds__(256) void k_conv_backward(ConvArgs a)
{
    constexpr int V = conv_vec<T, TAPS>();
    typedef typename Pack<T, V>::type Raw;
    __shared__ float red[256 * V];
    const int blocks_x = ((a.channels + V - 1) / V + a.tx - 1) / a.tx;
    const int c = (blockIdx.x % blocks_x * a.tx + threadIdx.x % a.tx) * V, n = a.channels - c;
    const int ty = 256 / a.tx, part = blockIdx.x / blocks_x;
    float w[TAPS][V], bias[V], x[TAPS][V], acc[TAPS][V], dw[TAPS][V], db[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        db[e] = 0.f;
#pragma unroll
        for (int j = 0; j < TAPS; ++j) dw[j][e] = 0.f;
    }
    const int64_t items = n > 0 ? (int64_t)a.batch * a.runs : 0;
    if (n > 0) load_weights<W, V, TAPS>(a, c, n, w, bias);
    for (int64_t item = (int64_t)part * ty + threadIdx.x / a.tx; item < items; item += (int64_t)a.parts * ty) {
        const int64_t b = item / a.runs;
        const int i = item % a.runs, t0 = i * a.run, t1 = min(t0 + a.run, a.plies);
        const int len = a.lengths ? min(max(a.lengths[b], 0), a.plies) : a.plies;
        const int end = min(t1, len), until = min(t1 + a.taps - 1, len);   // plies of this run; plies that see one
        const int from = i ? t0 : 1 - a.taps;                              // the first run has the state's gradients
        // acc[j]: the gradient of the input j plies before the one at hand
        auto give = [&](int t, const float (&g)[V]) {
            if (t < from || t >= end) return;
            if (t >= 0) {
                if (a.dx.data) store_floats<T, V>(row_at<T>(a.dx, b, t, 0) + c, n, g);
            } else if (a.d_initial)
                store_floats<T, V>(static_cast<T *>(a.d_initial) + (b * (a.taps - 1) + a.taps - 1 + t) * a.channels + c, n, g);
        };
        if (end > t0 || !i) {
#pragma unroll
            for (int j = 0; j < TAPS; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) x[j][e] = acc[j][e] = 0.f;
            int reach = a.taps - 1;
            for (int at = t0 - (a.taps - 1); at < until; at += CONV_AHEAD) {
                Raw raw[CONV_AHEAD], graw[CONV_AHEAD];
                bool start[CONV_AHEAD];
#pragma unroll
                for (int k = 0; k < CONV_AHEAD; ++k) {
                    const int t = min(at + k, until - 1);
                    raw[k] = conv_input<T, V>(a, b, t, c, n);
                    graw[k] = Raw{};
                    if (t >= t0) graw[k] = load_some<T, V>(row_at<const T>(a.d_out, b, t, 0) + c, n);
                    start[k] = conv_start(a, b, t);
                }
#pragma unroll
                for (int k = 0; k < CONV_AHEAD; ++k) {
                    const int t = at + k;
                    if (t >= until) continue;
                    if (start[k]) reach = -1;
                    reach = min(reach + 1, a.taps - 1);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
#pragma unroll
                        for (int j = 0; j + 1 < TAPS; ++j) x[j][e] = x[j + 1][e];
                        x[TAPS - 1][e] = (float)raw[k][e];
#pragma unroll
                        for (int j = TAPS - 1; j > 0; --j) acc[j][e] = acc[j - 1][e];
                        acc[0][e] = 0.f;
                    }
                    if (t >= t0) {
                        float g[V];
#pragma unroll
                        for (int e = 0; e < V; ++e) g[e] = (float)graw[k][e];
                        if (a.silu) {
                            float o[V];
#pragma unroll
                            for (int e = 0; e < V; ++e) o[e] = bias[e];
                            if (reach >= TAPS - 1) conv_sum<V, TAPS>(x, w, TAPS - 1, o);
                            else conv_sum<V, TAPS>(x, w, reach, o);
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                const float s = sigmoid(o[e]);
                                g[e] *= s * fmaf(o[e], 1.f - s, 1.f);
                            }
                        }
                        auto take = [&](int most) {
#pragma unroll
                            for (int j = 0; j < TAPS; ++j) {
                                if (TAPS - 1 - j > most) continue;
#pragma unroll
                                for (int e = 0; e < V; ++e) {
                                    acc[TAPS - 1 - j][e] = fmaf(w[j][e], g[e], acc[TAPS - 1 - j][e]);
                                    if (t < t1) dw[j][e] = fmaf(x[j][e], g[e], dw[j][e]);
                                }
                            }
                        };
                        if (reach >= TAPS - 1) take(TAPS - 1);
                        else take(reach);
                        if (t < t1)
#pragma unroll
                            for (int e = 0; e < V; ++e) db[e] += g[e];
                    }
                    if (t < until - 1 || until < len) {   // the last input that the next ply does not see
#pragma unroll
                        for (int j = 0; j < TAPS; ++j)
                            if (j == a.taps - 1) give(t - j, acc[j]);
                    }
                }
            }
            // what is left: all inputs up to the last ply, with what the state after it sends back
            const int at = until - 1;
            if (until == len) {
#pragma unroll
                for (int j = 0; j < TAPS; ++j) {
                    if (j > a.taps - 1) continue;
                    float g[V];
                    const bool kept = a.d_final && j < a.taps - 1 && (j <= reach || len == 0);
                    typename Pack<T, V>::type d{};
                    if (kept) d = load_some<T, V>(static_cast<const T *>(a.d_final) + (b * (a.taps - 1) + a.taps - 2 - j) * a.channels + c, n);
#pragma unroll
                    for (int e = 0; e < V; ++e) g[e] = acc[j][e] + (kept ? (float)d[e] : 0.f);
                    give(at - j, g);
                }
            } else {
#pragma unroll
                for (int j = 0; j < TAPS; ++j)
                    if (j < a.taps - 1) give(at - j, acc[j]);
            }
        }
        const Raw zero{};
        if (a.dx.data)
            for (int t = max(t0, end); t < t1; ++t) store_some<T, V>(row_at<T>(a.dx, b, t, 0) + c, n, zero);
    }
    if (!a.part) return;
    // the block's rows of threads summed in order
#pragma unroll
    for (int j = 0; j <= TAPS; ++j) {
        if (j < TAPS - a.taps) continue;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) red[threadIdx.x * V + e] = j < TAPS ? dw[j < TAPS ? j : 0][e] : db[e];
        __syncthreads();
        const int cols = a.tx * V, base = blockIdx.x % blocks_x * cols;
        float *to = a.part + ((int64_t)part * (a.taps + 1) + j - (TAPS - a.taps)) * a.channels + base;
        for (int q = threadIdx.x; q < cols; q += 256) {
            float s = 0.f;
            for (int y = 0; y < ty; ++y) s += red[y * cols + q];
            if (base + q < a.channels) to[q] = s;
        }
    }
}

// dweight (channels, taps) and dbias: the blocks' shares summed in a fixed order.
template <class W>
__global__ __launch_bounds__(256) void k_conv_join(const float *part, int parts, int taps, int channels, W *dweight, W *dbias)
{
    __shared__ float red[16][17];
    const int64_t cols = (int64_t)(taps + 1) * channels, col = (int64_t)blockIdx.x * 16 + threadIdx.x % 16;
    const int slice = threadIdx.x / 16;
    float s = 0.f;
    if (col < cols)
        for (int q = slice; q < parts; q += 16) s += part[q * cols + col];
    red[slice][threadIdx.x % 16] = s;
    __syncthreads();
    if (slice || col >= cols) return;
    s = 0.f;
    for (int q = 0; q < 16; ++q) s += red[q][threadIdx.x];
    const int j = col / channels, ch = col % channels;
    if (j < taps) {
        if (dweight) dweight[(int64_t)ch * taps + j] = from_float<W>(s);
    } else if (dbias) dbias[ch] = from_float<W>(s);
}

// ------------------------------------------------------------------ one ply
struct ConvStepArgs {
    ConvArgs c;   // x and out: (batch, channels); weights
    void *state;
    int64_t state_rows;
    const int64_t *rows;
    const uint8_t *starts;
};

template <class T, class W, int TAPS>
__global__ __launch_bounds__(256) void k_conv_step(ConvStepArgs s)
{
    constexpr int V = conv_vec<T, TAPS>();
    typedef typename Pack<T, V>::type Raw;
    const ConvArgs &a = s.c;
    const int blocks_x = ((a.channels + V - 1) / V + a.tx - 1) / a.tx;
    const int c = (blockIdx.x % blocks_x * a.tx + threadIdx.x % a.tx) * V, n = a.channels - c;
    if (n <= 0) return;
    const int ty = 256 / a.tx, part = blockIdx.x / blocks_x;
    float w[TAPS][V], bias[V];
    load_weights<W, V, TAPS>(a, c, n, w, bias);
    for (int64_t b = (int64_t)part * ty + threadIdx.x / a.tx; b < a.batch; b += (int64_t)a.parts * ty) {
        T *out = row_at<T>(a.out, b, 0, 0) + c;
        const int64_t row = s.rows ? s.rows[b] : b;
        if (row < 0 || row >= s.state_rows) {
            store_some<T, V>(out, n, Raw{});
            continue;
        }
        T *state = static_cast<T *>(s.state) + row * (a.taps - 1) * a.channels + c;
        const bool start = s.starts && s.starts[b];
        Raw x[TAPS];
#pragma unroll
        for (int j = 0; j + 1 < TAPS; ++j) {
            const int e = j - (TAPS - a.taps);
            x[j] = e >= 0 && !start ? load_some<T, V>(state + (int64_t)e * a.channels, n) : Raw{};
        }
        x[TAPS - 1] = load_some<T, V>(row_at<const T>(a.x, b, 0, 0) + c, n);
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = bias[e];
#pragma unroll
        for (int j = 0; j < TAPS; ++j) {
            if (TAPS - 1 - j > (start ? 0 : a.taps - 1)) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fmaf(w[j][e], (float)x[j][e], o[e]);
        }
        if (a.silu)
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] *= sigmoid(o[e]);
        store_floats<T, V>(out, n, o);
#pragma unroll
        for (int j = 1; j < TAPS; ++j) {
            const int e = j - 1 - (TAPS - a.taps);
            if (e >= 0) store_some<T, V>(state + (int64_t)e * a.channels, n, x[j]);
        }
    }
}

}  // namespace jq
