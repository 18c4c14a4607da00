// The causal convolution over a few plies, forward and backward, and its step of one ply.
#pragma once
#include "jq_memory.h"
#include "jq_scan.h"

namespace jq {

// out_t = bias + sum over j of weight[j] x_{t - taps + 1 + j}, then x sigmoid(x) where
// `silu`; inputs before a game's start are not there. A thread has V channels together and
// walks a run of plies with the last inputs in a ring of registers, so a row is read once but
// for the taps - 1 before a run, and the next step's rows are asked for before this one's
// results are stored: loads behind stores are seen only after these. Bound by the rows'
// traffic forward (1,024 games x 256 plies of 512 channels, four taps, bfloat16, 537 MB: 97
// us, 5.5 TB/s), by that and its products backward (805 MB: 228 us, 3.6 TB/s, VALU busy 56 %,
// 177 registers: two waves a SIMD, and one of 256 behind five to eight taps, 435 us).
// A row that ends inside a thread's channels takes that thread, and so its wave, element by
// element there: 501 channels 186 us forward and 639 with gradients, 512 97 and 301.
// With an address worked out for every access, and a step's loads behind the last one's
// stores, 164 and 332 us.
// Plies of a step, whose rows are on their way while the step before is computed: a
// multiple of the taps, so that the last inputs stay where they are in registers.
constexpr int conv_step(int taps) { return taps == 2 ? 4 : taps; }

// Channels of a thread, V: 4 of float32 and behind four taps, whose registers would not
// hold more. Of bfloat16 8 or 4, 1e8 elements of four taps, us with 8 / with 4:
//                            512 channels   500 (rows 8-byte aligned)   501 (2-byte aligned)
//   forward                     98 / 121           183 / 120                187 / 263
//   one ply, 32,768 games       46 / 40             59 / 50                  62 / 62
//   backward                   246 / 205           646 / 220                653 / 452
// (the backward pass holds four times the taps' registers). So: forward 8, unless rows lie
// at 8 bytes and not at 16; the others 4.
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

// The weights of a thread's channels by how far back they reach, 0 behind the last tap.
template <class W, int V, int TAPS>
__device__ __forceinline__ void load_weights(const ConvArgs &a, int c, int n, float (&w)[TAPS][V], float (&bias)[V])
{
    const W *weight = static_cast<const W *>(a.weight) + (int64_t)c * a.taps, *b = static_cast<const W *>(a.bias);
#pragma unroll
    for (int e = 0; e < V; ++e) bias[e] = 0.f;
    if (b) {
        const typename Pack<W, V>::type r = load_some<W, V>(b + c, n);
#pragma unroll
        for (int e = 0; e < V; ++e) bias[e] = (float)r[e];
    }
    if (n >= V && a.taps == TAPS) {   // V * TAPS of them together
#pragma unroll
        for (int i = 0; i < V * TAPS; i += V) {
            const typename Pack<W, V>::type r = load_some<W, V>(weight + i, V);
#pragma unroll
            for (int e = 0; e < V; ++e) w[TAPS - 1 - (i + e) % TAPS][(i + e) / TAPS] = (float)r[e];
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
#pragma unroll
        for (int j = 0; j < TAPS; ++j) w[j][e] = j < a.taps ? (float)weight[min(e, n - 1) * a.taps + a.taps - 1 - j] : 0.f;
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

// o += the sum over the taps that reach back at most `reach` plies, where x[(k + TAPS - j) % TAPS]
// is the input j plies back.
template <int V, int TAPS>
__device__ __forceinline__ void conv_sum(const float (&x)[TAPS][V], const float (&w)[TAPS][V], int k, int reach, float (&o)[V])
{
#pragma unroll
    for (int j = 0; j < TAPS; ++j) {
        if (j > reach) break;
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf(w[j][e], x[(k + TAPS - j) % TAPS][e], o[e]);
    }
}

// A thread's part in a pass: its channels from c on, n of them, and the items (game, run)
// part * rows + its row, every parts * rows.
struct ConvPlace {
    int c, n, rows, part, base;
    int64_t first;
    __device__ __forceinline__ ConvPlace(const ConvArgs &a, int v)
    {
        const int blocks_x = ((a.channels + v - 1) / v + a.tx - 1) / a.tx;
        base = blockIdx.x % blocks_x * a.tx * v;
        c = base + threadIdx.x % a.tx * v;
        n = a.channels - c;
        rows = 256 / a.tx;
        part = blockIdx.x / blocks_x;
        first = (int64_t)part * rows + threadIdx.x / a.tx;
    }
};

// The inputs before ply t0 into x[TAPS - j], j plies back; returns how far back those of
// ply t0 - 1's game reach.
template <class T, int V, int TAPS>
__device__ __forceinline__ int conv_before(const ConvArgs &a, int64_t b, int t0, int c, int n, float (&x)[TAPS][V])
{
    int reach = a.taps - 1;
    bool start[TAPS];
    typename Pack<T, V>::type raw[TAPS];
#pragma unroll
    for (int j = TAPS - 1; j > 0; --j) {
        raw[j] = j < a.taps ? conv_input<T, V>(a, b, t0 - j, c, n) : typename Pack<T, V>::type{};
        start[j] = j < a.taps && conv_start(a, b, t0 - j);
    }
#pragma unroll
    for (int j = TAPS - 1; j > 0; --j) {
        reach = start[j] ? 0 : min(reach + 1, a.taps - 1);
#pragma unroll
        for (int e = 0; e < V; ++e) x[TAPS - j][e] = (float)raw[j][e];
    }
    return reach;
}

// One ply's row after the other, for one thread.
template <class T> struct PlyPointer {
    T *at;
    int64_t step;
    __device__ __forceinline__ PlyPointer(const jq_rows &r, int64_t b, int64_t t, int c) : at(row_at<T>(r, b, t, 0) + c), step(r.ply) {}
};

template <class T, class W, int TAPS, int V>
__global__ __launch_bounds__(256) void k_conv_forward(ConvArgs a)
{
    constexpr int U = conv_step(TAPS);
    typedef typename Pack<T, V>::type Raw;
    const ConvPlace p(a, V);
    if (p.n <= 0) return;
    const int c = p.c, n = p.n;
    float w[TAPS][V], bias[V], x[TAPS][V];
    load_weights<W, V, TAPS>(a, c, n, w, bias);
    const int64_t items = (int64_t)a.batch * a.runs;
    for (int64_t item = p.first; item < items; item += (int64_t)a.parts * p.rows) {
        const int64_t b = item / a.runs;
        const int i = (int)(item - b * a.runs), t0 = i * a.run, t1 = min(t0 + a.run, a.plies);
        const int len = a.lengths ? min(max(a.lengths[b], 0), a.plies) : a.plies, end = min(t1, len);
        PlyPointer<T> out(a.out, b, t0, c);
        int reach = a.taps - 1;
        if (end > t0) {
            PlyPointer<const T> in(a.x, b, t0, c);
            const uint8_t *starts = a.starts ? a.starts + b * a.starts_batch + t0 * a.starts_ply : nullptr;
            struct Step { Raw raw[U]; uint8_t start[U]; } next;
            auto load = [&](int at, Step &s) {
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    s.start[k] = 0;
                    if (at + k >= end) continue;
                    s.raw[k] = load_some<T, V>(in.at, n);
                    in.at += in.step;
                    if (!starts) continue;
                    s.start[k] = *starts;
                    starts += a.starts_ply;
                }
            };
            load(t0, next);
            reach = conv_before<T, V, TAPS>(a, b, t0, c, n, x);
            for (int at = t0; at < end; at += U) {
                const Step s = next;
                load(at + U, next);
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    if (at + k >= end) break;
                    reach = s.start[k] ? 0 : min(reach + 1, a.taps - 1);
                    float o[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        x[k % TAPS][e] = (float)s.raw[k][e];
                        o[e] = bias[e];
                    }
                    if (reach >= TAPS - 1) conv_sum<V, TAPS>(x, w, k, TAPS - 1, o);
                    else conv_sum<V, TAPS>(x, w, k, reach, o);
                    if (a.silu)
#pragma unroll
                        for (int e = 0; e < V; ++e) o[e] *= sigmoid(o[e]);
                    store_floats<T, V>(out.at, n, o);
                    out.at += out.step;
                }
            }
        }
        if (a.s_out && i == max(len - 1, 0) / a.run)   // the inputs before ply len that its game has
            for (int j = 1; j < a.taps; ++j) {
                const Raw r = j - 1 <= reach || !len ? conv_input<T, V>(a, b, len - j, c, n) : Raw{};
                store_some<T, V>(static_cast<T *>(a.s_out) + (b * (a.taps - 1) + a.taps - 1 - j) * a.channels + c, n, r);
            }
        const Raw zero{};
        for (int t = max(t0, end); t < t1; ++t, out.at += out.step) store_some<T, V>(out.at, n, zero);
    }
}

// Backward over a run: with g the gradient of the sum at ply t (from the inputs again),
// the plies that it reaches back to gain weight g, and each one's gradient is given out
// when the last ply that sees it is done; dweight and dbias stay in registers over a
// block's runs.
template <class T, class W, int TAPS>
__global__ __launch_bounds__(256) void k_conv_backward(ConvArgs a)
{
    constexpr int V = 4, U = conv_step(TAPS);
    typedef typename Pack<T, V>::type Raw;
    __shared__ float red[256 * V];
    const ConvPlace p(a, V);
    const int c = p.c, n = p.n;
    float w[TAPS][V], bias[V], x[TAPS][V], acc[TAPS][V], dw[TAPS][V], db[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        db[e] = 0.f;
#pragma unroll
        for (int j = 0; j < TAPS; ++j) dw[j][e] = 0.f;
    }
    const int64_t items = n > 0 ? (int64_t)a.batch * a.runs : 0;
    if (n > 0) load_weights<W, V, TAPS>(a, c, n, w, bias);
    for (int64_t item = p.first; item < items; item += (int64_t)a.parts * p.rows) {
        const int64_t b = item / a.runs;
        const int i = (int)(item - b * a.runs), t0 = i * a.run, t1 = min(t0 + a.run, a.plies);
        const int len = a.lengths ? min(max(a.lengths[b], 0), a.plies) : a.plies;
        const int end = min(t1, len), until = min(t1 + a.taps - 1, len);   // plies of this run; plies that see one
        const int from = i ? t0 : 1 - a.taps;                              // the first run has the state's gradients
        if (end > t0 || !i) {
            PlyPointer<const T> in(a.x, b, t0, c), gin(a.d_out, b, t0, c);
            PlyPointer<T> out(a.dx, b, t0, c);
            const uint8_t *starts = a.starts ? a.starts + b * a.starts_batch + t0 * a.starts_ply : nullptr;
            struct Step { Raw raw[U], g[U]; uint8_t start[U]; } next;
            auto load = [&](int at, Step &s) {
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    s.start[k] = 0;
                    if (at + k >= until) continue;
                    s.raw[k] = load_some<T, V>(in.at, n);
                    s.g[k] = load_some<T, V>(gin.at, n);
                    in.at += in.step, gin.at += gin.step;
                    if (!starts) continue;
                    s.start[k] = *starts;
                    starts += a.starts_ply;
                }
            };
            load(t0, next);
            int reach = conv_before<T, V, TAPS>(a, b, t0, c, n, x);
#pragma unroll
            for (int j = 0; j < TAPS; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[j][e] = 0.f;
            // the last input is given out TAPS - 1 plies later
            for (int at = t0; at < end + TAPS - 1; at += U) {
                const Step s = next;
                load(at + U, next);
#pragma unroll
                for (int k = 0; k < U; ++k) {
                    const int t = at + k;
#pragma unroll
                    for (int e = 0; e < V; ++e) acc[k % TAPS][e] = 0.f;
                    if (t < until) {
                        reach = s.start[k] ? 0 : min(reach + 1, a.taps - 1);
                        float g[V];
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            x[k % TAPS][e] = (float)s.raw[k][e];
                            g[e] = (float)s.g[k][e];
                        }
                        if (a.silu) {
                            float o[V];
#pragma unroll
                            for (int e = 0; e < V; ++e) o[e] = bias[e];
                            if (reach >= TAPS - 1) conv_sum<V, TAPS>(x, w, k, TAPS - 1, o);
                            else conv_sum<V, TAPS>(x, w, k, reach, o);
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                const float s = sigmoid(o[e]);
                                g[e] *= s * fmaf(o[e], 1.f - s, 1.f);
                            }
                        }
                        const bool own = t < t1;
                        auto take = [&](int most) {
#pragma unroll
                            for (int j = 0; j < TAPS; ++j) {
                                if (j > most) break;
#pragma unroll
                                for (int e = 0; e < V; ++e) acc[(k + TAPS - j) % TAPS][e] = fmaf(w[j][e], g[e], acc[(k + TAPS - j) % TAPS][e]);
                                if (own)
#pragma unroll
                                    for (int e = 0; e < V; ++e) dw[j][e] = fmaf(x[(k + TAPS - j) % TAPS][e], g[e], dw[j][e]);
                            }
                        };
                        if (reach >= TAPS - 1) take(TAPS - 1);
                        else take(reach);
                        if (own)
#pragma unroll
                            for (int e = 0; e < V; ++e) db[e] += g[e];
                    }
                    // the input that no later ply sees, with what the state after the last ply sends back
                    const int s_ply = t - (TAPS - 1), back = len - 1 - s_ply;
                    if (s_ply < from || s_ply >= end) continue;
                    float (&g)[V] = acc[(k + 1) % TAPS];
                    if (a.d_final && back < a.taps - 1 && (back <= reach || !len)) {
                        const Raw d = load_some<T, V>(static_cast<const T *>(a.d_final) + (b * (a.taps - 1) + a.taps - 2 - back) * a.channels + c, n);
#pragma unroll
                        for (int e = 0; e < V; ++e) g[e] += (float)d[e];
                    }
                    if (s_ply >= 0) {
                        if (a.dx.data) store_floats<T, V>(out.at, n, g);
                        out.at += out.step;
                    } else if (a.d_initial)
                        store_floats<T, V>(static_cast<T *>(a.d_initial) + (b * (a.taps - 1) + a.taps - 1 + s_ply) * a.channels + c, n, g);
                }
            }
        }
        if (a.dx.data) {
            const Raw zero{};
            PlyPointer<T> out(a.dx, b, max(t0, end), c);
            for (int t = max(t0, end); t < t1; ++t, out.at += out.step) store_some<T, V>(out.at, n, zero);
        }
    }
    if (!a.part) return;
    // the block's rows of threads summed in order
#pragma unroll
    for (int j = 0; j <= TAPS; ++j) {
        if (j < TAPS && j >= a.taps) continue;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) red[threadIdx.x * V + e] = j < TAPS ? dw[j < TAPS ? j : 0][e] : db[e];
        __syncthreads();
        const int cols = a.tx * V, row = j < TAPS ? a.taps - 1 - j : a.taps;
        float *to = a.part + ((int64_t)p.part * (a.taps + 1) + row) * a.channels + p.base;
        for (int q = threadIdx.x; q < cols; q += 256) {
            float s = 0.f;
            for (int y = 0; y < p.rows; ++y) s += red[y * cols + q];
            if (p.base + q < a.channels) to[q] = s;
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

// A thread walks games with its channels' weights in registers and the next game's inputs
// on their way.
template <class T, class W, int TAPS>
__global__ __launch_bounds__(256) void k_conv_step(ConvStepArgs s)
{
    constexpr int V = 4;
    typedef typename Pack<T, V>::type Raw;
    const ConvArgs &a = s.c;
    const ConvPlace p(a, V);
    if (p.n <= 0) return;
    const int c = p.c, n = p.n;
    float w[TAPS][V], bias[V];
    load_weights<W, V, TAPS>(a, c, n, w, bias);
    struct Game { T *state; Raw x[TAPS]; bool start; };   // x[j]: the input j plies back
    auto load = [&](int64_t b, Game &g) {
        const int64_t row = s.rows ? s.rows[b] : b;
        g.state = row < 0 || row >= s.state_rows ? nullptr : static_cast<T *>(s.state) + row * (a.taps - 1) * a.channels + c;
        g.start = s.starts && s.starts[b];
        const bool there = row >= 0 && row < s.state_rows;
        g.x[0] = load_some<T, V>(row_at<const T>(a.x, b, 0, 0) + c, n);
#pragma unroll
        for (int j = 1; j < TAPS; ++j) g.x[j] = there && j < a.taps && !g.start ? load_some<T, V>(g.state + (int64_t)(a.taps - 1 - j) * a.channels, n) : Raw{};
    };
    const int64_t step = (int64_t)a.parts * p.rows;
    Game next;
    if (p.first < a.batch) load(p.first, next);
    for (int64_t b = p.first; b < a.batch; b += step) {
        const Game g = next;
        if (b + step < a.batch) load(b + step, next);
        T *out = row_at<T>(a.out, b, 0, 0) + c;
        const int64_t row = s.rows ? s.rows[b] : b;
        if (row < 0 || row >= s.state_rows) {
            store_some<T, V>(out, n, Raw{});
            continue;
        }
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = bias[e];
#pragma unroll
        for (int j = 0; j < TAPS; ++j) {
            if (j > (g.start ? 0 : a.taps - 1)) break;
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fmaf(w[j][e], (float)g.x[j][e], o[e]);
        }
        if (a.silu)
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] *= sigmoid(o[e]);
        store_floats<T, V>(out, n, o);
#pragma unroll
        for (int j = 0; j + 1 < TAPS; ++j)
            if (j < a.taps - 1) store_some<T, V>(g.state + (int64_t)(a.taps - 2 - j) * a.channels, n, g.x[j]);
    }
}

}  // namespace jq
