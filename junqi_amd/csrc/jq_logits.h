// Penalties, biases and legal masks on the logits of the actions, and their gradients.
#pragma once
#include <type_traits>

#include "jq_conv.h"

namespace jq {

// For each row and action, with count how often the row's recent actions name it:
//   x = logit; where count > 0: x = (x > 0 ? x / repetition : x * repetition) - frequency count - presence;
//   x += bias; where the mask has the action: out = x, else -infinity
// Bound by the rows' traffic. A wave has a row's columns (parts of them where rows are few)
// and streams them: their mask first, as bits in LDS of the wave's own, then vectors of 16
// bytes, the next ones' logits asked for before this ones' results are stored, because
// loads behind stores are seen only after these. Where none of a lane's columns is legal it
// reads no logits: a policy's masks leave a few dozen of 16,641. The columns are written
// without the penalties; where a recent action is legal, the wave counts these in a table
// of its own in LDS and writes their columns again. 32,768 rows of 16,641 in bfloat16: 385 us
// (1.09 GB written, 0.28 GB read; waves wait three quarters of the time); 705 with the counts of a tile's actions in LDS and
// barriers around them, 611 with a wave for four vectors a lane, 513 with loads behind
// stores. Vectors that straddle 16 bytes, as odd rows' do, cost nothing here (stores of
// nothing but -infinity 228 us, aligned 251).
constexpr int LOGITS_AHEAD = 2;   // vectors of a lane on their way together (1 / 2 / 3: 435 / 400 / 419 us a call)
constexpr int LOGITS_TILE = 32768;   // most columns of a wave

struct LogitsArgs {
    const void *x, *d;   // logits; gradient of the result (backward)
    void *o;             // result, or gradient of the logits
    int64_t x_stride, d_stride, o_stride;
    int64_t rows;
    int actions, tile, tiles;   // columns of a wave, a multiple of 32; tiles of a row
    int mask_words;             // of a wave's mask in LDS, before its table
    int slots;                  // of a wave's table: a power of two, at least twice the actions that it can get
    const float *bias;
    const uint32_t *words;    // legal, packed: bit j of word i is column 32 i + j
    const uint8_t *dense;     // legal, a byte a column
    int64_t mask_stride;      // between rows, in words or bytes
    const void *recent;       // (rows, recent_count) ids; others than 0 .. actions - 1 are passed over
    int64_t recent_stride;
    int recent_count;
    bool recent64;
    const int32_t *recent_lengths;
    float repetition, frequency, presence;               // of every row,
    const float *repetitions, *frequencies, *presences;  // or of each
    float *part;   // (parts, actions): each block's share of dbias
    int parts;
};

// Bit e: column c + e is legal, e < n: 1, 4 or 8.
__device__ __forceinline__ uint32_t legal_bits(const LogitsArgs &a, int64_t row, int c, int n)
{
    const uint32_t all = (1u << n) - 1;
    if (a.words) {
        const uint32_t *w = a.words + row * a.mask_stride;
        const uint64_t lo = w[c / 32], hi = w[(c + n - 1) / 32];
        return (uint32_t)((lo | hi << 32) >> c % 32) & all;
    }
    if (a.dense) {
        const uint8_t *m = a.dense + row * a.mask_stride + c;
        uint32_t bits = 0;
        if (n >= 4) {
            typedef uint32_t At __attribute__((aligned(1)));
            for (int q = 0; q < n; q += 4) {
                const uint32_t v = *reinterpret_cast<const At *>(m + q);
#pragma unroll
                for (int e = 0; e < 4; ++e) bits |= (uint32_t)((v >> e * 8 & 0xFF) != 0) << (q + e);
            }
        } else
            for (int e = 0; e < n; ++e) bits |= (uint32_t)(m[e] != 0) << e;
        return bits;
    }
    return all;
}

// The few named columns of a row are divided, not multiplied by a reciprocal: one rounding,
// and no infinity where the repetition is below 2^-128.
struct Penalty {
    float repetition, frequency, presence;
    __device__ __forceinline__ Penalty(const LogitsArgs &a, int64_t row)
    {
        repetition = a.repetitions ? a.repetitions[row] : a.repetition;
        frequency = a.frequencies ? a.frequencies[row] : a.frequency;
        presence = a.presences ? a.presences[row] : a.presence;
    }
};

// A wave's columns of a row, their mask and the recent actions in them.
struct Tile {
    int64_t row;
    int c0, c1, count, *table;
    uint32_t *mask;   // bit j of word i: column c0 + 32 i + j
    __device__ __forceinline__ Tile(const LogitsArgs &a, int64_t item, float *lds)
    {
        row = item / a.tiles;
        c0 = (int)(item - row * a.tiles) * a.tile;
        c1 = c0 + min(a.tile, a.actions - c0);   // c0 + a.tile may not fit 32 bits
        count = !a.recent_count ? 0 : a.recent_lengths ? min(max(a.recent_lengths[row], 0), a.recent_count) : a.recent_count;
        mask = reinterpret_cast<uint32_t *>(lds) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * (a.mask_words + 2 * a.slots);
        table = reinterpret_cast<int *>(mask + a.mask_words);
        const int words = (c1 - c0 + 31) / 32;
        for (int i = threadIdx.x % 64; i < words; i += 64) {
            const int c = c0 + 32 * i, n = min(c1 - c, 32);
            uint32_t bits = 0;
            if (a.words) bits = a.words[row * a.mask_stride + c / 32];
            else if (!a.dense) bits = ~0u;
            else if (n == 32) {
                typedef u32x4 At __attribute__((aligned(1)));
                const At *m = reinterpret_cast<const At *>(a.dense + row * a.mask_stride + c);
                const u32x4 v[2] = {m[0], m[1]};
#pragma unroll
                for (int e = 0; e < 32; ++e) bits |= (uint32_t)((v[e / 16][e / 4 % 4] >> e % 4 * 8 & 0xFF) != 0) << e;
            } else
                for (int e = 0; e < n; ++e) bits |= (uint32_t)(a.dense[row * a.mask_stride + c + e] != 0) << e;
            mask[i] = n < 32 ? bits & ((1u << n) - 1) : bits;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    // bit e: column c + e is legal, e < n; c - c0 is a multiple of n, n of 1, 4 or 8
    __device__ __forceinline__ uint32_t legal(int c, int n) const { return mask[(c - c0) / 32] >> (c - c0) % 32 & ((1u << n) - 1); }
    // recent action i where it is a legal one of the tile, else -1
    __device__ __forceinline__ int recent(const LogitsArgs &a, int i) const
    {
        const int64_t at = row * a.recent_stride + i;
        const int64_t id = a.recent64 ? static_cast<const int64_t *>(a.recent)[at] : static_cast<const int32_t *>(a.recent)[at];
        return id >= c0 && id < c1 && legal((int)id, 1) ? (int)id : -1;
    }
    __device__ __forceinline__ bool penalised(const LogitsArgs &a) const
    {
        bool any = false;
        for (int i = threadIdx.x % 64; i < count; i += 64) any |= recent(a, i) >= 0;
        return __builtin_amdgcn_ballot_w64(any) != 0;
    }
    // f(column, count), each once: an open table, which has more slots than it gets keys
    template <class F> __device__ __forceinline__ void each_recent(const LogitsArgs &a, F &&f) const
    {
        const int lane = threadIdx.x % 64;
        int *keys = table, *counts = table + a.slots;
        for (int i = lane; i < a.slots; i += 64) keys[i] = -1, counts[i] = 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int i = lane; i < count; i += 64) {
            const int key = recent(a, i);
            if (key < 0) continue;
            for (uint32_t s = (uint32_t)key * 0x9E3779B1u >> 16;; ++s) {
                s &= a.slots - 1;
                const int old = atomicCAS(&keys[s], -1, key);
                if (old != -1 && old != key) continue;
                atomicAdd(&counts[s], 1);
                break;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int i = lane; i < a.slots; i += 64)
            if (keys[i] >= 0) f(keys[i], counts[i]);
    }
};

// BACK: the gradient of the logits: g where the action is legal, times what the
// repetition's penalty multiplies by; else the result.
template <class T, bool BACK>
__global__ __launch_bounds__(256) void k_logits(LogitsArgs a)
{
    constexpr int N = Vec<T>::N, AHEAD = LOGITS_AHEAD;
    typedef typename Pack<T, N>::type R;
    typedef typename Pack<float, N>::type B;
    extern __shared__ float lds[];   // the waves' masks and tables
    const bool biased = !BACK && a.bias;
    const int waves = blockDim.x / 64, lane = threadIdx.x % 64;
    const int64_t items = a.rows * a.tiles;
    for (int64_t item = (int64_t)blockIdx.x * waves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64); item < items; item += (int64_t)gridDim.x * waves) {
        const Tile t(a, item, lds);
        const T *x = static_cast<const T *>(a.x) + t.row * a.x_stride, *d = static_cast<const T *>(a.d) + t.row * a.d_stride;
        const T *in = (BACK ? d : x) + t.c0;
        T *o = static_cast<T *>(a.o) + t.row * a.o_stride;
        const bool again = t.count && t.penalised(a);
        const int vectors = (t.c1 - t.c0) / N;
        struct Ahead { uint32_t legal[AHEAD]; R raw[AHEAD]; B bias[AHEAD]; } next;
        auto load = [&](int v0, Ahead &q) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int v = v0 + u * 64;
                q.legal[u] = v < vectors ? t.legal(t.c0 + v * N, N) : 0;
                if (q.legal[u]) {
                    q.raw[u] = load_some<T, N>(in + (int64_t)v * N, N);
                    if (biased) q.bias[u] = load_some<float, N>(a.bias + t.c0 + (int64_t)v * N, N);
                }
            }
        };
        load(lane, next);
        for (int v0 = lane; v0 - lane < vectors; v0 += 64 * AHEAD) {
            const Ahead q = next;
            load(v0 + 64 * AHEAD, next);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int v = v0 + u * 64, c = t.c0 + v * N;
                if (v >= vectors) break;
                R r;
#pragma unroll
                for (int e = 0; e < N; ++e) r[e] = BACK ? T(0.f) : T(-__builtin_inff());
                if (q.legal[u])
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (q.legal[u] >> e & 1) r[e] = biased ? from_float<T>((float)q.raw[u][e] + q.bias[u][e]) : q.raw[u][e];
                store_some<T, N>(o + c, N, r);
            }
        }
        const int single = t.c0 + vectors * N + lane;   // the columns behind the last vector
        if (single < t.c1) {
            float y = BACK ? 0.f : -__builtin_inff();
            if (t.legal(single, 1)) y = (float)in[single - t.c0] + (biased ? a.bias[single] : 0.f);
            o[single] = from_float<T>(y);
        }
        if (!again) continue;
        __builtin_amdgcn_s_waitcnt(0);   // the row is written before its named columns are written again
        const Penalty p(a, t.row);
        t.each_recent(a, [&](int c, int count) {
            const float y = (float)x[c], v = BACK ? (float)d[c] : y, held = y > 0.f ? v / p.repetition : v * p.repetition;
            o[c] = from_float<T>(BACK ? held : held - fmaf(p.frequency, (float)count, p.presence) + (biased ? a.bias[c] : 0.f));
        });
    }
}

// The gradient of the bias: g summed over the rows where the action is legal. A thread has
// N columns of every parts-th row.
template <class T>
__global__ __launch_bounds__(256) void k_logits_bias(LogitsArgs a)
{
    constexpr int N = Vec<T>::N, AHEAD = 4;   // rows on their way together
    const int c = (blockIdx.x % a.tiles * 256 + threadIdx.x) * N, part = blockIdx.x / a.tiles;
    const int n = a.actions - c;
    if (n <= 0) return;
    float sum[N];
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = 0.f;
    const T *d = static_cast<const T *>(a.d) + c;
    for (int64_t row = part; row < a.rows; row += (int64_t)a.parts * AHEAD) {
        uint32_t legal[AHEAD];
        typename Pack<T, N>::type raw[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int64_t r = row + (int64_t)u * a.parts;
            legal[u] = 0;
            if (r >= a.rows) continue;
            if (n >= N) legal[u] = legal_bits(a, r, c, N);
            else
                for (int e = 0; e < n; ++e) legal[u] |= legal_bits(a, r, c + e, 1) << e;
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (legal[u]) raw[u] = load_some<T, N>(d + (row + (int64_t)u * a.parts) * a.d_stride, n);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (legal[u])
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (legal[u] >> e & 1) sum[e] += (float)raw[u][e];
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e < n) a.part[(int64_t)part * a.actions + c + e] = sum[e];
}

// dbias: the blocks' shares summed in a fixed order, 16 columns a block at a time: a block for
// each 16 would be 2^32 threads, more than a launch may have, from 2^28 actions on.
constexpr int LOGITS_JOIN_BLOCKS = 1 << 20;
__global__ __launch_bounds__(256) void k_logits_join(const float *part, int parts, int actions, float *dbias)
{
    __shared__ float red[16][17];
    const int lane = threadIdx.x % 16, slice = threadIdx.x / 16;
    for (int64_t c0 = (int64_t)blockIdx.x * 16; c0 < actions; c0 += (int64_t)gridDim.x * 16) {
        const int64_t col = c0 + lane;
        float s = 0.f;
        if (col < actions)
            for (int q = slice; q < parts; q += 16) s += part[(int64_t)q * actions + col];
        red[slice][lane] = s;
        __syncthreads();
        if (!slice && col < actions) {
            s = 0.f;
            for (int q = 0; q < 16; ++q) s += red[q][lane];
            dbias[col] = s;
        }
        __syncthreads();   // red is written anew
    }
}

}  // namespace jq
