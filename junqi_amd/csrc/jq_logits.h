// Penalties, biases and legal masks on the logits of the actions, and their gradients.
#pragma once
#include <type_traits>

#include "jq_conv.h"

namespace jq {

// For each row and action, with count how often the row's recent actions name it:
//   x = logit; where count > 0: x = (x > 0 ? x / repetition : x * repetition) - frequency count - presence;
//   x += bias; where the mask has the action: out = x, else -infinity
// A block has a tile of a row's columns. Where none of a thread's columns is legal it
// reads no logits: a policy's masks leave a few dozen of 16,641 actions.
constexpr int LOGITS_TILE = 4096;

struct LogitsArgs {
    const void *x, *d;   // logits; gradient of the result (backward)
    void *o;             // result, or gradient of the logits
    int64_t x_stride, d_stride, o_stride;
    int64_t rows;
    int actions, tiles;
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

// Which of a tile's columns the recent actions of a row name, and how often.
struct Named {
    uint32_t any[LOGITS_TILE / 32 + 1];
    int count[LOGITS_TILE];
};

// The ids of a row that lie in [c0, c1): f(column - c0).
template <class F>
__device__ __forceinline__ void each_recent(const LogitsArgs &a, int64_t row, int c0, int c1, F &&f)
{
    const int count = a.recent_lengths ? min(max(a.recent_lengths[row], 0), a.recent_count) : a.recent_count;
    for (int i = threadIdx.x; i < count; i += 256) {
        const int64_t at = row * a.recent_stride + i;
        const int64_t id = a.recent64 ? static_cast<const int64_t *>(a.recent)[at] : static_cast<const int32_t *>(a.recent)[at];
        if (id >= c0 && id < c1) f((int)id - c0);
    }
}

__device__ __forceinline__ void count_recent(const LogitsArgs &a, Named &named, int64_t row, int c0, int c1)
{
    __syncthreads();   // the row before is done
    for (int i = threadIdx.x; i < LOGITS_TILE / 32 + 1; i += 256) named.any[i] = 0;
    each_recent(a, row, c0, c1, [&](int c) { named.count[c] = 0; });
    __syncthreads();
    each_recent(a, row, c0, c1, [&](int c) {
        atomicAdd(&named.count[c], 1);
        atomicOr(&named.any[c / 32], 1u << c % 32);
    });
    __syncthreads();
}

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

struct Penalty {
    float repetition, inverse, frequency, presence;
    __device__ __forceinline__ Penalty(const LogitsArgs &a, int64_t row)
    {
        repetition = a.repetitions ? a.repetitions[row] : a.repetition;
        frequency = a.frequencies ? a.frequencies[row] : a.frequency;
        presence = a.presences ? a.presences[row] : a.presence;
        inverse = 1.f / repetition;
    }
};

// The first column of a tile's vectors: out's rows are written in whole aligned vectors of
// N, whatever their length, with the columns before and after one by one.
template <class T, int N>
__device__ __forceinline__ int first_whole(const T *row, int c0, int c1)
{
    const int off = (int)(((uintptr_t)(row + c0) / sizeof(T)) % N);
    return min(off ? c0 + N - off : c0, c1);
}

// f(first column, count) for this thread's columns of [c0, c1): vectors of N, and single ones at the ends.
template <class T, int N, class F>
__device__ __forceinline__ void each_vector(const T *row, int c0, int c1, F &&f)
{
    const int head = first_whole<T, N>(row, c0, c1), vectors = (c1 - head) / N, tail = head + vectors * N;
    if (threadIdx.x < N && c0 + (int)threadIdx.x < head) f(c0 + (int)threadIdx.x, 1);
    for (int v = threadIdx.x; v < vectors; v += 256) f(head + v * N, N);
    if (threadIdx.x >= 256 - N && tail + 255 - (int)threadIdx.x < c1) f(tail + 255 - (int)threadIdx.x, 1);
}

// Which of n columns from c on the recent actions name (bit e: column c + e).
__device__ __forceinline__ uint32_t named_bits(const Named &named, int at, int n)
{
    const uint64_t lo = named.any[at / 32], hi = named.any[at / 32 + 1];
    return (uint32_t)((lo | hi << 32) >> at % 32) & ((1u << n) - 1);
}

template <class T, bool RECENT>
__global__ __launch_bounds__(256) void k_logits_forward(LogitsArgs a)
{
    constexpr int N = Vec<T>::N;
    __shared__ typename std::conditional<RECENT, Named, int>::type named;
    const int64_t items = a.rows * a.tiles;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t row = item / a.tiles;
        const int c0 = item % a.tiles * LOGITS_TILE, c1 = min(c0 + LOGITS_TILE, a.actions);
        if constexpr (RECENT) count_recent(a, named, row, c0, c1);
        const Penalty p(a, row);
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
        T *o = static_cast<T *>(a.o) + row * a.o_stride;
        each_vector<T, N>(o, c0, c1, [&](int c, int n) {
            const uint32_t legal = legal_bits(a, row, c, n);
            typename Pack<T, N>::type r;
#pragma unroll
            for (int e = 0; e < N; ++e) r[e] = T(-__builtin_inff());
            if (legal) {
                const typename Pack<T, N>::type raw = load_some<T, N>(x + c, n);
                float y[N];
#pragma unroll
                for (int e = 0; e < N; ++e) y[e] = (float)raw[e];
                if constexpr (RECENT) {
                    const uint32_t again = named_bits(named, c - c0, n);
                    if (again)
#pragma unroll
                        for (int e = 0; e < N; ++e)
                            if (again >> e & 1)
                                y[e] = (y[e] > 0.f ? y[e] * p.inverse : y[e] * p.repetition) - fmaf(p.frequency, (float)named.count[c - c0 + e], p.presence);
                }
                if (a.bias)
#pragma unroll
                    for (int e = 0; e < N; ++e) y[e] += a.bias[e < n ? c + e : c];
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (legal >> e & 1) r[e] = from_float<T>(y[e]);
            }
            store_some<T, N>(o + c, n, r);
        });
    }
}

// Gradients: of the logits, g where the action is legal, times what the repetition's
// penalty multiplies by; of the bias, g summed over the rows. A block has one tile of
// every parts-th row, and a thread adds to sums of the tile in LDS: which thread has a
// column changes with the rows' alignment, so a barrier parts the rows.
template <class T, bool RECENT>
__global__ __launch_bounds__(256) void k_logits_backward(LogitsArgs a)
{
    constexpr int N = Vec<T>::N;
    __shared__ typename std::conditional<RECENT, Named, int>::type named;
    extern __shared__ float sums[];   // LOGITS_TILE, where dbias is wanted
    const int tile = blockIdx.x % a.tiles, part = blockIdx.x / a.tiles;
    const int c0 = tile * LOGITS_TILE, c1 = min(c0 + LOGITS_TILE, a.actions);
    if (a.part)
        for (int i = threadIdx.x; i < LOGITS_TILE; i += 256) sums[i] = 0.f;
    for (int64_t row = part; row < a.rows; row += a.parts) {
        if constexpr (RECENT) count_recent(a, named, row, c0, c1);
        else if (a.part) __syncthreads();
        const Penalty p(a, row);
        const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
        const T *d = static_cast<const T *>(a.d) + row * a.d_stride;
        T *o = static_cast<T *>(a.o) + row * a.o_stride;
        each_vector<T, N>(a.o ? o : d, c0, c1, [&](int c, int n) {
            const uint32_t legal = legal_bits(a, row, c, n);
            typename Pack<T, N>::type r{};
            if (legal) {
                const typename Pack<T, N>::type raw = load_some<T, N>(d + c, n);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    if (!(legal >> e & 1)) continue;
                    const float g = (float)raw[e];
                    r[e] = raw[e];
                    if (a.part) sums[c - c0 + e] += g;
                    if constexpr (RECENT)
                        if (named_bits(named, c - c0 + e, 1)) r[e] = from_float<T>((float)x[c + e] > 0.f ? g * p.inverse : g * p.repetition);
                }
            }
            if (a.o) store_some<T, N>(o + c, n, r);
        });
    }
    if (!a.part) return;
    __syncthreads();
    for (int i = threadIdx.x; c0 + i < c1; i += 256) a.part[(int64_t)part * a.actions + c0 + i] = sums[i];
}

// dbias: the blocks' shares summed in a fixed order.
__global__ __launch_bounds__(256) void k_logits_join(const float *part, int parts, int actions, float *dbias)
{
    __shared__ float red[16][17];
    const int64_t col = (int64_t)blockIdx.x * 16 + threadIdx.x % 16;
    const int slice = threadIdx.x / 16;
    float s = 0.f;
    if (col < actions)
        for (int q = slice; q < parts; q += 16) s += part[(int64_t)q * actions + col];
    red[slice][threadIdx.x % 16] = s;
    __syncthreads();
    if (slice || col >= actions) return;
    s = 0.f;
    for (int q = 0; q < 16; ++q) s += red[q][threadIdx.x];
    dbias[col] = s;
}

}  // namespace jq
