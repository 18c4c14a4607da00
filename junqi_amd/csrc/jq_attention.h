// Linear attention with a decay for each head: the passes over segments of plies
// and the step of one ply.
#pragma once
#include "jq_memory.h"

namespace jq {

// One pass over the plies of every game and head. Forward in time it is
//   S <- (start ? 0 : lambda S) + in_scale k v^T,   o = out_scale q S
// and in reverse, with the state carried from the plies after,
//   full = S + in_scale k v^T,   o = out_scale q full,   S <- start ? 0 : lambda full.
// All passes are this one with the tensors in other places:
//   out: q, k, v forward           dq: d_out, v, k forward, on the transposed state
//   dv:  k, q, d_out in reverse    dk: v, d_out, q in reverse, on the transposed state
struct ScanArgs {
    jq_rows q, k, v, o;
    int batch, plies, heads, kd, vd;   // kd: dim of q and k, vd: dim of v and o
    const float *log_decay;
    const uint8_t *starts;
    int64_t starts_batch, starts_ply;
    const int32_t *lengths;
    const float *s_in;                 // element (i, j) of a head's state at i * s_row + j * s_col
    float *s_out;
    int s_row, s_col;
    float in_scale, out_scale;
    bool reverse;
};

// One block per game and head, one thread per column of the state, which stays in
// registers; q and k of a ply are shared through LDS.
template <class T, int K>
__global__ __launch_bounds__(128) void k_attention_scan(ScanArgs a)
{
    __shared__ float qs[2][K], ks[2][K];
    const int b = blockIdx.x / a.heads, h = blockIdx.x % a.heads, c = threadIdx.x;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.plies) : a.plies;
    const float lam = expf(a.log_decay[h]);
    const bool on = c < a.vd;
    const int64_t sbase = (int64_t)blockIdx.x * a.kd * a.vd;
    float s[K];
#pragma unroll
    for (int i = 0; i < K; ++i) s[i] = a.s_in && on && i < a.kd ? a.s_in[sbase + i * a.s_row + c * a.s_col] : 0.f;
    for (int n = 0; n < len; ++n) {
        const int t = a.reverse ? len - 1 - n : n;
        float *qb = qs[n & 1], *kb = ks[n & 1];
        if (c < K) {
            qb[c] = c < a.kd ? (float)row_at<const T>(a.q, b, t, h)[c] : 0.f;
            kb[c] = c < a.kd ? a.in_scale * (float)row_at<const T>(a.k, b, t, h)[c] : 0.f;
        }
        const float v = on ? (float)row_at<const T>(a.v, b, t, h)[c] : 0.f;
        const bool start = a.starts && a.starts[b * a.starts_batch + t * a.starts_ply];
        __syncthreads();   // two buffers: the next ply's writes are to the other one
        float o = 0.f;
#pragma unroll
        for (int i = 0; i < K; ++i) {
            if (!a.reverse) s[i] = start ? 0.f : lam * s[i];
            s[i] += kb[i] * v;
            o += qb[i] * s[i];
            if (a.reverse) s[i] = start ? 0.f : lam * s[i];
        }
        if (on) row_at<T>(a.o, b, t, h)[c] = from_float<T>(a.out_scale * o);
    }
    for (int t = len; t < a.plies; ++t)
        if (on) row_at<T>(a.o, b, t, h)[c] = from_float<T>(0.f);
    if (a.s_out && on)
#pragma unroll
        for (int i = 0; i < K; ++i)
            if (i < a.kd) a.s_out[sbase + i * a.s_row + c * a.s_col] = s[i];
}

struct StepArgs {
    jq_rows q, k, v, o;
    int heads, dk, dv;
    float scale;
    const float *log_decay;
    float *state;
    int64_t state_rows;
    const int64_t *rows;
    const uint8_t *starts;
};

// One ply of every game: one block per game and head, one thread per column.
template <class T>
__global__ __launch_bounds__(128) void k_attention_step(StepArgs a)
{
    const int b = blockIdx.x / a.heads, h = blockIdx.x % a.heads, c = threadIdx.x;
    if (c >= a.dv) return;
    T *o = row_at<T>(a.o, b, 0, h);
    const int64_t row = a.rows ? a.rows[b] : b;
    if (row < 0 || row >= a.state_rows) {
        o[c] = from_float<T>(0.f);
        return;
    }
    float *s = a.state + (row * a.heads + h) * a.dk * a.dv;
    const T *q = row_at<const T>(a.q, b, 0, h), *k = row_at<const T>(a.k, b, 0, h);
    const float v = (float)row_at<const T>(a.v, b, 0, h)[c], lam = expf(a.log_decay[h]);
    const bool start = a.starts && a.starts[b];
    float sum = 0.f;
    for (int i = 0; i < a.dk; ++i) {
        const float x = (start ? 0.f : lam * s[i * a.dv + c]) + (float)k[i] * v;
        s[i * a.dv + c] = x;
        sum += (float)q[i] * x;
    }
    o[c] = from_float<T>(a.scale * sum);
}

}  // namespace jq
