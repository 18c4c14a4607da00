// The selective state space scan, forward and backward, and its step of one ply.
#pragma once
#include <utility>

#include "jq_memory.h"

namespace jq {

// For each game, channel d and state n, with dt = softplus(delta + bias):
//   h_t = exp(dt_t a) h_{t-1} + dt_t u_t b_t;   y_t = sum over n of c_t h_t, + skip u_t;   out = y silu(gate)
// A lane has a channel and NS of its states in registers; a wave has 64 channels of one
// group, and the SG waves of a block the states of these. b_t and c_t, the same for all
// channels of a group, lie in lanes 0 .. NS - 1 of each row of 16 and reach the products
// as their row-broadcast operands, without an instruction of their own.
constexpr int SCAN_STATES = 64;   // largest states
constexpr int SCAN_PLIES = 4;     // plies whose rows are on their way while the ones before are computed
constexpr int SCAN_CHUNK = 8;     // plies of a chunk of the backward pass, which starts from a saved state

struct SelectArgs {
    jq_rows u, delta, gate, b, c, out;
    int batch, plies, channels, states, groups, per, waves;   // per: channels of a group, waves: of 64 of them
    bool softplus;
    const float *a, *skip, *bias;
    const uint8_t *starts;
    int64_t starts_batch, starts_ply;
    const int32_t *lengths;
    const float *s_in;   // states before, (batch, channels, states)
    float *s_out;        // states after
    float *saved;        // states before each chunk, (batch, chunks, states, channels)
    int segments, seg_plies;        // a long axis in parts: seg_plies is a multiple of SCAN_CHUNK
    float *seg_state, *seg_sum;     // (batch, segments, states, channels): what a part adds, then the state before it;
                                    // (batch, segments, channels): sum of its dt, NaN where a game starts in it
    // backward
    jq_rows d_out, du, ddelta, dgate;
    const float *d_final;
    float *d_initial;
    float *part_bc;   // (waves, batch, plies, groups, 2, states): each wave's share of db and dc
    float *part_a;    // (parts, states + 2, channels): each block's share of da, dskip, dbias
    int parts;        // blocks that share the items (game, segment)
    bool want_bc, want_a;
};

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(-LOG2E * x)); }

// log(1 + e^x) = max(x, 0) + 2 atanh(e / (2 + e)), e = e^-|x|: s = e / (2 + e) is at most
// 1/3, and the series to s^15 is off by less than 2^-26 of the result; small results keep
// all their digits.
__device__ __forceinline__ float softplus(float x)
{
    const float e = exp2_fast(-LOG2E * fabsf(x)), s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float p = 1.f / 15;
    p = fmaf(p, q, 1.f / 13);
    p = fmaf(p, q, 1.f / 11);
    p = fmaf(p, q, 1.f / 9);
    p = fmaf(p, q, 1.f / 7);
    p = fmaf(p, q, 1.f / 5);
    p = fmaf(p, q, 1.f / 3);
    p = fmaf(p, q, 1.f);
    return fmaxf(x, 0.f) + 2.f * s * p;
}

// f(integral_constant<int, 0>()), ..., f(integral_constant<int, N - 1>())
template <class F, int... I> __device__ __forceinline__ void each_of(F &&f, std::integer_sequence<int, I...>)
{
    (f(std::integral_constant<int, I>()), ...);
}
template <int N, class F> __device__ __forceinline__ void each_of(F &&f) { each_of(f, std::make_integer_sequence<int, N>()); }

// x of lane I of each row of 16 lanes, as an operand.
template <int I> __device__ __forceinline__ float row_lane(float x)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x150 + I, 0xF, 0xF, true));
}

template <int HOW> __device__ __forceinline__ float across(float x)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), HOW, 0xF, 0xF, true));
}

// The sums of N values over the wave's lanes, value i in lanes i * 64 / N on: each step
// adds two halves of the lanes for one half of the values, and so halves both.
template <int N>
__device__ __forceinline__ float lane_sums(float (&v)[N])
{
    static_assert(N == 4 || N == 8 || N == 16);
    const int lane = threadIdx.x % 64;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v[i]), __builtin_bit_cast(int, v[i + N / 2]), false, false);
        const uint32_t lo = r[0], hi = r[1];
        v[i] = __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, v[i]), __builtin_bit_cast(int, v[i + N / 4]), false, false);
        const uint32_t lo = r[0], hi = r[1];
        v[i] = __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
    }
    if constexpr (N >= 8) {
        const bool up = lane & 8;
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            const float mine = up ? v[i + N / 8] : v[i], other = up ? v[i] : v[i + N / 8];
            v[i] = mine + across<0x128>(other);   // 8 lanes on, around the row
        }
    } else v[0] += across<0x128>(v[0]);
    if constexpr (N >= 16) {
        const bool up = lane & 4;
        const float mine = up ? v[1] : v[0], other = up ? v[0] : v[1];
        v[0] = mine + across<0x141>(other);   // the other four of eight, mirrored: their sum is taken next
    } else v[0] += across<0x141>(v[0]);
    v[0] += across<0xB1>(v[0]);
    v[0] += across<0x4E>(v[0]);
    return v[0];
}

// Where this wave's lanes are: channel, states, rows.
template <class T, int NS>
struct Place {
    int lane, sg, group, ch, n0, row_n;
    bool on, row_on;
    __device__ __forceinline__ Place(const SelectArgs &a, int cw)
    {
        lane = threadIdx.x % 64;
        sg = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        group = cw / a.waves;
        const int at = (cw % a.waves) * 64 + lane;
        on = at < a.per;
        ch = group * a.per + (on ? at : a.per - 1);
        n0 = sg * NS;
        row_n = n0 + lane % 16;
        row_on = lane % 16 < NS && row_n < a.states;
    }
    template <class F> __device__ __forceinline__ void a2(const SelectArgs &a, F &&f) const
    {
#pragma unroll
        for (int i = 0; i < NS; ++i) f(i, n0 + i < a.states ? a.a[(int64_t)ch * a.states + n0 + i] * LOG2E : 0.f);
    }
};

template <class T> __device__ __forceinline__ const T *at_ply(const jq_rows &r, int64_t b, int64_t t, int64_t h)
{
    return row_at<const T>(r, b, t, h);
}

__device__ __forceinline__ int live_plies(const SelectArgs &a, int b)
{
    return a.lengths ? min(max(a.lengths[b], 0), a.plies) : a.plies;
}

// Bit k: a game starts at ply t0 + k, k < 8.
__device__ __forceinline__ uint32_t starts_of(const SelectArgs &a, int b, int t0, int end, int lane)
{
    if (!a.starts) return 0;
    const int t = min(t0 + (lane & 7), end - 1);
    return __builtin_amdgcn_ballot_w64(a.starts[b * a.starts_batch + t * a.starts_ply] != 0) & 0xFF;
}

template <class T, int NS, bool EXACT, bool OUT>
__global__ __launch_bounds__(256) void k_scan_forward(SelectArgs a)
{
    extern __shared__ float lds[];   // more than one wave of states: [2][SG][SCAN_PLIES][64] shares of y
    const int SG = blockDim.x / 64, CW = a.waves * a.groups;
    const Place<T, NS> p(a, blockIdx.x % CW);
    float A[NS], h[NS];
    p.a2(a, [&](int i, float x) { A[i] = x; });
    const float skip = a.skip ? a.skip[p.ch] : 0.f, bias = a.bias ? a.bias[p.ch] : 0.f;
    const bool gated = OUT && a.gate.data;
    struct Raw { T u[SCAN_PLIES], delta[SCAN_PLIES], gate[SCAN_PLIES], b[SCAN_PLIES], c[SCAN_PLIES]; };
    const int64_t items = (int64_t)a.batch * a.segments;
    int turn = 0;
    for (int64_t item = blockIdx.x / CW; item < items; item += gridDim.x / CW) {
        const int b = item / a.segments, seg = item % a.segments;
        const int len = live_plies(a, b), begin = seg * a.seg_plies, stop = min(begin + a.seg_plies, a.plies);
        const int end = min(stop, len);
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            h[i] = 0.f;
            const int n = p.n0 + i;
            if (!OUT || n >= a.states) continue;
            if (seg) h[i] = a.seg_state[((int64_t)(b * (int64_t)a.segments + seg) * a.states + n) * a.channels + p.ch];
            else if (a.s_in) h[i] = a.s_in[((int64_t)b * a.channels + p.ch) * a.states + n];
        }
        float total = 0.f;
        auto fetch = [&](int t0, Raw &r) {
#pragma unroll
            for (int k = 0; k < SCAN_PLIES; ++k) {
                const int t = min(t0 + k, end - 1);
                r.u[k] = at_ply<T>(a.u, b, t, 0)[p.ch];
                r.delta[k] = at_ply<T>(a.delta, b, t, 0)[p.ch];
                if (gated) r.gate[k] = at_ply<T>(a.gate, b, t, 0)[p.ch];
                r.b[k] = r.c[k] = T(0.f);
                if (p.row_on) {
                    r.b[k] = at_ply<T>(a.b, b, t, p.group)[p.row_n];
                    if (OUT) r.c[k] = at_ply<T>(a.c, b, t, p.group)[p.row_n];
                }
            }
        };
        Raw next;
        uint32_t next_starts = 0;
        if (begin < end) {
            fetch(begin, next);
            next_starts = starts_of(a, b, begin, end, p.lane);
        }
        for (int t0 = begin; t0 < end; t0 += SCAN_PLIES) {
            const Raw r = next;
            const uint32_t starts = next_starts;
            if (t0 + SCAN_PLIES < end) {
                fetch(t0 + SCAN_PLIES, next);
                next_starts = starts_of(a, b, t0 + SCAN_PLIES, end, p.lane);
            }
            if (OUT && a.saved && t0 % SCAN_CHUNK == 0 && p.on) {
                const int chunks = (a.plies + SCAN_CHUNK - 1) / SCAN_CHUNK;
                float *to = a.saved + ((int64_t)b * chunks + t0 / SCAN_CHUNK) * a.states * a.channels + p.ch;
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    if (p.n0 + i < a.states) to[(int64_t)(p.n0 + i) * a.channels] = h[i];
            }
            float y[SCAN_PLIES];
#pragma unroll
            for (int k = 0; k < SCAN_PLIES; ++k) {
                y[k] = 0.f;
                if (t0 + k >= end) continue;
                const float u = (float)r.u[k], pre = (float)r.delta[k] + bias, dt = a.softplus ? softplus(pre) : pre;
                const float push = dt * u, bt = (float)r.b[k], ct = (float)r.c[k];
                if (starts >> k & 1) {
#pragma unroll
                    for (int i = 0; i < NS; ++i) h[i] = 0.f;
                    if (!OUT) total = __builtin_nanf("");
                }
                if (!OUT) total += dt;
                each_of<NS>([&](auto i) {
                    h[i] = fmaf(row_lane<i>(bt), push, exp2_fast(dt * A[i]) * h[i]);
                    if (!EXACT && p.n0 + i >= a.states) h[i] = 0.f;
                    if (OUT) y[k] = fmaf(row_lane<i>(ct), h[i], y[k]);
                });
            }
            if (!OUT) continue;
            if (SG > 1) {
                float *mine = lds + (turn & 1) * SG * SCAN_PLIES * 64;
#pragma unroll
                for (int k = 0; k < SCAN_PLIES; ++k) mine[(p.sg * SCAN_PLIES + k) * 64 + p.lane] = y[k];
                __syncthreads();
            }
#pragma unroll
            for (int k = 0; k < SCAN_PLIES; ++k) {
                if (t0 + k >= end) continue;
                if (SG > 1) {
                    if (k % SG != p.sg) continue;
                    const float *all = lds + (turn & 1) * SG * SCAN_PLIES * 64 + k * 64 + p.lane;
                    y[k] = 0.f;
                    for (int g = 0; g < SG; ++g) y[k] += all[g * SCAN_PLIES * 64];
                }
                float o = a.skip ? fmaf(skip, (float)r.u[k], y[k]) : y[k];
                if (gated) {
                    const float z = (float)r.gate[k];
                    o *= z * sigmoid(z);
                }
                if (p.on) row_at<T>(a.out, b, t0 + k, 0)[p.ch] = from_float<T>(o);
            }
            ++turn;   // the other buffer: the one before is read by then
        }
        if (OUT) {
            for (int t = max(begin, end) + p.sg; t < stop; t += SG)
                if (p.on) row_at<T>(a.out, b, t, 0)[p.ch] = T(0.f);
            if (a.s_out && seg == a.segments - 1 && p.on)
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    if (p.n0 + i < a.states) a.s_out[((int64_t)b * a.channels + p.ch) * a.states + p.n0 + i] = h[i];
        } else if (p.on) {
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (p.n0 + i < a.states) a.seg_state[(item * a.states + p.n0 + i) * a.channels + p.ch] = h[i];
            if (p.sg == 0) a.seg_sum[item * a.channels + p.ch] = total;
        }
    }
}

// What each part of a split axis adds becomes the state before it (BACK: the gradient
// behind it): one thread for each game, state and channel.
template <bool BACK>
__global__ __launch_bounds__(256) void k_scan_join(SelectArgs a)
{
    const int64_t all = (int64_t)a.batch * a.states * a.channels;
    const int64_t step = (int64_t)a.states * a.channels;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int ch = i % a.channels, n = i / a.channels % a.states;
        const int64_t b = i / step, home = ((int64_t)b * a.channels + ch) * a.states + n;
        const float *in = BACK ? a.d_final : a.s_in;
        float h = in ? in[home] : 0.f;
        const float A = a.a[(int64_t)ch * a.states + n] * LOG2E;
        for (int s = 0; s < a.segments; ++s) {
            const int64_t seg = b * a.segments + (BACK ? a.segments - 1 - s : s);
            float *at = a.seg_state + seg * step + (int64_t)n * a.channels + ch;
            const float add = *at, sum = a.seg_sum[seg * a.channels + ch];
            *at = h;
            // an infinity stays one over any number of plies: no power is 0
            h = sum != sum ? add : fmaf(fmaxf(exp2_fast(sum * A), 0x1p-126f), h, add);
        }
    }
}

// Backward over a part of the axis: what its gradients of y send to the state before it
// (seg_state, seg_sum), in reverse.
template <class T, int NS, bool EXACT>
__global__ __launch_bounds__(256) void k_scan_carry(SelectArgs a)
{
    const int CW = a.waves * a.groups;
    const Place<T, NS> p(a, blockIdx.x % CW);
    float A[NS], dh[NS];
    p.a2(a, [&](int i, float x) { A[i] = x; });
    const float bias = a.bias ? a.bias[p.ch] : 0.f;
    const int64_t items = (int64_t)a.batch * a.segments;
    for (int64_t item = blockIdx.x / CW; item < items; item += gridDim.x / CW) {
        const int b = item / a.segments, seg = item % a.segments;
        const int begin = seg * a.seg_plies, end = min(min(begin + a.seg_plies, a.plies), live_plies(a, b));
#pragma unroll
        for (int i = 0; i < NS; ++i) dh[i] = 0.f;
        float total = 0.f;
        for (int t0 = begin + (max(end - begin, 1) - 1) / 8 * 8; t0 >= begin && begin < end; t0 -= 8) {
            const uint32_t starts = starts_of(a, b, t0, end, p.lane);
            T delta[8], gate[8], d_out[8], c[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int t = min(t0 + k, end - 1);
                delta[k] = at_ply<T>(a.delta, b, t, 0)[p.ch];
                d_out[k] = at_ply<T>(a.d_out, b, t, 0)[p.ch];
                if (a.gate.data) gate[k] = at_ply<T>(a.gate, b, t, 0)[p.ch];
                c[k] = p.row_on ? at_ply<T>(a.c, b, t, p.group)[p.row_n] : T(0.f);
            }
#pragma unroll
            for (int k = 7; k >= 0; --k) {
                if (t0 + k >= end) continue;
                const float pre = (float)delta[k] + bias, dt = a.softplus ? softplus(pre) : pre, ct = (float)c[k];
                float dy = (float)d_out[k];
                if (a.gate.data) {
                    const float z = (float)gate[k];
                    dy *= z * sigmoid(z);
                }
                each_of<NS>([&](auto i) {
                    dh[i] = exp2_fast(dt * A[i]) * fmaf(row_lane<i>(ct), dy, dh[i]);
                    if (!EXACT && p.n0 + i >= a.states) dh[i] = 0.f;
                });
                total += dt;
                if (starts >> k & 1) {
#pragma unroll
                    for (int i = 0; i < NS; ++i) dh[i] = 0.f;
                    total = __builtin_nanf("");
                }
            }
        }
        if (!p.on) continue;
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (p.n0 + i < a.states) a.seg_state[(item * a.states + p.n0 + i) * a.channels + p.ch] = dh[i];
        if (p.sg == 0) a.seg_sum[item * a.channels + p.ch] = total;
    }
}

// Backward, chunks of 8 plies from the last one on: the states of a chunk again, from the
// saved one before it, into registers; then its gradients in reverse. With dh the gradient
// of h_t from all that follows:
//   dh += c dy;  db = sum over channels of dh dt u;  dc = sum over channels of dy h;
//   through = sum over n of b dh;  dh = exp(dt a) dh;  w = dh h_{t-1};  da += w dt;
//   du = dt through + skip dy;  ddt = u through + sum over n of w a
template <class T, int NS, bool EXACT>
__global__ __launch_bounds__(256) void k_scan_backward(SelectArgs a)
{
    extern __shared__ float lds[];   // more than one wave of states: [3][SG][8][64] shares of y, through and sum of w a
    constexpr int K = SCAN_CHUNK;
    const int SG = blockDim.x / 64, CW = a.waves * a.groups, cw = blockIdx.x % CW;
    const Place<T, NS> p(a, cw);
    const int part = blockIdx.x / CW;
    float A[NS], dA[NS], dh[NS], h[NS];
    p.a2(a, [&](int i, float x) { A[i] = x, dA[i] = 0.f; });
    const float skip = a.skip ? a.skip[p.ch] : 0.f, bias = a.bias ? a.bias[p.ch] : 0.f;
    float dskip = 0.f, dbias = 0.f;
    const bool gated = a.gate.data;
    const int chunks = (a.plies + K - 1) / K;
    const int64_t items = (int64_t)a.batch * a.segments;
    for (int64_t item = part; item < items; item += a.parts) {
        const int b = item / a.segments, seg = item % a.segments;
        const int begin = seg * a.seg_plies, stop = min(begin + a.seg_plies, a.plies), end = min(stop, live_plies(a, b));
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int n = p.n0 + i;
            dh[i] = 0.f;
            if (n >= a.states) continue;
            if (a.segments > 1) dh[i] = a.seg_state[(item * a.states + n) * a.channels + p.ch];
            else if (a.d_final) dh[i] = a.d_final[((int64_t)b * a.channels + p.ch) * a.states + n];
        }
        for (int t = max(begin, end) + p.sg; t < stop; t += SG) {
            if (!p.on) continue;
            if (a.du.data) row_at<T>(a.du, b, t, 0)[p.ch] = T(0.f);
            if (a.ddelta.data) row_at<T>(a.ddelta, b, t, 0)[p.ch] = T(0.f);
            if (a.dgate.data) row_at<T>(a.dgate, b, t, 0)[p.ch] = T(0.f);
        }
        for (int t0 = begin + (max(end - begin, 1) - 1) / K * K; t0 >= begin && begin < end; t0 -= K) {
            const uint32_t starts = starts_of(a, b, t0, end, p.lane);
            T u[K], delta[K], gate[K], d_out[K], bb[K], cc[K];
            float hist[K][NS], dt[K], dy[K], y[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int t = min(t0 + k, end - 1);
                u[k] = at_ply<T>(a.u, b, t, 0)[p.ch];
                delta[k] = at_ply<T>(a.delta, b, t, 0)[p.ch];
                d_out[k] = at_ply<T>(a.d_out, b, t, 0)[p.ch];
                if (gated) gate[k] = at_ply<T>(a.gate, b, t, 0)[p.ch];
                bb[k] = cc[k] = T(0.f);
                if (p.row_on) {
                    bb[k] = at_ply<T>(a.b, b, t, p.group)[p.row_n];
                    cc[k] = at_ply<T>(a.c, b, t, p.group)[p.row_n];
                }
            }
            const float *from = a.saved + ((int64_t)b * chunks + t0 / K) * a.states * a.channels + p.ch;
#pragma unroll
            for (int i = 0; i < NS; ++i) h[i] = p.n0 + i < a.states ? from[(int64_t)(p.n0 + i) * a.channels] : 0.f;
            float *bc = a.part_bc + ((((int64_t)(cw % a.waves) * a.batch + b) * a.plies + t0) * a.groups + p.group) * 2 * a.states;
            const int64_t bc_ply = (int64_t)a.groups * 2 * a.states;
            const int sum_n = p.n0 + p.lane / (64 / NS);
            const bool sum_on = p.lane % (64 / NS) == 0 && sum_n < a.states;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                y[k] = 0.f;
                if (t0 + k >= end) continue;
                const float pre = (float)delta[k] + bias, bt = (float)bb[k], ct = (float)cc[k];
                dt[k] = a.softplus ? softplus(pre) : pre;
                const float push = dt[k] * (float)u[k];
                dy[k] = (float)d_out[k];
                if (gated) dy[k] *= (float)gate[k] * sigmoid((float)gate[k]);
                if (starts >> k & 1)
#pragma unroll
                    for (int i = 0; i < NS; ++i) h[i] = 0.f;
                float q[NS];
                each_of<NS>([&](auto i) {
                    hist[k][i] = h[i];
                    h[i] = fmaf(row_lane<i>(bt), push, exp2_fast(dt[k] * A[i]) * h[i]);
                    if (!EXACT && p.n0 + i >= a.states) h[i] = 0.f;
                    y[k] = fmaf(row_lane<i>(ct), h[i], y[k]);
                    q[i] = EXACT || p.on ? dy[k] * h[i] : 0.f;
                });
                if (a.want_bc) {
                    const float s = lane_sums<NS>(q);
                    if (sum_on) bc[k * bc_ply + a.states + sum_n] = s;
                }
            }
            float s1[K], s2[K];
#pragma unroll
            for (int k = K - 1; k >= 0; --k) {
                s1[k] = s2[k] = 0.f;
                if (t0 + k >= end) continue;
                const float push = dt[k] * (float)u[k], bt = (float)bb[k], ct = (float)cc[k];
                const bool start = starts >> k & 1;
                float q[NS];
                each_of<NS>([&](auto i) {
                    dh[i] = fmaf(row_lane<i>(ct), dy[k], dh[i]);
                    if (!EXACT && p.n0 + i >= a.states) dh[i] = 0.f;
                    s1[k] = fmaf(row_lane<i>(bt), dh[i], s1[k]);
                    q[i] = EXACT || p.on ? dh[i] * push : 0.f;
                });
                if (a.want_bc) {
                    const float s = lane_sums<NS>(q);
                    if (sum_on) bc[k * bc_ply + sum_n] = s;
                }
                if (start) {
#pragma unroll
                    for (int i = 0; i < NS; ++i) dh[i] = 0.f;
                } else {
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        dh[i] *= exp2_fast(dt[k] * A[i]);
                        const float w = dh[i] * hist[k][i];
                        s2[k] = fmaf(w, A[i], s2[k]);
                        dA[i] = fmaf(w, dt[k], dA[i]);
                    }
                }
            }
            if (SG > 1) {
                __syncthreads();   // the shares of the chunk before have been read
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    lds[(p.sg * K + k) * 64 + p.lane] = y[k];
                    lds[((SG + p.sg) * K + k) * 64 + p.lane] = s1[k];
                    lds[((2 * SG + p.sg) * K + k) * 64 + p.lane] = s2[k];
                }
                __syncthreads();
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (t0 + k >= end || (SG > 1 && k % SG != p.sg)) continue;
                if (SG > 1) {
                    y[k] = s1[k] = s2[k] = 0.f;
                    for (int g = 0; g < SG; ++g) {
                        y[k] += lds[(g * K + k) * 64 + p.lane];
                        s1[k] += lds[((SG + g) * K + k) * 64 + p.lane];
                        s2[k] += lds[((2 * SG + g) * K + k) * 64 + p.lane];
                    }
                }
                const float uu = (float)u[k], pre = (float)delta[k] + bias;
                float d_pre = fmaf(s1[k], uu, s2[k] * LN2), d_u = s1[k] * dt[k];
                if (a.softplus) d_pre *= sigmoid(pre);
                if (a.skip) {
                    d_u = fmaf(skip, dy[k], d_u);
                    y[k] = fmaf(skip, uu, y[k]);
                    dskip = fmaf(dy[k], uu, dskip);
                }
                dbias += d_pre;
                if (!p.on) continue;
                if (a.du.data) row_at<T>(a.du, b, t0 + k, 0)[p.ch] = from_float<T>(d_u);
                if (a.ddelta.data) row_at<T>(a.ddelta, b, t0 + k, 0)[p.ch] = from_float<T>(d_pre);
                if (a.dgate.data) {
                    const float z = (float)gate[k], s = sigmoid(z);
                    row_at<T>(a.dgate, b, t0 + k, 0)[p.ch] = from_float<T>((float)d_out[k] * y[k] * s * fmaf(z, 1.f - s, 1.f));
                }
            }
        }
        if (a.d_initial && seg == 0 && p.on)
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (p.n0 + i < a.states) a.d_initial[((int64_t)b * a.channels + p.ch) * a.states + p.n0 + i] = dh[i];
    }
    if (!a.want_a) return;
    float *to = a.part_a + (int64_t)part * (a.states + 2) * a.channels + p.ch;
    if (SG > 1) {   // each wave has some plies' share of dskip and dbias
        __syncthreads();
        lds[p.sg * 64 + p.lane] = dskip;
        lds[(SG + p.sg) * 64 + p.lane] = dbias;
        __syncthreads();
        dskip = dbias = 0.f;
        for (int g = 0; g < SG; ++g) {
            dskip += lds[g * 64 + p.lane];
            dbias += lds[(SG + g) * 64 + p.lane];
        }
    }
    if (!p.on) return;
#pragma unroll
    for (int i = 0; i < NS; ++i)
        if (p.n0 + i < a.states) to[(int64_t)(p.n0 + i) * a.channels] = dA[i];
    if (p.sg == 0) {
        to[(int64_t)a.states * a.channels] = dskip;
        to[(int64_t)(a.states + 1) * a.channels] = dbias;
    }
}

// db and dc: the waves' shares summed in a fixed order; 0 from a game's length on.
template <class T>
__global__ __launch_bounds__(256) void k_scan_join_bc(SelectArgs a, jq_rows db, jq_rows dc)
{
    const int n2 = 2 * a.states;
    const int64_t tokens = (int64_t)a.batch * a.plies, all = tokens * a.groups * n2;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int j = i % n2, g = i / n2 % a.groups;
        const int64_t token = i / n2 / a.groups, b = token / a.plies;
        const int t = token % a.plies;
        float s = 0.f;
        if (t < live_plies(a, b))
            for (int w = 0; w < a.waves; ++w) s += a.part_bc[w * all + i];
        const jq_rows &r = j < a.states ? db : dc;
        if (r.data) row_at<T>(r, b, t, g)[j < a.states ? j : j - a.states] = from_float<T>(s);
    }
}

// da (channels, states), dskip and dbias: the blocks' shares summed in a fixed order, 16
// columns and 16 parts of the sum a block.
__global__ __launch_bounds__(256) void k_scan_join_a(SelectArgs a, float *da, float *dskip, float *dbias)
{
    __shared__ float red[16][17];
    const int64_t cols = (int64_t)(a.states + 2) * a.channels, col = (int64_t)blockIdx.x * 16 + threadIdx.x % 16;
    const int slice = threadIdx.x / 16;
    float s = 0.f;
    if (col < cols)
        for (int q = slice; q < a.parts; q += 16) s += a.part_a[q * cols + col];
    red[slice][threadIdx.x % 16] = s;
    __syncthreads();
    if (slice || col >= cols) return;
    s = 0.f;
    for (int q = 0; q < 16; ++q) s += red[q][threadIdx.x];
    const int n = col / a.channels, ch = col % a.channels;
    if (n < a.states) {
        if (da) da[(int64_t)ch * a.states + n] = s;
    } else {
        float *to = n == a.states ? dskip : dbias;
        if (to) to[ch] = s;
    }
}

// ------------------------------------------------------------------ one ply
struct SelectStepArgs {
    jq_rows u, delta, gate, b, c, out;
    int batch, channels, states, groups, per;
    bool softplus;
    const float *a, *skip, *bias;
    float *state;
    int64_t state_rows;
    const int64_t *rows;
    const uint8_t *starts;
};

// L lanes a channel, four states each: a wave walks games with its channels' a in
// registers, so what it moves is the states.
template <class T, int L>
__global__ __launch_bounds__(256) void k_scan_step(SelectStepArgs a, int channel_waves, int at_once)
{
    constexpr int PER = 64 / L;
    typedef f32x4 At __attribute__((aligned(4)));
    const int lane = threadIdx.x % 64;
    const int64_t wave = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (wave >= (int64_t)channel_waves * at_once) return;
    const int cw = wave % channel_waves;
    const int ch = cw * PER + lane / L, n = lane % L * 4, left = min(a.states - n, 4);
    const bool on = ch < a.channels, mine = on && left > 0;
    const int at = on ? ch : 0, group = at / a.per;
    float A[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) A[e] = mine && e < left ? a.a[(int64_t)at * a.states + n + e] * LOG2E : 0.f;
    const float skip = a.skip ? a.skip[at] : 0.f, bias = a.bias ? a.bias[at] : 0.f;
    for (int64_t game = wave / channel_waves; game < a.batch; game += at_once) {
        const int64_t row = a.rows ? a.rows[game] : game;
        if (row < 0 || row >= a.state_rows) {
            if (on && n == 0) row_at<T>(a.out, game, 0, 0)[ch] = T(0.f);
            continue;
        }
        float *s = a.state + (row * a.channels + at) * a.states + n;
        const bool start = a.starts && a.starts[game];
        float h[4], bt[4], ct[4];
        const T *pb = row_at<const T>(a.b, game, 0, group) + n, *pc = row_at<const T>(a.c, game, 0, group) + n;
        if (left >= 4) {
            const f32x4 v = *reinterpret_cast<const At *>(s);
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = v[e], bt[e] = (float)pb[e], ct[e] = (float)pc[e];
        } else
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool there = e < left;
                h[e] = there ? s[e] : 0.f;
                bt[e] = there ? (float)pb[e] : 0.f;
                ct[e] = there ? (float)pc[e] : 0.f;
            }
        const float u = (float)row_at<const T>(a.u, game, 0, 0)[at], pre = (float)row_at<const T>(a.delta, game, 0, 0)[at] + bias;
        const float dt = a.softplus ? softplus(pre) : pre, push = dt * u;
        float y = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float old = start ? 0.f : exp2_fast(dt * A[e]) * h[e];
            h[e] = fmaf(bt[e], push, old);
            if (e < left) y = fmaf(ct[e], h[e], y);
        }
        if (mine) {
            if (left >= 4) *reinterpret_cast<At *>(s) = At{h[0], h[1], h[2], h[3]};
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < left) s[e] = h[e];
        }
        y = group_total<L>(y);
        if (a.skip) y = fmaf(skip, u, y);
        if (a.gate.data) {
            const float z = (float)row_at<const T>(a.gate, game, 0, 0)[at];
            y *= z * sigmoid(z);
        }
        if (on && n == 0) row_at<T>(a.out, game, 0, 0)[ch] = from_float<T>(y);
    }
}

}  // namespace jq
