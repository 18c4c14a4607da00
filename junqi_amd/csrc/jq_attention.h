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
//
// A chunk of plies a .. a + n at a time, with P_ij = lambda^(i - j) q_i.k_j for the
// plies j <= i that i sees (in reverse: j >= i, lambda^(j - i)):
//   o_i = out_scale (in_scale sum_j P_ij v_j + lambda^(i - a + 1) q_i S)
//   S  <- lambda^n S + in_scale sum_j lambda^(a + n - 1 - j) k_j v_j^T
// with the state's term left out where a game starts in between.
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
    // a long axis is split into segments of seg_plies (whole chunks) that run side by
    // side: seg_states[(b, h)][g] (kd, vd) is the state before segment g, seg_carry
    // what a segment leaves of it
    int segments, seg_plies;
    float *seg_states, *seg_carry;
    int seg_row, seg_col;              // strides of a seg_states' element
    bool stream;                       // the rows go past the caches
};

// ---- products of 16 x 16 tiles -------------------------------------------------
// A product takes two fragments: lane l holds row (or column) l % 16 and, with
// g = l / 16, the depths that its e-th elements stand for. The result has column
// l % 16 and rows 4g .. 4g + 3 in lane l. Depths may be taken in any order that
// both fragments share; here it is the order in which a result's rows lie in its
// lanes (depth), so that the state and P go from result to operand without leaving
// their registers.
template <class T> struct Mma;

template <> struct Mma<bf16> {
    typedef bf16x8 Frag;
    static constexpr int KB = 32;   // depth of a fragment
    static __device__ __forceinline__ f32x4 mul(Frag a, Frag b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ int depth(int g, int e) { return 16 * (e >> 2) + 4 * g + (e & 3); }
    // depths = elements p[0 .. KB) of this lane's row
    static __device__ __forceinline__ Frag row(const bf16 *p, int g)
    {
        const bf16x4 x = *reinterpret_cast<const bf16x4 *>(p + 4 * g), y = *reinterpret_cast<const bf16x4 *>(p + 16 + 4 * g);
        return Frag{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    }
    // depths = rows p[0 .. KB) of stride ld, this lane's column l % 16: each 16 lanes
    // read a 4 x 16 block with its columns turned to the lanes
    static __device__ __forceinline__ Frag col(const bf16 *p, int ld, int l)
    {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
        const bf16 *at = p + (l >> 2) * ld + 4 * (l & 3);
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)at);
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + 16 * ld));
        return __builtin_bit_cast(Frag, s16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]});
    }
    // x as a sum of N terms: 8 bits each
    template <int N> static __device__ __forceinline__ void split(const float (&x)[8], Frag (&part)[N])
    {
        // (-1, 0) and (0, -1) from registers: as an operand's inline constant, -1 lands in the other half
        uint32_t first = 0x0000BF80u, second = 0xBF800000u;
        asm("" : "+s"(first), "+s"(second));
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            float a = x[e], b = x[e + 1];
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const bf16x2 h{(bf16)a, (bf16)b};
                part[u][e] = h[0];
                part[u][e + 1] = h[1];
                if (u + 1 < N) {   // what is left: exact
                    a = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, first), a, false);
                    b = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, second), b, false);
                }
            }
        }
    }
};

template <> struct Mma<float> {
    typedef f32x4 Frag;
    static constexpr int KB = 16;
    static __device__ __forceinline__ f32x4 mul(Frag a, Frag b, f32x4 c)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ int depth(int g, int e) { return 4 * g + e; }
    static __device__ __forceinline__ Frag row(const float *p, int g) { return *reinterpret_cast<const Frag *>(p + 4 * g); }
    static __device__ __forceinline__ Frag col(const float *p, int ld, int l)
    {
        const float *at = p + 4 * (l >> 4) * ld + (l & 15);
        return Frag{at[0], at[ld], at[2 * ld], at[3 * ld]};
    }
    template <int N> static __device__ __forceinline__ void split(const float (&x)[4], Frag (&part)[N])
    {
        part[0] = Frag{x[0], x[1], x[2], x[3]};
    }
};

// Terms that a float32 operand is split into. In bfloat16, three hold all of a
// float32: sums that come out in float32, the states. Two hold 16 bits: operands (P,
// and the state where it is read) of sums that are rounded to bfloat16, 8 bits. Against
// the definition in 64 bits these outputs are off by 1.66e-3 in the mean, as much as
// its own rounding to bfloat16, with two terms and with three, which take 8 % longer
// (training 1,024 x 256 plies 559 -> 599 us, two records of 65,537 plies 540 -> 594).
// One term for P is off by 1.8e-3 to 2.4e-3; two cost nothing where the card is full, and
// what their products take where each wave waits for its own chunk alone (512 heads of 64
// over 1,024 plies 81 -> 87 us, 4,096 plies 297 -> 333).
template <class T, int N> constexpr int PARTS = sizeof(T) == 2 ? N : 1;

// log2 lambda, and lambda^d from it: lambda = 0 has a logarithm whose products with
// whole numbers are finite, so that lambda^0 is 1.
__device__ __forceinline__ float log2_lambda(float log_decay)
{
    const float x = log_decay * 1.44269504088896340736f;
    return x < -1e30f ? -1e30f : x;
}
__device__ __forceinline__ float power(float log2_lam, int d) { return __builtin_amdgcn_exp2f(log2_lam * (float)d); }

// Four elements of a result in T.
__device__ __forceinline__ void store4(bf16 *p, f32x4 x)
{
    *reinterpret_cast<bf16x4 *>(p) = bf16x4{(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]};
}
__device__ __forceinline__ void store4(float *p, f32x4 x) { *reinterpret_cast<f32x4 *>(p) = x; }

// The games of a chunk of n plies: bit i of `starts` where one starts at ply i. The
// same in all lanes.
struct Games {
    uint32_t starts;
    int n;
    static __device__ __forceinline__ uint32_t upto(int i) { return (2u << i) - 1; }   // plies 0 .. i
    __device__ __forceinline__ bool from_begin(int i) const { return i < n && !(starts & upto(i)); }   // i sees the begin
    __device__ __forceinline__ bool to_end(int i) const { return i < n && !(starts & ~upto(i)); }      // the end sees i
    __device__ __forceinline__ bool same(int i, int j) const { return !(starts & upto(i) & ~upto(j)); }   // j <= i
};

// A wave's part of a pass for heads of D elements: the state's columns c0 .. c0 + CW
// in registers, and all that has those columns. Chunks have the depth of one
// fragment, and each wave computes P for itself, so that P goes from its product's
// registers into the next product as an operand and the waves of a head exchange
// nothing but its tiles in LDS. One wave for heads up to 32, two up to 64; eight for
// heads of 128, whose state would otherwise leave no registers for the rows on their
// way (four waves: 256 registers and spills, 575 us against 504 for the outputs of
// 2 x 65,537 plies of 8 heads). Chunks of 64 plies, P shared through LDS by four
// waves of 16 columns each, took 185 us for the outputs of 1,024 x 256 plies of 4 heads
// of 64 in bfloat16 (165 now), and the gradients of k and v 338 (291): three barriers
// and twice the LDS traffic a chunk. With P of one term, 160 us, the same loads, stores
// and barriers without the products took 150, the products without the loads 140: memory
// and issue are balanced (VALU 46 % busy, MFMA 18 %, LDS 22 %).
constexpr int pass_waves(int dim) { return dim == 128 ? 8 : dim / 32; }
template <class T, int D, bool REV>
struct Chunk {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    static constexpr int WAVES = pass_waves(D), CW = D / WAVES;
    static constexpr int KB = M::KB, CH = KB, NT = CH / 16, KT = D / 16, CT = CW / 16, FE = KB / 4;
    static constexpr int LD = D + Vec<T>::N;   // 16 bytes of padding turn a tile's rows over the banks

    f32x4 s[KT][CT];   // state (16t + 4g + r, c0 + 16c + l % 16)
    float g2;          // log2 lambda
    float in_scale, out_scale;
    int l, lc, g, c0;
    // of a whole chunk in which no game starts: lambda's powers with their scales, for
    // P's tiles u tiles beside the diagonal (0 where a ply is not seen), for what a ply
    // sees of the state before, and for what is left of it after
    f32x4 apart[NT];
    float sees[NT], left[FE];

    __device__ __forceinline__ Chunk(float log_decay, float in_scale_, float out_scale_, int wave)
        : g2(log2_lambda(log_decay)), in_scale(in_scale_), out_scale(out_scale_), l(threadIdx.x & 63), lc(l & 15), g(l >> 4), c0(wave * CW)
    {
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 16 * u + (REV ? 4 * g + r - lc : lc - 4 * g - r);
                apart[u][r] = d >= 0 ? in_scale * out_scale * power(g2, d) : 0.f;
            }
        const Games gm{0, CH};
        reach(gm, lc, g, sees, left);
    }

    // what the plies of a chunk see of the state before it, and what is left of them after
    __device__ __forceinline__ void reach(const Games &gm, int lc, int g, float (&see)[NT], float (&leave)[FE]) const
    {
#pragma unroll
        for (int it = 0; it < NT; ++it) {
            const int i = 16 * it + lc;
            const float f = out_scale * power(g2, REV ? gm.n - 1 - i : i + 1);
            see[it] = (REV ? gm.to_end(i) : gm.from_begin(i)) ? f : 0.f;
        }
#pragma unroll
        for (int e = 0; e < FE; ++e) {
            const int j = M::depth(g, e);
            const float f = in_scale * power(g2, REV ? j + 1 : gm.n - 1 - j);
            leave[e] = (REV ? gm.from_begin(j) : gm.to_end(j)) ? f : 0.f;
        }
    }

    // f(t, c, r, offset) for this lane's part of a (rows, cols) state
    template <class F>
    __device__ __forceinline__ void each(int rows, int cols, int s_row, int s_col, F &&f)
    {
        int i0 = 4 * g, j0 = c0 + lc;
        asm("" : "+v"(i0), "+v"(j0));   // the offsets are made where they are used, not kept over the pass
#pragma unroll
        for (int c = 0; c < CT; ++c)
            if (j0 + 16 * c < cols)
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (i0 + 16 * t + r < rows) f(t, c, r, (i0 + 16 * t + r) * s_row + (j0 + 16 * c) * s_col);
    }
    __device__ __forceinline__ void load_state(const float *p, int rows, int cols, int s_row, int s_col)
    {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int c = 0; c < CT; ++c) s[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (p) each(rows, cols, s_row, s_col, [&](int t, int c, int r, int at) { s[t][c][r] = p[at]; });
    }
    __device__ __forceinline__ void store_state(float *p, int rows, int cols, int s_row, int s_col)
    {
        each(rows, cols, s_row, s_col, [&](int t, int c, int r, int at) { p[at] = s[t][c][r]; });
    }

    // o[c][it] (rows: value columns c0 + 16c .., column: ply 16it + l % 16) = the
    // chunk's outputs (OUT), and the state after it, from its tiles in LDS.
    template <bool OUT>
    __device__ __forceinline__ void run(const T *q, const T *k, const T *v, const Games &gm, f32x4 (&o)[CT][NT])
    {
        float see[NT], leave[FE];
#pragma unroll
        for (int it = 0; it < NT; ++it) see[it] = sees[it];
#pragma unroll
        for (int e = 0; e < FE; ++e) leave[e] = left[e];
        const bool whole = !gm.starts && gm.n == CH;
        if (!whole) {
            int lc_ = lc, g_ = g;
            asm volatile("" : "+v"(lc_), "+v"(g_));   // made here, not kept over the pass for chunks that are few
            reach(gm, lc_, g_, see, leave);
        }
        Frag p[NT][PARTS<T, 2>];
        if constexpr (OUT) {
            // P's products, and what the state before the chunk answers, a depth of q at a time
            f32x4 acc[NT][NT];   // [it][jt]
#pragma unroll
            for (int it = 0; it < NT; ++it) {
#pragma unroll
                for (int jt = 0; jt < NT; ++jt) acc[it][jt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < CT; ++c) o[c][it] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int d = 0; d < D / KB; ++d) {
                Frag x[NT];
#pragma unroll
                for (int it = 0; it < NT; ++it) x[it] = M::row(q + (16 * it + lc) * LD + d * KB, g);
#pragma unroll
                for (int jt = 0; jt < NT; ++jt) {
                    const Frag y = M::row(k + (16 * jt + lc) * LD + d * KB, g);
#pragma unroll
                    for (int it = 0; it < NT; ++it)
                        if (REV ? jt >= it : jt <= it) acc[it][jt] = M::mul(y, x[it], acc[it][jt]);
                }
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    constexpr int N = PARTS<T, 2>;
                    Frag part[N];
                    float y[FE];
#pragma unroll
                    for (int e = 0; e < FE; ++e) y[e] = s[(d * KB + 4 * e) / 16][c][e & 3];
                    M::template split<N>(y, part);
#pragma unroll
                    for (int u = 0; u < N; ++u)   // no product waits for the one just before it
#pragma unroll
                        for (int it = 0; it < NT; ++it) o[c][it] = M::mul(part[u], x[it], o[c][it]);
                }
            }
            weigh(acc, gm, p);
            if (!whole) {   // a state that is not seen may hold NaN
                int lc_ = lc;
                asm volatile("" : "+v"(lc_));
#pragma unroll
                for (int it = 0; it < NT; ++it) {
                    const bool on = REV ? gm.to_end(16 * it + lc_) : gm.from_begin(16 * it + lc_);
#pragma unroll
                    for (int c = 0; c < CT; ++c)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[c][it][r] = on ? o[c][it][r] : 0.f;
                }
            }
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int it = 0; it < NT; ++it)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[c][it][r] *= see[it];
        }
        if (gm.starts) {   // nothing is left of the state
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int c = 0; c < CT; ++c) s[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
        } else {
            const float carry = power(g2, gm.n);
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[t][c][r] *= carry;
        }
        Frag x[CT], part[CT][PARTS<T, 3>];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            x[c] = M::col(v + c0 + 16 * c, LD, l);
            float y[FE];
#pragma unroll
            for (int e = 0; e < FE; ++e) y[e] = (float)x[c][e] * leave[e];
            M::template split<PARTS<T, 3>>(y, part[c]);
        }
#pragma unroll
        for (int t = 0; t < KT; t += 2) {
            const Frag z0 = M::col(k + 16 * t, LD, l), z1 = M::col(k + 16 * t + 16, LD, l);
#pragma unroll
            for (int u = 0; u < PARTS<T, 3>; ++u)
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    s[t][c] = M::mul(z0, part[c][u], s[t][c]);
                    s[t + 1][c] = M::mul(z1, part[c][u], s[t + 1][c]);
                }
        }
        if constexpr (OUT)
#pragma unroll
            for (int u = 0; u < PARTS<T, 2>; ++u)
#pragma unroll
                for (int it = 0; it < NT; ++it)
#pragma unroll
                    for (int c = 0; c < CT; ++c) o[c][it] = M::mul(x[c], p[it][u], o[c][it]);
    }

    // p[it] = P's columns i = 16it + l % 16 as an operand over the plies j, times the
    // scales, from its products.
    __device__ __forceinline__ void weigh(f32x4 (&acc)[NT][NT], const Games &gm, Frag (&p)[NT][PARTS<T, 2>]) const
    {
        // a ply that is not seen leaves 0, whatever its product is
#pragma unroll
        for (int it = 0; it < NT; ++it)
#pragma unroll
            for (int jt = 0; jt < NT; ++jt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int u = REV ? jt - it : it - jt;
                    float y = 0.f;
                    if (u >= 0) {
                        y = acc[it][jt][r] * apart[u < 0 ? 0 : u][r];
                        if (u == 0) y = (REV ? 4 * g + r >= lc : lc >= 4 * g + r) ? y : 0.f;
                    }
                    acc[it][jt][r] = y;
                }
        if (gm.starts) {
            int lc_ = lc, g_ = g;
            asm volatile("" : "+v"(lc_), "+v"(g_));
#pragma unroll
            for (int it = 0; it < NT; ++it)
#pragma unroll
                for (int jt = 0; jt < NT; ++jt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int i = 16 * it + lc_, j = 16 * jt + 4 * g_ + r;
                        acc[it][jt][r] = (REV ? gm.same(j, i) : gm.same(i, j)) ? acc[it][jt][r] : 0.f;
                    }
        }
#pragma unroll
        for (int it = 0; it < NT; ++it) {
            float y[FE];
#pragma unroll
            for (int e = 0; e < FE; ++e) y[e] = acc[it][e >> 2][e & 3];
            M::template split<PARTS<T, 2>>(y, p[it]);
        }
    }

    // whether an element of this wave's part of the state is infinite
    __device__ __forceinline__ bool infinite() const
    {
        float m = 0.f;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) m = fmaxf(m, fabsf(s[t][c][r]));
        return __ballot(m == __builtin_inff()) != 0;
    }

    // The chunk ply by ply as the definition says, for tiles with infinities or NaN (a
    // product with 0 in their place is not 0, and a ply must get nothing of those it does
    // not see) and for states with infinities (which are no sum of two terms, and whose
    // product with a power that has become 0 is not 0).
    // put(i, c, x): x = value column c0 + 16c + l % 16 of ply i.
    template <class F>
    __device__ __forceinline__ void singly(const T *q, const T *k, const T *v, const Games &gm, int rows, int cols, F &&put)
    {
        const float lam = power(g2, 1);
        for (int m = 0; m < gm.n; ++m) {
            const int i = REV ? gm.n - 1 - m : m;
            const bool start = (gm.starts >> i) & 1;
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const float x = in_scale * (float)v[i * LD + c0 + 16 * c + lc];
                float o = 0.f;
                // beside the state's elements nothing is added: 0 times an infinity is not 0
                int own = c0 + 16 * c + lc < cols ? rows - 4 * g : 0;
                asm volatile("" : "+v"(own));   // compared here, the results not kept over the pass: 5 % of its time
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int at = i * LD + 16 * t + 4 * g + r;
                        float y = s[t][c][r];
                        if (!REV) y = start ? 0.f : lam * y;
                        if (16 * t + r < own) y += (float)k[at] * x;
                        o += (float)q[at] * y;
                        if (REV) y = start ? 0.f : lam * y;
                        s[t][c][r] = y;
                    }
                o += __shfl_xor(o, 16);
                o += __shfl_xor(o, 32);
                put(i, c, out_scale * o);
            }
        }
    }
};

// sum + 0 for finite elements, NaN where one is infinite or NaN.
__device__ __forceinline__ float probe(bf16x8 x, float sum)
{
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        sum = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{x[i], x[i + 1]}, bf16x2{bf16(0.f), bf16(0.f)}, sum, false);
    return sum;
}
__device__ __forceinline__ float probe(f32x4 x, float sum)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = fmaf(x[i], 0.f, sum);
    return sum;
}

// Waves of a block that share its tiles wait for each other; a wave alone only keeps
// its own order.
template <int WAVES>
__device__ __forceinline__ void meet()
{
    if constexpr (WAVES > 1) __syncthreads();
    else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// Rows of one game and head that a block of THREADS reads or writes, a chunk of
// plies at a time. FAST: through a buffer descriptor of the chunk's plies, whose
// bounds give zeros for (and drop) rows past the chunk's end without a branch; rows
// are whole aligned 16-byte vectors and a chunk spans less than 2 GiB (the host's
// check). Otherwise element by element.
template <class T, int D, int THREADS, bool FAST>
struct Plies {
    using V = typename Vec<T>::type;
    static constexpr int N = Vec<T>::N, PER_ROW = D / N, CH = Mma<T>::KB, LD = D + N;
    static constexpr int NV = CH * PER_ROW / THREADS, ROWS = THREADS / PER_ROW;   // vectors of a thread, ROWS rows apart
    static_assert(NV * ROWS == CH, "a tile is NV vectors a thread");
    T *base;
    int64_t ply;
    int dim;
    bool stream;   // past the caches

    static __device__ __forceinline__ int me() { return threadIdx.x % THREADS; }   // a block's halves read different tiles

    __device__ __forceinline__ Plies(const jq_rows &r, int b, int h, int dim_, bool stream_)
        : base(row_at<T>(r, b, 0, h)), ply(r.ply), dim(dim_), stream(stream_)
    {
    }

    __device__ __forceinline__ __amdgpu_buffer_rsrc_t chunk(int t0, int n) const
    {
        return __builtin_amdgcn_make_buffer_rsrc(base + t0 * ply, 0, (int)(((n - 1) * ply + dim) * sizeof(T)), 0x00020000);
    }
    // byte offset of this thread's first vector in a chunk; past any bound where it is beside the row
    __device__ __forceinline__ int first() const
    {
        const int row = me() / PER_ROW, c = me() % PER_ROW * N;
        return c < dim ? (row * (int)ply + c) * (int)sizeof(T) : INT32_MIN;
    }
    __device__ __forceinline__ int step() const { return me() % PER_ROW * N < dim ? ROWS * (int)ply * (int)sizeof(T) : 0; }

    // this thread's vectors of the tile of plies t0 .. t0 + n; zeros elsewhere
    __device__ __forceinline__ void load(int t0, int n, V (&x)[NV]) const
    {
        if constexpr (FAST) {
            const __amdgpu_buffer_rsrc_t r = chunk(t0, n);
            int at = first();
            const int by = step();
            if (stream)
#pragma unroll
                for (int u = 0; u < NV; ++u, at += by)
                    x[u] = __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 2));
            else
#pragma unroll
                for (int u = 0; u < NV; ++u, at += by)
                    x[u] = __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
        } else {
            const int row = me() / PER_ROW, c = me() % PER_ROW * N;
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                x[u] = V{};
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (row + u * ROWS < n && c + e < dim) x[u][e] = base[(t0 + row + u * ROWS) * ply + c + e];
            }
        }
    }
    // a tile in LDS out to plies t0 .. t0 + n
    __device__ __forceinline__ void store(int t0, int n, const T *lds) const
    {
        const T *p = lds + me() / PER_ROW * LD + me() % PER_ROW * N;
        if constexpr (FAST) {
            const __amdgpu_buffer_rsrc_t r = chunk(t0, n);
            int at = first();
            const int by = step();
            V y[NV];
#pragma unroll
            for (int u = 0; u < NV; ++u) y[u] = *reinterpret_cast<const V *>(p + u * ROWS * LD);
            if (stream)
#pragma unroll
                for (int u = 0; u < NV; ++u, at += by)
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y[u]), r, at, 0, 2);
            else
#pragma unroll
                for (int u = 0; u < NV; ++u, at += by)
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y[u]), r, at, 0, 0);
        } else {
            const int row = me() / PER_ROW, c = me() % PER_ROW * N;
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (row + u * ROWS < n && c + e < dim) base[(t0 + row + u * ROWS) * ply + c + e] = p[u * ROWS * LD + e];
        }
    }
    // zeros from ply t0 to t1
    __device__ __forceinline__ void clear(int t0, int t1) const
    {
        for (int t = t0 + me() / 64; t < t1; t += THREADS / 64)
            for (int c = me() % 64; c < dim; c += 64) base[t * ply + c] = from_float<T>(0.f);
    }
    // a thread's vectors of a tile into LDS
    static __device__ __forceinline__ void stage(T *lds, const V (&x)[NV])
    {
        T *p = lds + me() / PER_ROW * LD + me() % PER_ROW * N;
#pragma unroll
        for (int u = 0; u < NV; ++u) *reinterpret_cast<V *>(p + u * ROWS * LD) = x[u];
    }
    static __device__ __forceinline__ float probe_all(const V (&x)[NV])
    {
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < NV; ++u) sum = probe(x[u], sum);
        return sum;
    }
};

// The plies of one segment of one game and head.
struct Segment {
    int b, h, seg, s0, s1, end, chunks;   // s0 .. s1 of all plies, s0 .. end of the game's
    __device__ __forceinline__ Segment(const ScanArgs &a, int seg_, int ch) : b(blockIdx.x / a.heads), h(blockIdx.x % a.heads), seg(seg_)
    {
        const int len = a.lengths ? min(max(a.lengths[b], 0), a.plies) : a.plies;
        s0 = seg * a.seg_plies;
        s1 = a.plies - s0 > a.seg_plies ? s0 + a.seg_plies : a.plies;
        end = max(s0, min(s1, len));
        chunks = (end - s0 + ch - 1) / ch;
    }
};

// A pass over one segment of one game and head by one block: chunks in turn, the
// state in registers; every row is read and written once. 670 MB (1,024 x 256 plies of
// 4 heads of 64 in bfloat16 with their states) in 165 us: 4.1 TB/s, where a plain copy
// reaches 6.0. While a chunk is worked on, the next one's rows are on their way (of two
// chunks: no faster). OUT: the plies' outputs, from the state before the segment; else only the
// state that the segment's own plies leave, for the states before the others.
template <class T, int D, bool REV, bool FAST, bool OUT>
__global__ __launch_bounds__(64 * pass_waves(D), 2) void k_attention_pass(ScanArgs a)
{
    using C = Chunk<T, D, REV>;
    constexpr int CH = C::CH, LD = C::LD, WAVES = C::WAVES;
    using P = Plies<T, D, 64 * WAVES, FAST>;
    using V = typename P::V;
    __shared__ __align__(16) T qs[OUT ? CH * LD : 1], ks[CH * LD], vs[CH * LD];
    __shared__ int bad[2];
    const Segment sg(a, blockIdx.y + (!OUT && REV ? 1 : 0), CH);   // the last segment's own state goes nowhere
    C ch(a.log_decay[sg.h], a.in_scale, a.out_scale, WAVES > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
    const int64_t size = (int64_t)a.kd * a.vd;
    float *slot = a.seg_states + ((int64_t)blockIdx.x * a.segments + sg.seg) * size;
    if (!OUT) ch.load_state(nullptr, 0, 0, 0, 0);
    else if (a.segments > 1) ch.load_state(slot, a.kd, a.vd, a.seg_row, a.seg_col);
    else ch.load_state(a.s_in ? a.s_in + blockIdx.x * size : nullptr, a.kd, a.vd, a.s_row, a.s_col);
    const P q(a.q, sg.b, sg.h, a.kd, a.stream), k(a.k, sg.b, sg.h, a.kd, a.stream), v(a.v, sg.b, sg.h, a.vd, a.stream), o(a.o, sg.b, sg.h, a.vd, a.stream);
    const uint8_t *starts = a.starts ? a.starts + sg.b * a.starts_batch : nullptr;
    bool wild = ch.infinite();
    if (WAVES > 1) {
        if (threadIdx.x < 2) bad[threadIdx.x] = 0;
        meet<WAVES>();
    }

    V qt[P::NV], kt[P::NV], vt[P::NV];
    bool start = false, any_start = false;
    const auto begin = [&](int m) { return sg.s0 + (REV ? sg.chunks - 1 - m : m) * CH; };
    const auto fetch = [&](int m) {
        const int t0 = begin(m), n = min(CH, sg.end - t0);
        start = starts && ch.l < n && starts[(t0 + ch.l) * a.starts_ply];
        if (OUT) q.load(t0, n, qt);
        k.load(t0, n, kt);
        v.load(t0, n, vt);
    };
    if (sg.chunks) fetch(0);
    for (int m = 0; m < sg.chunks; ++m) {
        const int t0 = begin(m);
        const Games gm{(uint32_t)__ballot(start), min(CH, sg.end - t0)};
        any_start |= gm.starts != 0;
        if (OUT) P::stage(qs, qt);
        P::stage(ks, kt);
        P::stage(vs, vt);
        float sum = P::probe_all(kt) + P::probe_all(vt);
        if (OUT) sum += P::probe_all(qt);
        bool singly = wild || __ballot(sum != sum) != 0;
        if (WAVES > 1 && singly) bad[m & 1] = 1;
        meet<WAVES>();
        if (WAVES > 1) {
            singly = bad[m & 1];
            if (threadIdx.x == 0) bad[(m + 1) & 1] = 0;
        }
        if (m + 1 < sg.chunks) fetch(m + 1);
        f32x4 acc[C::CT][C::NT];
        if (singly) {
            meet<WAVES>();   // bad is read
            ch.singly(OUT ? qs : ks, ks, vs, gm, a.kd, a.vd, [&](int i, int c, float x) {
                const int j = ch.c0 + 16 * c + ch.lc;
                if (OUT && ch.g == 0 && j < a.vd) o.base[(t0 + i) * o.ply + j] = from_float<T>(x);
            });
            wild = ch.infinite();
            meet<WAVES>();
        } else {
            ch.template run<OUT>(qs, ks, vs, gm, acc);
            meet<WAVES>();
            if constexpr (OUT) {   // out through LDS, a row's bytes together
#pragma unroll
                for (int c = 0; c < C::CT; ++c)
#pragma unroll
                    for (int it = 0; it < C::NT; ++it)
                        store4(qs + (16 * it + ch.lc) * LD + ch.c0 + 16 * c + 4 * ch.g, acc[c][it]);
                meet<WAVES>();
                o.store(t0, gm.n, qs);   // the elements that this thread's next rows replace
            }
        }
    }
    if constexpr (OUT) {
        o.clear(sg.end, sg.s1);
        if (a.s_out && sg.seg == (REV ? 0 : a.segments - 1))
            ch.store_state(a.s_out + blockIdx.x * size, a.kd, a.vd, a.s_row, a.s_col);
    } else {
        ch.store_state(slot, a.kd, a.vd, a.vd, 1);
        if (threadIdx.x == 0)
            a.seg_carry[(int64_t)blockIdx.x * a.segments + sg.seg] = any_start ? -1.f : power(ch.g2, sg.end - sg.s0);
    }
}

// The gradients of k and v over one segment of one game and head, in reverse, from
// one reading of q, k, v and d_out: two passes side by side on the same tiles, dv
// (k, q, d_out) by one half of the block's waves and dk (v, d_out, q), on the
// transposed state, by the other.
struct GradArgs {
    ScanArgs scan;       // q: k, k: q, v: d_out, o: dv
    jq_rows values, dk;  // v and the gradient of k
};
template <class T, int D, bool FAST>
__global__ __launch_bounds__(128 * pass_waves(D), 2) void k_attention_kv(GradArgs ga)
{
    using C = Chunk<T, D, true>;
    constexpr int CH = C::CH, LD = C::LD, WAVES = 2 * C::WAVES;
    using P = Plies<T, D, 64 * WAVES, FAST>;
    using V = typename P::V;
    const ScanArgs &a = ga.scan;
    __shared__ __align__(16) T ks[CH * LD], qs[CH * LD], ds[CH * LD], vs[CH * LD];
    __shared__ int bad[2];
    const Segment sg(a, blockIdx.y, CH);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool second = wave >= C::WAVES;   // dk
    C ch(a.log_decay[sg.h], a.in_scale, 1.f, wave % C::WAVES);
    const int64_t size = (int64_t)a.kd * a.vd;
    const float *init = a.segments > 1 ? a.seg_states + ((int64_t)blockIdx.x * a.segments + sg.seg) * size
                                       : a.s_in ? a.s_in + blockIdx.x * size : nullptr;
    if (second) ch.load_state(init, a.vd, a.kd, 1, a.vd);
    else ch.load_state(init, a.kd, a.vd, a.vd, 1);
    const P k(a.q, sg.b, sg.h, a.kd, a.stream), q(a.k, sg.b, sg.h, a.kd, a.stream), d(a.v, sg.b, sg.h, a.vd, a.stream), v(ga.values, sg.b, sg.h, a.vd, a.stream);
    const P dv(a.o, sg.b, sg.h, a.vd, a.stream), dk(ga.dk, sg.b, sg.h, a.kd, a.stream);
    const uint8_t *starts = a.starts ? a.starts + sg.b * a.starts_batch : nullptr;
    if (threadIdx.x < 2) bad[threadIdx.x] = 0;
    __syncthreads();

    V kt[P::NV], qt[P::NV], dt[P::NV], vt[P::NV];
    bool start = false, wild = ch.infinite();
    const auto begin = [&](int m) { return sg.s0 + (sg.chunks - 1 - m) * CH; };
    const auto fetch = [&](int m) {
        const int t0 = begin(m), n = min(CH, sg.end - t0);
        start = starts && ch.l < n && starts[(t0 + ch.l) * a.starts_ply];
        k.load(t0, n, kt);
        q.load(t0, n, qt);
        d.load(t0, n, dt);
        v.load(t0, n, vt);
    };
    if (sg.chunks) fetch(0);
    for (int m = 0; m < sg.chunks; ++m) {
        const int t0 = begin(m);
        const Games gm{(uint32_t)__ballot(start), min(CH, sg.end - t0)};
        P::stage(ks, kt);
        P::stage(qs, qt);
        P::stage(ds, dt);
        P::stage(vs, vt);
        const float sum = (P::probe_all(kt) + P::probe_all(qt)) + (P::probe_all(dt) + P::probe_all(vt));
        if (wild || __ballot(sum != sum)) bad[m & 1] = 1;
        __syncthreads();
        const bool singly = bad[m & 1];
        if (threadIdx.x == 0) bad[(m + 1) & 1] = 0;
        if (m + 1 < sg.chunks) fetch(m + 1);
        const T *x = second ? vs : ks, *y = second ? ds : qs, *z = second ? qs : ds;
        f32x4 acc[C::CT][C::NT];
        if (singly) {
            T *out = second ? dk.base : dv.base;
            const int64_t ply = second ? dk.ply : dv.ply;
            const int dim = second ? a.kd : a.vd;
            ch.singly(x, y, z, gm, second ? a.vd : a.kd, dim, [&](int i, int c, float value) {
                const int j = ch.c0 + 16 * c + ch.lc;
                if (ch.g == 0 && j < dim) out[(t0 + i) * ply + j] = from_float<T>(value);
            });
            wild = ch.infinite();
            __syncthreads();
        } else {
            ch.template run<true>(x, y, z, gm, acc);
            __syncthreads();
            T *to = second ? ks : vs;   // the tiles that this thread's next rows replace
#pragma unroll
            for (int c = 0; c < C::CT; ++c)
#pragma unroll
                for (int it = 0; it < C::NT; ++it)
                    store4(to + (16 * it + ch.lc) * LD + ch.c0 + 16 * c + 4 * ch.g, acc[c][it]);
            __syncthreads();
            dv.store(t0, gm.n, vs);
            dk.store(t0, gm.n, ks);
        }
    }
    dv.clear(sg.end, sg.s1);
    dk.clear(sg.end, sg.s1);
    if (a.s_out && sg.seg == 0 && !second) ch.store_state(a.s_out + blockIdx.x * size, a.kd, a.vd, a.vd, 1);
}

// What the segments leave, in their order: seg_states[g] becomes the state before
// segment g. One thread per element of a head's state.
template <bool REV>
__global__ __launch_bounds__(256) void k_attention_join(ScanArgs a)
{
    const int size = a.kd * a.vd, e = blockIdx.y * 256 + threadIdx.x;
    if (e >= size) return;
    const int i = e / a.vd, j = e % a.vd;
    float s = a.s_in ? a.s_in[(int64_t)blockIdx.x * size + i * a.s_row + j * a.s_col] : 0.f;
    float *slots = a.seg_states + (int64_t)blockIdx.x * a.segments * size + e;
    const float *carry = a.seg_carry + (int64_t)blockIdx.x * a.segments;
    const bool fades = power(log2_lambda(a.log_decay[blockIdx.x % a.heads]), 1) > 0.f;   // lambda is not 0, whatever its power has become
#pragma unroll 4
    for (int m = 0; m < a.segments - 1; ++m) {
        const int g = REV ? a.segments - 1 - m : m;
        const float own = slots[(int64_t)g * size], c = carry[g];
        slots[(int64_t)g * size] = s;
        s = c < 0.f ? own : (c == 0.f && fades && fabsf(s) == __builtin_inff() ? s : c * s) + own;
    }
    slots[(int64_t)(REV ? 0 : a.segments - 1) * size] = s;
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

// One ply of every game, a wave for each game and head. L lanes hold a row's columns,
// four each (ODD: rows that are not whole vectors, the last lane with what is left);
// the 64 / L groups of lanes take a part of the rows each, STEP_ROWS at a time
// with all their loads on their way, and their sums are joined by shuffles: no
// barriers, the state is read and written once. Bound by that: 32,768 games of 4 heads
// of 64 x 64 (4.36 GB) in 744 us, 5.9 TB/s (one thread per column: 1,858);
// 4,693 games of 4 heads of 50 x 50 in float32 (188 MB, which the caches hold) in 66 us
// (284), 60,000 (2.4 GB) in 1,234 us, 3.9 TB/s.
constexpr int STEP_ROWS = 16, STEP_WAVES = 4;
template <class T, int L, bool STREAM, bool ODD>
__global__ __launch_bounds__(64 * STEP_WAVES) void k_attention_step_wave(StepArgs a, int count)
{
    typedef f32x4 At __attribute__((aligned(4)));   // states lie at any alignment of their elements
    const int at = blockIdx.x * STEP_WAVES + (threadIdx.x >> 6);
    if (at >= count) return;
    const int b = at / a.heads, h = at % a.heads, l = threadIdx.x & 63, c = 4 * (l % L), g = l / L;
    const bool on = c < a.dv;
    const int n = ODD ? min(4, a.dv - c) : 4;   // columns of this lane
    const int64_t row = a.rows ? a.rows[b] : b;
    const bool live = row >= 0 && row < a.state_rows;
    f32x4 sum{0.f, 0.f, 0.f, 0.f};
    if (live && on) {
        float *s = a.state + (row * a.heads + h) * a.dk * a.dv + c;
        const T *q = row_at<const T>(a.q, b, 0, h), *k = row_at<const T>(a.k, b, 0, h), *vp = row_at<const T>(a.v, b, 0, h) + c;
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)vp[min(e, n - 1)];
        const float lam = expf(a.log_decay[h]);
        const bool start = a.starts && a.starts[b];
        const int each = (a.dk + 64 / L - 1) / (64 / L), end = min(a.dk, (g + 1) * each);
        for (int i0 = g * each; i0 < end; i0 += STEP_ROWS) {
            f32x4 x[STEP_ROWS];
            float qs[STEP_ROWS], ks[STEP_ROWS];
#pragma unroll
            for (int i = 0; i < STEP_ROWS; ++i) {
                const int r = min(i0 + i, end - 1);
                const float *at = s + r * a.dv;
                if (n == 4) x[i] = STREAM ? __builtin_nontemporal_load(reinterpret_cast<const At *>(at)) : *reinterpret_cast<const At *>(at);
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[i][e] = at[min(e, n - 1)];
                qs[i] = (float)q[r];
                ks[i] = (float)k[r];
            }
#pragma unroll
            for (int i = 0; i < STEP_ROWS; ++i) {
                if (i0 + i >= end) break;
                f32x4 y;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y[e] = fmaf(ks[i], v[e], start ? 0.f : lam * x[i][e]);
                    sum[e] = fmaf(qs[i], y[e], sum[e]);
                }
                float *at = s + (i0 + i) * a.dv;
                if (n < 4)
#pragma unroll
                    for (int e = 0; e < 3; ++e) {
                        if (e < n) at[e] = y[e];
                    }
                else if (STREAM) __builtin_nontemporal_store(y, reinterpret_cast<At *>(at));
                else *reinterpret_cast<At *>(at) = y;
            }
        }
    }
#pragma unroll
    for (int o = L; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], o);
    if (g == 0 && on) {
        T *o = row_at<T>(a.o, b, 0, h) + c;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) o[e] = from_float<T>(live ? a.scale * sum[e] : 0.f);
    }
}

}  // namespace jq
