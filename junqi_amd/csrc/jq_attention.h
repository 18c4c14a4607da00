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
    // a long axis is split into segments of seg_plies (whole chunks) that run side by
    // side: seg_states[(b, h)][g] (kd, vd) is the state before segment g, seg_carry
    // what a segment leaves of it
    int segments, seg_plies;
    float *seg_states, *seg_carry;
};

// ---- products of 16 x 16 tiles -------------------------------------------------
// A product takes two fragments: lane l holds row (or column) l % 16 and, with
// g = l / 16, the depths that its e-th elements stand for. The result has column
// l % 16 and rows 4g .. 4g + 3 in lane l. Depths may be taken in any order that
// both fragments share. `deep`, `col` and the split state take them in the order in
// which a result's rows lie in its lanes (depth), so that a state goes from result
// to operand without leaving its registers; `row` takes them as they lie.
template <class T> struct Mma;

template <> struct Mma<bf16> {
    typedef bf16x8 Frag;
    static constexpr int CH = 64;   // plies of a chunk
    static constexpr int KB = 32;   // depth of a fragment
    static __device__ __forceinline__ f32x4 mul(Frag a, Frag b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ int depth(int g, int e) { return 16 * (e >> 2) + 4 * g + (e & 3); }
    // where depths d .. d + 3, d % 4 == 0, of a row stored for `row` lie, for `row` to give them in `depth`'s order
    static __device__ __forceinline__ int place(int d) { return (d & ~31) + 2 * (d & 15) + ((d & 16) >> 2); }
    static __device__ __forceinline__ Frag row(const bf16 *p, int g) { return *reinterpret_cast<const Frag *>(p + 8 * g); }
    static __device__ __forceinline__ Frag deep(const bf16 *p, int g)
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
    static constexpr int CH = 32;
    static constexpr int KB = 16;
    static __device__ __forceinline__ f32x4 mul(Frag a, Frag b, f32x4 c)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ int depth(int g, int e) { return 4 * g + e; }
    static __device__ __forceinline__ int place(int d) { return d; }
    static __device__ __forceinline__ Frag row(const float *p, int g) { return *reinterpret_cast<const Frag *>(p + 4 * g); }
    static __device__ __forceinline__ Frag deep(const float *p, int g) { return row(p, g); }
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
// float32: sums that come out in float32. Two hold 16 bits: operands of sums that
// are rounded to bfloat16.
template <class T, int N> constexpr int PARTS = sizeof(T) == 2 ? N : 1;

// log2 lambda, and lambda^d from it: lambda = 0 has a logarithm whose products with
// whole numbers are finite, so that lambda^0 is 1.
__device__ __forceinline__ float log2_lambda(float log_decay)
{
    const float x = log_decay * 1.44269504088896340736f;
    return x < -1e30f ? -1e30f : x;
}
__device__ __forceinline__ float power(float log2_lam, float d) { return __builtin_amdgcn_exp2f(log2_lam * d); }

// What the plies of a chunk need to know of it, made once for each chunk.
template <int CH>
struct alignas(16) Marks {
    float sees[CH];    // lambda's power from the chunk's begin (REV: end) to the ply; -1: it sees nothing from there
    float leaves[CH];  // lambda's power from the ply to the chunk's end (REV: begin) times in_scale; 0: nothing is left
    int game[CH];      // games that start in the chunk up to the ply
    float carry;       // lambda's power over the chunk; -1: a game starts in it
    int n;             // plies
    bool starts;       // a game starts in it
};

// One chunk of a pass for D columns: D / 16 waves, each with 16 columns of the
// value-side and of the state.
template <class T, int D, bool REV>
struct Chunk {
    using M = Mma<T>;
    using Frag = typename M::Frag;
    static constexpr int CH = M::CH, KB = M::KB, NT = CH / 16, WAVES = D / 16, THREADS = 64 * WAVES;
    static constexpr int LD = D + Vec<T>::N, PLD = CH + Vec<T>::N;   // 16 bytes of padding turn the rows over the banks
    static constexpr int FE = KB / 4;                                // elements of a fragment

    f32x4 s[D / 16];   // state (16t + 4g + r, 16w + l % 16)
    float g2;          // log2 lambda
    int w, l, lc, g;

    __device__ __forceinline__ Chunk(float log_decay)
        : g2(log2_lambda(log_decay)), w(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), l(threadIdx.x & 63), lc(l & 15), g(l >> 4)
    {
    }

    // f(register t, r of the state, its offset) for this lane's part of a (rows, cols) state
    template <class F>
    __device__ __forceinline__ void each(int rows, int cols, int s_row, int s_col, F &&f)
    {
        int i0 = 4 * g, c = 16 * w + lc;
        asm("" : "+v"(i0), "+v"(c));   // the offsets are made where they are used, not kept over the pass
        const int at = i0 * s_row + c * s_col;
        if (c >= cols) rows = 0;
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (i0 + 16 * t + r < rows) f(t, r, at + (16 * t + r) * s_row);
    }
    __device__ __forceinline__ void load_state(const float *p, int rows, int cols, int s_row, int s_col)
    {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (p) each(rows, cols, s_row, s_col, [&](int t, int r, int at) { s[t][r] = p[at]; });
    }
    __device__ __forceinline__ void store_state(float *p, int rows, int cols, int s_row, int s_col)
    {
        each(rows, cols, s_row, s_col, [&](int t, int r, int at) { p[at] = s[t][r]; });
    }

    // Lane i: ply i of a chunk of n plies, `start` where a game starts there. One wave.
    __device__ __forceinline__ void mark(Marks<CH> &mk, bool start, int n, float in_scale) const
    {
        const uint64_t mask = __ballot(start);
        const int i = l, game = __popcll(mask & ((2ull << i) - 1)), games = __popcll(mask);
        if (i < CH) {
            const bool from = game == 0, to = game == games;   // sees the begin; is seen from the end
            mk.sees[i] = i < n && (REV ? to : from) ? power(g2, REV ? n - 1 - i : i + 1) : -1.f;
            mk.leaves[i] = i < n && (REV ? from : to) ? in_scale * power(g2, REV ? i + 1 : n - 1 - i) : 0.f;
            mk.game[i] = game;
        }
        if (i == 0) {
            mk.carry = games ? -1.f : power(g2, n);
            mk.n = n;
            mk.starts = games != 0;
        }
    }

    // p[i][j] = scale lambda^|i - j| q_i.k_j for the plies j that i sees, else 0, of N
    // pairs q, k; the tiles on the diagonal and on one side of it, shared out over the
    // waves.
    template <int N>
    __device__ __forceinline__ void scores(const T *const (&q)[N], const T *const (&k)[N], T *const (&p)[N],
                                           const Marks<CH> &mk, float scale) const
    {
        const bool starts = __builtin_amdgcn_readfirstlane(mk.starts);
        for (int m = w; m < NT * (NT + 1) / 2; m += WAVES) {
            const int a = m < 1 ? 0 : m < 3 ? 1 : m < 6 ? 2 : 3, b = m - a * (a + 1) / 2;
            const int it = REV ? b : a, jt = REV ? a : b, i = 16 * it + lc, j0 = 16 * jt + 4 * g;
            f32x4 acc[N];
#pragma unroll
            for (int u = 0; u < N; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < D; c += KB)
#pragma unroll
                for (int u = 0; u < N; ++u)
                    acc[u] = M::mul(M::row(k[u] + (16 * jt + lc) * LD + c, g), M::row(q[u] + i * LD + c, g), acc[u]);
            const float d0 = (float)(REV ? j0 - i : i - j0);
            const int game = starts ? mk.game[i] : 0;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float d = REV ? d0 + r : d0 - r, f = scale * power(g2, d);
                const bool seen = d >= 0.f && (!starts || game == mk.game[j0 + r]);
#pragma unroll
                for (int u = 0; u < N; ++u) acc[u][r] = seen ? acc[u][r] * f : 0.f;
            }
#pragma unroll
            for (int u = 0; u < N; ++u) store4(p[u] + i * PLD + M::place(j0), acc[u]);
        }
    }

    static __device__ __forceinline__ void store4(bf16 *p, f32x4 x)
    {
        *reinterpret_cast<bf16x4 *>(p) = bf16x4{(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]};
    }
    static __device__ __forceinline__ void store4(float *p, f32x4 x) { *reinterpret_cast<f32x4 *>(p) = x; }

    // o[it] (columns i = 16it + l % 16, rows: this wave's value columns) = what the
    // state before the chunk answers to q_i.
    __device__ __forceinline__ void inter(const T *q, const Marks<CH> &mk, float scale, f32x4 (&o)[NT]) const
    {
#pragma unroll
        for (int it = 0; it < NT; ++it) o[it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < D / KB; ++c) {
            constexpr int N = PARTS<T, 2>;
            Frag part[N];
            float x[FE];
#pragma unroll
            for (int e = 0; e < FE; ++e) x[e] = s[(c * KB + 4 * e) / 16][e & 3];
            M::template split<N>(x, part);
#pragma unroll
            for (int it = 0; it < NT; ++it) {
                const Frag y = M::deep(q + (16 * it + lc) * LD + c * KB, g);
#pragma unroll
                for (int u = 0; u < N; ++u) o[it] = M::mul(part[u], y, o[it]);
            }
        }
        seen(mk, scale, o);
    }

    // o += P v (OUT), and the state after the chunk (STATE).
    template <bool OUT, bool STATE>
    __device__ __forceinline__ void apply(const T *k, const T *v, const T *p, const Marks<CH> &mk, f32x4 (&o)[NT])
    {
        if constexpr (STATE) {
            const float carry = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, mk.carry)));
            if (carry >= 0.f) {
#pragma unroll
                for (int t = 0; t < D / 16; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[t][r] *= carry;
            } else {
#pragma unroll
                for (int t = 0; t < D / 16; ++t) s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
#pragma unroll
        for (int c = 0; c < CH / KB; ++c) {
            const Frag x = M::col(v + c * KB * LD + 16 * w, LD, l);
#pragma unroll
            for (int it = 0; it < NT; ++it) {
                if (!OUT || (REV ? c * KB + KB <= 16 * it : c * KB >= 16 * it + 16)) continue;   // nothing to see there
                o[it] = M::mul(x, M::row(p + (16 * it + lc) * PLD + c * KB, g), o[it]);
            }
            if constexpr (STATE) {
                // the plies' values times what is left of them after the chunk
                constexpr int N = PARTS<T, 3>;
                Frag part[N];
                float left[FE];
#pragma unroll
                for (int e = 0; e < FE; ++e) left[e] = (float)x[e] * mk.leaves[c * KB + M::depth(g, e)];
                M::template split<N>(left, part);
#pragma unroll
                for (int t = 0; t < D / 16; ++t) {
                    const Frag y = M::col(k + c * KB * LD + 16 * t, LD, l);
#pragma unroll
                    for (int u = 0; u < N; ++u) s[t] = M::mul(y, part[u], s[t]);
                }
            }
        }
    }

    // ---- the state turned over, for the pass that needs both of its sides: as terms in
    // LDS, turned[u][c][i] for element (i, c)
    static constexpr int TURNED = PARTS<T, 2>;
    __device__ __forceinline__ void turn(T *turned) const
    {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
            f32x4 x = s[t];
#pragma unroll
            for (int u = 0; u < TURNED; ++u) {
                T *at = turned + (u * D + 16 * w + lc) * LD + 16 * t + 4 * g;
                store4(at, x);
                if (u + 1 < TURNED)
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[r] -= (float)from_float<T>(x[r]);
            }
        }
    }

    // like inter, for the turned state: rows of o are this wave's columns of its other side
    __device__ __forceinline__ void inter_turned(const T *turned, const T *q, const Marks<CH> &mk, float scale,
                                                 f32x4 (&o)[NT]) const
    {
#pragma unroll
        for (int it = 0; it < NT; ++it) o[it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < D / KB; ++c) {
            Frag part[TURNED];
#pragma unroll
            for (int u = 0; u < TURNED; ++u) part[u] = M::col(turned + (u * D + c * KB) * LD + 16 * w, LD, l);
#pragma unroll
            for (int it = 0; it < NT; ++it) {
                const Frag y = M::deep(q + (16 * it + lc) * LD + c * KB, g);
#pragma unroll
                for (int u = 0; u < TURNED; ++u) o[it] = M::mul(part[u], y, o[it]);
            }
        }
        seen(mk, scale, o);
    }

    // o times what is left of the state at its plies
    __device__ __forceinline__ void seen(const Marks<CH> &mk, float scale, f32x4 (&o)[NT]) const
    {
#pragma unroll
        for (int it = 0; it < NT; ++it) {
            const float f = mk.sees[16 * it + lc];
#pragma unroll
            for (int r = 0; r < 4; ++r) o[it][r] = f >= 0.f ? o[it][r] * (f * scale) : 0.f;
        }
    }

    // The chunk ply by ply, for tiles with infinities or NaN: a product with 0 in
    // their place is not 0, and a ply must get nothing of those it does not see.
    // put(i, x): x = this wave's value column l % 16 of ply i. each(i, t, r, y): y = the
    // state's element (16t + 4g + r, 16w + l % 16) that ply i sees.
    template <class F, class E>
    __device__ __forceinline__ void singly(const T *q, const T *k, const T *v, const Marks<CH> &mk, float in_scale,
                                           float out_scale, F &&put, E &&each)
    {
        const float lam = power(g2, 1);
        for (int m = 0; m < mk.n; ++m) {
            const int i = REV ? mk.n - 1 - m : m;
            const bool start = mk.game[i] != (i ? mk.game[i - 1] : 0);
            const float x = in_scale * (float)v[i * LD + 16 * w + lc];
            float o = 0.f;
#pragma unroll
            for (int t = 0; t < D / 16; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int c = 16 * t + 4 * g + r;
                    float y = s[t][r];
                    if (!REV) y = start ? 0.f : lam * y;
                    y += (float)k[i * LD + c] * x;
                    o += (float)q[i * LD + c] * y;
                    each(i, t, r, y);
                    if (REV) y = start ? 0.f : lam * y;
                    s[t][r] = y;
                }
            o += __shfl_xor(o, 16);
            o += __shfl_xor(o, 32);
            put(i, out_scale * o);
        }
    }
};

// sum + 0 for finite elements, NaN where one is infinite or NaN.
__device__ __forceinline__ float probe(bf16x8 x, float sum)
{
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        sum = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{x[i], x[i + 1]}, bf16x2{bf16(0.f), bf16(0.f)}, sum, false);
    }
    return sum;
}
__device__ __forceinline__ float probe(f32x4 x, float sum)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = fmaf(x[i], 0.f, sum);
    return sum;
}

// Rows of one game and head that a block reads or writes, a chunk of plies at a
// time. FAST: through a buffer descriptor of the chunk's plies, whose bounds give
// zeros for (and drop) rows past the chunk's end without a branch; rows are whole
// aligned 16-byte vectors and a chunk spans less than 2 GiB (the host's check).
// Otherwise element by element.
template <class T, int D, bool FAST>
struct Plies {
    using V = typename Vec<T>::type;
    static constexpr int N = Vec<T>::N, PER_ROW = D / N, CH = Mma<T>::CH;
    T *base;
    int64_t ply;
    int dim;

    __device__ __forceinline__ Plies(const jq_rows &r, int b, int h, int dim_) : base(row_at<T>(r, b, 0, h)), ply(r.ply), dim(dim_) {}

    __device__ __forceinline__ __amdgpu_buffer_rsrc_t chunk(int t0, int n) const
    {
        return __builtin_amdgcn_make_buffer_rsrc(base + t0 * ply, 0, (int)(((n - 1) * ply + dim) * sizeof(T)), 0x00020000);
    }

    // this thread's two vectors of the tile of plies t0 .. t0 + n, CH / 2 rows apart; zeros elsewhere
    __device__ __forceinline__ void load(int t0, int n, V (&x)[2]) const
    {
        const int row = threadIdx.x / PER_ROW, c = threadIdx.x % PER_ROW * N;
        if constexpr (FAST) {
            const __amdgpu_buffer_rsrc_t r = chunk(t0, n);
            const int step = (int)ply * (int)sizeof(T);
            const int at = c < dim ? row * step + c * (int)sizeof(T) : INT32_MIN;   // past any bound
            x[0] = __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
            x[1] = __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, c < dim ? at + CH / 2 * step : INT32_MIN, 0, 0));
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int i = row + u * (CH / 2);
                x[u] = V{};
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (i < n && c + e < dim) x[u][e] = base[(t0 + i) * ply + c + e];
            }
        }
    }

    // rows 16 it + l % 16, columns c .. c + 3 of the chunk, from a product's result
    template <int NT>
    __device__ __forceinline__ void put(int t0, int n, int lc, int c, const f32x4 (&x)[NT]) const
    {
        if constexpr (FAST) {
            const __amdgpu_buffer_rsrc_t r = chunk(t0, n);
            const int step = (int)ply * (int)sizeof(T);
            int at = c < dim ? lc * step + c * (int)sizeof(T) : INT32_MIN;
#pragma unroll
            for (int it = 0; it < NT; ++it) {
                if constexpr (sizeof(T) == 2) {
                    const bf16x4 y{(bf16)x[it][0], (bf16)x[it][1], (bf16)x[it][2], (bf16)x[it][3]};
                    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, y), r, at, 0, 0);
                } else {
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x[it]), r, at, 0, 0);
                }
                at = c < dim ? at + 16 * step : at;
            }
        } else {
#pragma unroll
            for (int it = 0; it < NT; ++it)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * it + lc < n && c + r < dim)
                        base[(t0 + 16 * it + lc) * ply + c + r] = from_float<T>(x[it][r]);
        }
    }

    // zeros from ply t0 to t1
    __device__ __forceinline__ void clear(int t0, int t1) const
    {
        for (int t = t0 + (int)(threadIdx.x >> 6); t < t1; t += D / 16)
            for (int c = threadIdx.x & 63; c < dim; c += 64) base[t * ply + c] = from_float<T>(0.f);
    }

    // a thread's two vectors of a tile into LDS
    static __device__ __forceinline__ void stage(T *lds, const V (&x)[2])
    {
        T *p = lds + threadIdx.x / PER_ROW * (D + N) + threadIdx.x % PER_ROW * N;
        *reinterpret_cast<V *>(p) = x[0];
        *reinterpret_cast<V *>(p + CH / 2 * (D + N)) = x[1];
    }
};

// A pass over one segment of one game and head by one block: chunks in turn, the
// state in registers. While a chunk is worked on, the next one's tiles are on
// their way. OUT: the plies' outputs, from the state before the segment; else only
// the state that the segment's own plies leave, for the states before the others.
template <class T, int D, bool REV, bool FAST, bool OUT>
__global__ __launch_bounds__(4 * D, D == 32 ? 3 : 4) void k_attention_pass(ScanArgs a)
{
    using C = Chunk<T, D, REV>;
    using P = Plies<T, D, FAST>;
    using V = typename P::V;
    constexpr int CH = C::CH, LD = C::LD, NT = C::NT;
    __shared__ __align__(16) T qs[OUT ? CH * LD : 1], ks[CH * LD], vs[CH * LD], ps[OUT ? CH * C::PLD : 1];
    __shared__ Marks<CH> mk;
    __shared__ int bad[2];
    const int b = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
    const int seg = blockIdx.y + (!OUT && REV ? 1 : 0);   // the last segment's own state goes nowhere
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.plies) : a.plies;
    const int s0 = seg * a.seg_plies, s1 = a.plies - s0 > a.seg_plies ? s0 + a.seg_plies : a.plies, end = min(s1, len);
    const int chunks = end > s0 ? (end - s0 + CH - 1) / CH : 0;
    C ch(a.log_decay[h]);
    const int64_t size = (int64_t)a.kd * a.vd;
    float *slot = a.seg_states + ((int64_t)blockIdx.x * a.segments + seg) * size;
    if (!OUT) ch.load_state(nullptr, 0, 0, 0, 0);
    else if (a.segments > 1) ch.load_state(slot, a.kd, a.vd, a.vd, 1);
    else ch.load_state(a.s_in ? a.s_in + blockIdx.x * size : nullptr, a.kd, a.vd, a.s_row, a.s_col);
    const P q(a.q, b, h, a.kd), k(a.k, b, h, a.kd), v(a.v, b, h, a.vd), o(a.o, b, h, a.vd);
    const uint8_t *starts = a.starts ? a.starts + b * a.starts_batch : nullptr;
    if (OUT)
        for (int x = threadIdx.x; x < CH * C::PLD; x += C::THREADS) ps[x] = T(0.f);   // tiles beside the diagonal stay 0
    if (threadIdx.x < 2) bad[threadIdx.x] = 0;
    __syncthreads();

    V qt[2], kt[2], vt[2];
    bool start = false, any_start = false;
    const auto begin = [&](int m) { return s0 + (REV ? chunks - 1 - m : m) * CH; };
    const auto fetch = [&](int m) {
        const int t0 = begin(m), n = min(CH, end - t0);
        if (OUT) q.load(t0, n, qt);
        k.load(t0, n, kt);
        v.load(t0, n, vt);
        start = starts && ch.l < n && starts[(t0 + ch.l) * a.starts_ply];
    };
    if (chunks) fetch(0);
    for (int m = 0; m < chunks; ++m) {
        const int t0 = begin(m), n = min(CH, end - t0);
        if (ch.w == 0) ch.mark(mk, start, n, a.in_scale);
        if (!OUT) any_start |= __ballot(start) != 0;
        if (OUT) P::stage(qs, qt);
        P::stage(ks, kt);
        P::stage(vs, vt);
        const float sum = probe(vt[1], probe(vt[0], probe(kt[1], probe(kt[0], 0.f))));
        if (sum != sum) bad[m & 1] = 1;
        __syncthreads();
        if (m + 1 < chunks) fetch(m + 1);
        if (threadIdx.x == 0) bad[(m + 1) & 1] = 0;
        if (bad[m & 1]) {
            ch.singly(OUT ? qs : ks, ks, vs, mk, a.in_scale, a.out_scale, [&](int i, float x) {
                const int c = 16 * ch.w + ch.lc;
                if (OUT && ch.g == 0 && c < a.vd) o.base[(t0 + i) * o.ply + c] = from_float<T>(x);
            }, [](int, int, int, float) {});
        } else if constexpr (OUT) {
            f32x4 acc[NT];
            ch.template scores<1>({qs}, {ks}, {ps}, mk, a.in_scale * a.out_scale);
            ch.inter(qs, mk, a.out_scale, acc);
            __syncthreads();
            ch.template apply<true, true>(ks, vs, ps, mk, acc);
            o.put(t0, n, ch.lc, 16 * ch.w + 4 * ch.g, acc);
        } else {
            f32x4 none[NT];
            ch.template apply<false, true>(ks, vs, nullptr, mk, none);
        }
        __syncthreads();
    }
    if constexpr (OUT) {
        o.clear(max(s0, len), s1);
        if (a.s_out && seg == (REV ? 0 : a.segments - 1)) ch.store_state(a.s_out + blockIdx.x * size, a.kd, a.vd, a.s_row, a.s_col);
    } else {
        ch.store_state(slot, a.kd, a.vd, a.vd, 1);
        if (threadIdx.x == 0)
            a.seg_carry[(int64_t)blockIdx.x * a.segments + seg] = any_start ? -1.f : power(ch.g2, max(end - s0, 0));
    }
}

// The gradients of k and v over one segment of one game and head, in reverse, from
// one reading of q, k, v and d_out. With R the gradient of the state after a ply,
//   dv_j = R^T k_j and dk_j = R v_j   where R = scale sum_{i >= j} lambda^(i - j) q_i d_i^T + ...
// are two passes with one state: dv is the pass (k, q, d_out), whose state stays in
// registers; dk is (v, d_out, q) on its transpose, which the waves leave for each
// other in LDS, as terms. Both share the plies' weights.
struct GradArgs {
    ScanArgs scan;       // q: k, k: q, v: d_out, o: dv
    jq_rows values, dk;  // v and the gradient of k
};
template <class T, int D> constexpr int kv_lds()
{
    using C = Chunk<T, D, true>;
    return (4 * C::CH * C::LD + 2 * C::CH * C::PLD + C::TURNED * D * C::LD) * (int)sizeof(T);
}
template <class T, int D, bool FAST>
__global__ __launch_bounds__(4 * D, 2) void k_attention_kv(GradArgs ga)
{
    using C = Chunk<T, D, true>;
    using P = Plies<T, D, FAST>;
    using V = typename P::V;
    constexpr int CH = C::CH, LD = C::LD, NT = C::NT, PLD = C::PLD;
    const ScanArgs &a = ga.scan;
    extern __shared__ __align__(16) char dynamic[];
    T *ks = reinterpret_cast<T *>(dynamic), *qs = ks + CH * LD, *ds = qs + CH * LD, *vs = ds + CH * LD;
    T *p1 = vs + CH * LD, *p2 = p1 + CH * PLD, *turned = p2 + CH * PLD;
    __shared__ Marks<CH> mk;
    __shared__ int bad[2];
    const int b = blockIdx.x / a.heads, h = blockIdx.x % a.heads, seg = blockIdx.y;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.plies) : a.plies;
    const int s0 = seg * a.seg_plies, s1 = a.plies - s0 > a.seg_plies ? s0 + a.seg_plies : a.plies, end = min(s1, len);
    const int chunks = end > s0 ? (end - s0 + CH - 1) / CH : 0;
    C ch(a.log_decay[h]);
    const int64_t size = (int64_t)a.kd * a.vd;
    if (a.segments > 1) ch.load_state(a.seg_states + ((int64_t)blockIdx.x * a.segments + seg) * size, a.kd, a.vd, a.vd, 1);
    else ch.load_state(a.s_in ? a.s_in + blockIdx.x * size : nullptr, a.kd, a.vd, a.vd, 1);
    const P k(a.q, b, h, a.kd), q(a.k, b, h, a.kd), d(a.v, b, h, a.vd), v(ga.values, b, h, a.vd);
    const P dv(a.o, b, h, a.vd), dk(ga.dk, b, h, a.kd);
    const uint8_t *starts = a.starts ? a.starts + b * a.starts_batch : nullptr;
    for (int x = threadIdx.x; x < 2 * CH * PLD; x += C::THREADS) p1[x] = T(0.f);   // tiles beside the diagonal stay 0
    ch.turn(turned);
    if (threadIdx.x < 2) bad[threadIdx.x] = 0;
    __syncthreads();

    V kt[2], qt[2], dt[2], vt[2];
    bool start = false;
    const auto begin = [&](int m) { return s0 + (chunks - 1 - m) * CH; };
    const auto fetch = [&](int m) {
        const int t0 = begin(m), n = min(CH, end - t0);
        k.load(t0, n, kt);
        q.load(t0, n, qt);
        d.load(t0, n, dt);
        v.load(t0, n, vt);
        start = starts && ch.l < n && starts[(t0 + ch.l) * a.starts_ply];
    };
    if (chunks) fetch(0);
    for (int m = 0; m < chunks; ++m) {
        const int t0 = begin(m), n = min(CH, end - t0);
        if (ch.w == 0) ch.mark(mk, start, n, a.in_scale);
        P::stage(ks, kt);
        P::stage(qs, qt);
        P::stage(ds, dt);
        P::stage(vs, vt);
        const float sum = probe(dt[1], probe(dt[0], probe(qt[1], probe(qt[0], 0.f))));
        if (sum != sum) bad[m & 1] = 1;
        __syncthreads();
        if (m + 1 < chunks) fetch(m + 1);
        if (threadIdx.x == 0) bad[(m + 1) & 1] = 0;
        if (bad[m & 1]) {
            float *red = reinterpret_cast<float *>(p1);   // [wave][D], for the sums over all columns
            static_assert(C::WAVES * D * sizeof(float) <= CH * PLD * sizeof(T));
            ch.singly(ks, qs, ds, mk, a.in_scale, 1.f, [&](int i, float x) {
                const int c = 16 * ch.w + ch.lc;
                if (ch.g == 0 && c < a.vd) dv.base[(t0 + i) * dv.ply + c] = from_float<T>(x);
                __syncthreads();
                if (threadIdx.x < a.kd) {
                    float y = 0.f;
                    for (int u = 0; u < C::WAVES; ++u) y += red[u * D + threadIdx.x];
                    dk.base[(t0 + i) * dk.ply + threadIdx.x] = from_float<T>(y);
                }
                __syncthreads();
            }, [&](int i, int t, int r, float y) {
                y *= (float)vs[i * LD + 16 * ch.w + ch.lc];
#pragma unroll
                for (int o = 8; o; o >>= 1) y += __shfl_xor(y, o);
                if (ch.lc == 0) red[ch.w * D + 16 * t + 4 * ch.g + r] = y;
            });
            for (int x = threadIdx.x; x < CH * PLD; x += C::THREADS) p1[x] = T(0.f);
        } else {
            f32x4 o1[NT], o2[NT];
            ch.template scores<2>({ks, vs}, {qs, ds}, {p1, p2}, mk, a.in_scale);
            ch.inter(ks, mk, 1.f, o1);
            ch.inter_turned(turned, vs, mk, 1.f, o2);
            __syncthreads();
            ch.template apply<true, true>(qs, ds, p1, mk, o1);
            ch.template apply<true, false>(nullptr, qs, p2, mk, o2);
            dv.put(t0, n, ch.lc, 16 * ch.w + 4 * ch.g, o1);
            dk.put(t0, n, ch.lc, 16 * ch.w + 4 * ch.g, o2);
        }
        ch.turn(turned);
        __syncthreads();
    }
    dv.clear(max(s0, len), s1);
    dk.clear(max(s0, len), s1);
    if (a.s_out && seg == 0) ch.store_state(a.s_out + blockIdx.x * size, a.kd, a.vd, a.vd, 1);
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
#pragma unroll 4
    for (int m = 0; m < a.segments - 1; ++m) {
        const int g = REV ? a.segments - 1 - m : m;
        const float own = slots[(int64_t)g * size], c = carry[g];
        slots[(int64_t)g * size] = s;
        s = c >= 0.f ? c * s + own : own;
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

// One ply of every game, for value dims that are not whole vectors: one block per
// game and head, one thread per column.
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

// The same with a wave for each game and head. L lanes hold a row's columns, four
// each; the 64 / L groups of lanes take a part of the rows each, STEP_ROWS at a time
// with all their loads on their way, and their sums are joined by shuffles: no
// barriers, the state is read and written once.
constexpr int STEP_ROWS = 16, STEP_WAVES = 4;
template <class T, int L>
__global__ __launch_bounds__(64 * STEP_WAVES) void k_attention_step_wave(StepArgs a, int count)
{
    const int at = blockIdx.x * STEP_WAVES + (threadIdx.x >> 6);
    if (at >= count) return;
    const int b = at / a.heads, h = at % a.heads, l = threadIdx.x & 63, c = 4 * (l % L), g = l / L;
    const bool on = c < a.dv;
    const int64_t row = a.rows ? a.rows[b] : b;
    const bool live = row >= 0 && row < a.state_rows;
    f32x4 sum{0.f, 0.f, 0.f, 0.f};
    if (live && on) {
        float *s = a.state + (row * a.heads + h) * a.dk * a.dv + c;
        const T *q = row_at<const T>(a.q, b, 0, h), *k = row_at<const T>(a.k, b, 0, h), *vp = row_at<const T>(a.v, b, 0, h) + c;
        const f32x4 v{(float)vp[0], (float)vp[1], (float)vp[2], (float)vp[3]};
        const float lam = expf(a.log_decay[h]);
        const bool start = a.starts && a.starts[b];
        const int each = (a.dk + 64 / L - 1) / (64 / L), end = min(a.dk, (g + 1) * each);
        for (int i0 = g * each; i0 < end; i0 += STEP_ROWS) {
            f32x4 x[STEP_ROWS];
            float qs[STEP_ROWS], ks[STEP_ROWS];
#pragma unroll
            for (int i = 0; i < STEP_ROWS; ++i) {
                const int r = min(i0 + i, end - 1);
                x[i] = *reinterpret_cast<const f32x4 *>(s + r * a.dv);
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
                *reinterpret_cast<f32x4 *>(s + (i0 + i) * a.dv) = y;
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
        for (int e = 0; e < 4; ++e) o[e] = from_float<T>(live ? a.scale * sum[e] : 0.f);
    }
}

}  // namespace jq
