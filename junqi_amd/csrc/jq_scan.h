// The selective state space scan, forward and backward, and its step of one ply.
#pragma once
#include "jq_memory.h"

namespace jq {

// For each game, channel d and state n, with dt = softplus(delta + bias):
//   h_t = exp(dt_t a) h_{t-1} + dt_t u_t b_t;   y_t = sum over n of c_t h_t, + skip u_t;   out = y silu(gate)
// A lane has a channel and NS of its states in registers; a wave has 64 channels of one
// group, and more than 16 states are parted among the waves of a block. b_t and c_t, the
// same for all channels of a group, lie in lanes 0 .. NS - 1 of each row of 16 and reach
// the products as their row-broadcast operands, without an instruction of their own.
// Bound by the vector units: a state of a ply takes five instructions (of which the
// exponential as long as two) forward and thirteen backward, with the sums of db and dc
// over channels 17.5. 512 games x 256 plies of 512 channels of 16 states in bfloat16:
// forward 334 us (121 instructions a ply and wave, of which 80 the states', the units busy
// 77 % of the time; the rows and saved states are 1.1 GB), backward 1,115 us (393 a ply
// and wave, busy 74 %, 86 while its waves live), times under the profiler; 1,419 us in all
// without it. Without these operands, with 64-bit addresses in vector registers and the
// arguments of a dozen tensors held over the pass: 3,160 us in all.
constexpr int SCAN_PLIES = 4;     // plies whose rows are on their way while the ones before are computed
constexpr int SCAN_CHUNK = 8;     // plies of a chunk of the backward pass, which starts from a saved state
constexpr int scan_far(int ns) { return ns > 8 ? 2 : 0; }   // plies of a chunk whose states wait in LDS: registers would spill

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

// log(1 + e^x) = max(x, 0) + 2 atanh(e / (2 + e)), e = e^-|x|, so small results keep all
// their digits. s = e / (2 + e) is at most 1/3; atanh(s) / s as a polynomial in s^2 of the
// fourth degree, fitted for the least largest relative error: below 1e-8 with these
// coefficients (the series to s^14 takes three terms more).
__device__ __forceinline__ float softplus(float x)
{
    const float e = exp2_fast(-LOG2E * fabsf(x)), s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    float p = 0.14089167f;
    p = fmaf(p, q, 0.13980301f);
    p = fmaf(p, q, 0.20012455f);
    p = fmaf(p, q, 0.33333157f);
    p = fmaf(p, q, 1.f);
    return fmaf(s + s, p, fmaxf(x, 0.f));
}

// Products whose one factor is x of lane i of each row of 16 lanes (row_newbcast), as an
// operand: the compiler folds it into products, not into fused ones, which would take a
// move for each. The two wait states after x's write come first.
#define JQ_ROW_FMAC(d, i, s) "v_fmac_f32_dpp " d ", %[x], " s " row_newbcast:" #i " row_mask:0xf bank_mask:0xf\n"

// y + the sum of x of lane i times h[i]
__device__ __forceinline__ float row_dot(float y, float x, const float (&h)[4])
{
    asm("s_nop 1\n" JQ_ROW_FMAC("%[y]", 0, "%[a]") JQ_ROW_FMAC("%[y]", 1, "%[b]") JQ_ROW_FMAC("%[y]", 2, "%[c]") JQ_ROW_FMAC("%[y]", 3, "%[d]")
        : [y] "+v"(y) : [x] "v"(x), [a] "v"(h[0]), [b] "v"(h[1]), [c] "v"(h[2]), [d] "v"(h[3]));
    return y;
}
__device__ __forceinline__ float row_dot(float y, float x, const float (&h)[8])
{
    asm("s_nop 1\n" JQ_ROW_FMAC("%[y]", 0, "%[a]") JQ_ROW_FMAC("%[y]", 1, "%[b]") JQ_ROW_FMAC("%[y]", 2, "%[c]") JQ_ROW_FMAC("%[y]", 3, "%[d]")
        JQ_ROW_FMAC("%[y]", 4, "%[e]") JQ_ROW_FMAC("%[y]", 5, "%[f]") JQ_ROW_FMAC("%[y]", 6, "%[g]") JQ_ROW_FMAC("%[y]", 7, "%[h]")
        : [y] "+v"(y) : [x] "v"(x), [a] "v"(h[0]), [b] "v"(h[1]), [c] "v"(h[2]), [d] "v"(h[3]), [e] "v"(h[4]), [f] "v"(h[5]),
          [g] "v"(h[6]), [h] "v"(h[7]));
    return y;
}
__device__ __forceinline__ float row_dot(float y, float x, const float (&h)[16])
{
    asm("s_nop 1\n" JQ_ROW_FMAC("%[y]", 0, "%[a]") JQ_ROW_FMAC("%[y]", 1, "%[b]") JQ_ROW_FMAC("%[y]", 2, "%[c]") JQ_ROW_FMAC("%[y]", 3, "%[d]")
        JQ_ROW_FMAC("%[y]", 4, "%[e]") JQ_ROW_FMAC("%[y]", 5, "%[f]") JQ_ROW_FMAC("%[y]", 6, "%[g]") JQ_ROW_FMAC("%[y]", 7, "%[h]")
        JQ_ROW_FMAC("%[y]", 8, "%[i]") JQ_ROW_FMAC("%[y]", 9, "%[j]") JQ_ROW_FMAC("%[y]", 10, "%[k]") JQ_ROW_FMAC("%[y]", 11, "%[l]")
        JQ_ROW_FMAC("%[y]", 12, "%[m]") JQ_ROW_FMAC("%[y]", 13, "%[n]") JQ_ROW_FMAC("%[y]", 14, "%[o]") JQ_ROW_FMAC("%[y]", 15, "%[p]")
        : [y] "+v"(y) : [x] "v"(x), [a] "v"(h[0]), [b] "v"(h[1]), [c] "v"(h[2]), [d] "v"(h[3]), [e] "v"(h[4]), [f] "v"(h[5]),
          [g] "v"(h[6]), [h] "v"(h[7]), [i] "v"(h[8]), [j] "v"(h[9]), [k] "v"(h[10]), [l] "v"(h[11]), [m] "v"(h[12]),
          [n] "v"(h[13]), [o] "v"(h[14]), [p] "v"(h[15]));
    return y;
}

// v[i] += x of lane i times y
__device__ __forceinline__ void row_add(float (&v)[4], float x, float y)
{
    asm("s_nop 1\n" JQ_ROW_FMAC("%[a]", 0, "%[y]") JQ_ROW_FMAC("%[b]", 1, "%[y]") JQ_ROW_FMAC("%[c]", 2, "%[y]") JQ_ROW_FMAC("%[d]", 3, "%[y]")
        : [a] "+v"(v[0]), [b] "+v"(v[1]), [c] "+v"(v[2]), [d] "+v"(v[3]) : [x] "v"(x), [y] "v"(y));
}
__device__ __forceinline__ void row_add(float (&v)[8], float x, float y)
{
    asm("s_nop 1\n" JQ_ROW_FMAC("%[a]", 0, "%[y]") JQ_ROW_FMAC("%[b]", 1, "%[y]") JQ_ROW_FMAC("%[c]", 2, "%[y]") JQ_ROW_FMAC("%[d]", 3, "%[y]")
        JQ_ROW_FMAC("%[e]", 4, "%[y]") JQ_ROW_FMAC("%[f]", 5, "%[y]") JQ_ROW_FMAC("%[g]", 6, "%[y]") JQ_ROW_FMAC("%[h]", 7, "%[y]")
        : [a] "+v"(v[0]), [b] "+v"(v[1]), [c] "+v"(v[2]), [d] "+v"(v[3]), [e] "+v"(v[4]), [f] "+v"(v[5]), [g] "+v"(v[6]),
          [h] "+v"(v[7]) : [x] "v"(x), [y] "v"(y));
}
__device__ __forceinline__ void row_add(float (&v)[16], float x, float y)
{
    asm("s_nop 1\n" JQ_ROW_FMAC("%[a]", 0, "%[y]") JQ_ROW_FMAC("%[b]", 1, "%[y]") JQ_ROW_FMAC("%[c]", 2, "%[y]") JQ_ROW_FMAC("%[d]", 3, "%[y]")
        JQ_ROW_FMAC("%[e]", 4, "%[y]") JQ_ROW_FMAC("%[f]", 5, "%[y]") JQ_ROW_FMAC("%[g]", 6, "%[y]") JQ_ROW_FMAC("%[h]", 7, "%[y]")
        JQ_ROW_FMAC("%[i]", 8, "%[y]") JQ_ROW_FMAC("%[j]", 9, "%[y]") JQ_ROW_FMAC("%[k]", 10, "%[y]") JQ_ROW_FMAC("%[l]", 11, "%[y]")
        JQ_ROW_FMAC("%[m]", 12, "%[y]") JQ_ROW_FMAC("%[n]", 13, "%[y]") JQ_ROW_FMAC("%[o]", 14, "%[y]") JQ_ROW_FMAC("%[p]", 15, "%[y]")
        : [a] "+v"(v[0]), [b] "+v"(v[1]), [c] "+v"(v[2]), [d] "+v"(v[3]), [e] "+v"(v[4]), [f] "+v"(v[5]), [g] "+v"(v[6]),
          [h] "+v"(v[7]), [i] "+v"(v[8]), [j] "+v"(v[9]), [k] "+v"(v[10]), [l] "+v"(v[11]), [m] "+v"(v[12]), [n] "+v"(v[13]),
          [o] "+v"(v[14]), [p] "+v"(v[15]) : [x] "v"(x), [y] "v"(y));
}
#undef JQ_ROW_FMAC

// A game starts: nothing of the plies before. Rare, so a branch, not a selection in every ply.
template <int N> __device__ __forceinline__ void forget(float (&v)[N])
{
    asm volatile("");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
}
// The step that such a ply's decays are taken with: so small that no rate makes an infinity of
// them, which would make NaN of the zeros; of dt's sign, so that a rate of -infinity is none either.
__device__ __forceinline__ float no_step(float dt) { return copysignf(0x1p-126f, dt); }

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

// The arguments, read where they are used: held in scalar registers over a pass, those of
// a dozen tensors would be spilled to vector registers. `hidden` keeps the compiler from
// moving the reads up to the pass's start. The backward pass spills all the same (nine rows'
// cursors and steps, its flags): 202 scalars of bfloat16 and 16 states whose lanes all have
// a channel, 11 % of its vector instructions; 632 and 30 % where some have none, for then
// each state's check is a condition to keep, too.
typedef const __attribute__((address_space(4))) SelectArgs *SelectArgsPtr;
typedef const __attribute__((address_space(4))) jq_rows *RowsPtr;
__device__ __forceinline__ SelectArgsPtr hidden(SelectArgsPtr a)
{
    asm volatile("" : "+s"(a));
    return a;
}
__device__ __forceinline__ SelectArgsPtr select_arguments() { return (SelectArgsPtr)__builtin_amdgcn_kernarg_segment_ptr(); }

// Memory behind a wave's own address, at each lane's offset and one for the wave: a lane's
// offset of NOWHERE reads 0 and writes nothing, as all do where `really` is false.
constexpr uint32_t NOWHERE = 0x80000000u;
struct Window {
    char *base;
    template <class T> __device__ __forceinline__ T get(uint32_t at, uint32_t more = 0, bool really = true) const
    {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(base, 0, really ? (int)(NOWHERE - 1) : 0, 0x00020000);
        if constexpr (sizeof(T) == 2) return __builtin_bit_cast(T, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at, more, 0));
        else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(r, at, more, 0));
    }
    template <class T> __device__ __forceinline__ void put(uint32_t at, T x, uint32_t more = 0) const
    {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(base, 0, (int)(NOWHERE - 1), 0x00020000);
        if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, x), r, at, more, 0);
        else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), r, at, more, 0);
    }
};

// What a call has and wants, in one scalar register: a truth value of each would take two.
enum : uint32_t { HAS_SKIP = 1, HAS_GATE = 2, SOFTPLUS = 4, SAVES = 8, WANT_BC = 16, WANT_GATE = 32, WANT_U = 64, WANT_DELTA = 128 };
struct Has {
    uint32_t bits;
    __device__ __forceinline__ explicit Has(SelectArgsPtr a)
        : bits((a->skip ? HAS_SKIP : 0) | (a->gate.data ? HAS_GATE : 0) | (a->softplus ? SOFTPLUS : 0) | (a->saved ? SAVES : 0) |
               (a->want_bc ? WANT_BC : 0) | (a->dgate.data ? WANT_GATE : 0) | (a->du.data ? WANT_U : 0) | (a->ddelta.data ? WANT_DELTA : 0))
    {
        asm volatile("" : "+s"(bits));
    }
    __device__ __forceinline__ bool operator()(uint32_t what) const
    {
        uint32_t b = bits;
        asm volatile("" : "+s"(b));   // looked at anew each time
        return b & what;
    }
};

// A tensor's rows from ply t on; `step` bytes part two plies' rows. A chunk's rows are
// reached by 32-bit offsets: plies are less than SCAN_STEP bytes apart.
constexpr int64_t SCAN_STEP = 1 << 28;
struct PlyRows : Window {
    uint32_t step;
    template <class T> __device__ __forceinline__ PlyRows(T, RowsPtr r, int64_t b, int64_t t, int64_t h)
        : Window{static_cast<char *>(r->data) + (b * r->batch + t * r->ply + h * r->head) * (int64_t)sizeof(T)},
          step((uint32_t)r->ply * (uint32_t)sizeof(T)) {}
    __device__ __forceinline__ void on(int plies) { base += (uint64_t)step * plies; }
    __device__ __forceinline__ void back(int plies) { base -= (uint64_t)step * plies; }
};

// Where this wave's lanes are: channel, states, rows. EXACT: every lane has a channel and
// each of its states (one flag for both: 500 channels of 16 states take the states' checks
// as well, 160 against 134 us forward and 872 against 694 with gradients). MANY: a block's waves have the states of one wave's channels; else
// channels of their own, four waves a block so that each SIMD of a CU gets one (blocks of
// one wave leave some SIMDs with more waves than others).
template <class T, int NS, bool EXACT, bool MANY>
struct Place {
    int lane, sg, cw, part, parts,   // parts share the items (game, part of the axis)
         group, ch, n0, states;
    uint32_t at, row_at, at4;   // bytes into a row of channels, of a group's states, and of channels in float32
    bool on_;
    __device__ __forceinline__ Place(SelectArgsPtr a)
    {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64, CW = a->waves * a->groups;
        const int w = MANY ? blockIdx.x : blockIdx.x * waves + wave;
        lane = threadIdx.x % 64;
        sg = MANY ? wave : 0;
        cw = w % CW;
        part = w / CW;
        parts = a->parts;
        group = cw / a->waves;
        states = a->states;
        const int c = (cw % a->waves) * 64 + lane;
        on_ = c < a->per;
        ch = group * a->per + (on_ ? c : a->per - 1);
        n0 = sg * NS;
        const int n = n0 + lane % 16;
        at = on_ ? (uint32_t)ch * sizeof(T) : NOWHERE;
        at4 = on_ ? (uint32_t)ch * 4 : NOWHERE;
        row_at = lane % 16 < NS && n < a->states ? (uint32_t)n * sizeof(T) : NOWHERE;
    }
    __device__ __forceinline__ bool on() const { return EXACT || on_; }
    __device__ __forceinline__ bool has(int i) const { return EXACT || n0 + i < states; }
    // a, in powers of 2
    __device__ __forceinline__ void rates(SelectArgsPtr a, float (&A)[NS]) const
    {
#pragma unroll
        for (int i = 0; i < NS; ++i) A[i] = has(i) ? a->a[(int64_t)ch * states + n0 + i] * LOG2E : 0.f;
    }
};

// The same for the wave, which a load alone does not say.
__device__ __forceinline__ int live_plies(const int32_t *lengths, int b, int plies)
{
    return lengths ? min(max(__builtin_amdgcn_readfirstlane(lengths[b]), 0), plies) : plies;
}

// Where a game's plies start games. Bit k: one starts at ply t0 + k, k < 8; plies from
// `end` on are not looked at.
struct Starts {
    const uint8_t *row;
    int64_t step;
    __device__ __forceinline__ Starts(SelectArgsPtr a, int b) : row(a->starts ? a->starts + b * a->starts_batch : nullptr), step(a->starts_ply) {}
    __device__ __forceinline__ uint32_t at(int t0, int end, int lane) const
    {
        if (!row) return 0;
        const int k = lane & 7, t = min(t0 + k, end - 1);
        return __builtin_amdgcn_ballot_w64(row[t * step] != 0 && t0 + k < end) & 0xFF;
    }
};

// The states of this lane in a (.., channels, states) tensor's row, or in a (.., states, channels) one's.
template <class T, int NS, bool EXACT, bool MANY>
__device__ __forceinline__ void load_states(const Place<T, NS, EXACT, MANY> &p, float (&h)[NS], const float *row)
{
#pragma unroll
    for (int i = 0; i < NS; ++i) h[i] = row && p.has(i) ? row[(int64_t)p.ch * p.states + p.n0 + i] : 0.f;
}
template <class T, int NS, bool EXACT, bool MANY>
__device__ __forceinline__ void store_states(const Place<T, NS, EXACT, MANY> &p, const float (&h)[NS], float *row)
{
    if (p.on())
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (p.has(i)) row[(int64_t)p.ch * p.states + p.n0 + i] = h[i];
}
template <class T, int NS, bool EXACT, bool MANY>
__device__ __forceinline__ void load_apart(const Place<T, NS, EXACT, MANY> &p, float (&h)[NS], const float *row, int channels, bool really = true)
{
    const Window from{reinterpret_cast<char *>(const_cast<float *>(row))};
    uint32_t step = channels * 4, more = p.n0 * step;
    asm volatile("" : "+s"(step));   // its multiples are not worth registers over the pass
#pragma unroll
    for (int i = 0; i < NS; ++i, more += step) h[i] = p.has(i) ? from.get<float>(p.at4, more, really) : 0.f;
}
template <class T, int NS, bool EXACT, bool MANY>
__device__ __forceinline__ void store_apart(const Place<T, NS, EXACT, MANY> &p, const float (&h)[NS], float *row, int channels)
{
    const Window to{reinterpret_cast<char *>(row)};
    uint32_t step = channels * 4, more = p.n0 * step;
    asm volatile("" : "+s"(step));
#pragma unroll
    for (int i = 0; i < NS; ++i, more += step)
        if (p.has(i)) to.put(p.at4, h[i], more);
}

template <class T, int NS, bool EXACT, bool MANY, bool OUT>
__global__ __launch_bounds__(256) void k_scan_forward(SelectArgs)
{
    constexpr int K = SCAN_PLIES;
    extern __shared__ float lds[];   // more than one wave of states: [2][SG][K][64] shares of y
    const SelectArgsPtr a = hidden(select_arguments());
    const int SG = MANY ? blockDim.x / 64 : 1;
    const Place<T, NS, EXACT, MANY> p(a);
    float A[NS], h[NS];
    p.rates(a, A);
    const Has has(a);
    const float skip = a->skip ? a->skip[p.ch] : 0.f, bias = a->bias ? a->bias[p.ch] : 0.f;
    struct Raw { T u[K], delta[K], gate[K], b[K], c[K]; };
    const int items = a->batch * a->segments, channels = a->channels;
    const int64_t state_bytes = (int64_t)p.states * channels * 4;
    int turn = 0;
    if (p.part >= p.parts) return;
    for (int item = p.part; item < items; item += p.parts) {
        SelectArgsPtr q = hidden(a);
        const int b = item / q->segments, seg = item % q->segments;
        const int begin = seg * q->seg_plies, stop = min(begin + q->seg_plies, q->plies), end = min(stop, live_plies(q->lengths, b, q->plies));
        if (OUT && seg) load_apart(p, h, q->seg_state + (int64_t)item * p.states * channels, channels);
        else load_states(p, h, OUT && q->s_in ? q->s_in + (int64_t)b * channels * p.states : nullptr);
        float total = 0.f;
        const Starts game(q, b);
        PlyRows ru(T(), &q->u, b, begin, 0), rd(T(), &q->delta, b, begin, 0), rz(T(), &q->gate, b, begin, 0), rb(T(), &q->b, b, begin, p.group),
            rc(T(), &q->c, b, begin, p.group), ro(T(), &q->out, b, begin, 0);
        Window save{reinterpret_cast<char *>(q->saved) + ((int64_t)b * ((q->plies + SCAN_CHUNK - 1) / SCAN_CHUNK) + begin / SCAN_CHUNK) * state_bytes};
        auto fetch = [&](int t0, Raw &r, uint32_t &starts) {
            const int last = end - 1 - t0;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const uint32_t at = min(k, last);   // behind the end the last row again
                r.u[k] = ru.get<T>(p.at, at * ru.step);
                r.delta[k] = rd.get<T>(p.at, at * rd.step);
                if (OUT && has(HAS_GATE)) r.gate[k] = rz.get<T>(p.at, at * rz.step);
                r.b[k] = rb.get<T>(p.row_at, at * rb.step);
                if (OUT) r.c[k] = rc.get<T>(p.row_at, at * rc.step);
            }
            ru.on(K), rd.on(K), rz.on(K), rb.on(K), rc.on(K);
            starts = game.at(t0, end, p.lane);
        };
        Raw next;
        uint32_t next_starts = 0;
        if (begin < end) fetch(begin, next, next_starts);
        for (int t0 = begin; t0 < end; t0 += K) {
            const Raw r = next;
            const uint32_t starts = next_starts;
            if (t0 + K < end) fetch(t0 + K, next, next_starts);
            if (OUT && has(SAVES) && t0 % SCAN_CHUNK == 0) {
                store_apart(p, h, reinterpret_cast<float *>(save.base), channels);
                save.base += state_bytes;
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (t0 + k >= end) break;
                const float u = (float)r.u[k], pre = (float)r.delta[k] + bias;
                float dt = has(SOFTPLUS) ? softplus(pre) : pre;
                const float push = dt * u, bt = (float)r.b[k];
                if (!OUT) total += dt;
                if (starts >> k & 1) {
                    forget(h);
                    dt = no_step(dt);
                    if (!OUT) total = __builtin_nanf("");
                }
#pragma unroll
                for (int i = 0; i < NS; ++i) h[i] *= exp2_fast(dt * A[i]);
                row_add(h, bt, push);
#pragma unroll
                for (int i = 0; i < NS; ++i)
                    if (!p.has(i)) h[i] = 0.f;
                if (!OUT) continue;
                const float y = row_dot(0.f, (float)r.c[k], h);
                if (MANY) lds[(((turn & 1) * SG + p.sg) * K + k) * 64 + p.lane] = y;
                else {
                    float o = has(HAS_SKIP) ? fmaf(skip, u, y) : y;
                    if (OUT && has(HAS_GATE)) o *= (float)r.gate[k] * sigmoid((float)r.gate[k]);
                    ro.put<T>(p.at, from_float<T>(o), k * ro.step);
                }
            }
            if (!OUT) continue;
            if (!MANY) {
                ro.on(K);
                continue;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (t0 + k >= end) break;
                if (k % SG == p.sg) {
                    float o = 0.f;
                    for (int g = 0; g < SG; ++g) o += lds[(((turn & 1) * SG + g) * K + k) * 64 + p.lane];
                    if (has(HAS_SKIP)) o = fmaf(skip, (float)r.u[k], o);
                    if (OUT && has(HAS_GATE)) o *= (float)r.gate[k] * sigmoid((float)r.gate[k]);
                    ro.put<T>(p.at, from_float<T>(o), k * ro.step);
                }
            }
            ro.on(K);
            ++turn;   // the other buffer: the one before is read by then
        }
        q = hidden(a);
        if (OUT) {
            for (int t = max(begin, end); t < stop; ++t)
                if (t % SG == p.sg) PlyRows(T(), &q->out, b, t, 0).template put<T>(p.at, T(0.f));
            if (q->s_out && seg == q->segments - 1) store_states(p, h, q->s_out + (int64_t)b * channels * p.states);
        } else {
            store_apart(p, h, q->seg_state + (int64_t)item * p.states * channels, channels);
            if (p.sg == 0 && p.on()) q->seg_sum[(int64_t)item * channels + p.ch] = total;
        }
    }
}

// h 2^x as the product of what is returned, h times a whole power, and frac, in [1, 2). The
// power of a whole part, 64 plies or more, may be past either end of float32 where each
// ply's is a common number: so it is never taken by itself. 0 stays 0 and an infinity one
// behind any power, a tiny h grows, and a large one decays to 0. Past 2^+-1024 nothing
// but 0 and the infinities is left of any h.
__device__ __forceinline__ float times_power(float h, float x, float &frac)
{
    x = fminf(fmaxf(x, -1024.f), 1024.f);
    const float whole = floorf(x);
    frac = exp2_fast(x - whole);
    return ldexpf(h, (int)whole);
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
        // parts are asked for AHEAD at a time: one after the other, each waits for the last
        constexpr int AHEAD = 16;
        float *first = a.seg_state + (b * a.segments + (BACK ? a.segments - 1 : 0)) * step + (int64_t)n * a.channels + ch;
        const float *sums = a.seg_sum + (b * a.segments + (BACK ? a.segments - 1 : 0)) * a.channels + ch;
        const int64_t by = BACK ? -step : step, sum_by = BACK ? -a.channels : a.channels;
        for (int s0 = 0; s0 < a.segments; s0 += AHEAD) {
            float add[AHEAD], keep[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int s = min(s0 + k, a.segments - 1);
                add[k] = first[s * by], keep[k] = sums[s * sum_by];
            }
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                if (s0 + k >= a.segments) break;
                float frac;
                first[(s0 + k) * by] = h;
                h = keep[k] != keep[k] ? add[k] : fmaf(times_power(h, keep[k] * A, frac), frac, add[k]);
            }
        }
    }
}

// Backward over a part of the axis: what its gradients of y send to the state before it
// (seg_state, seg_sum), in reverse.
template <class T, int NS, bool EXACT, bool MANY>
__global__ __launch_bounds__(256) void k_scan_carry(SelectArgs)
{
    constexpr int K = SCAN_CHUNK;
    const SelectArgsPtr a = hidden(select_arguments());
    const int items = a->batch * a->segments, channels = a->channels;
    const Place<T, NS, EXACT, MANY> p(a);
    if (p.part >= p.parts) return;
    float A[NS], dh[NS];
    p.rates(a, A);
    const Has has(a);
    const float bias = a->bias ? a->bias[p.ch] : 0.f;
    for (int item = p.part; item < items; item += p.parts) {
        SelectArgsPtr q = hidden(a);
        const int b = item / q->segments, seg = item % q->segments;
        const int begin = seg * q->seg_plies, end = min(min(begin + q->seg_plies, q->plies), live_plies(q->lengths, b, q->plies));
#pragma unroll
        for (int i = 0; i < NS; ++i) dh[i] = 0.f;
        float total = 0.f;
        const int top = begin + (max(end - begin, 1) - 1) / K * K;
        for (int t0 = top; t0 >= begin && begin < end; t0 -= K) {
            T delta[K], gate[K], d_out[K], c[K];
            q = hidden(a);
            const uint32_t starts = Starts(q, b).at(t0, end, p.lane);
            const PlyRows rd(T(), &q->delta, b, t0, 0), rz(T(), &q->gate, b, t0, 0), rg(T(), &q->d_out, b, t0, 0), rc(T(), &q->c, b, t0, p.group);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const uint32_t at = min(k, end - 1 - t0);
                delta[k] = rd.get<T>(p.at, at * rd.step);
                d_out[k] = rg.get<T>(p.at, at * rg.step);
                if (has(HAS_GATE)) gate[k] = rz.get<T>(p.at, at * rz.step);
                c[k] = rc.get<T>(p.row_at, at * rc.step);
            }
#pragma unroll
            for (int k = K - 1; k >= 0; --k) {
                if (t0 + k >= end) continue;
                const float pre = (float)delta[k] + bias, dt = has(SOFTPLUS) ? softplus(pre) : pre;
                float dy = (float)d_out[k];
                if (has(HAS_GATE)) dy *= (float)gate[k] * sigmoid((float)gate[k]);
                row_add(dh, (float)c[k], dy);
#pragma unroll
                for (int i = 0; i < NS; ++i) dh[i] = p.has(i) ? dh[i] * exp2_fast(dt * A[i]) : 0.f;
                total += dt;
                if (starts >> k & 1) {
                    forget(dh);
                    total = __builtin_nanf("");
                }
            }
        }
        q = hidden(a);
        store_apart(p, dh, q->seg_state + (int64_t)item * p.states * channels, channels);
        if (p.sg == 0 && p.on()) q->seg_sum[(int64_t)item * channels + p.ch] = total;
    }
}

// Backward, chunks of 8 plies from the last one on: the states of a chunk again, from the
// saved one before it, into registers; then its gradients in reverse. With dh the gradient
// of h_t from all that follows:
//   dh += c dy;  db = sum over channels of dh dt u;  dc = sum over channels of dy h;
//   through = sum over n of b dh;  dh = exp(dt a) dh;  w = dh h_{t-1};  da += w dt;
//   du = dt through + skip dy;  ddt = u through + sum over n of w a
// MANY: more than one wave of states, whose shares of y, through and the sum of w a meet in
// LDS. Registers are what it is short of: two waves a SIMD leave 256, of which 96 hold six
// plies' states of 16 (the first two plies' wait in LDS), so the way back reads its rows
// again (from the caches), and the next chunk's are asked for when half of the states are
// done with.
template <class T, int NS, bool EXACT, bool MANY>
__global__ __launch_bounds__(256, 2) void k_scan_backward(SelectArgs)
{
    extern __shared__ float lds[];   // [waves][FAR][NS / 4][64][4] states, then, of MANY, [3][SG][8][64] shares
    constexpr int K = SCAN_CHUNK, FAR = scan_far(NS);
    const SelectArgsPtr a = hidden(select_arguments());
    const int SG = MANY ? blockDim.x / 64 : 1;
    const Place<T, NS, EXACT, MANY> p(a);
    if (p.part >= p.parts) return;   // never of MANY: its waves meet
    float A[NS], dA[NS], dh[NS];
    p.rates(a, A);
#pragma unroll
    for (int i = 0; i < NS; ++i) dA[i] = 0.f;
    const Has has(a);
    const float skip = a->skip ? a->skip[p.ch] : 0.f, bias = a->bias ? a->bias[p.ch] : 0.f;
    float dskip = 0.f, dbias = 0.f;
    const int items = a->batch * a->segments, channels = a->channels;
    const int sum_n = p.n0 + p.lane / (64 / NS);
    const uint32_t sum_at = p.lane % (64 / NS) == 0 && (EXACT || sum_n < p.states) ? sum_n * 4 : NOWHERE;
    struct Raw { T u[K], delta[K], gate[K], d_out[K], b[K], c[K]; };
    float *const far = lds + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * FAR * NS * 64, *const shares = lds + SG * FAR * NS * 64;
    auto share = [&](int j, int g, int k) -> float & { return shares[((j * SG + g) * K + k) * 64 + p.lane]; };
    for (int item = p.part; item < items; item += p.parts) {
        SelectArgsPtr q = hidden(a);
        const int b = item / q->segments, seg = item % q->segments;
        const int begin = seg * q->seg_plies, stop = min(begin + q->seg_plies, q->plies), end = min(stop, live_plies(q->lengths, b, q->plies));
        if (q->segments > 1) load_apart(p, dh, q->seg_state + (int64_t)item * p.states * channels, channels);
        else load_states(p, dh, q->d_final ? q->d_final + (int64_t)b * channels * p.states : nullptr);
        for (int t = max(begin, end) + p.sg; t < stop; t += SG) {
            if (has(WANT_U)) PlyRows(T(), &q->du, b, t, 0).template put<T>(p.at, T(0.f));
            if (has(WANT_DELTA)) PlyRows(T(), &q->ddelta, b, t, 0).template put<T>(p.at, T(0.f));
            if (has(WANT_GATE)) PlyRows(T(), &q->dgate, b, t, 0).template put<T>(p.at, T(0.f));
        }
        const int top = begin + (max(end - begin, 1) - 1) / K * K;
        const Starts game(q, b);
        PlyRows ru(T(), &q->u, b, top, 0), rd(T(), &q->delta, b, top, 0), rz(T(), &q->gate, b, top, 0), rg(T(), &q->d_out, b, top, 0),
            rb(T(), &q->b, b, top, p.group), rc(T(), &q->c, b, top, p.group), to_u(T(), &q->du, b, top, 0), to_delta(T(), &q->ddelta, b, top, 0),
            to_gate(T(), &q->dgate, b, top, 0);
        const int64_t state_bytes = (int64_t)p.states * channels * 4, sum_step = (int64_t)q->groups * 2 * p.states * 4;
        const char *saved = reinterpret_cast<const char *>(q->saved) + ((int64_t)b * ((q->plies + K - 1) / K) + top / K) * state_bytes;
        Window sums{reinterpret_cast<char *>(q->part_bc) + (((int64_t)(p.cw % q->waves) * q->batch + b) * q->plies + top) * sum_step +
                    (int64_t)p.group * 2 * p.states * 4};
        // the rows of the chunk `plies` before the one at hand, whose first ply is t0; nothing is read where not `really`
        auto load = [&](int t0, int plies, Raw &r, uint32_t &starts, bool really) {
            PlyRows lu = ru, ld = rd, lz = rz, lg = rg, lb = rb, lc = rc;
            lu.back(plies), ld.back(plies), lz.back(plies), lg.back(plies), lb.back(plies), lc.back(plies);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const uint32_t at = min(k, end - 1 - t0);   // behind the end the last row again
                r.u[k] = lu.get<T>(p.at, at * lu.step, really);
                r.delta[k] = ld.get<T>(p.at, at * ld.step, really);
                r.d_out[k] = lg.get<T>(p.at, at * lg.step, really);
                if (has(HAS_GATE)) r.gate[k] = lz.get<T>(p.at, at * lz.step, really);
                r.b[k] = lb.get<T>(p.row_at, at * lb.step, really);
                r.c[k] = lc.get<T>(p.row_at, at * lc.step, really);
            }
            starts = really ? game.at(t0, end, p.lane) : 0;
        };
        // the gradient of a gate and the ones of u and delta, their rows as they lie in memory
        auto give_gate = [&](const PlyRows &to, int k, T u, T gate, T d_out, float y) {
            const float z = (float)gate, s = sigmoid(z);
            to.put<T>(p.at, from_float<T>((float)d_out * (has(HAS_SKIP) ? fmaf(skip, (float)u, y) : y) * s * fmaf(z, 1.f - s, 1.f)), k * to.step);
        };
        auto give = [&](const PlyRows &to_u, const PlyRows &to_delta, int k, T u, T delta, float dt, float dy, float s1, float s2) {
            float d_pre = fmaf(s1, (float)u, s2 * LN2);
            if (has(SOFTPLUS)) d_pre *= sigmoid((float)delta + bias);
            if (p.on()) {   // lanes without a channel have read zeros: their sums are not looked at
                dbias += d_pre;
                dskip = fmaf(dy, (float)u, dskip);
            }
            if (has(WANT_U)) to_u.put<T>(p.at, from_float<T>(has(HAS_SKIP) ? fmaf(s1, dt, skip * dy) : s1 * dt), k * to_u.step);
            if (has(WANT_DELTA)) to_delta.put<T>(p.at, from_float<T>(d_pre), k * to_delta.step);
        };
        Raw next;
        float h[NS];
        uint32_t next_starts = 0;
        if (begin < end) {
            load(top, 0, next, next_starts, true);
            load_apart(p, h, reinterpret_cast<const float *>(saved), channels);
        }
        // the chunk from ply t0 on; whole: K plies
        auto chunk = [&](int t0, auto whole) {
            const uint32_t starts = next_starts;
            const int count = whole ? K : min(end - t0, K);
            float hist[K - FAR][NS], dt[K], dy[K];
            {
                Window to{sums.base + p.states * 4};
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (k >= count) break;
                    const float pre = (float)next.delta[k] + bias, bt = (float)next.b[k], u = (float)next.u[k];
                    dt[k] = has(SOFTPLUS) ? softplus(pre) : pre;
                    dy[k] = (float)next.d_out[k];
                    if (has(HAS_GATE)) dy[k] *= (float)next.gate[k] * sigmoid((float)next.gate[k]);
                    float step = dt[k];
                    if (starts >> k & 1) {
                        forget(h);
                        step = no_step(step);
                    }
                    const float push = dt[k] * u;
                    float v[NS];
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        if (k < FAR) far[(k * NS + i / 4 * 4) * 64 + p.lane * 4 + i % 4] = h[i];
                        else hist[k < FAR ? 0 : k - FAR][i] = h[i];
                    }
#pragma unroll
                    for (int i = 0; i < NS; ++i) h[i] *= exp2_fast(step * A[i]);
                    row_add(h, bt, push);
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        if (!p.has(i)) h[i] = 0.f;
                        v[i] = p.on() ? dy[k] * h[i] : 0.f;
                    }
                    if (has(WANT_GATE)) {
                        const float y = row_dot(0.f, (float)next.c[k], h);
                        if (MANY) share(0, p.sg, k) = y;
                        else give_gate(to_gate, k, next.u[k], next.gate[k], next.d_out[k], y);
                    }
                    if (has(WANT_BC)) {
                        to.put(sum_at, lane_sums<NS>(v));
                        to.base += sum_step;
                    }
                }
            }
            {
                Window to{sums.base + (count - 1) * sum_step};
                const uint32_t last = count - 1;
                T u = ru.get<T>(p.at, last * ru.step), delta = rd.get<T>(p.at, last * rd.step), bb = rb.get<T>(p.row_at, last * rb.step),
                  cc = rc.get<T>(p.row_at, last * rc.step);
#pragma unroll
                for (int k = K - 1; k >= 0; --k) {
                    if (k == K / 2 - 1) {
                        load(t0 - K, K, next, next_starts, t0 > begin);
                        load_apart(p, h, reinterpret_cast<const float *>(saved - state_bytes), channels, t0 > begin);
                    }
                    if (k >= count) continue;
                    const T u0 = u, delta0 = delta, b0 = bb, c0 = cc;
                    if (k) {
                        const uint32_t at = k - 1;
                        u = ru.get<T>(p.at, at * ru.step), delta = rd.get<T>(p.at, at * rd.step), bb = rb.get<T>(p.row_at, at * rb.step);
                        cc = rc.get<T>(p.row_at, at * rc.step);
                    }
                    asm("" : "+v"(dt[k]));   // the decays once more: kept from the way there they would take 128 registers
                    const float push = dt[k] * (float)u0;
                    row_add(dh, (float)c0, dy[k]);
                    float v[NS];
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        if (!p.has(i)) dh[i] = 0.f;
                        v[i] = p.on() ? dh[i] * push : 0.f;
                    }
                    const float s1 = row_dot(0.f, (float)b0, dh);
                    float s2 = 0.f;
                    if (has(WANT_BC)) {
                        to.put(sum_at, lane_sums<NS>(v));
                        to.base -= sum_step;
                    }
                    if (starts >> k & 1) forget(dh);
                    else {
#pragma unroll
                        for (int i = 0; i < NS; ++i) {
                            dh[i] *= exp2_fast(dt[k] * A[i]);
                            const float w = dh[i] * (k < FAR ? far[(k * NS + i / 4 * 4) * 64 + p.lane * 4 + i % 4] : hist[k < FAR ? 0 : k - FAR][i]);
                            s2 = fmaf(w, A[i], s2);
                            dA[i] = fmaf(w, dt[k], dA[i]);
                        }
                    }
                    if (MANY) share(1, p.sg, k) = s1, share(2, p.sg, k) = s2;
                    else give(to_u, to_delta, k, u0, delta0, dt[k], dy[k], s1, s2);
                }
            }
            if constexpr (MANY) {
                __syncthreads();
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (k >= count) break;
                    if (k % SG != p.sg) continue;
                    float all[3] = {0.f, 0.f, 0.f};
                    for (int g = 0; g < SG; ++g) {
                        if (has(WANT_GATE)) all[0] += share(0, g, k);
                        all[1] += share(1, g, k);
                        all[2] += share(2, g, k);
                    }
                    const T u = ru.get<T>(p.at, k * ru.step);
                    if (has(WANT_GATE)) give_gate(to_gate, k, u, rz.get<T>(p.at, k * rz.step), rg.get<T>(p.at, k * rg.step), all[0]);
                    give(to_u, to_delta, k, u, rd.get<T>(p.at, k * rd.step), dt[k], dy[k], all[1], all[2]);
                }
                __syncthreads();   // the next chunk's shares take their place
            }
            ru.back(K), rd.back(K), rz.back(K), rg.back(K), rb.back(K), rc.back(K), to_u.back(K), to_delta.back(K), to_gate.back(K);
            saved -= state_bytes;
            sums.base -= K * sum_step;
        };
        if (begin < end) {
            // only the last chunk may have fewer plies: the others take code without a way round each
            int t0 = top;
            if (end - top < K) chunk(t0, std::false_type()), t0 -= K;
            for (; t0 >= begin; t0 -= K) chunk(t0, std::true_type());
        }
        if (seg == 0) {
            float *to = hidden(a)->d_initial;
            if (to) store_states(p, dh, to + (int64_t)b * channels * p.states);
        }
    }
    const SelectArgsPtr q = hidden(a);
    if (!q->want_a) return;
    if constexpr (MANY) {   // each wave has some plies' share of dskip and dbias
        __syncthreads();
        share(0, p.sg, 0) = dskip;
        share(1, p.sg, 0) = dbias;
        __syncthreads();
        dskip = dbias = 0.f;
        for (int g = 0; g < SG; ++g) {
            dskip += share(0, g, 0);
            dbias += share(1, g, 0);
        }
    }
    float *to = q->part_a + (int64_t)p.part * (p.states + 2) * channels;
    store_apart(p, dA, to, channels);
    if (p.sg == 0 && p.on()) {
        to[(int64_t)p.states * channels + p.ch] = dskip;
        to[(int64_t)(p.states + 1) * channels + p.ch] = dbias;
    }
}

// db and dc: the waves' shares summed in a fixed order; 0 from a game's length on. N values
// a thread, which lie together: states is a multiple of N.
template <class T, int N>
__global__ __launch_bounds__(256) void k_scan_join_bc(SelectArgs a, jq_rows db, jq_rows dc)
{
    typedef float V __attribute__((ext_vector_type(N)));
    const int n2 = 2 * a.states / N;
    const int64_t tokens = (int64_t)a.batch * a.plies, all = tokens * a.groups * n2;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t of = i / n2, token = of / a.groups, b = token / a.plies;
        const int j = (int)(i - of * n2) * N, g = (int)(of - token * a.groups), t = (int)(token - b * a.plies);
        const int len = a.lengths ? min(max(a.lengths[b], 0), a.plies) : a.plies;
        V s{};
        if (t < len)
#pragma unroll 4
            for (int w = 0; w < a.waves; ++w) s += reinterpret_cast<const V *>(a.part_bc)[w * all + i];
        const jq_rows &r = j < a.states ? db : dc;
        if (!r.data) continue;
        T *to = row_at<T>(r, b, t, g) + (j < a.states ? j : j - a.states);
#pragma unroll
        for (int e = 0; e < N; ++e) to[e] = from_float<T>(s[e]);
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

// L lanes a channel, four states each. Bound by the states, read and written once: a wave
// walks games with its channels' a in registers and the next game's state, rows and flags
// on their way; the states of calls that the caches would not hold to the next ply go past
// them.
template <class T, int L, bool STREAM>
__global__ __launch_bounds__(256) void k_scan_step(SelectStepArgs a, int channel_waves, int at_once)
{
    constexpr int PER = 64 / L;
    typedef f32x4 At __attribute__((aligned(4)));
    const int lane = threadIdx.x % 64;
    const int wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    if (wave >= channel_waves * at_once) return;
    const int cw = wave % channel_waves;
    const int ch = cw * PER + lane / L, n = lane % L * 4, left = min(a.states - n, 4);
    const bool on = ch < a.channels, mine = on && left > 0;
    const int at = on ? ch : a.channels - 1, group = at / a.per;
    float A[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) A[e] = mine && e < left ? a.a[(int64_t)at * a.states + n + e] * LOG2E : 0.f;
    const float skip = a.skip ? a.skip[at] : 0.f, bias = a.bias ? a.bias[at] : 0.f;
    struct Game { int64_t row; f32x4 h; T b[4], c[4], u, delta, gate; bool start, there; };
    auto load = [&](int game, Game &g) {
        g.row = a.rows ? a.rows[game] : game;
        g.there = g.row >= 0 && g.row < a.state_rows;
        g.start = a.starts && a.starts[game];
        g.u = row_at<const T>(a.u, game, 0, 0)[at];
        g.delta = row_at<const T>(a.delta, game, 0, 0)[at];
        if (a.gate.data) g.gate = row_at<const T>(a.gate, game, 0, 0)[at];
        const T *pb = row_at<const T>(a.b, game, 0, group) + n, *pc = row_at<const T>(a.c, game, 0, group) + n;
        g.h = f32x4{};
#pragma unroll
        for (int e = 0; e < 4; ++e) g.b[e] = g.c[e] = T(0.f);
        if (!mine) return;
        const float *s = a.state + (g.row * a.channels + at) * a.states + n;
        if (left >= 4) {
            if (g.there) g.h = STREAM ? __builtin_nontemporal_load(reinterpret_cast<const At *>(s)) : *reinterpret_cast<const At *>(s);
            const typename Pack<T, 4>::type vb = load_some<T, 4>(pb, 4), vc = load_some<T, 4>(pc, 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) g.b[e] = vb[e], g.c[e] = vc[e];
        } else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < left) {
                    if (g.there) g.h[e] = s[e];
                    g.b[e] = pb[e], g.c[e] = pc[e];
                }
    };
    int game = wave / channel_waves;
    Game next;
    if (game < a.batch) load(game, next);
    for (; game < a.batch; game += at_once) {
        const Game g = next;
        if (game + at_once < a.batch) load(game + at_once, next);
        T *out = row_at<T>(a.out, game, 0, 0) + at;
        if (!g.there) {
            if (on && n == 0) *out = T(0.f);
            continue;
        }
        const float u = (float)g.u, pre = (float)g.delta + bias, dt = a.softplus ? softplus(pre) : pre, push = dt * u;
        f32x4 h;
        float y = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float old = g.start ? 0.f : exp2_fast(dt * A[e]) * g.h[e];
            h[e] = fmaf((float)g.b[e], push, old);
            if (e < left) y = fmaf((float)g.c[e], h[e], y);
        }
        if (mine) {
            float *s = a.state + (g.row * a.channels + at) * a.states + n;
            if (left >= 4) {
                if (STREAM) __builtin_nontemporal_store(h, reinterpret_cast<At *>(s));
                else *reinterpret_cast<At *>(s) = h;
            } else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < left) s[e] = h[e];
        }
        y = group_total<L>(y);
        if (a.skip) y = fmaf(skip, u, y);
        if (a.gate.data) y *= (float)g.gate * sigmoid((float)g.gate);
        if (on && n == 0) *out = from_float<T>(y);
    }
}

}  // namespace jq
