// C entry points of the operators of a policy's memory over plies: linear
// attention, rotary positions, layer norm. Declarations and contracts live in
// include/junqi_amd.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "junqi_amd.h"
#include "jq_error.h"
#include "jq_memory.h"
#include "jq_attention.h"
#include "jq_rotary.h"
#include "jq_norm.h"

using namespace jq;

namespace {

hipStream_t strm(void *s) { return reinterpret_cast<hipStream_t>(s); }

// Calls over more bytes than that go past the caches, which would not hold them to
// their next use; what smaller ones touch is found there. One ply, 4 heads of 64 x 64
// in bfloat16, through the caches / past them: 1,024 games (67 MB of states) 24.5 /
// 26.0 us, 4,096 (268 MB) 83.8 / 95.8, 8,192 (537 MB) 211 / 190, 32,768 846 / 749
// (5.7 TB/s). Segments of 256 plies, 4 heads of 64, forward, the same rows again: 512
// games (268 MB) 56 / 64 us, 1,024 135 / 126.
constexpr int64_t STREAM_BYTES = 400ll << 20;

int check_dtype(int32_t dtype)
{
    if (dtype != JQ_F32 && dtype != JQ_BF16) return fail(JQ_E_ARG, "element type %d is neither JQ_F32 nor JQ_BF16", dtype);
    return JQ_OK;
}

size_t elem_bytes(int32_t dtype) { return dtype == JQ_F32 ? 4 : 2; }

bool aligned(const void *p, size_t to) { return (uintptr_t)p % to == 0; }

int check_rows(const jq_rows &r, int32_t dtype, const char *name)
{
    if (!r.data) return fail(JQ_E_ARG, "null %s", name);
    if (!aligned(r.data, elem_bytes(dtype))) return fail(JQ_E_ARG, "%s must be aligned to its element size", name);
    return JQ_OK;
}

#define TRY(expr)                  \
    do {                           \
        const int rc_ = (expr);    \
        if (rc_) return rc_;       \
    } while (0)

int check_dims(int32_t batch, int32_t heads, int32_t dk, int32_t dv)
{
    if (batch < 0 || heads <= 0) return fail(JQ_E_ARG, "bad shapes (batch %d, heads %d)", batch, heads);
    if (dk <= 0 || dv <= 0 || dk > JQ_ATTENTION_MAX_DIM || dv > JQ_ATTENTION_MAX_DIM)
        return fail(JQ_E_ARG, "key_dim %d and value_dim %d must be in [1, %d]", dk, dv, JQ_ATTENTION_MAX_DIM);
    if ((int64_t)batch * heads >= 1 << 23)   // a launch holds fewer than 2^32 threads
        return fail(JQ_E_ARG, "batch * heads %lld is too large", (long long)batch * heads);
    return JQ_OK;
}

int check_attention(const jq_attention *a)
{
    if (!a) return fail(JQ_E_ARG, "null arguments");
    TRY(check_dtype(a->dtype));
    TRY(check_dims(a->batch, a->heads, a->key_dim, a->value_dim));
    if (a->plies < 0 || a->plies > INT_MAX - 1024) return fail(JQ_E_ARG, "plies %d out of range", a->plies);
    return JQ_OK;
}

int check_attention_inputs(const jq_attention *a)
{
    if (!a->log_decay) return fail(JQ_E_ARG, "null log_decay");
    if (a->plies == 0) return JQ_OK;
    TRY(check_rows(a->q, a->dtype, "q"));
    TRY(check_rows(a->k, a->dtype, "k"));
    return check_rows(a->v, a->dtype, "v");
}

// Whether a pass may take r's rows as whole aligned vectors of `bytes` through a
// buffer descriptor of `plies` of them: no two rows share bytes, and they span less
// than 2 GiB.
bool whole_vectors(const jq_rows &r, int dim, size_t elem, size_t bytes, int plies)
{
    const int64_t n = (int64_t)(bytes / elem);
    return aligned(r.data, bytes) && dim % n == 0 && r.batch % n == 0 && r.ply % n == 0 && r.head % n == 0 &&
           r.ply >= dim && r.ply < ((int64_t)1 << 31) / (int64_t)elem / (plies + 1);
}

// The states before the segments of a split axis.
template <class T, int D, bool REV, bool FAST>
int launch_states(const ScanArgs &s, hipStream_t stream)
{
    const int heads = s.batch * s.heads;
    if (s.segments < 2) return JQ_OK;
    hipLaunchKernelGGL((k_attention_pass<T, D, REV, FAST, false>), dim3(heads, s.segments - 1), dim3(64 * pass_waves(D)), 0, stream, s);
    TRY(launch_check("k_attention_pass (states)"));
    hipLaunchKernelGGL(k_attention_join<REV>, dim3(heads, (s.kd * s.vd + 255) / 256), dim3(256), 0, stream, s);
    return launch_check("k_attention_join");
}

template <class T, int D, bool REV, bool FAST>
int launch_pass(const ScanArgs &s, hipStream_t stream)
{
    hipLaunchKernelGGL((k_attention_pass<T, D, REV, FAST, true>), dim3(s.batch * s.heads, s.segments),
                       dim3(64 * pass_waves(D)), 0, stream, s);
    return launch_check("k_attention_pass");
}

template <class T, int D, bool FAST>
int launch_kv(const GradArgs &g, hipStream_t stream)
{
    TRY((launch_states<T, D, true, FAST>(g.scan, stream)));
    if constexpr (D == 128) {
        // both passes' waves in one block would have half the registers that they need
        TRY((launch_pass<T, D, true, FAST>(g.scan, stream)));
        ScanArgs s = g.scan;
        s.q = g.values, s.k = g.scan.v, s.v = g.scan.k, s.o = g.dk;
        s.kd = g.scan.vd, s.vd = g.scan.kd;
        s.s_row = 1, s.s_col = s.kd, s.s_out = nullptr;
        s.seg_row = 1, s.seg_col = s.kd;
        return launch_pass<T, D, true, FAST>(s, stream);
    } else {
        hipLaunchKernelGGL((k_attention_kv<T, D, FAST>), dim3(g.scan.batch * g.scan.heads, g.scan.segments),
                           dim3(128 * pass_waves(D)), 0, stream, g);
        return launch_check("k_attention_kv");
    }
}

// Whether a pass may take all of these as whole vectors.
template <class T>
bool all_whole(std::initializer_list<std::pair<const jq_rows *, int>> rows, size_t bytes)
{
    for (const auto &r : rows)
        if (!whole_vectors(*r.first, r.second, sizeof(T), bytes, Mma<T>::KB)) return false;
    return true;
}

template <class T, int D>
int scan_width(const ScanArgs &s, hipStream_t stream)
{
    const bool fast = all_whole<T>({{&s.q, s.kd}, {&s.k, s.kd}, {&s.v, s.vd}}, 16) && all_whole<T>({{&s.o, s.vd}}, 16);
    if (fast) {
        TRY((launch_states<T, D, false, true>(s, stream)));
        return launch_pass<T, D, false, true>(s, stream);
    }
    TRY((launch_states<T, D, false, false>(s, stream)));
    return launch_pass<T, D, false, false>(s, stream);
}

template <class T, int D>
int kv_width(const GradArgs &g, hipStream_t stream)
{
    const ScanArgs &s = g.scan;
    const bool fast = all_whole<T>({{&s.q, s.kd}, {&s.k, s.kd}, {&s.v, s.vd}, {&g.values, s.vd}}, 16) &&
                      all_whole<T>({{&s.o, s.vd}, {&g.dk, s.kd}}, 16);
    return fast ? launch_kv<T, D, true>(g, stream) : launch_kv<T, D, false>(g, stream);
}

// The pass forward in time for its wider dim.
template <class T>
int scan_as(const ScanArgs &s, hipStream_t stream)
{
    const int d = std::max(s.kd, s.vd);
    return d <= 32 ? scan_width<T, 32>(s, stream) : d <= 64 ? scan_width<T, 64>(s, stream) : scan_width<T, 128>(s, stream);
}
int scan(int32_t dtype, const ScanArgs &s, hipStream_t stream)
{
    return dtype == JQ_F32 ? scan_as<float>(s, stream) : scan_as<bf16>(s, stream);
}

template <class T>
int scan_kv_as(const GradArgs &g, hipStream_t stream)
{
    const int d = std::max(g.scan.kd, g.scan.vd);
    return d <= 32 ? kv_width<T, 32>(g, stream) : d <= 64 ? kv_width<T, 64>(g, stream) : kv_width<T, 128>(g, stream);
}
int scan_kv(int32_t dtype, const GradArgs &g, hipStream_t stream)
{
    return dtype == JQ_F32 ? scan_kv_as<float>(g, stream) : scan_kv_as<bf16>(g, stream);
}

// How a call's plies are split: few games and heads, a block each, leave the card's 256
// CUs idle unless parts of a long axis run side by side, at the price of reading k and v
// twice, of the states between and of two more launches. Split / in one piece, us:
//                   forward, plies                     with the gradients
//   heads      blocks   512     1,024     8,192         512       1,024       8,192
//   128 bf16     64    40/48    60/90    286/694      165/192    228/360   1,037/2,753
//                96    59/48    83/90    417/696      213/191    302/360   1,531/2,763
//               128    62/48    90/90    525/696      226/194    337/361   1,906/2,768
//   128 f32     128   115/128  200/250 1,376/1,966    431/511    747/1,003 5,156/7,876
//    64 bf16    128    34/35    38/63    209/473      161/135    156/198     700/1,469
//               192    37/35    58/64    284/475      160/136    191/198     980/1,470
//               256    39/35    71/64    357/474      162/136    238/199   1,249/1,474
//    64 f32     192    59/76    98/147   581/1,131    202/228    334/444   2,009/3,473
//               256    76/75   121/146   761/1,135    259/230    409/445   2,619/3,490
//    32 bf16    256    25/26    41/48    329/349      160/130    157/151   1,096/1,094
//               384    33/28    59/51    466/381      159/129    191/172   1,571/1,320
//    32 f32     384    39/49    72/92    522/711      164/172    247/333   1,752/2,570
// So: below 512 waves, 255 heads of 64 and 511 of 32, from four segments of
// SPLIT_MIN_CHUNKS chunks on; heads of 128, eight waves each, up to 128 of them, of which
// four segments take SPLIT_WAVES waves, but above 64 only from 32 chunks on. 2 x 65,537
// plies of 8 heads of 128 in 2,048 / 4,096 / 8,192 / 16,384 waves: 692 / 678 / 708 / 755 us
// of kernels.
constexpr int SPLIT_WAVES = 4096, SPLIT_MIN_CHUNKS = 4, SPLIT_LONG_CHUNKS = 32;
constexpr int split_blocks(int dim, int64_t chunks) { return dim > 64 ? (chunks < SPLIT_LONG_CHUNKS ? 64 : 128) : dim > 32 ? 255 : 511; }
struct Split { int segments, seg_plies; };
Split split_of(const jq_attention *a)
{
    const int ch = a->dtype == JQ_F32 ? Mma<float>::KB : Mma<bf16>::KB, dim = std::max(a->key_dim, a->value_dim);
    const int64_t blocks = std::max<int64_t>(1, (int64_t)a->batch * a->heads);
    const int64_t waves = blocks * pass_waves(dim <= 32 ? 32 : dim <= 64 ? 64 : 128);
    const int64_t chunks = ((int64_t)a->plies + ch - 1) / ch;
    const int64_t want = blocks <= split_blocks(dim, chunks) ? std::min(SPLIT_WAVES / waves, chunks / SPLIT_MIN_CHUNKS) : 1;
    if (want < 4) return {1, (int)std::max<int64_t>(chunks, 1) * ch};
    const int64_t each = (chunks + want - 1) / want;
    return {(int)((chunks + each - 1) / each), (int)each * ch};
}

int64_t split_bytes(const jq_attention *a)
{
    const Split s = split_of(a);
    if (s.segments < 2) return 0;
    const int64_t n = (int64_t)a->batch * a->heads * s.segments;
    return n * ((int64_t)a->key_dim * a->value_dim + 1) * (int64_t)sizeof(float);
}

ScanArgs scan_args(const jq_attention *a)
{
    ScanArgs s{};
    s.batch = a->batch;
    s.plies = a->plies;
    s.heads = a->heads;
    s.log_decay = a->log_decay;
    s.starts = a->starts;
    s.starts_batch = a->starts_batch;
    s.starts_ply = a->starts_ply;
    s.lengths = a->lengths;
    s.in_scale = s.out_scale = 1.f;
    s.seg_col = 1;
    s.stream = (int64_t)a->batch * a->plies * a->heads * (a->key_dim + a->value_dim) * 2 * (int64_t)elem_bytes(a->dtype) > STREAM_BYTES;
    const Split split = split_of(a);
    s.segments = split.segments;
    s.seg_plies = split.seg_plies;
    s.seg_states = static_cast<float *>(a->workspace);
    s.seg_carry = s.seg_states ? s.seg_states + (int64_t)a->batch * a->heads * split.segments * a->key_dim * a->value_dim : nullptr;
    return s;
}

int check_workspace(const jq_attention *a)
{
    const int64_t need = split_bytes(a);
    if (a->workspace_bytes < need || (need && !a->workspace))
        return fail(JQ_E_ARG, "workspace of %lld bytes, %lld are needed", (long long)a->workspace_bytes, (long long)need);
    if (!aligned(a->workspace, 16)) return fail(JQ_E_ARG, "workspace must be 16-byte aligned");
    return JQ_OK;
}

template <class T, bool STREAM, bool ODD>
void step_waves(const StepArgs &a, int count, hipStream_t stream)
{
    const dim3 grid((count + STEP_WAVES - 1) / STEP_WAVES), block(64 * STEP_WAVES);
    if (a.dv <= 16) hipLaunchKernelGGL((k_attention_step_wave<T, 4, STREAM, ODD>), grid, block, 0, stream, a, count);
    else if (a.dv <= 32) hipLaunchKernelGGL((k_attention_step_wave<T, 8, STREAM, ODD>), grid, block, 0, stream, a, count);
    else if (a.dv <= 64) hipLaunchKernelGGL((k_attention_step_wave<T, 16, STREAM, ODD>), grid, block, 0, stream, a, count);
    else hipLaunchKernelGGL((k_attention_step_wave<T, 32, STREAM, ODD>), grid, block, 0, stream, a, count);
}

template <class T>
void step(const StepArgs &a, int count, hipStream_t stream)
{
    const int64_t bytes = (int64_t)count * a.dk * a.dv * (int64_t)sizeof(float);
    // rows that end inside a vector share cache lines with the next: past the caches they
    // take longer at any size (20,000 games of 8 heads of 50 x 50 in bfloat16, 3.2 GB of
    // traffic: 920 us, through them 801)
    if (a.dv % 4) step_waves<T, false, true>(a, count, stream);
    else if (bytes > STREAM_BYTES) step_waves<T, true, false>(a, count, stream);
    else step_waves<T, false, false>(a, count, stream);
}

// Blocks for that much work: kernels over rows and tokens take the rest a grid's
// stride on (a launch holds fewer than 2^32 threads).
int grid_of(int64_t blocks) { return (int)std::min<int64_t>(blocks, 1 << 20); }

template <class T, int N, bool INTERLEAVED>
int launch_rotary(const RotaryArgs &a, int64_t all, hipStream_t stream)
{
    // about four items a thread, the tables within their share of LDS
    const int items = std::max(1, a.dim / N * a.heads);
    const int tokens = std::max(1, std::min(1024 / items, ROTARY_TABLE / std::max(1, a.pairs)));
    hipLaunchKernelGGL((k_rotary<T, N, INTERLEAVED>), dim3(grid_of((all + tokens - 1) / tokens)), dim3(256),
                       tokens * (2 * sizeof(int64_t) + 2 * sizeof(float) * a.pairs), stream, a, all, tokens);
    return launch_check("k_rotary");
}

template <class T>
int rotary(const RotaryArgs &a, int64_t all, hipStream_t stream)
{
    // whole vectors where the pairs are made of them, else pair by pair
    constexpr int N = Vec<T>::N;
    if (a.interleaved)
        return 2 * a.pairs % N == 0 ? launch_rotary<T, N, true>(a, all, stream) : launch_rotary<T, 2, true>(a, all, stream);
    return a.pairs % N == 0 ? launch_rotary<T, N, false>(a, all, stream) : launch_rotary<T, 1, false>(a, all, stream);
}

// f(group, vectors a lane) for the narrowest group that holds a row in registers;
// false for a row that is wider than that.
template <class T, class F>
bool norm_shape(int width, F &&f)
{
    const int vectors = (width + Vec<T>::N - 1) / Vec<T>::N;
    using std::integral_constant;
    if (vectors <= 4) f(integral_constant<int, 4>(), integral_constant<int, 1>());
    else if (vectors <= 8) f(integral_constant<int, 8>(), integral_constant<int, 1>());
    else if (vectors <= 16) f(integral_constant<int, 16>(), integral_constant<int, 1>());
    else if (vectors <= 32) f(integral_constant<int, 32>(), integral_constant<int, 1>());
    else if (vectors <= 64) f(integral_constant<int, 64>(), integral_constant<int, 1>());
    else if (vectors <= 128) f(integral_constant<int, 64>(), integral_constant<int, 2>());
    else if (vectors <= 256) f(integral_constant<int, 256>(), integral_constant<int, 1>());
    else if (vectors <= 512) f(integral_constant<int, 256>(), integral_constant<int, 2>());
    else if (vectors <= 1024) f(integral_constant<int, 256>(), integral_constant<int, 4>());
    else if (vectors <= 2048) f(integral_constant<int, 1024>(), integral_constant<int, 2>());
    else return false;
    return true;
}

// Blocks of the backward pass, each with its own sums of the weights' gradients:
// four blocks a CU, and four rows a group at least, so that the sums' traffic stays
// below the rows'.
constexpr int NORM_BLOCKS = 1024, NORM_ROWS = 4;
// Threads of the forward pass: all that the card's CUs hold, so that a block goes over
// many rows (262,144 rows of 256 in bfloat16: a block for every eight rows, with weight
// and bias read again for each, took 244 us where this took 62, 49 since).
constexpr int NORM_FORWARD_THREADS = 2048 * 256;

template <class T>
int norm_parts(int64_t rows, int32_t width)
{
    int64_t parts = std::min<int64_t>((rows + NORM_ROWS - 1) / NORM_ROWS, NORM_BLOCKS);
    norm_shape<T>(width, [&](auto g, auto nv) {
        const int64_t each = (int64_t)NORM_ROWS * NormRow<T, g(), nv()>::GROUPS;
        parts = std::min<int64_t>((rows + each - 1) / each, NORM_BLOCKS);
    });
    return (int)parts;
}

template <class T, class W>
int norm_backward(NormArgs a, void *dweight, void *dbias, hipStream_t stream)
{
    const bool sums = dweight || dbias;
    if (!sums) a.part = nullptr;
    const int parts = norm_parts<T>(a.rows, a.width);
    if (a.rows && (a.o || sums)) {
        const bool fits = norm_shape<T>(a.width, [&](auto g, auto nv) {
            hipLaunchKernelGGL((k_norm_backward<T, W, g(), nv()>), dim3(parts), dim3(NormRow<T, g(), nv()>::BLOCK), 0,
                               stream, a);
        });
        if (!fits && a.o) hipLaunchKernelGGL((k_norm_dx_wide<T, W>), dim3(grid_of(a.rows)), dim3(1024), 0, stream, a);
        if (!fits && sums) hipLaunchKernelGGL((k_norm_dw_wide<T>), dim3((a.width + 255) / 256, parts), dim3(256), 0, stream, a);
        TRY(launch_check("k_norm_backward"));
    }
    if (!sums) return JQ_OK;
    hipLaunchKernelGGL((k_norm_join<W>), dim3((a.width + 15) / 16, 2), dim3(256), 0, stream, a.part, parts, a.width,
                       static_cast<W *>(dweight), static_cast<W *>(dbias));
    return launch_check("k_norm_join");
}

template <class T, class W>
int norm_forward(const NormArgs &a, hipStream_t stream)
{
    const bool fits = norm_shape<T>(a.width, [&](auto g, auto nv) {
        using R = NormRow<T, g(), nv()>;
        hipLaunchKernelGGL((k_norm_forward<T, W, g(), nv()>), dim3(std::min<int64_t>((a.rows + R::GROUPS - 1) / R::GROUPS, NORM_FORWARD_THREADS / R::BLOCK)),
                           dim3(R::BLOCK), 0, stream, a);
    });
    if (!fits) hipLaunchKernelGGL((k_norm_forward_wide<T, W>), dim3(grid_of(a.rows)), dim3(1024), 0, stream, a);
    return launch_check("k_norm_forward");
}

int check_norm(int32_t dtype, int32_t weight_dtype, int64_t rows, int32_t width)
{
    TRY(check_dtype(dtype));
    if (weight_dtype != JQ_F32 && weight_dtype != dtype)
        return fail(JQ_E_ARG, "weights are float32 or of the rows' type");
    if (rows < 0 || rows > INT_MAX) return fail(JQ_E_ARG, "rows %lld out of range", (long long)rows);
    if (width <= 0 || width > INT_MAX - 1024)   // the kernels walk a row's columns up to 1,024 past its end
        return fail(JQ_E_ARG, "width %d out of range", width);
    return JQ_OK;
}

}  // namespace

extern "C" {

int jq_attention_workspace(const jq_attention *a, int32_t backward, int64_t *bytes)
{
    TRY(check_attention(a));
    if (!bytes) return fail(JQ_E_ARG, "null output");
    *bytes = split_bytes(a);
    return JQ_OK;
}

int jq_attention_forward(const jq_attention *a, void *stream)
{
    TRY(check_attention(a));
    if (a->batch == 0) return JQ_OK;
    TRY(check_attention_inputs(a));
    if (a->plies) TRY(check_rows(a->out, a->dtype, "out"));
    TRY(check_workspace(a));
    ScanArgs s = scan_args(a);
    s.q = a->q, s.k = a->k, s.v = a->v, s.o = a->out;
    s.kd = a->key_dim, s.vd = a->value_dim;
    s.s_in = a->initial_state, s.s_out = a->final_state, s.s_row = a->value_dim, s.s_col = 1;
    s.out_scale = a->scale;
    s.seg_row = s.vd;
    return scan(a->dtype, s, strm(stream));
}

int jq_attention_backward(const jq_attention *a, void *stream)
{
    TRY(check_attention(a));
    if (a->batch == 0) return JQ_OK;
    TRY(check_attention_inputs(a));
    if (a->plies) TRY(check_rows(a->d_out, a->dtype, "d_out"));
    TRY(check_workspace(a));
    if (!a->dk.data != !a->dv.data) return fail(JQ_E_ARG, "dk and dv go together");
    if (a->d_initial && !a->dk.data && a->plies) return fail(JQ_E_ARG, "d_initial comes with dk and dv");
    if (a->dq.data) {
        TRY(check_rows(a->dq, a->dtype, "dq"));
        ScanArgs s = scan_args(a);
        s.q = a->d_out, s.k = a->v, s.v = a->k, s.o = a->dq;
        s.kd = a->value_dim, s.vd = a->key_dim;
        s.s_in = a->initial_state, s.s_row = 1, s.s_col = a->value_dim;
        s.seg_row = s.vd;
        s.out_scale = a->scale;
        TRY(scan(a->dtype, s, strm(stream)));
    }
    if (a->dk.data || a->d_initial) {
        if (a->plies) {
            TRY(check_rows(a->dk, a->dtype, "dk"));
            TRY(check_rows(a->dv, a->dtype, "dv"));
        }
        GradArgs g{scan_args(a), a->v, a->dk};
        ScanArgs &s = g.scan;
        s.in_scale = a->scale;
        s.q = a->k, s.k = a->q, s.v = a->d_out, s.o = a->dv;
        s.kd = a->key_dim, s.vd = a->value_dim;
        s.s_in = a->d_final, s.s_out = a->d_initial, s.s_row = a->value_dim, s.s_col = 1;
        s.seg_row = s.vd;
        TRY(scan_kv(a->dtype, g, strm(stream)));
    }
    return JQ_OK;
}

int jq_attention_step(int32_t dtype, int32_t batch, int32_t heads, int32_t key_dim, int32_t value_dim, float scale,
                      const float *log_decay, const jq_rows *q, const jq_rows *k, const jq_rows *v,
                      const jq_rows *out, float *state, int64_t state_rows, const int64_t *rows,
                      const uint8_t *starts, void *stream)
{
    TRY(check_dtype(dtype));
    TRY(check_dims(batch, heads, key_dim, value_dim));
    if (state_rows < 0) return fail(JQ_E_ARG, "negative state_rows");
    if (batch == 0) return JQ_OK;
    if (!log_decay || !q || !k || !v || !out) return fail(JQ_E_ARG, "null device pointer");
    TRY(check_rows(*q, dtype, "q"));
    TRY(check_rows(*k, dtype, "k"));
    TRY(check_rows(*v, dtype, "v"));
    TRY(check_rows(*out, dtype, "out"));
    if (state_rows && !state) return fail(JQ_E_ARG, "null state");
    if (!aligned(state, 4)) return fail(JQ_E_ARG, "state must be 4-byte aligned");
    const StepArgs a{*q, *k, *v, *out, heads, key_dim, value_dim, scale, log_decay, state, state_rows, rows, starts};
    if (dtype == JQ_F32) step<float>(a, batch * heads, strm(stream));
    else step<bf16>(a, batch * heads, strm(stream));
    return launch_check("k_attention_step");
}

int jq_rotary(int32_t dtype, int64_t n0, int64_t n1, int32_t heads, int32_t dim, int32_t pairs, const jq_rows *x,
              const jq_rows *out, const void *positions, int32_t positions64, int64_t positions_n0,
              int64_t positions_n1, int32_t axes, const int32_t *section_ends, const float *frequencies,
              int32_t interleaved, int32_t inverse, void *stream)
{
    TRY(check_dtype(dtype));
    if (n0 < 0 || n1 < 0 || heads < 0 || dim <= 0 || pairs < 0 || 2 * (int64_t)pairs > dim)
        return fail(JQ_E_ARG, "bad shapes (%lld x %lld tokens, heads %d, dim %d, pairs %d)", (long long)n0, (long long)n1,
                    heads, dim, pairs);
    if (pairs > JQ_ROTARY_MAX_PAIRS || (int64_t)heads * dim > INT_MAX)
        return fail(JQ_E_ARG, "%d pairs (at most %d) and %d heads of %d elements are too many", pairs, JQ_ROTARY_MAX_PAIRS, heads, dim);
    if (axes < 1 || axes > JQ_ROTARY_MAX_AXES) return fail(JQ_E_ARG, "axes %d not in [1, %d]", axes, JQ_ROTARY_MAX_AXES);
    if (!section_ends) return fail(JQ_E_ARG, "null section_ends");
    for (int i = 0; i < axes; ++i)
        if (section_ends[i] < (i ? section_ends[i - 1] : 0))
            return fail(JQ_E_ARG, "section ends must not fall: %d at axis %d", section_ends[i], i);
    if (section_ends[axes - 1] != pairs)
        return fail(JQ_E_ARG, "the sections hold %d pairs, not %d", section_ends[axes - 1], pairs);
    if (n0 == 0 || n1 == 0 || heads == 0) return JQ_OK;
    if (n0 > INT_MAX / n1) return fail(JQ_E_ARG, "%lld x %lld tokens are too many", (long long)n0, (long long)n1);
    if (!x || !out || (pairs && (!positions || !frequencies))) return fail(JQ_E_ARG, "null device pointer");
    TRY(check_rows(*x, dtype, "x"));
    TRY(check_rows(*out, dtype, "out"));
    if (!aligned(positions, positions64 ? 8 : 4)) return fail(JQ_E_ARG, "positions must be aligned to their element size");
    RotaryArgs a{*x, *out, n1, heads, dim, pairs, axes, positions, positions_n0, positions_n1, {}, frequencies,
                 positions64 != 0, interleaved != 0, inverse != 0};
    std::copy(section_ends, section_ends + axes, a.ends);
    return dtype == JQ_F32 ? rotary<float>(a, n0 * n1, strm(stream)) : rotary<bf16>(a, n0 * n1, strm(stream));
}

int jq_layer_norm_forward(int32_t dtype, int32_t weight_dtype, int64_t rows, int32_t width, const void *x,
                          int64_t x_stride, const void *weight, const void *bias, float eps, void *out,
                          int64_t out_stride, float *mean, float *rstd, void *stream)
{
    TRY(check_norm(dtype, weight_dtype, rows, width));
    if (rows == 0) return JQ_OK;
    if (!x || !out) return fail(JQ_E_ARG, "null device pointer");
    if (!aligned(x, elem_bytes(dtype)) || !aligned(out, elem_bytes(dtype)))
        return fail(JQ_E_ARG, "rows must be aligned to their element size");
    const NormArgs a{x, weight, bias, nullptr, out, x_stride, out_stride, 0, rows, width, eps, mean, rstd, nullptr};
    if (dtype == JQ_F32) return norm_forward<float, float>(a, strm(stream));
    return weight_dtype == JQ_F32 ? norm_forward<bf16, float>(a, strm(stream)) : norm_forward<bf16, bf16>(a, strm(stream));
}

int jq_layer_norm_workspace(int64_t rows, int32_t width, int64_t *bytes)
{
    TRY(check_norm(JQ_F32, JQ_F32, rows, width));
    if (!bytes) return fail(JQ_E_ARG, "null output");
    *bytes = (int64_t)std::max(norm_parts<float>(rows, width), norm_parts<bf16>(rows, width)) * 2 * width * (int64_t)sizeof(float);
    return JQ_OK;
}

int jq_layer_norm_backward(int32_t dtype, int32_t weight_dtype, int64_t rows, int32_t width, const void *x,
                           int64_t x_stride, const void *weight, const float *mean, const float *rstd,
                           const void *d_out, int64_t d_out_stride, void *dx, int64_t dx_stride, void *dweight,
                           void *dbias, void *workspace, int64_t workspace_bytes, void *stream)
{
    TRY(check_norm(dtype, weight_dtype, rows, width));
    if (rows && (!x || !mean || !rstd || !d_out)) return fail(JQ_E_ARG, "null device pointer");
    if (!aligned(x, elem_bytes(dtype)) || !aligned(d_out, elem_bytes(dtype)) || !aligned(dx, elem_bytes(dtype)))
        return fail(JQ_E_ARG, "rows must be aligned to their element size");
    if (dweight || dbias) {
        int64_t need = 0;
        TRY(jq_layer_norm_workspace(rows, width, &need));
        if (workspace_bytes < need || (need && !workspace))
            return fail(JQ_E_ARG, "workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)need);
        if (!aligned(workspace, 4)) return fail(JQ_E_ARG, "workspace must be 4-byte aligned");
    }
    const NormArgs a{x, weight, nullptr, d_out, dx, x_stride, dx_stride, d_out_stride, rows, width, 0.f,
                     const_cast<float *>(mean), const_cast<float *>(rstd), static_cast<float *>(workspace)};
    if (dtype == JQ_F32) return norm_backward<float, float>(a, dweight, dbias, strm(stream));
    return weight_dtype == JQ_F32 ? norm_backward<bf16, float>(a, dweight, dbias, strm(stream))
                                  : norm_backward<bf16, bf16>(a, dweight, dbias, strm(stream));
}

}  // extern "C"
