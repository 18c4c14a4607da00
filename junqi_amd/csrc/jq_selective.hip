// C entry points of a policy's selective memory (state space scan, causal convolution)
// and of its masked logits. Declarations and contracts live in include/junqi_amd.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "junqi_amd.h"
#include "jq_entry.h"
#include "jq_memory.h"
#include "jq_scan.h"
#include "jq_conv.h"
#include "jq_logits.h"

using namespace jq;

namespace {

constexpr int MOST_CHANNELS = 1 << 20, MOST_PLIES = 1 << 30, MOST_BLOCKS = 1 << 20;
static_assert(SCAN_STEP == JQ_SCAN_MAX_PLY_STRIDE, "the header's limit");
constexpr int64_t MOST_ELEMENTS = 1ll << 42;   // of a segment's rows: every size below fits 64 bits
constexpr int MOST_GAMES = 1 << 30;            // with the parts of a split axis they fit 32

template <class F>
int by_type(int32_t dtype, F &&f)
{
    return dtype == JQ_F32 ? f(float()) : f(bf16());
}

int check_segment(int32_t dtype, int32_t batch, int32_t plies, int32_t channels)
{
    TRY(check_dtype(dtype));
    if (batch < 0 || batch > MOST_GAMES || plies < 0 || plies > MOST_PLIES || channels <= 0 || channels > MOST_CHANNELS)
        return fail(JQ_E_ARG, "bad shapes (batch %d, plies %d, channels %d)", batch, plies, channels);
    if ((int64_t)batch * std::max(1, plies) > MOST_ELEMENTS / channels)
        return fail(JQ_E_ARG, "%d games of %d plies of %d channels are too many", batch, plies, channels);
    return JQ_OK;
}

// ------------------------------------------------------------------ scan
int check_states(int32_t channels, int32_t states, int32_t groups)
{
    if (states <= 0 || states > JQ_SCAN_MAX_STATES) return fail(JQ_E_ARG, "states %d not in [1, %d]", states, JQ_SCAN_MAX_STATES);
    if (groups <= 0 || channels % groups) return fail(JQ_E_ARG, "%d channels do not part into %d groups", channels, groups);
    return JQ_OK;
}

int check_scan(const jq_scan *a)
{
    if (!a) return fail(JQ_E_ARG, "null arguments");
    TRY(check_segment(a->dtype, a->batch, a->plies, a->channels));
    return check_states(a->channels, a->states, a->groups);
}

// Rows of a segment whose plies a chunk's 32-bit offsets reach.
int check_ply_rows(const jq_scan *a, const jq_rows &r, const char *name)
{
    TRY(check_rows(r, a->dtype, name));
    if (a->plies > 1 && (r.ply < 0 || r.ply > JQ_SCAN_MAX_PLY_STRIDE / (int64_t)elem_bytes(a->dtype)))
        return fail(JQ_E_ARG, "the plies of %s are %lld elements apart", name, (long long)r.ply);
    return JQ_OK;
}

int check_scan_inputs(const jq_scan *a)
{
    if (!a->a) return fail(JQ_E_ARG, "null a");
    TRY(check_pointer(a->a, 4, "a"));
    TRY(check_pointer(a->skip, 4, "skip"));
    TRY(check_pointer(a->delta_bias, 4, "delta_bias"));
    if (a->plies == 0 || a->batch == 0) return JQ_OK;
    TRY(check_ply_rows(a, a->u, "u"));
    TRY(check_ply_rows(a, a->delta, "delta"));
    TRY(check_ply_rows(a, a->b, "b"));
    TRY(check_ply_rows(a, a->c, "c"));
    if (a->gate.data) TRY(check_ply_rows(a, a->gate, "gate"));
    return JQ_OK;
}

// States of a lane and waves of states, and the parts of a split axis.
struct ScanShape { int ns, sg, waves, segments, seg_plies; bool exact; };

// Few games and channels leave most of the card's 1,024 SIMDs idle unless parts of a long
// axis run side by side, at the price of its states taken twice. Split / in one piece, us,
// 16 states in bfloat16:
//                    forward, plies            with the gradients
//   waves          512          2,048          512           2,048
//      64        55 / 213      79 / 832      221 / 941      288 / 3,629
//     256        78 / 212     242 / 872      287 / 943      961 / 3,788
//     512       129 / 213     468 / 901      513 / 977    1,853 / 3,859
//   1,024       247 / 215     919 / 910      974 / 1,017  3,625 / 4,033
// So: below 1,024 waves, from four parts of 64 plies on. Shorter parts and fewer of them, which
// would split axes of less than 256 plies, are not measured: there one piece takes about 0.4
// us a ply forward and 1.8 with the gradients. Waves of all parts (two records of
// 65,537 plies, us at 2,048 / 4,096 / 8,192): 605 / 520 / 509; the middle one, for the third
// doubles the states kept between them.
constexpr int SPLIT_BELOW = 1024, SPLIT_WAVES = 4096, SPLIT_PLIES = 64;
ScanShape scan_shape(const jq_scan *a)
{
    ScanShape s;
    const int per = a->channels / a->groups;
    s.waves = (per + 63) / 64;
    s.ns = a->states <= 4 ? 4 : a->states <= 8 ? 8 : 16;
    s.sg = (a->states + s.ns - 1) / s.ns;
    const int64_t waves = std::max<int64_t>(1, (int64_t)a->batch * a->groups * s.waves);
    int64_t want = waves * s.sg < SPLIT_BELOW ? std::min<int64_t>(SPLIT_WAVES / (waves * s.sg), a->plies / SPLIT_PLIES) : 1;
    if (want < 4) want = 1;
    const int64_t each = ((a->plies + want - 1) / want + SCAN_CHUNK - 1) / SCAN_CHUNK * SCAN_CHUNK;
    s.seg_plies = (int)std::max<int64_t>(each, SCAN_CHUNK);
    s.segments = want == 1 ? 1 : (int)((a->plies + each - 1) / each);
    s.exact = s.ns * s.sg == a->states && per % 64 == 0;
    return s;
}

// Waves that share the backward pass's items, each with its own sums of da, dskip and dbias:
// as many as its registers let live (training, us at 1,024 / 2,048 / 4,096: 1,852 / 1,416 /
// 1,402, the last with twice the sums to keep and join).
constexpr int BACKWARD_WAVES = 2048;
int64_t scan_parts(const jq_scan *a)
{
    const ScanShape s = scan_shape(a);
    const int64_t items = (int64_t)a->batch * s.segments, blocks = (int64_t)s.waves * a->groups;
    return std::max<int64_t>(1, std::min(items, BACKWARD_WAVES / (blocks * s.sg)));
}

// One ply: waves that walk the games (32,768 games of 512 channels of 16 states, us at 8,192 /
// 16,384 / 32,768 / 131,072 waves and one game each: 563 / 491 / 459 / 468 / 832), and the
// bytes of states past which they would not be found in the caches at the next ply (that call
// through them 550).
constexpr int STEP_GAME_WAVES = 32768;
constexpr int64_t STEP_STREAM_BYTES = 400ll << 20;

struct ScanBytes { int64_t state, sum, bc, a; int64_t all() const { return state + sum + bc + a; } };
ScanBytes scan_bytes(const jq_scan *a, bool backward)
{
    const ScanShape s = scan_shape(a);
    ScanBytes n{0, 0, 0, 0};
    if (s.segments > 1) {
        n.sum = (int64_t)a->batch * s.segments * a->channels * 4;
        n.state = n.sum * a->states;
    }
    if (backward) {
        if (a->db.data || a->dc.data) n.bc = (int64_t)s.waves * a->batch * a->plies * a->groups * 2 * a->states * 4;
        if (a->da || a->dskip || a->ddelta_bias) n.a = scan_parts(a) * (a->states + 2) * a->channels * 4;
    }
    return n;
}

int check_scan_workspace(const jq_scan *a, bool backward)
{
    const int64_t need = scan_bytes(a, backward).all();
    if (a->workspace_bytes < need || (need && !a->workspace))
        return fail(JQ_E_ARG, "workspace of %lld bytes, %lld are needed", (long long)a->workspace_bytes, (long long)need);
    if (!aligned(a->workspace, 16)) return fail(JQ_E_ARG, "workspace must be 16-byte aligned");
    return JQ_OK;
}

SelectArgs select_args(const jq_scan *a, bool backward)
{
    SelectArgs s{};
    const ScanShape shape = scan_shape(a);
    s.u = a->u, s.delta = a->delta, s.gate = a->gate, s.b = a->b, s.c = a->c, s.out = a->out;
    s.batch = a->batch, s.plies = a->plies, s.channels = a->channels, s.states = a->states, s.groups = a->groups;
    s.per = a->channels / a->groups, s.waves = shape.waves, s.softplus = a->softplus != 0;
    s.a = a->a, s.skip = a->skip, s.bias = a->delta_bias;
    s.starts = a->starts, s.starts_batch = a->starts_batch, s.starts_ply = a->starts_ply;
    s.lengths = a->lengths;
    s.s_in = a->initial_state, s.s_out = a->final_state, s.saved = a->saved;
    s.segments = shape.segments, s.seg_plies = shape.seg_plies;
    const ScanBytes n = scan_bytes(a, backward);
    char *w = static_cast<char *>(a->workspace);
    s.part_bc = reinterpret_cast<float *>(w);   // first: read in vectors
    s.seg_state = reinterpret_cast<float *>(w + n.bc);
    s.seg_sum = reinterpret_cast<float *>(w + n.bc + n.state);
    s.part_a = reinterpret_cast<float *>(w + n.bc + n.state + n.sum);
    s.want_bc = n.bc, s.want_a = n.a;
    return s;
}

// f(states of a lane, exact, more than one wave of states)
template <class F>
int by_shape(const ScanShape &s, F &&f)
{
    using std::integral_constant;
    auto go = [&](auto ns, auto many) { return s.exact ? f(ns, std::true_type(), many) : f(ns, std::false_type(), many); };
    if (s.sg > 1) return go(integral_constant<int, 16>(), std::true_type());
    return s.ns == 4 ? go(integral_constant<int, 4>(), std::false_type())
           : s.ns == 8 ? go(integral_constant<int, 8>(), std::false_type()) : go(integral_constant<int, 16>(), std::false_type());
}

int grid_over(int64_t threads) { return (int)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, 1 << 16)); }

template <bool BACK>
int launch_join(const SelectArgs &s, hipStream_t stream)
{
    hipLaunchKernelGGL(k_scan_join<BACK>, dim3(grid_over((int64_t)s.batch * s.states * s.channels)), dim3(256), 0, stream, s);
    return launch_check("k_scan_join");
}

// Blocks and threads of a pass in which `parts` share the items, and s.parts set to them.
constexpr int SCAN_BLOCK_WAVES = 4;
struct ScanGrid { dim3 grid, block; };
ScanGrid scan_grid(SelectArgs &s, const ScanShape &shape, int64_t parts)
{
    const int cw = s.waves * s.groups;
    s.parts = (int)std::max<int64_t>(1, std::min<int64_t>(parts, MOST_BLOCKS / cw));
    const int64_t waves = (int64_t)cw * s.parts;
    if (shape.sg > 1) return {dim3((int)waves), dim3(64 * shape.sg)};
    return {dim3((int)((waves + SCAN_BLOCK_WAVES - 1) / SCAN_BLOCK_WAVES)), dim3(64 * SCAN_BLOCK_WAVES)};
}

// ------------------------------------------------------------------ convolution
int check_taps(int32_t dtype, int32_t weight_dtype, int32_t taps)
{
    if (weight_dtype != JQ_F32 && weight_dtype != dtype) return fail(JQ_E_ARG, "weights are float32 or of the rows' type");
    if (taps <= 0 || taps > JQ_CONV_MAX_TAPS) return fail(JQ_E_ARG, "taps %d not in [1, %d]", taps, JQ_CONV_MAX_TAPS);
    return JQ_OK;
}

int check_conv(const jq_conv *a)
{
    if (!a) return fail(JQ_E_ARG, "null arguments");
    TRY(check_segment(a->dtype, a->batch, a->plies, a->channels));
    return check_taps(a->dtype, a->weight_dtype, a->taps);
}

int check_conv_inputs(const jq_conv *a)
{
    if (!a->weight) return fail(JQ_E_ARG, "null weight");
    TRY(check_pointer(a->weight, elem_bytes(a->weight_dtype), "weight"));
    TRY(check_pointer(a->bias, elem_bytes(a->weight_dtype), "bias"));
    TRY(check_pointer(a->initial_state, elem_bytes(a->dtype), "initial_state"));
    TRY(check_pointer(a->lengths, 4, "lengths"));
    if (a->plies && a->batch) TRY(check_rows(a->x, a->dtype, "x"));
    return JQ_OK;
}

// Whether r's rows lie at multiples of `bytes`.
bool rows_at(const jq_rows &r, int32_t dtype, int64_t bytes)
{
    const int64_t n = bytes / (int64_t)elem_bytes(dtype);
    return aligned(r.data, bytes) && r.batch % n == 0 && r.ply % n == 0;
}
int conv_forward_vec(const jq_conv *a)
{
    if (a->dtype == JQ_F32 || a->taps > 4) return 4;
    const bool eight = rows_at(a->x, a->dtype, 8) && rows_at(a->out, a->dtype, 8), sixteen = rows_at(a->x, a->dtype, 16) && rows_at(a->out, a->dtype, 16);
    return eight && !sixteen ? 4 : 8;
}

// Threads across channels, and plies of a run: as many runs as keep the card's threads
// busy, none so short that the taps before it are most of what it reads (1,024 games of 256
// plies of 512 channels, training, us at 64 K / 128 K / 256 K / 512 K threads: 361 / 318 /
// 356 / 378). Blocks of the backward pass, each with its own sums, and of one ply.
constexpr int CONV_THREADS = 128 * 1024, CONV_RUN = 16, CONV_BACKWARD_BLOCKS = 1024, CONV_STEP_BLOCKS = 4096;
struct ConvShape { int blocks_x, v; };
ConvShape conv_shape(ConvArgs &c, int v)
{
    const int64_t vectors = (c.channels + v - 1) / v;
    c.tx = vectors <= 8 ? 8 : vectors <= 16 ? 16 : vectors <= 32 ? 32 : 64;
    const int64_t across = (vectors + c.tx - 1) / c.tx * c.tx;
    const int64_t want = std::max<int64_t>(1, CONV_THREADS / across / std::max(1, c.batch));
    c.run = (int)std::max<int64_t>(CONV_RUN, (c.plies + want - 1) / want);
    c.runs = std::max(1, (c.plies + c.run - 1) / c.run);
    return {(int)(across / c.tx), v};
}
int64_t conv_parts(const ConvArgs &c, const ConvShape &s, int64_t items, int64_t most)
{
    const int64_t rows = 256 / c.tx;
    return std::max<int64_t>(1, std::min((items + rows - 1) / rows, most / s.blocks_x));
}

ConvArgs conv_args(const jq_conv *a)
{
    ConvArgs c{};
    c.x = a->x, c.out = a->out;
    c.batch = a->batch, c.plies = a->plies, c.channels = a->channels, c.taps = a->taps, c.silu = a->silu != 0;
    c.weight = a->weight, c.bias = a->bias;
    c.starts = a->starts, c.starts_batch = a->starts_batch, c.starts_ply = a->starts_ply;
    c.lengths = a->lengths;
    c.s_in = a->initial_state, c.s_out = a->final_state;
    return c;
}

int64_t conv_bytes(const jq_conv *a)
{
    ConvArgs c = conv_args(a);
    if (!a->dweight && !a->dbias) return 0;
    const ConvShape s = conv_shape(c, 4);
    return conv_parts(c, s, (int64_t)c.batch * c.runs, CONV_BACKWARD_BLOCKS) * (c.taps + 1) * c.channels * 4;
}

// f(rows' type, weights' type, taps)
template <class F>
int by_taps(int32_t dtype, int32_t weight_dtype, int taps, F &&f)
{
    auto go = [&](auto t, auto w) {
        using std::integral_constant;
        return taps <= 2 ? f(t, w, integral_constant<int, 2>()) : taps == 3 ? f(t, w, integral_constant<int, 3>())
               : taps == 4 ? f(t, w, integral_constant<int, 4>()) : f(t, w, integral_constant<int, 8>());
    };
    if (dtype == JQ_F32) return go(float(), float());
    return weight_dtype == JQ_F32 ? go(bf16(), float()) : go(bf16(), bf16());
}

// ------------------------------------------------------------------ logits
constexpr int LOGITS_MOST_ACTIONS = INT_MAX - 4096;   // a lane's columns are walked that far past the last
int check_logits(const jq_logits *a)
{
    if (!a) return fail(JQ_E_ARG, "null arguments");
    TRY(check_dtype(a->dtype));
    if (a->rows < 0 || a->rows > INT_MAX || a->actions <= 0 || a->actions > LOGITS_MOST_ACTIONS || a->recent_count < 0 || a->recent_count > INT_MAX - 256)
        return fail(JQ_E_ARG, "bad shapes (rows %lld, actions %d, recent %d)", (long long)a->rows, a->actions, a->recent_count);
    if (a->mask && a->mask_kind != JQ_LOGITS_MASK_WORDS && a->mask_kind != JQ_LOGITS_MASK_BYTES) return fail(JQ_E_ARG, "mask kind %d", a->mask_kind);
    if (a->mask && a->mask_kind == JQ_LOGITS_MASK_WORDS && !aligned(a->mask, 4)) return fail(JQ_E_ARG, "mask words must be 4-byte aligned");
    if (a->recent_count && !a->recent) return fail(JQ_E_ARG, "null recent");
    if (!aligned(a->recent, a->recent64 ? 8 : 4)) return fail(JQ_E_ARG, "recent must be aligned to its element size");
    if (!aligned(a->bias, 4)) return fail(JQ_E_ARG, "bias must be 4-byte aligned");
    TRY(check_pointer(a->recent_lengths, 4, "recent_lengths"));
    TRY(check_pointer(a->repetitions, 4, "repetitions"));
    TRY(check_pointer(a->frequencies, 4, "frequencies"));
    return check_pointer(a->presences, 4, "presences");
}

LogitsArgs logits_args(const jq_logits *a)
{
    LogitsArgs l{};
    l.x = a->logits, l.x_stride = a->logits_stride;
    l.rows = a->rows, l.actions = a->actions;
    l.bias = a->bias;
    if (a->mask && a->mask_kind == JQ_LOGITS_MASK_WORDS) l.words = static_cast<const uint32_t *>(a->mask);
    else l.dense = static_cast<const uint8_t *>(a->mask);
    l.mask_stride = a->mask_stride;
    l.recent = a->recent, l.recent_stride = a->recent_stride, l.recent_count = a->recent_count, l.recent64 = a->recent64 != 0;
    l.recent_lengths = a->recent_lengths;
    l.repetition = a->repetition, l.frequency = a->frequency, l.presence = a->presence;
    l.repetitions = a->repetitions, l.frequencies = a->frequencies, l.presences = a->presences;
    return l;
}

// Columns of a wave: whole rows where there are enough for the card's waves, else parts of
// them, and no more than LDS has a mask for. Blocks of as many waves as LDS has tables for
// (a wave gets at most as many actions as it has columns).
constexpr int LOGITS_WAVES = 4096, LOGITS_TABLE_TILE = 2048;
constexpr size_t LOGITS_LDS = 64 << 10;
struct LogitsGrid { dim3 grid, block; size_t lds; };
template <class T>
LogitsGrid logits_grid(LogitsArgs &l)
{
    constexpr int64_t STEP = 64 * Vec<T>::N;   // a vector for each lane
    const int64_t want = std::max<int64_t>(1, LOGITS_WAVES / std::max<int64_t>(1, l.rows));
    int64_t tile = std::min<int64_t>((l.actions / want + STEP) / STEP * STEP, LOGITS_TILE);
    if (l.recent_count > LOGITS_TABLE_TILE) tile = std::min<int64_t>(tile, LOGITS_TABLE_TILE);
    l.tile = (int)tile;
    l.tiles = (int)((l.actions + tile - 1) / tile);
    l.mask_words = (int)((std::min<int64_t>(tile, l.actions) + 31) / 32);
    l.slots = 0;
    if (l.recent_count)
        for (l.slots = 64; l.slots < 2 * std::min(l.recent_count, l.tile); l.slots *= 2) {}
    const size_t each = 4 * ((size_t)l.mask_words + 2 * l.slots);
    int waves = 4;
    while (waves > 1 && waves * each > LOGITS_LDS) waves /= 2;
    return {dim3((unsigned)std::min<int64_t>((l.rows * l.tiles + waves - 1) / waves, 1 << 23)), dim3(64 * waves), waves * each};
}

// Blocks along the rows that sum dbias (4,096 rows of 16,641, training, us at 1,024 / 2,048 /
// 4,096: 272 / 248 / 252).
constexpr int LOGITS_BIAS_BLOCKS = 2048;
int bias_tiles(const jq_logits *a)
{
    const int64_t columns = 256 * (a->dtype == JQ_F32 ? 4 : 8);
    return (int)((a->actions + columns - 1) / columns);
}
int64_t logits_parts(const jq_logits *a)
{
    return std::max<int64_t>(1, std::min<int64_t>((a->rows + 3) / 4, LOGITS_BIAS_BLOCKS / bias_tiles(a)));
}

}  // namespace

extern "C" {

int jq_scan_workspace(const jq_scan *a, int32_t backward, int64_t *bytes)
{
    TRY(check_scan(a));
    if (!bytes) return fail(JQ_E_ARG, "null output");
    *bytes = scan_bytes(a, backward != 0).all();
    return JQ_OK;
}

int jq_scan_saved(const jq_scan *a, int64_t *bytes)
{
    TRY(check_scan(a));
    if (!bytes) return fail(JQ_E_ARG, "null output");
    *bytes = (int64_t)a->batch * ((a->plies + SCAN_CHUNK - 1) / SCAN_CHUNK) * a->states * a->channels * 4;
    return JQ_OK;
}

int jq_scan_forward(const jq_scan *a, void *stream)
{
    TRY(check_scan(a));
    if (a->batch == 0) return JQ_OK;
    TRY(check_scan_inputs(a));
    if (a->plies) TRY(check_ply_rows(a, a->out, "out"));
    TRY(check_pointer(a->lengths, 4, "lengths"));
    TRY(check_pointer(a->initial_state, 4, "initial_state"));
    TRY(check_pointer(a->final_state, 4, "final_state"));
    TRY(check_pointer(a->saved, 4, "saved"));
    TRY(check_scan_workspace(a, false));
    SelectArgs s = select_args(a, false);
    const ScanShape shape = scan_shape(a);
    const hipStream_t q = strm(stream);
    const ScanGrid g = scan_grid(s, shape, (int64_t)s.batch * s.segments);
    return by_type(a->dtype, [&](auto t) {
        using T = decltype(t);
        return by_shape(shape, [&](auto ns, auto exact, auto many) {
            if (s.segments > 1) {
                hipLaunchKernelGGL((k_scan_forward<T, ns(), exact(), many(), false>), g.grid, g.block, 0, q, s);
                TRY(launch_check("k_scan_forward (states)"));
                TRY(launch_join<false>(s, q));
            }
            const size_t lds = many() ? 2 * shape.sg * SCAN_PLIES * 64 * sizeof(float) : 0;
            hipLaunchKernelGGL((k_scan_forward<T, ns(), exact(), many(), true>), g.grid, g.block, lds, q, s);
            return launch_check("k_scan_forward");
        });
    });
}

int jq_scan_backward(const jq_scan *a, void *stream)
{
    TRY(check_scan(a));
    TRY(check_scan_inputs(a));
    if (a->plies && a->batch) TRY(check_ply_rows(a, a->d_out, "d_out"));
    if (a->plies && a->batch && !a->saved) return fail(JQ_E_ARG, "null saved");
    if (a->dgate.data && !a->gate.data) return fail(JQ_E_ARG, "dgate without a gate");
    for (const jq_rows *r : {&a->du, &a->ddelta, &a->dgate, &a->db, &a->dc})
        if (r->data) TRY(check_ply_rows(a, *r, "a gradient"));   // absent ones are not wanted
    TRY(check_pointer(a->lengths, 4, "lengths"));
    TRY(check_pointer(a->saved, 4, "saved"));
    TRY(check_pointer(a->da, 4, "da"));
    TRY(check_pointer(a->dskip, 4, "dskip"));
    TRY(check_pointer(a->ddelta_bias, 4, "ddelta_bias"));
    TRY(check_pointer(a->d_final, 4, "d_final"));
    TRY(check_pointer(a->d_initial, 4, "d_initial"));
    TRY(check_scan_workspace(a, true));
    SelectArgs s = select_args(a, true);
    s.d_out = a->d_out, s.du = a->du, s.ddelta = a->ddelta, s.dgate = a->dgate;
    s.d_final = a->d_final, s.d_initial = a->d_initial;
    const ScanShape shape = scan_shape(a);
    const hipStream_t q = strm(stream);
    const int64_t parts = scan_parts(a);
    return by_type(a->dtype, [&](auto t) {
        using T = decltype(t);
        return by_shape(shape, [&](auto ns, auto exact, auto many) {
            if (s.segments > 1) {
                const ScanGrid g = scan_grid(s, shape, (int64_t)s.batch * s.segments);
                hipLaunchKernelGGL((k_scan_carry<T, ns(), exact(), many()>), g.grid, g.block, 0, q, s);
                TRY(launch_check("k_scan_carry"));
                TRY(launch_join<true>(s, q));
            }
            const ScanGrid g = scan_grid(s, shape, parts);
            const size_t far = (size_t)g.block.x * scan_far(ns()) * ns() * sizeof(float);
            const size_t shares = many() ? 3 * shape.sg * SCAN_CHUNK * 64 * sizeof(float) : 0;
            hipLaunchKernelGGL((k_scan_backward<T, ns(), exact(), many()>), g.grid, g.block, far + shares, q, s);
            TRY(launch_check("k_scan_backward"));
            if (s.want_bc && s.batch && s.plies) {
                const int64_t n = (int64_t)s.batch * s.plies * s.groups * 2 * s.states;
                if (s.states % 4 == 0) hipLaunchKernelGGL((k_scan_join_bc<T, 4>), dim3(grid_over(n / 4)), dim3(256), 0, q, s, a->db, a->dc);
                else hipLaunchKernelGGL((k_scan_join_bc<T, 1>), dim3(grid_over(n)), dim3(256), 0, q, s, a->db, a->dc);
                TRY(launch_check("k_scan_join_bc"));
            }
            if (!s.want_a) return JQ_OK;
            hipLaunchKernelGGL(k_scan_join_a, dim3((int)(((int64_t)(s.states + 2) * s.channels + 15) / 16)), dim3(256), 0, q, s, a->da, a->dskip,
                               a->ddelta_bias);
            return launch_check("k_scan_join_a");
        });
    });
}

int jq_scan_step(const jq_scan *a, float *state, int64_t state_rows, const int64_t *rows, const uint8_t *starts, void *stream)
{
    TRY(check_scan(a));
    if (state_rows < 0) return fail(JQ_E_ARG, "negative state_rows");
    if (a->plies != 1) return fail(JQ_E_ARG, "a step has one ply, not %d", a->plies);
    if (a->batch == 0) return JQ_OK;
    TRY(check_scan_inputs(a));
    TRY(check_rows(a->out, a->dtype, "out"));
    if (state_rows && !state) return fail(JQ_E_ARG, "null state");
    TRY(check_pointer(rows, 8, "rows"));
    if (!aligned(state, 4)) return fail(JQ_E_ARG, "state must be 4-byte aligned");
    const SelectStepArgs s{a->u, a->delta, a->gate, a->b, a->c, a->out, a->batch, a->channels, a->states, a->groups,
                           a->channels / a->groups, a->softplus != 0, a->a, a->skip, a->delta_bias, state, state_rows, rows, starts};
    return by_type(a->dtype, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto l) {
            const int per = 64 / l(), cw = (a->channels + per - 1) / per;
            const int at_once = (int)std::max<int64_t>(1, std::min<int64_t>(a->batch, STEP_GAME_WAVES / cw));
            const dim3 grid((int)(((int64_t)cw * at_once + 3) / 4));
            if ((int64_t)a->batch * a->channels * a->states * 4 > STEP_STREAM_BYTES)
                hipLaunchKernelGGL((k_scan_step<T, l(), true>), grid, dim3(256), 0, strm(stream), s, cw, at_once);
            else hipLaunchKernelGGL((k_scan_step<T, l(), false>), grid, dim3(256), 0, strm(stream), s, cw, at_once);
            return launch_check("k_scan_step");
        };
        using std::integral_constant;
        return a->states <= 4 ? go(integral_constant<int, 1>()) : a->states <= 8 ? go(integral_constant<int, 2>())
               : a->states <= 16 ? go(integral_constant<int, 4>()) : a->states <= 32 ? go(integral_constant<int, 8>())
               : go(integral_constant<int, 16>());
    });
}

int jq_conv_workspace(const jq_conv *a, int64_t *bytes)
{
    TRY(check_conv(a));
    if (!bytes) return fail(JQ_E_ARG, "null output");
    *bytes = conv_bytes(a);
    return JQ_OK;
}

int jq_conv_forward(const jq_conv *a, void *stream)
{
    TRY(check_conv(a));
    if (a->batch == 0) return JQ_OK;
    TRY(check_conv_inputs(a));
    if (a->plies) TRY(check_rows(a->out, a->dtype, "out"));
    TRY(check_pointer(a->final_state, elem_bytes(a->dtype), "final_state"));
    ConvArgs c = conv_args(a);
    const ConvShape s = conv_shape(c, conv_forward_vec(a));
    c.parts = (int)conv_parts(c, s, (int64_t)c.batch * c.runs, MOST_BLOCKS);
    return by_taps(a->dtype, a->weight_dtype, a->taps, [&](auto t, auto w, auto taps) {
        using T = decltype(t);
        using W = decltype(w);
        const dim3 grid(c.parts * s.blocks_x);
        if constexpr (conv_vec<T, taps()>() == 8)
            if (s.v == 8) {
                hipLaunchKernelGGL((k_conv_forward<T, W, taps(), 8>), grid, dim3(256), 0, strm(stream), c);
                return launch_check("k_conv_forward");
            }
        hipLaunchKernelGGL((k_conv_forward<T, W, taps(), 4>), grid, dim3(256), 0, strm(stream), c);
        return launch_check("k_conv_forward");
    });
}

int jq_conv_backward(const jq_conv *a, void *stream)
{
    TRY(check_conv(a));
    TRY(check_conv_inputs(a));
    if (a->plies && a->batch) TRY(check_rows(a->d_out, a->dtype, "d_out"));
    if (a->dx.data) TRY(check_rows(a->dx, a->dtype, "dx"));
    TRY(check_pointer(a->d_final, elem_bytes(a->dtype), "d_final"));
    TRY(check_pointer(a->d_initial, elem_bytes(a->dtype), "d_initial"));
    TRY(check_pointer(a->dweight, elem_bytes(a->weight_dtype), "dweight"));
    TRY(check_pointer(a->dbias, elem_bytes(a->weight_dtype), "dbias"));
    const int64_t need = conv_bytes(a);
    if (a->workspace_bytes < need || (need && !a->workspace))
        return fail(JQ_E_ARG, "workspace of %lld bytes, %lld are needed", (long long)a->workspace_bytes, (long long)need);
    if (!aligned(a->workspace, 4)) return fail(JQ_E_ARG, "workspace must be 4-byte aligned");
    ConvArgs c = conv_args(a);
    c.d_out = a->d_out, c.dx = a->dx, c.d_final = a->d_final, c.d_initial = a->d_initial;
    c.part = need ? static_cast<float *>(a->workspace) : nullptr;
    const ConvShape s = conv_shape(c, 4);
    c.parts = (int)conv_parts(c, s, (int64_t)c.batch * c.runs, CONV_BACKWARD_BLOCKS);
    return by_taps(a->dtype, a->weight_dtype, a->taps, [&](auto t, auto w, auto taps) {
        using W = decltype(w);
        hipLaunchKernelGGL((k_conv_backward<decltype(t), W, taps()>), dim3(c.parts * s.blocks_x), dim3(256), 0, strm(stream), c);
        TRY(launch_check("k_conv_backward"));
        if (!c.part) return JQ_OK;
        hipLaunchKernelGGL(k_conv_join<W>, dim3((int)(((int64_t)(c.taps + 1) * c.channels + 15) / 16)), dim3(256), 0, strm(stream), c.part, c.parts, c.taps,
                           c.channels, static_cast<W *>(a->dweight), static_cast<W *>(a->dbias));
        return launch_check("k_conv_join");
    });
}

int jq_conv_step(const jq_conv *a, void *state, int64_t state_rows, const int64_t *rows, const uint8_t *starts, void *stream)
{
    TRY(check_conv(a));
    if (state_rows < 0) return fail(JQ_E_ARG, "negative state_rows");
    if (a->plies != 1) return fail(JQ_E_ARG, "a step has one ply, not %d", a->plies);
    if (a->batch == 0) return JQ_OK;
    TRY(check_conv_inputs(a));
    TRY(check_rows(a->out, a->dtype, "out"));
    if (state_rows && !state && a->taps > 1) return fail(JQ_E_ARG, "null state");
    TRY(check_pointer(rows, 8, "rows"));
    TRY(check_pointer(state, elem_bytes(a->dtype), "state"));
    ConvStepArgs s{conv_args(a), state, state_rows, rows, starts};
    const ConvShape shape = conv_shape(s.c, 4);
    s.c.parts = (int)conv_parts(s.c, shape, a->batch, CONV_STEP_BLOCKS);
    return by_taps(a->dtype, a->weight_dtype, a->taps, [&](auto t, auto w, auto taps) {
        hipLaunchKernelGGL((k_conv_step<decltype(t), decltype(w), taps()>), dim3(s.c.parts * shape.blocks_x), dim3(256), 0, strm(stream), s);
        return launch_check("k_conv_step");
    });
}

int jq_logits_forward(const jq_logits *a, void *out, int64_t out_stride, void *stream)
{
    TRY(check_logits(a));
    if (a->rows == 0) return JQ_OK;
    if (!a->logits || !out) return fail(JQ_E_ARG, "null device pointer");
    if (!aligned(a->logits, elem_bytes(a->dtype)) || !aligned(out, elem_bytes(a->dtype)))
        return fail(JQ_E_ARG, "rows must be aligned to their element size");
    LogitsArgs l = logits_args(a);
    l.o = out, l.o_stride = out_stride;
    return by_type(a->dtype, [&](auto t) {
        using T = decltype(t);
        const LogitsGrid g = logits_grid<T>(l);
        hipLaunchKernelGGL((k_logits<T, false>), g.grid, g.block, g.lds, strm(stream), l);
        return launch_check("k_logits");
    });
}

int jq_logits_workspace(const jq_logits *a, int64_t *bytes)
{
    TRY(check_logits(a));
    if (!bytes) return fail(JQ_E_ARG, "null output");
    *bytes = logits_parts(a) * a->actions * 4;
    return JQ_OK;
}

int jq_logits_backward(const jq_logits *a, const void *d_out, int64_t d_out_stride, void *d_logits, int64_t d_logits_stride,
                       float *d_bias, void *workspace, int64_t workspace_bytes, void *stream)
{
    TRY(check_logits(a));
    if (a->rows && (!d_out || (a->recent_count && d_logits && !a->logits))) return fail(JQ_E_ARG, "null device pointer");
    if (!aligned(a->logits, elem_bytes(a->dtype)) || !aligned(d_out, elem_bytes(a->dtype)) || !aligned(d_logits, elem_bytes(a->dtype)))
        return fail(JQ_E_ARG, "rows must be aligned to their element size");
    if (!d_logits && !d_bias) return JQ_OK;
    LogitsArgs l = logits_args(a);
    l.d = d_out, l.d_stride = d_out_stride, l.o = d_logits, l.o_stride = d_logits_stride;
    if (d_bias) {
        l.parts = (int)logits_parts(a);
        const int64_t need = (int64_t)l.parts * l.actions * 4;
        if (workspace_bytes < need || !workspace)
            return fail(JQ_E_ARG, "workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)need);
        if (!aligned(workspace, 4)) return fail(JQ_E_ARG, "workspace must be 4-byte aligned");
        TRY(check_pointer(d_bias, 4, "d_bias"));
        l.part = static_cast<float *>(workspace);
    }
    return by_type(a->dtype, [&](auto t) {
        using T = decltype(t);
        if (d_logits && l.rows) {
            const LogitsGrid g = logits_grid<T>(l);
            hipLaunchKernelGGL((k_logits<T, true>), g.grid, g.block, g.lds, strm(stream), l);
            TRY(launch_check("k_logits (gradient)"));
        }
        if (!d_bias) return JQ_OK;
        LogitsArgs sums = l;
        sums.tiles = bias_tiles(a);
        hipLaunchKernelGGL((k_logits_bias<T>), dim3(sums.tiles * sums.parts), dim3(256), 0, strm(stream), sums);
        TRY(launch_check("k_logits_bias"));
        hipLaunchKernelGGL(k_logits_join, dim3(std::min((l.actions + 15) / 16, LOGITS_JOIN_BLOCKS)), dim3(256), 0, strm(stream), l.part, l.parts, l.actions, d_bias);
        return launch_check("k_logits_join");
    });
}

}  // extern "C"
