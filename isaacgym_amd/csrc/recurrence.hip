// Gated linear recurrence h[t] = gate[t] h[t-1] + inp[t] over rollouts [T, N, D], and its gradients.
//
// Channels are independent and adjacent in memory, so a lane owns a vector of channels (16 bytes) and walks the steps with
// the carried value in fp32 registers.  A call moves 3 elements per (t, n, d) forward and 5 backward and does 2 - 3
// operations on each: HBM bounds it where there are enough channels to fill the card (32 x 65 536 x 64 bf16 forward and
// backward: 2.25 GB in 387 us, 5.8 TB/s; one step of 262 144 x 64 with its fp32 state: 235 MB in 40 us, 5.9 TB/s).  Arrays
// that nothing reads again soon go past the caches' replacement (non-temporal; loads too where a lane walks alone: 387 us
// against 438).  All times here are device times of graph replays on one set of buffers.
//
// With fewer channels the time is split, for the recurrence is a composition of maps h -> A h + B that is associative:
//   - within a workgroup SEG groups of lanes take a few consecutive steps each of the same channels, reduce them to
//     (A, B) in registers, exchange those - between the groups of a wave in registers, between waves through LDS - and then
//     walk their steps from the value that reaches them, so every element is still read and written once;
//   - across workgroups a first kernel reduces every span of the time to its (A, B) in a workspace, and each workgroup of
//     the second composes the spans before its own, while its first steps are on their way.  That reads gate and inp twice
//     (the second time mostly from the caches), so it is done only where the channels alone leave CUs without work: 8 192
//     steps of 512 channels in bf16 take 17 us forward and 20 us backward, bound by the latency of two launches and the
//     exchange (a lane for every 8 channels needs 10 600 us).
#include "igx_recurrence.hpp"

namespace igx {
namespace {

// nothing but the carried value goes through a call without steps
__global__ void carry_through_kernel(const float *from, float *to, int64_t n)
{
    const int64_t i = (int64_t)blockIdx.x * kRecBlock + threadIdx.x;
    if (i < n) to[i] = from ? from[i] : 0.0f;
}

int check(const igx_recurrence *r, const char *who)
{
    if (!r) return fail(IGX_E_NULL, "%s: r is NULL", who);
    if (!known_dtype(r->dtype)) return fail(IGX_E_PARAM, "%s: dtype %d is not IGX_F32, IGX_F16 or IGX_BF16", who, r->dtype);
    if (r->steps < 0 || r->envs < 0 || r->width < 0)
        return fail(IGX_E_SIZE, "%s: steps, envs and width must not be negative", who);
    const int64_t most = (int64_t)1 << 31;  // the grid's limit
    if (r->steps > most || r->envs > most || r->width > most || (r->width && r->envs > most / r->width))
        return fail(IGX_E_SIZE, "%s: %lld environments of %lld channels or %lld steps are more than 2^31", who,
                    (long long)r->envs, (long long)r->width, (long long)r->steps);
    if (r->gate_stride[2] != 0 && r->gate_stride[2] != 1)
        return fail(IGX_E_PARAM, "%s: the gate's channel stride must be 1 or 0, not %lld", who, (long long)r->gate_stride[2]);
    return IGX_OK;
}

// are environments n and n + 1 adjacent in this array?
bool follows(const igx_recurrence *r, int64_t stride_n) { return r->envs == 1 || stride_n == r->width; }

// How the time is split (both sides measured, forward + backward).  131 072 lanes and more walk the steps alone (64 x 16 384 x
// 64 fp32: 367 us, 441 in four groups).  With fewer, four groups share a workgroup's steps (32 x 4 096 x 64 fp32, 65 536
// lanes: 49 us, 89 alone), below 16 384 lanes sixteen.  A sequence goes to several workgroups in spans only where the
// channels fill fewer than 256 of them, one for each CU (300 x 64 x 256 fp32 fills 256: 45 us in one span, 64 in two, for
// gate and inp are then read twice); 512 workgroups in all are enough.  Where they fill 256 and the sequence is long,
// sixty-four groups keep a CU's waves busy (2 048 x 16 x 1 024 bf16: 134 us, 173 in sixteen; 1 024 x 64 x 256 fp32: 107, 123),
// unless a lane needs more than one flag a step, which takes the registers (1 000 x 200 x 105 bf16: 263, 207 in sixteen).
// Rollouts kept environment by environment have their next steps next to each other: four groups, however many lanes there
// are, and the caches, which complete the lines that narrow rows share (32 x 20 000 x 60 fp32: 290 us, 481 with lanes that walk
// alone past the caches).
void split(Plan &p)
{
    const int64_t vectors = p.a.vectors, T = p.a.T;
    p.spans = 1;
    p.a.span = T;
    p.seg = T <= steps_of(16) || (vectors >= 131072 && !p.apart) ? 1 : vectors >= 16384 ? 4 : 16;
    if (p.seg != 16) return;
    const int64_t strips = ceil_div(vectors, lanes_of(16)), tile = 16 * steps_of(16);
    if (strips >= 256) {
        if (T >= 512 && p.flags <= kOneFlag) p.seg = 64;
        return;
    }
    if (T <= tile) return;
    const int64_t want = ceil_div(512, strips), most = ceil_div(T, tile);
    const int64_t spans = want < most ? want : most;
    p.a.span = ceil_div(ceil_div(T, spans), tile) * tile;
    p.spans = ceil_div(T, p.a.span);
}

void make_plan(const igx_recurrence *r, const igx_recurrence_grad *g, const igx_recurrence_rest *rest, Plan &p)
{
    RecArgs &a = p.a;
    a = RecArgs();
    const int64_t e = element_size(r->dtype), T = r->steps, N = r->envs, D = r->width;
    const bool shared = r->gate_stride[2] == 0 && D > 1;
    bool flat;
    if (!g) {
        flat = follows(r, r->inp_stride[1]) && follows(r, r->out_stride[1]);
    } else {
        flat = (!g->d_out || follows(r, g->d_out_stride[1])) && (!g->d_inp || follows(r, g->d_inp_stride[1])) &&
               (!g->d_gate || (follows(r, g->d_gate_stride[1]) && follows(r, r->out_stride[1])));
    }
    if (g && !g->d_gate) rest = nullptr;  // not read
    if (rest) flat = flat && follows(r, rest->stride[1]);
    p.apart = !flat;
    a.past = flat;
    // one gate for everything (all strides 0 beyond time) keeps the environments in one run
    const bool one_gate = (r->gate_stride[1] == 0 || N == 1) && (r->gate_stride[2] == 0 || D == 1);
    flat = flat && (one_gate || (!shared && follows(r, r->gate_stride[1])));
    a.T = T;
    a.D = (uint32_t)D;
    a.run = (uint32_t)(flat ? N * D : D);
    a.splat = one_gate || shared;
    auto lanes = [&](int vec) {
        p.vec = a.run >= (uint32_t)vec ? vec : 1;
        a.per_run = (uint32_t)ceil_div(a.run, p.vec);
        a.vectors = (uint32_t)(flat ? 1 : N) * a.per_run;
        p.flags = !r->reset ? kNoFlags : (p.vec == 1 || !flat || D % p.vec == 0 || N == 1) ? kOneFlag : D >= p.vec ? kTwoFlags : kFlagEach;
        split(p);
    };
    lanes(r->dtype == IGX_F32 ? 4 : 8);
    if (r->dtype != IGX_F32 && p.seg > 1) {  // too few lanes: twice as many with half the bytes (8 192 x 1 x 512 bf16: 37 us, 51 with 8 channels)
        lanes(4);
        if (p.seg == 1) p.seg = 4;
    }

    // forward order: as stored, or turned round for reverse; the backward pass goes the other way through the same order
    const bool down = (r->reverse != 0) != (g != nullptr);
    auto turn = [&](const void *base, int64_t st, int64_t sn, int64_t size, int64_t &bt, int64_t &bn) -> const char * {
        const char *q = static_cast<const char *>(base);
        bt = (down ? -st : st) * size;
        bn = sn * size;
        return q && down ? q + (T - 1) * st * size : q;
    };
    a.gate = turn(r->gate, r->gate_stride[0], r->gate_stride[1], e, a.gate_t, a.gate_n);
    a.reset = turn(r->reset, r->reset_stride[0], r->reset_stride[1], 8, a.reset_t, a.reset_n);
    if (!g) {
        a.add = turn(r->inp, r->inp_stride[0], r->inp_stride[1], e, a.add_t, a.add_n);
        a.to = const_cast<char *>(turn(r->out, r->out_stride[0], r->out_stride[1], e, a.to_t, a.to_n));
        if (rest) a.rest = const_cast<char *>(turn(rest->codes, rest->stride[0], rest->stride[1], 1, a.rest_t, a.rest_n));
        a.start = r->state;
        a.end = r->last;
    } else {
        a.add = turn(g->d_out, g->d_out_stride[0], g->d_out_stride[1], e, a.add_t, a.add_n);
        a.to = const_cast<char *>(turn(g->d_inp, g->d_inp_stride[0], g->d_inp_stride[1], e, a.to_t, a.to_n));
        a.d_gate = const_cast<char *>(turn(g->d_gate, g->d_gate_stride[0], g->d_gate_stride[1], e, a.d_gate_t, a.d_gate_n));
        if (a.d_gate) {  // the value before a step is one step further on in out, counted backwards
            a.before = turn(r->out, r->out_stride[0], r->out_stride[1], e, a.before_t, a.before_n);
            a.before += a.before_t;
            if (rest) {
                a.rest = const_cast<char *>(turn(rest->codes, rest->stride[0], rest->stride[1], 1, a.rest_t, a.rest_n));
                a.rest += a.rest_t;
            }
            a.state = r->state;
        }
        a.start = g->d_last;
        a.end = g->d_state;
    }
}

template <bool BACKWARD> int launch(const igx_recurrence *r, Plan &p, hipStream_t s, const char *who)
{
    const int64_t need = p.workspace();
    if (need) {
        if (!r->workspace) return fail(IGX_E_NULL, "%s: workspace is NULL", who);
        if (!aligned16(r->workspace)) return fail(IGX_E_ALIGN, "%s: workspace must be 16-byte aligned", who);
        if (r->workspace_bytes < need)
            return fail(IGX_E_SIZE, "%s: workspace of %lld bytes is smaller than igx_linear_recurrence_workspace()", who,
                        (long long)r->workspace_bytes);
        p.a.spans = static_cast<float *>(r->workspace);
    }
    launch_recurrence<BACKWARD>(r->dtype, p, s);
    return launch_status(who);
}

int carry_through(const float *from, float *to, int64_t n, hipStream_t s, const char *who)
{
    if (!to || n == 0 || to == from) return IGX_OK;
    carry_through_kernel<<<dim3((unsigned)ceil_div(n, kRecBlock)), dim3(kRecBlock), 0, s>>>(from, to, n);
    return launch_status(who);
}

}  // namespace
}  // namespace igx

extern "C" int64_t igx_linear_recurrence_workspace(const igx_recurrence *r)
{
    const int rc = igx::check(r, __func__);
    if (rc) return rc;
    // which environments follow each other decides how many lanes there are, and that differs with the arrays of the two
    // passes: the most that either could need, from lanes per environment and lanes over all of them
    int64_t most = 0;
    if (r->steps == 0 || r->envs == 0 || r->width == 0) return 0;
    igx_recurrence q = *r;
    for (int apart = 0; apart < 2; apart++) {
        q.inp_stride[1] = q.out_stride[1] = r->width + apart;
        igx::Plan p;
        igx::make_plan(&q, nullptr, nullptr, p);
        if (p.workspace() > most) most = p.workspace();
    }
    return most;
}

namespace igx {
namespace {

int check_rest(const igx_recurrence *r, const igx_recurrence_rest *rest, const char *who)
{
    if (!rest) return IGX_OK;
    if (r->dtype == IGX_F32) return fail(IGX_E_PARAM, "%s: float32 results are not rounded, there is no rest", who);
    return IGX_OK;
}

int forward(const igx_recurrence *r, const igx_recurrence_rest *rest, igx_stream_t stream, const char *who)
{
    int rc = check(r, who);
    if (!rc) rc = check_rest(r, rest, who);
    if (rc) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t channels = r->envs * r->width;
    if (channels == 0) return IGX_OK;
    if (r->steps == 0) return carry_through(r->state, r->last, channels, s, who);
    if (!r->gate) return fail(IGX_E_NULL, "%s: gate is NULL", who);
    if (!r->inp) return fail(IGX_E_NULL, "%s: inp is NULL", who);
    if (!r->out) return fail(IGX_E_NULL, "%s: out is NULL", who);
    if (rest && !rest->codes) return fail(IGX_E_NULL, "%s: codes is NULL", who);
    Plan p;
    make_plan(r, nullptr, rest, p);
    return launch<false>(r, p, s, who);
}

int backward(const igx_recurrence *r, const igx_recurrence_grad *g, const igx_recurrence_rest *rest, igx_stream_t stream,
             const char *who)
{
    int rc = check(r, who);
    if (!rc) rc = check_rest(r, rest, who);
    if (rc) return rc;
    if (!g) return fail(IGX_E_NULL, "%s: g is NULL", who);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t channels = r->envs * r->width;
    if (channels == 0 || (!g->d_gate && !g->d_inp && !g->d_state)) return IGX_OK;
    if (r->steps == 0) return carry_through(g->d_last, g->d_state, channels, s, who);
    if (!r->gate) return fail(IGX_E_NULL, "%s: gate is NULL", who);
    if (g->d_gate && !r->out) return fail(IGX_E_NULL, "%s: out is NULL", who);
    if (g->d_gate && rest && !rest->codes) return fail(IGX_E_NULL, "%s: codes is NULL", who);
    Plan p;
    make_plan(r, g, rest, p);
    return launch<true>(r, p, s, who);
}

}  // namespace
}  // namespace igx

extern "C" int igx_linear_recurrence(const igx_recurrence *r, igx_stream_t stream)
{
    return igx::forward(r, nullptr, stream, __func__);
}

extern "C" int igx_linear_recurrence_backward(const igx_recurrence *r, const igx_recurrence_grad *g, igx_stream_t stream)
{
    return igx::backward(r, g, nullptr, stream, __func__);
}

extern "C" int igx_linear_recurrence_with_rest(const igx_recurrence *r, const igx_recurrence_rest *rest, igx_stream_t stream)
{
    return igx::forward(r, rest, stream, __func__);
}

extern "C" int igx_linear_recurrence_backward_with_rest(const igx_recurrence *r, const igx_recurrence_grad *g,
                                                        const igx_recurrence_rest *rest, igx_stream_t stream)
{
    return igx::backward(r, g, rest, stream, __func__);
}
