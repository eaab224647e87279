// Gated linear recurrence h[t] = gate[t] h[t-1] + inp[t] over rollouts [T, N, D], and its gradients.
//
// Channels are independent and adjacent in memory, so a lane owns one 16-byte vector of channels and walks the steps
// with the state in fp32 registers.  A call moves 3 elements per (t, n, d) forward and 5 backward and does 2 - 3
// operations on each: HBM bounds it.
#include "igx_seq.hpp"

namespace igx {
namespace {

constexpr int kUnroll = 8;   // steps whose loads are in flight together: they do not depend on the state
constexpr int kBlock = 256;

enum Flags { kNoFlags = 0, kOneFlag = 1, kFlagEach = 2 };

// One call as the kernels see it.  The steps are numbered in the order they are computed (the host turns an array
// round by pointing at its last step and negating its stride), strides are in bytes.
struct RecArgs {
    const char *gate, *inp, *reset, *out_r;
    char *out;
    const float *state;
    float *last;
    const char *d_out;
    char *d_gate, *d_inp;
    const float *d_last;
    float *d_state;
    int64_t gate_t, gate_n, inp_t, inp_n, reset_t, reset_n, out_t, out_n;
    int64_t d_out_t, d_out_n, d_gate_t, d_gate_n, d_inp_t, d_inp_n;
    int64_t T, D;
    int64_t run;      // channels that are adjacent in every array: N * D where the environments follow each other, else D
    int64_t per_run;  // vectors in a run
    int64_t vectors;  // vectors in all
    int splat;        // one gate for all channels of a run
};

// Which channels a lane owns: V of them from `col` of run `row`.  The last vector of a run that V does not divide is
// moved back to end with the run: its first `skip` channels belong to the lane before and are computed but not stored.
struct Lane {
    int64_t row, col;
    int skip;
};

template <int V> __device__ __forceinline__ Lane lane_of(const RecArgs &a, int64_t v)
{
    Lane l;
    l.row = a.per_run == a.vectors ? 0 : v / a.per_run;
    l.col = (v - l.row * a.per_run) * V;
    l.skip = 0;
    if (l.col + V > a.run) {
        l.skip = (int)(l.col + V - a.run);
        l.col = a.run - V;
    }
    return l;
}

template <typename T, int V> __device__ __forceinline__ void store_from(char *p, const float (&f)[V], int skip)
{
    if (V == 1 || skip == 0) {
        store_vec<T, V>(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i >= skip) reinterpret_cast<T *>(p)[i] = (T)f[i];
    }
}

// Reset flags of the lane's channels for one step: one environment for all of them (a single flag), or one each.
template <int V, int FL> struct LaneFlags {
    const char *p[FL == kFlagEach ? V : 1];
    __device__ __forceinline__ LaneFlags(const RecArgs &a, const Lane &l)
    {
        if constexpr (FL == kNoFlags) return;
        const int64_t first = l.row * (a.run / a.D);  // run = D: the run's environment; run = N * D: row is 0
        if constexpr (FL == kOneFlag) {
            p[0] = a.reset + (first + l.col / a.D) * a.reset_n;
        } else if constexpr (FL == kFlagEach) {
#pragma unroll
            for (int i = 0; i < V; i++) p[i] = a.reset + (first + (l.col + i) / a.D) * a.reset_n;
        }
    }
};

template <int V, int FL> struct StepFlags {
    int64_t f[FL == kFlagEach ? V : 1];
    __device__ __forceinline__ void load(const LaneFlags<V, FL> &lf, int64_t off)
    {
        if constexpr (FL != kNoFlags) {
#pragma unroll
            for (int i = 0; i < (FL == kFlagEach ? V : 1); i++) f[i] = *reinterpret_cast<const int64_t *>(lf.p[i] + off);
        }
    }
    __device__ __forceinline__ bool begins(int i) const
    {
        if constexpr (FL == kNoFlags) return false;
        return f[FL == kFlagEach ? i : 0] != 0;
    }
};

template <typename T, int V> __device__ __forceinline__ void load_gate(Raw<T, V> &g, const char *p, int splat)
{
    if (V == 1 || !splat) {
        g = load_raw<T, V>(p);
    } else if constexpr (V > 1) {
        const T one = *reinterpret_cast<const T *>(p);
#pragma unroll
        for (int i = 0; i < V; i++) g.v[i] = one;
    }
}

template <typename T, int V, int FL> __global__ __launch_bounds__(kBlock) void recurrence_kernel(RecArgs a)
{
    const int64_t v = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (v >= a.vectors) return;
    const Lane l = lane_of<V>(a, v);
    const LaneFlags<V, FL> lf(a, l);
    const char *gate = a.gate + l.row * a.gate_n + (a.splat ? 0 : l.col * (int64_t)sizeof(T));
    const char *inp = a.inp + l.row * a.inp_n + l.col * sizeof(T);
    char *out = a.out + l.row * a.out_n + l.col * sizeof(T);
    const int64_t c = l.row * a.run + l.col;
    float h[V];
#pragma unroll
    for (int i = 0; i < V; i++) h[i] = a.state ? a.state[c + i] : 0.0f;
    for (int64_t t0 = 0; t0 < a.T; t0 += kUnroll) {
        Raw<T, V> g[kUnroll], x[kUnroll];
        StepFlags<V, FL> f[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; k++) {
            const int64_t t = t0 + k < a.T ? t0 + k : a.T - 1;
            load_gate<T, V>(g[k], gate + t * a.gate_t, a.splat);
            x[k] = load_raw<T, V>(inp + t * a.inp_t);
            f[k].load(lf, t * a.reset_t);
        }
#pragma unroll
        for (int k = 0; k < kUnroll; k++) {
            if (t0 + k >= a.T) break;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float add = raw_at(x[k], i);
                h[i] = f[k].begins(i) ? add : fmaf(raw_at(g[k], i), h[i], add);
            }
            store_from<T, V>(out + (t0 + k) * a.out_t, h, l.skip);
        }
    }
    if (a.last) {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i >= l.skip) a.last[c + i] = h[i];
    }
}

// Backward: the steps are numbered from the last computed one, `carry` is what the later steps hand back.
//     d = d_out + carry;  d_inp = d;  d_gate = d * before;  carry = gate * d
template <typename T, int V, int FL> __global__ __launch_bounds__(kBlock) void recurrence_backward_kernel(RecArgs a)
{
    const int64_t v = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (v >= a.vectors) return;
    const Lane l = lane_of<V>(a, v);
    const LaneFlags<V, FL> lf(a, l);
    const char *gate = a.gate + l.row * a.gate_n + (a.splat ? 0 : l.col * (int64_t)sizeof(T));
    const char *before = a.out_r + l.row * a.out_n + l.col * sizeof(T);
    const char *d_out = a.d_out ? a.d_out + l.row * a.d_out_n + l.col * sizeof(T) : nullptr;
    char *d_gate = a.d_gate ? a.d_gate + l.row * a.d_gate_n + l.col * sizeof(T) : nullptr;
    char *d_inp = a.d_inp ? a.d_inp + l.row * a.d_inp_n + l.col * sizeof(T) : nullptr;
    const int64_t c = l.row * a.run + l.col;
    float carry[V];
#pragma unroll
    for (int i = 0; i < V; i++) carry[i] = a.d_last ? a.d_last[c + i] : 0.0f;
    for (int64_t t0 = 0; t0 < a.T; t0 += kUnroll) {
        Raw<T, V> g[kUnroll], y[kUnroll], hb[kUnroll];
        StepFlags<V, FL> f[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; k++) {
            const int64_t t = t0 + k < a.T ? t0 + k : a.T - 1;
            load_gate<T, V>(g[k], gate + t * a.gate_t, a.splat);
            f[k].load(lf, t * a.reset_t);
        }
        if (d_out) {
#pragma unroll
            for (int k = 0; k < kUnroll; k++) {
                const int64_t t = t0 + k < a.T ? t0 + k : a.T - 1;
                y[k] = load_raw<T, V>(d_out + t * a.d_out_t);
            }
        }
        if (d_gate) {
#pragma unroll
            for (int k = 0; k < kUnroll; k++) {  // the value before the first step is `state`, not in out
                const int64_t t = t0 + k < a.T - 1 ? t0 + k : a.T - 2;
                if (a.T > 1) hb[k] = load_raw<T, V>(before + t * a.out_t);
            }
        }
#pragma unroll
        for (int k = 0; k < kUnroll; k++) {
            if (t0 + k >= a.T) break;
            float d[V], dg[V];
            const bool first = t0 + k == a.T - 1;
#pragma unroll
            for (int i = 0; i < V; i++) {
                d[i] = (d_out ? raw_at(y[k], i) : 0.0f) + carry[i];
                const bool begins = f[k].begins(i);
                if (d_gate) {
                    const float h = first ? (a.state ? a.state[c + i] : 0.0f) : raw_at(hb[k], i);
                    dg[i] = begins ? 0.0f : d[i] * h;
                }
                carry[i] = begins ? 0.0f : raw_at(g[k], i) * d[i];
            }
            if (d_inp) store_from<T, V>(d_inp + (t0 + k) * a.d_inp_t, d, l.skip);
            if (d_gate) store_from<T, V>(d_gate + (t0 + k) * a.d_gate_t, dg, l.skip);
        }
    }
    if (a.d_state) {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i >= l.skip) a.d_state[c + i] = carry[i];
    }
}

// nothing but the carried value goes through a call without steps
__global__ void carry_through_kernel(const float *from, float *to, int64_t n)
{
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i < n) to[i] = from ? from[i] : 0.0f;
}

struct Plan {
    RecArgs a;
    int vec;    // channels per lane: the type's 16 bytes, or 1 where a run is shorter than that
    int flags;
};

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

void make_plan(const igx_recurrence *r, const igx_recurrence_grad *g, Plan &p)
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
    // one gate for everything (all strides 0 beyond time) keeps the environments in one run
    const bool one_gate = (r->gate_stride[1] == 0 || N == 1) && (r->gate_stride[2] == 0 || D == 1);
    flat = flat && (one_gate || (!shared && follows(r, r->gate_stride[1])));
    a.T = T;
    a.D = D;
    a.run = flat ? N * D : D;
    a.splat = one_gate || shared;
    p.vec = a.run >= (r->dtype == IGX_F32 ? 4 : 8) ? (r->dtype == IGX_F32 ? 4 : 8) : 1;
    a.per_run = ceil_div(a.run, p.vec);
    a.vectors = (flat ? 1 : N) * a.per_run;
    p.flags = !r->reset ? kNoFlags : (p.vec == 1 || !flat || D % p.vec == 0 || N == 1) ? kOneFlag : kFlagEach;

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
    a.state = r->state;
    if (!g) {
        a.inp = turn(r->inp, r->inp_stride[0], r->inp_stride[1], e, a.inp_t, a.inp_n);
        a.out = const_cast<char *>(turn(r->out, r->out_stride[0], r->out_stride[1], e, a.out_t, a.out_n));
        a.last = r->last;
    } else {
        // the value before the step that comes first backwards (the last computed) is one step further on in out
        a.out_r = turn(r->out, r->out_stride[0], r->out_stride[1], e, a.out_t, a.out_n);
        if (a.out_r) a.out_r += a.out_t;
        a.d_out = turn(g->d_out, g->d_out_stride[0], g->d_out_stride[1], e, a.d_out_t, a.d_out_n);
        a.d_gate = const_cast<char *>(turn(g->d_gate, g->d_gate_stride[0], g->d_gate_stride[1], e, a.d_gate_t, a.d_gate_n));
        a.d_inp = const_cast<char *>(turn(g->d_inp, g->d_inp_stride[0], g->d_inp_stride[1], e, a.d_inp_t, a.d_inp_n));
        a.d_last = g->d_last;
        a.d_state = g->d_state;
    }
}

template <int DT> void launch(const Plan &p, bool backward, hipStream_t s)
{
    using T = typename Elem<DT>::type;
    constexpr int V = Elem<DT>::vec;
    const dim3 grid((unsigned)ceil_div(p.a.vectors, kBlock)), block(kBlock);
#define IGX_REC_GO(VV, FF)                                                                       \
    do {                                                                                         \
        if (backward) recurrence_backward_kernel<T, VV, FF><<<grid, block, 0, s>>>(p.a);         \
        else recurrence_kernel<T, VV, FF><<<grid, block, 0, s>>>(p.a);                           \
    } while (0)
    if (p.vec == 1) {
        if (p.flags == kNoFlags) IGX_REC_GO(1, kNoFlags);
        else IGX_REC_GO(1, kOneFlag);
    } else {
        if (p.flags == kNoFlags) IGX_REC_GO(V, kNoFlags);
        else if (p.flags == kOneFlag) IGX_REC_GO(V, kOneFlag);
        else IGX_REC_GO(V, kFlagEach);
    }
#undef IGX_REC_GO
}

void launch_any(int dtype, const Plan &p, bool backward, hipStream_t s)
{
    if (dtype == IGX_F32) launch<IGX_F32>(p, backward, s);
    else if (dtype == IGX_F16) launch<IGX_F16>(p, backward, s);
    else launch<IGX_BF16>(p, backward, s);
}

int carry_through(const float *from, float *to, int64_t n, hipStream_t s, const char *who)
{
    if (!to || n == 0 || to == from) return IGX_OK;
    carry_through_kernel<<<dim3((unsigned)ceil_div(n, kBlock)), dim3(kBlock), 0, s>>>(from, to, n);
    return launch_status(who);
}

}  // namespace
}  // namespace igx

extern "C" int64_t igx_linear_recurrence_workspace(const igx_recurrence *r)
{
    const int rc = igx::check(r, __func__);
    return rc ? rc : 0;
}

extern "C" int igx_linear_recurrence(const igx_recurrence *r, igx_stream_t stream)
{
    int rc = igx::check(r, __func__);
    if (rc) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t channels = r->envs * r->width;
    if (channels == 0) return IGX_OK;
    if (r->steps == 0) return igx::carry_through(r->state, r->last, channels, s, __func__);
    IGX_REQUIRE_PTR(r->gate, "gate");
    IGX_REQUIRE_PTR(r->inp, "inp");
    IGX_REQUIRE_PTR(r->out, "out");
    igx::Plan p;
    igx::make_plan(r, nullptr, p);
    igx::launch_any(r->dtype, p, false, s);
    return igx::launch_status(__func__);
}

extern "C" int igx_linear_recurrence_backward(const igx_recurrence *r, const igx_recurrence_grad *g, igx_stream_t stream)
{
    int rc = igx::check(r, __func__);
    if (rc) return rc;
    IGX_REQUIRE_PTR(g, "g");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t channels = r->envs * r->width;
    if (channels == 0 || (!g->d_gate && !g->d_inp && !g->d_state)) return IGX_OK;
    if (r->steps == 0) return igx::carry_through(g->d_last, g->d_state, channels, s, __func__);
    IGX_REQUIRE_PTR(r->gate, "gate");
    if (g->d_gate) IGX_REQUIRE_PTR(r->out, "out");
    igx::Plan p;
    igx::make_plan(r, g, p);
    igx::launch_any(r->dtype, p, true, s);
    return igx::launch_status(__func__);
}
