// The linear recurrence's kernels (recurrence.hip instantiates the forward, recurrence_backward.hip the backward ones).
#pragma once
#include <type_traits>

#include "igx_seq.hpp"

namespace igx {

constexpr int kRecBlock = 256;

// reset flags a lane needs for a step: its channels belong to one environment, to two, or to any number
enum Flags { kNoFlags = 0, kOneFlag = 1, kTwoFlags = 2, kFlagEach = 3 };

// One call as the kernels see it.  The steps are numbered in the order they are computed (the host turns an array
// round by pointing at its last step and negating its stride), strides are in bytes.  Forward reads gate and `add` = inp;
// backward runs the other way, add = d_out, before = out one step further on.
struct RecArgs {
    const char *gate, *add, *reset, *before;
    char *rest;                 // what out's rounding took: forward writes it, backward reads it beside `before`; NULL: not kept
    char *to, *d_gate;          // forward: out; backward: d_inp, d_gate (NULL: not wanted)
    const float *start;         // forward: state, backward: d_last; NULL: zeros
    float *end;                 // forward: last, backward: d_state; NULL: not wanted
    const float *state;         // backward: what stands before the first step; NULL: zeros
    float *spans;               // [0]: start; [1 + 2 s], [2 + 2 s]: A and B of span s; rows of `vectors` lane vectors
    int64_t gate_t, gate_n, add_t, add_n, reset_t, reset_n, before_t, before_n, rest_t, rest_n, to_t, to_n, d_gate_t, d_gate_n;
    int64_t T, span;            // steps in all, and in a span
    uint32_t D;
    uint32_t run;      // channels that are adjacent in every array: N * D where the environments follow each other, else D
    uint32_t per_run;  // vectors in a run
    uint32_t vectors;  // vectors in all
    int splat;         // one gate for all channels of a run
    int past;          // what is written goes past the caches' replacement
};

// Which channels a lane owns: V of them from `col` of run `row`.  The last vector of a run that V does not divide is
// moved back to end with the run: its first `skip` channels belong to the lane before and are computed but not stored.
struct Lane {
    uint32_t row, col;
    int skip;
    int64_t channel;  // of state, last and their gradients
};

template <int V> __device__ __forceinline__ Lane lane_of(const RecArgs &a, uint32_t v)
{
    Lane l;
    l.row = a.per_run == a.vectors ? 0 : v / a.per_run;
    l.col = (v - l.row * a.per_run) * V;
    l.skip = 0;
    if (V > 1 && a.run - l.col < V) {
        l.skip = (int)(V - (a.run - l.col));
        l.col = a.run - V;
    }
    l.channel = (int64_t)l.row * a.run + l.col;
    return l;
}

template <typename T, int V, bool STREAM = false> __device__ __forceinline__ void store_from(char *p, const float (&f)[V], int skip)
{
    if (V == 1 || skip == 0) {
        store_vec<T, V, STREAM>(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i >= skip) reinterpret_cast<T *>(p)[i] = (T)f[i];
    }
}

template <typename T, int V> __device__ __forceinline__ void store_step(const RecArgs &a, char *p, const float (&f)[V], int skip)
{
    if (a.past) store_from<T, V, true>(p, f, skip);
    else store_from<T, V>(p, f, skip);
}

// What the rounding to a 16-bit type took from a value, as 8 more bits: numbers of one sign order like their fp32 bit patterns,
// so it is the difference of the value's and the rounded value's patterns, counted in 1/256 of the type's step (2^16 patterns
// in bf16, 2^13 in fp16) and rounded to that: value and sum differ by at most 2^-7 of the half step that out is off by, and not
// at all where out is the value.  fp16's subnormals, whose steps are wider, gain less.  Beside inf and NaN it is 0.  8 bits, not
// the 16 that would be fp32: what is computed from the sum is itself rounded to T, a step 2^8 times as wide.  They take half
// of an array's bytes each way and go through the caches even where the arrays go past them (32 x 65 536 x 64 bf16, a training
// pass: 427 us, 469 past the caches, 398 without codes).
template <typename T> constexpr int kRestShift = sizeof(T) == 4 ? 0 : std::is_same<T, __bf16>::value ? 8 : 5;

template <typename T> __device__ __forceinline__ int rest_code(float h)
{
    constexpr int S = kRestShift<T>;
    const uint32_t o = __float_as_uint((float)(T)h);
    const int d = (int)(__float_as_uint(h) - o);
    const int code = min(max((d + (1 << S >> 1)) >> S, -128), 127);
    return (o & 0x7f800000u) == 0x7f800000u ? 0 : code;
}

template <int V> struct RestWords {
    static constexpr int kCount = V >= 4 ? V / 4 : 1;
    uint32_t w[kCount];
    __device__ __forceinline__ int at(int i) const { return (int8_t)(w[i / 4] >> (8 * (i % 4))); }
};

template <int V> __device__ __forceinline__ RestWords<V> load_rest(const char *p)
{
    RestWords<V> r;
    if constexpr (V == 1) {
        r.w[0] = *reinterpret_cast<const uint8_t *>(p);
    } else {
        typedef uint32_t Word __attribute__((aligned(1)));
#pragma unroll
        for (int j = 0; j < V / 4; j++) {
            r.w[j] = reinterpret_cast<const Word *>(p)[j];
        }
    }
    return r;
}

template <typename T, int V> __device__ __forceinline__ void store_rest(char *p, const float (&h)[V], int skip)
{
    if (V == 1 || skip) {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i >= skip) p[i] = (char)rest_code<T>(h[i]);
    } else if constexpr (V > 1) {
        typedef uint32_t Word __attribute__((aligned(1)));
#pragma unroll
        for (int j = 0; j < V / 4; j++) {
            uint32_t c[4];
#pragma unroll
            for (int i = 0; i < 4; i++) c[i] = (uint32_t)rest_code<T>(h[4 * j + i]);
            const uint32_t low = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400), high = __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400);
            reinterpret_cast<Word *>(p)[j] = __builtin_amdgcn_perm(high, low, 0x05040100);
        }
    }
}

// Reset flags of the lane's channels for one step: one environment's, that of the first and the last (the environment
// changes at channel `cut`), or each channel's.
template <int V, int FL> struct LaneFlags {
    static constexpr int kCount = FL == kFlagEach ? V : FL == kTwoFlags ? 2 : 1;
    const char *p[kCount];
    int cut;
    __device__ __forceinline__ LaneFlags(const RecArgs &a, const Lane &l)
    {
        if constexpr (FL == kNoFlags) return;
        // a run of D channels is one environment; the only run of N * D holds them all
#pragma unroll
        for (int i = 0; i < kCount; i++) {
            const uint32_t env = l.row + (l.col + (FL == kTwoFlags && i ? V - 1 : i)) / a.D;
            p[i] = a.reset + (int64_t)env * a.reset_n;
            if (FL == kTwoFlags && i) cut = (int)((env - l.row) * a.D - l.col);
        }
    }
};

// Steps whose loads a lane has in flight, by the groups that share a workgroup's channels (device time of forward and
// backward): with a lane for all steps 1, since thousands of waves are in flight and fewer rows [N, D] open at a time suit
// HBM better (32 x 65 536 x 64 bf16: 387 us with 1, 408 with 2, 413 with 4, 467 with 8); with four groups 2 (32 x 4 096 x 64
// fp32: 49 us, 50 with 4, 53 with 8); with sixteen, where waves are few, 8 (256 x 16 x 1 024 bf16: 27 us, 34 with 4); with
// sixty-four, whose 16 waves leave 128 registers each, 4.
constexpr int steps_of(int seg) { return seg == 1 ? 1 : seg == 4 ? 2 : seg == 16 ? 8 : 4; }

template <int V, int FL> struct StepFlags {
    using Places = LaneFlags<V, FL>;
    int64_t f[Places::kCount];
    int cut;
    __device__ __forceinline__ void load(const Places &lf, int64_t off)
    {
        if constexpr (FL != kNoFlags) {
#pragma unroll
            for (int i = 0; i < Places::kCount; i++) f[i] = *reinterpret_cast<const int64_t *>(lf.p[i] + off);
            if (FL == kTwoFlags) cut = lf.cut;
        }
    }
    __device__ __forceinline__ bool begins(int i) const
    {
        if constexpr (FL == kNoFlags) return false;
        if constexpr (FL == kTwoFlags) return i < cut ? f[0] != 0 : f[1] != 0;
        return f[FL == kFlagEach ? i : 0] != 0;
    }
};

template <typename T, int V, bool STREAM> __device__ __forceinline__ void load_gate(Raw<T, V> &g, const char *p, int splat)
{
    if (V == 1 || !splat) {
        g = load_raw<T, V, STREAM>(p);
    } else if constexpr (V > 1) {
        const T one = *reinterpret_cast<const T *>(p);
#pragma unroll
        for (int i = 0; i < V; i++) g.v[i] = one;
    }
}

// The map of some steps, h -> A h + B.  Behind an episode's start nothing of h is left, not even an inf or NaN times 0:
// such a map has kDropped for A, a NaN that arithmetic does not produce.  And where nothing is carried in, the result is
// B, also where A has left fp32's range.
constexpr uint32_t kDropped = 0x7fc0d209u;
__device__ __forceinline__ bool dropped(float A) { return __float_as_uint(A) == kDropped; }
__device__ __forceinline__ float through(float A, float B, float h) { return h == 0.0f || dropped(A) ? B : fmaf(A, h, B); }
__device__ __forceinline__ float as_factor(float A, bool none)
{
    return __uint_as_float(none ? kDropped : A != A ? 0x7fc00000u : __float_as_uint(A));
}

// K consecutive steps of a lane's channels in registers.  `count` of them exist, the others repeat the last one and are
// neutral; whole steps of a full group cost no test (CHECK false).  REST: there may be codes of out's rounding.
template <typename T, int V, int FL, int K, bool BACKWARD, bool CHECK, bool STREAM, bool REST> struct Steps {
    Raw<T, V> g[K], x[K], hb[K];
    RestWords<V> rb[K];  // REST
    StepFlags<V, FL> f[K];
    int count;

    // The addresses run along by a stride: a product of 64 bits for every load would cost more than the recurrence.  Steps
    // that do not exist repeat the last one.
    __device__ __forceinline__ void load(const RecArgs &a, const LaneFlags<V, FL> &lf, const char *gate, const char *add,
                                         const char *before, const char *rest, int64_t t0, int64_t t1)
    {
        count = CHECK ? (t1 - t0 < K ? (int)(t1 - t0) : K) : K;
        const int64_t t = CHECK && t0 >= t1 ? t1 - 1 : t0;
        gate += t * a.gate_t;
        int64_t flag = t * a.reset_t;
#pragma unroll
        for (int k = 0; k < K; k++) {
            load_gate<T, V, STREAM>(g[k], gate, a.splat);
            f[k].load(lf, flag);
            gate += on(k) ? a.gate_t : 0;
            flag += on(k) ? a.reset_t : 0;
        }
        if (!BACKWARD || add) {
            add += t * a.add_t;
#pragma unroll
            for (int k = 0; k < K; k++) {
                x[k] = load_raw<T, V, STREAM>(add);
                add += on(k) ? a.add_t : 0;
            }
        } else {
#pragma unroll
            for (int k = 0; k < K; k++) x[k] = {};
        }
        if (BACKWARD && before) {
            before += t * a.before_t;
#pragma unroll
            for (int k = 0; k < K; k++) {  // before the first step stands `state`, which is not in out
                if (t + k < a.T - 1) hb[k] = load_raw<T, V, STREAM>(before);
                before += on(k) ? a.before_t : 0;
            }
            if constexpr (REST) {
#pragma unroll
                for (int k = 0; k < K; k++) rb[k] = {};
                if (rest) {
                    rest += t * a.rest_t;
#pragma unroll
                    for (int k = 0; k < K; k++) {
                        if (t + k < a.T - 1) rb[k] = load_rest<V>(rest);
                        rest += on(k) ? a.rest_t : 0;
                    }
                }
            }
        }
    }
    // the value before step k, from out (and what its rounding took)
    __device__ __forceinline__ float value_before(int k, int i) const
    {
        if constexpr (REST)
            return __uint_as_float(__float_as_uint(raw_at(hb[k], i)) + (uint32_t)(rb[k].at(i) << kRestShift<T>));
        else
            return raw_at(hb[k], i);
    }
    __device__ __forceinline__ bool on(int k) const { return !CHECK || k + 1 < count; }  // is there a step behind step k?
    __device__ __forceinline__ bool there(int k) const { return !CHECK || k < count; }

    // the steps as one map (A, B) after those already in it; `starts`: channels in which an episode began
    __device__ __forceinline__ void reduce(float (&A)[V], float (&B)[V], bool (&starts)[V]) const
    {
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                const bool begins = f[k].begins(i);
                const float gate = raw_at(g[k], i), x1 = raw_at(x[k], i);
                const float b = BACKWARD ? (begins ? 0.0f : gate * (B[i] + x1)) : (begins ? x1 : fmaf(gate, B[i], x1));
                A[i] = there(k) ? gate * A[i] : A[i];
                B[i] = there(k) ? b : B[i];
                starts[i] = starts[i] || (there(k) && begins);
            }
        }
    }

    // forward: h = gate h + inp -> out, rest.  backward: d = d_out + h -> d_inp, d * before -> d_gate, h = gate d
    __device__ __forceinline__ void walk(const RecArgs &a, const Lane &l, bool store, char *to, char *d_gate, char *rest,
                                         int64_t t0, float (&h)[V]) const
    {
        if (to) to += t0 * a.to_t;
        if (!BACKWARD && rest) rest += t0 * a.rest_t;
        if (BACKWARD && d_gate) d_gate += t0 * a.d_gate_t;
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (CHECK && !there(k)) break;
            if constexpr (!BACKWARD) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float x1 = raw_at(x[k], i);
                    h[i] = f[k].begins(i) ? x1 : fmaf(raw_at(g[k], i), h[i], x1);
                }
                if (store) store_step<T, V>(a, to, h, l.skip);
                if constexpr (REST) {
                    if (rest) {
                        if (store) store_rest<T, V>(rest, h, l.skip);
                        rest += a.rest_t;
                    }
                }
            } else {
                float d[V], dg[V];
#pragma unroll
                for (int i = 0; i < V; i++) {
                    d[i] = raw_at(x[k], i) + h[i];
                    dg[i] = 0.0f;
                    h[i] = f[k].begins(i) ? 0.0f : raw_at(g[k], i) * d[i];
                }
                if (d_gate) {
                    if (t0 + k < a.T - 1) {
#pragma unroll
                        for (int i = 0; i < V; i++) dg[i] = f[k].begins(i) ? 0.0f : d[i] * value_before(k, i);
                    } else if (a.state) {
#pragma unroll
                        for (int i = 0; i < V; i++) dg[i] = f[k].begins(i) ? 0.0f : d[i] * a.state[l.channel + i];
                    }
                    if (store) store_step<T, V>(a, d_gate, dg, l.skip);
                    d_gate += a.d_gate_t;
                }
                if (to && store) store_step<T, V>(a, to, d, l.skip);
            }
            if (to) to += a.to_t;
        }
    }
};

template <int V> __device__ __forceinline__ void identity(float (&A)[V], float (&B)[V], bool (&starts)[V])
{
#pragma unroll
    for (int i = 0; i < V; i++) A[i] = 1.0f, B[i] = 0.0f, starts[i] = false;
}

// A as the maps hold it
template <int V> __device__ __forceinline__ void mark(float (&A)[V], const bool (&starts)[V])
{
#pragma unroll
    for (int i = 0; i < V; i++) A[i] = as_factor(A[i], starts[i]);
}

// where a lane's channels lie in the arrays
template <typename T> struct Places {
    const char *gate, *add, *before;
    char *rest, *to, *d_gate;
    __device__ __forceinline__ Places(const RecArgs &a, const Lane &l)
    {
        const int64_t at = (int64_t)l.col * sizeof(T);
        gate = a.gate + l.row * a.gate_n + (a.splat ? 0 : at);
        add = a.add ? a.add + l.row * a.add_n + at : nullptr;
        before = a.before ? a.before + l.row * a.before_n + at : nullptr;
        rest = a.rest ? a.rest + l.row * a.rest_n + l.col : nullptr;
        to = a.to ? a.to + l.row * a.to_n + at : nullptr;
        d_gate = a.d_gate ? a.d_gate + l.row * a.d_gate_n + at : nullptr;
    }
};

// the carried values of a lane's channels, [N, D] fp32
template <int V> __device__ __forceinline__ void load_start(const float *p, const Lane &l, float (&h)[V])
{
    if (p) {
        widen(load_raw<float, V>(p + l.channel), h);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) h[i] = 0.0f;
    }
}

template <int V> __device__ __forceinline__ void store_end(const RecArgs &a, const Lane &l, const float (&h)[V])
{
    if (a.end) store_from<float, V>(reinterpret_cast<char *>(a.end + l.channel), h, l.skip);
}

// enough channels: a lane walks all the steps.  REST is an argument of the template here, for a branch around its loads costs
// calls without it 2 % (32 x 65 536 x 64 bf16, a training pass: 398 us, 408 with the branch).
template <typename T, int V, int FL, bool BACKWARD, bool REST>
__global__ __launch_bounds__(kRecBlock) void recurrence_kernel(RecArgs a)
{
    const uint32_t v = blockIdx.x * kRecBlock + threadIdx.x;
    if (v >= a.vectors) return;
    const Lane l = lane_of<V>(a, v);
    const LaneFlags<V, FL> lf(a, l);
    const Places<T> p(a, l);
    float h[V];
    load_start<V>(a.start, l, h);
    for (int64_t t = 0; t < a.T; t++) {
        Steps<T, V, FL, steps_of(1), BACKWARD, false, true, REST> s;
        s.load(a, lf, p.gate, p.add, p.before, p.rest, t, t + 1);
        s.walk(a, l, true, p.to, p.d_gate, p.rest, t, h);
    }
    store_end<V>(a, l, h);
}

// V floats (4 or 1) of each of a workgroup's lanes
template <int V, int LANES> struct Exchange {
    typedef typename Pack<float, V>::type Word __attribute__((aligned(4 * V)));
    Word w[LANES];
    __device__ __forceinline__ void put(int lane, const float (&f)[V])
    {
        if constexpr (V == 1) w[lane] = f[0];
        else w[lane] = {f[0], f[1], f[2], f[3]};
    }
    __device__ __forceinline__ void get(int lane, float (&f)[V]) const
    {
        const Word x = w[lane];
        if constexpr (V == 1) {
            f[0] = x;
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) f[i] = x[i];
        }
    }
};

// the map (A, B) behind (A1, B1), into the latter
template <int V> __device__ __forceinline__ void compose(float (&A1)[V], float (&B1)[V], const float (&A)[V], const float (&B)[V])
{
#pragma unroll
    for (int i = 0; i < V; i++) {
        B1[i] = through(A[i], B[i], B1[i]);
        A1[i] = as_factor(A[i] * A1[i], dropped(A[i]) || dropped(A1[i]));
    }
}

template <int V> __device__ __forceinline__ void load_span(const RecArgs &a, int64_t row, uint32_t v, float (&f)[V])
{
    const float *p = a.spans + (row * a.vectors + v) * V;
    if constexpr (V == 1) f[0] = *p;
    else widen(load_raw<float, V>(p), f);
}

// SEG groups of LANES lanes with the maps of consecutive parts of the time: groups of one wave scan theirs by exchanging
// registers, the waves' totals go through LDS.
template <int V, int LANES, int SEG> struct Chain {
    static constexpr int kInWave = 64 / LANES, kWaves = LANES * SEG / 64;
    Exchange<V, LANES> (*maps)[kWaves][2];  // [2]: two halves used in turn, so that one barrier a call is enough
    int lane, in_wave, wave, turn;
    __device__ __forceinline__ Chain(Exchange<V, LANES> (*lds)[kWaves][2])
        : maps(lds), lane(threadIdx.x % LANES), in_wave(threadIdx.x % 64 / LANES), wave(threadIdx.x / 64), turn(0)
    {
    }
    // (A, B) becomes the map of this group's part behind those of the groups in front of it in the wave
    __device__ __forceinline__ void scan_wave(float (&A)[V], float (&B)[V]) const
    {
#pragma unroll
        for (int d = 1; d < kInWave; d *= 2) {
            float A1[V], B1[V];
#pragma unroll
            for (int i = 0; i < V; i++) {
                A1[i] = __shfl_up(A[i], d * LANES);
                B1[i] = __shfl_up(B[i], d * LANES);
            }
            if (in_wave >= d) {
                compose<V>(A1, B1, A, B);
#pragma unroll
                for (int i = 0; i < V; i++) A[i] = A1[i], B[i] = B1[i];
            }
        }
    }
    __device__ __forceinline__ void publish(const float (&A)[V], const float (&B)[V])
    {
        if (in_wave == kInWave - 1) {
            maps[turn][wave][0].put(lane, A);
            maps[turn][wave][1].put(lane, B);
        }
        __syncthreads();
    }
    __device__ __forceinline__ void total(int w, float (&A)[V], float (&B)[V]) const
    {
        maps[turn][w][0].get(lane, A);
        maps[turn][w][1].get(lane, B);
    }
    // h goes through all parts; `from` is what reaches this group's
    __device__ __forceinline__ void run(float (&A)[V], float (&B)[V], float (&h)[V], float (&from)[V])
    {
        scan_wave(A, B);
        publish(A, B);
#pragma unroll
        for (int i = 0; i < V; i++) from[i] = 0.0f;
#pragma unroll 2
        for (int w = 0; w < kWaves; w++) {
            float A2[V], B2[V];
            total(w, A2, B2);
#pragma unroll
            for (int i = 0; i < V; i++) {
                from[i] = w == wave ? h[i] : from[i];
                h[i] = through(A2[i], B2[i], h[i]);
            }
        }
        if constexpr (kInWave > 1) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float A1 = __shfl_up(A[i], LANES), B1 = __shfl_up(B[i], LANES);
                from[i] = in_wave ? through(A1, B1, from[i]) : from[i];
            }
        }
        turn ^= 1;
    }
};

// Time split: SEG groups of lanes take steps_of(SEG) steps each of the same channels; blockIdx.y is the span.
constexpr int lanes_of(int seg) { return seg == 4 ? 64 : 16; }

template <typename T, int V, int FL, bool BACKWARD, int SEG>
__global__ __launch_bounds__(lanes_of(SEG) * SEG) void recurrence_split_kernel(RecArgs a)
{
    constexpr int LANES = lanes_of(SEG), kSteps = steps_of(SEG);
    using Links = Chain<V, LANES, SEG>;
    __shared__ Exchange<V, LANES> maps[2][Links::kWaves][2];
    Links chain(maps);
    const int seg = threadIdx.x / LANES;
    const uint32_t mine = blockIdx.x * LANES + chain.lane, v = mine < a.vectors ? mine : a.vectors - 1;
    const bool store = mine < a.vectors;  // the other lanes of the last workgroup repeat its last vector
    const Lane l = lane_of<V>(a, v);
    const LaneFlags<V, FL> lf(a, l);
    const Places<T> p(a, l);
    const int64_t first = (int64_t)blockIdx.y * a.span, t1 = first + a.span < a.T ? first + a.span : a.T;
    Steps<T, V, FL, kSteps, BACKWARD, true, false, sizeof(T) == 2> s;
    s.load(a, lf, p.gate, p.add, p.before, p.rest, first + seg * kSteps, t1);  // on its way while the spans are composed
    float h[V], A[V], B[V], from[V];
    bool starts[V];
    if (gridDim.y == 1) {
        load_start<V>(a.start, l, h);
    } else {  // each group composes its part of the spans before this one, then all go through the parts
        const int64_t spans = blockIdx.y, part = ceil_div(spans, SEG);
        identity<V>(A, B, starts);
        const int64_t end = (seg + 1) * part < spans ? (seg + 1) * part : spans;
#pragma unroll 2
        for (int64_t q = seg * part; q < end; q++) {
            float A2[V], B2[V];
            load_span<V>(a, 1 + 2 * q, v, A2);
            load_span<V>(a, 2 + 2 * q, v, B2);
            compose<V>(A, B, A2, B2);
        }
        load_span<V>(a, 0, v, h);
        chain.run(A, B, h, from);
    }
    for (int64_t t0 = first; t0 < t1; t0 += SEG * kSteps) {
        const int64_t ts = t0 + seg * kSteps, next = t0 + SEG * kSteps;
        identity<V>(A, B, starts);
        s.reduce(A, B, starts);
        mark<V>(A, starts);
        chain.run(A, B, h, from);
        s.walk(a, l, store, p.to, p.d_gate, p.rest, ts, from);
        if (store && ts < a.T && ts + kSteps >= a.T) store_end<V>(a, l, from);  // what the last step left: `out` is its rounding
        if (next < t1) s.load(a, lf, p.gate, p.add, p.before, p.rest, next + seg * kSteps, t1);
    }
}

// The (A, B) of every span: SEG groups of lanes reduce consecutive parts of it.
template <typename T, int V, int FL, bool BACKWARD>
__global__ __launch_bounds__(kRecBlock) void recurrence_spans_kernel(RecArgs a)
{
    constexpr int SEG = 16, LANES = kRecBlock / SEG, kSteps = 8;
    using Links = Chain<V, LANES, SEG>;
    __shared__ Exchange<V, LANES> maps[2][Links::kWaves][2];
    Links chain(maps);
    const int seg = threadIdx.x / LANES;
    const uint32_t mine = blockIdx.x * LANES + chain.lane, v = mine < a.vectors ? mine : a.vectors - 1;
    const Lane l = lane_of<V>(a, v);
    const LaneFlags<V, FL> lf(a, l);
    const Places<T> p(a, l);
    const int64_t first = (int64_t)blockIdx.y * a.span, last = first + a.span < a.T ? first + a.span : a.T;
    const int64_t part = ceil_div(a.span, SEG);
    const int64_t from = first + seg * part, to = from + part < last ? from + part : last;
    float A[V], B[V];
    bool starts[V];
    identity<V>(A, B, starts);
    for (int64_t t = from; t < to; t += kSteps) {
        Steps<T, V, FL, kSteps, BACKWARD, true, false, false> s;
        s.load(a, lf, p.gate, p.add, nullptr, nullptr, t, to);
        s.reduce(A, B, starts);
    }
    mark<V>(A, starts);
    chain.scan_wave(A, B);
    chain.publish(A, B);
    if (seg != 0 || mine >= a.vectors) return;
    chain.total(0, A, B);
#pragma unroll
    for (int w = 1; w < Links::kWaves; w++) {
        float A2[V], B2[V];
        chain.total(w, A2, B2);
        compose<V>(A, B, A2, B2);
    }
    const int64_t at = (int64_t)a.vectors * V;
    float *to_span = a.spans + (int64_t)v * V;
    store_vec<float, V>(to_span + (1 + 2 * (int64_t)blockIdx.y) * at, A);
    store_vec<float, V>(to_span + (2 + 2 * (int64_t)blockIdx.y) * at, B);
    if (blockIdx.y == 0) {  // the second kernel takes the start from here: `end` may be the array it comes from
        load_start<V>(a.start, l, A);
        store_vec<float, V>(to_span, A);
    }
}

struct Plan {
    RecArgs a;
    int vec;    // channels per lane: the type's 16 bytes, or 4, or 1 where a run is shorter than that
    int flags;
    int seg;    // groups of lanes that share a workgroup's channels: 4, 16 or 64; 1: a lane walks all steps
    int64_t spans;
    bool apart;  // an environment's steps are adjacent in memory rather than a step's environments
    int64_t workspace() const { return spans > 1 ? (1 + 2 * spans) * a.vectors * vec * (int64_t)sizeof(float) : 0; }
};

// Lanes that share the time hold 4 channels or 1, a lane that walks alone holds 16 bytes or 1 channel: the other kernels are
// not there.
template <typename T, int V, int FL, bool BACKWARD> void launch_as(const Plan &p, hipStream_t s)
{
    constexpr bool kAlone = V == 1 || V * sizeof(T) == 16, kShared = V <= 4;
    const dim3 block(kRecBlock);
    const uint32_t v = p.a.vectors;
    if constexpr (kAlone) {
        if (p.seg == 1) {
            const dim3 grid((unsigned)ceil_div(v, kRecBlock));
            if constexpr (sizeof(T) == 2) {
                if (p.a.rest) return recurrence_kernel<T, V, FL, BACKWARD, true><<<grid, block, 0, s>>>(p.a);
            }
            return recurrence_kernel<T, V, FL, BACKWARD, false><<<grid, block, 0, s>>>(p.a);
        }
    }
    if constexpr (kShared) {
        if (p.spans > 1)
            recurrence_spans_kernel<T, V, FL, BACKWARD><<<dim3((unsigned)ceil_div(v, kRecBlock / 16), (unsigned)p.spans), block, 0, s>>>(p.a);
        if (p.seg == 4)
            return recurrence_split_kernel<T, V, FL, BACKWARD, 4><<<dim3((unsigned)ceil_div(v, lanes_of(4))), block, 0, s>>>(p.a);
        const dim3 grid((unsigned)ceil_div(v, lanes_of(16)), (unsigned)p.spans);
        if constexpr (FL <= kOneFlag) {
            if (p.seg == 64) return recurrence_split_kernel<T, V, FL, BACKWARD, 64><<<grid, dim3(lanes_of(64) * 64), 0, s>>>(p.a);
        }
        recurrence_split_kernel<T, V, FL, BACKWARD, 16><<<grid, block, 0, s>>>(p.a);
    }
}

template <int DT, bool BACKWARD> void launch_type(const Plan &p, hipStream_t s)
{
    using T = typename Elem<DT>::type;
    constexpr int V = Elem<DT>::vec;
    if (p.vec == 4 && V != 4) {
        if (p.flags == kNoFlags) launch_as<T, 4, kNoFlags, BACKWARD>(p, s);
        else if (p.flags == kOneFlag) launch_as<T, 4, kOneFlag, BACKWARD>(p, s);
        else if (p.flags == kTwoFlags) launch_as<T, 4, kTwoFlags, BACKWARD>(p, s);
        else launch_as<T, 4, kFlagEach, BACKWARD>(p, s);
    } else if (p.vec == 1) {
        if (p.flags == kNoFlags) launch_as<T, 1, kNoFlags, BACKWARD>(p, s);
        else launch_as<T, 1, kOneFlag, BACKWARD>(p, s);
    } else {
        if (p.flags == kNoFlags) launch_as<T, V, kNoFlags, BACKWARD>(p, s);
        else if (p.flags == kOneFlag) launch_as<T, V, kOneFlag, BACKWARD>(p, s);
        else if (p.flags == kTwoFlags) launch_as<T, V, kTwoFlags, BACKWARD>(p, s);
        else launch_as<T, V, kFlagEach, BACKWARD>(p, s);
    }
}

template <bool BACKWARD> void launch_recurrence(int dtype, const Plan &p, hipStream_t s)
{
    if (dtype == IGX_F32) launch_type<IGX_F32, BACKWARD>(p, s);
    else if (dtype == IGX_F16) launch_type<IGX_F16, BACKWARD>(p, s);
    else launch_type<IGX_BF16, BACKWARD>(p, s);
}

extern template void launch_recurrence<true>(int dtype, const Plan &p, hipStream_t s);

}  // namespace igx
