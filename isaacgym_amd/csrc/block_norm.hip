// The norms before and after a residual block, fused with the branch's gate and residual scale, and their gradients:
//     out = x + scale * act(gate) * (rms(y) * weight),   next = rms(out) * next_weight
//
// Row-wise and bound by HBM: forward moves up to 5 elements per (row, column), backward up to 8, a few dozen operations
// each.  A row stays in the registers of the lanes that loaded it - 8 columns a lane, 8 to 64 lanes of one wave or the
// waves of a whole workgroup, whichever the width fills - so every array is read and written once and the statistics
// need no second pass.  Groups of lanes walk over the rows, which keeps the parameter vectors in registers and lets
// backward add up the column sums there: one partial row per workgroup, joined in a fixed order by a second kernel.
#include "igx_seq.hpp"

namespace igx {
namespace {

constexpr int kBlock = 256;   // of the kernels whose row fits one wave
constexpr int kColumns = 8;   // of a lane

struct NormArgs {
    const char *x, *y, *gate, *d_out, *d_next;
    const char *x_end, *y_end, *gate_end, *d_out_end, *d_next_end;  // behind each array's last element
    int64_t x_row, y_row, gate_row, d_out_row, d_next_row;          // bytes from row to row
    char *out, *next, *d_x, *d_y, *d_gate;
    const float *weight, *scale, *next_weight;
    float *y_inv, *out_inv;
    int8_t *y8, *gate8;
    float *y8_scale, *gate8_scale;
    float *partial;  // [sums][workgroups][width]
    int64_t rows;
    int width, groups, act;
    float eps;
    bool sum_weight, sum_scale, sum_next;
};

__device__ __forceinline__ float sigmoid(float z) { return 1.0f / (1.0f + expf(-z)); }

__device__ __forceinline__ float activate(float z, int act)
{
    if (act == IGX_GATE_NONE) return z;
    const float p = sigmoid(z);
    return act == IGX_GATE_SIGMOID ? p : z * p;
}

__device__ __forceinline__ void activate_slope(float z, int act, float &f, float &slope)
{
    if (act == IGX_GATE_NONE) {
        f = z;
        slope = 1.0f;
        return;
    }
    const float p = sigmoid(z), q = p * (1.0f - p);
    f = act == IGX_GATE_SIGMOID ? p : z * p;
    slope = act == IGX_GATE_SIGMOID ? q : fmaf(z, q, p);
}

// The lanes that share a row.  LANES 8 ... 64: that many lanes of a wave, kWorkgroup: the whole workgroup of up to 512,
// kLargest: one of 1024, which leaves a lane half as many registers.
constexpr int kWorkgroup = 0, kLargest = -1;
constexpr int block_of(int lanes) { return lanes > 0 ? kBlock : lanes == kWorkgroup ? 512 : 1024; }

template <typename T, int LANES> struct RowLanes {
    static constexpr int V = Elem<std::is_same<T, float>::value ? IGX_F32 : std::is_same<T, _Float16>::value ? IGX_F16 : IGX_BF16>::vec;
    static constexpr int K = kColumns / V;
    static constexpr bool kWide = LANES <= 0;
    int lane, lanes, rows_per_block, sub;
    __device__ __forceinline__ RowLanes()
    {
        lanes = kWide ? blockDim.x : LANES;
        lane = kWide ? threadIdx.x : threadIdx.x % (kWide ? 1 : LANES);
        sub = kWide ? 0 : threadIdx.x / (kWide ? 1 : LANES);
        rows_per_block = kWide ? 1 : kBlock / (kWide ? 1 : LANES);
    }
    __device__ __forceinline__ int col(int k) const { return (k * lanes + lane) * V; }

    // sum over the row's lanes, the same value in all of them; `slots`: LDS for the wide form, two halves used in turn so
    // that one barrier a sum is enough
    __device__ __forceinline__ float sum(float v, float *slots, int &turn) const
    {
#pragma unroll
        for (int m = 1; m < (kWide ? 64 : LANES); m *= 2) v += __shfl_xor(v, m);
        if constexpr (kWide) {
            float *s = slots + 16 * turn;
            turn ^= 1;
            if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = v;
            __syncthreads();
            v = 0.0f;
            for (int w = 0; w < (int)(blockDim.x / 64); w++) v += s[w];
        }
        return v;
    }
};

// A lane's vector of a row: `left` of its V columns exist.  Reading on into the next row is fine, past the array is not.
template <typename T, int V> __device__ __forceinline__ Raw<T, V> load_row(const char *p, const char *end, int left)
{
    Raw<T, V> r = {};
    if (left <= 0) return r;
    if (p + V * sizeof(T) <= end) {
        r = load_raw<T, V>(p);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < left) r.v[i] = reinterpret_cast<const T *>(p)[i];
    }
    return r;
}

template <typename T, int V> __device__ __forceinline__ void widen_row(const Raw<T, V> &r, int left, float (&f)[V])
{
    widen(r, f);
    if (left < V) {
#pragma unroll
        for (int i = 0; i < V; i++) f[i] = i < left ? f[i] : 0.0f;
    }
}

template <typename T, int V> __device__ __forceinline__ void store_row(char *p, const float (&f)[V], int left)
{
    if (left >= V) {
        store_vec<T, V>(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < left) reinterpret_cast<T *>(p)[i] = (T)f[i];
    }
}

template <int V> __device__ __forceinline__ void load_param(const float *p, int col, int left, float absent, float (&f)[V])
{
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = i < left ? (p ? p[col + i] : absent) : 0.0f;
}

// the row's 8-bit codes: a group's lanes sit next to each other (with 8 lanes of 4 columns, in both of their vectors)
template <int V, int K, int LANES>
__device__ __forceinline__ void checkpoint_row(const float (&f)[K][V], const int (&left)[K], const int (&col)[K], int8_t *codes,
                                               float *scales)
{
    constexpr int kSpan = (LANES <= 0 ? 64 : LANES) * V;  // columns of one vector of the wave's part
    constexpr bool kBoth = kSpan < IGX_PACK8_GROUP;
    constexpr int kLanes = kBoth ? LANES : IGX_PACK8_GROUP / V;
    uint32_t top[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        top[k] = 0;
#pragma unroll
        for (int i = 0; i < V; i++) top[k] = max(top[k], magnitude_bits(f[k][i]));
    }
    if constexpr (kBoth) {
#pragma unroll
        for (int k = 1; k < K; k++) top[0] = max(top[0], top[k]);
#pragma unroll
        for (int k = 1; k < K; k++) top[k] = top[0];
    }
#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
        for (int m = 1; m < kLanes; m *= 2) top[k] = max(top[k], (uint32_t)__shfl_xor((int)top[k], m));
        const GroupScale s = group_scale(top[k]);
        if (left[k] >= V) {
            store_codes<V>(codes + col[k], f[k], s.inverse);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (i < left[k]) codes[col[k] + i] = (int8_t)code_of(f[k][i], s.inverse);
        }
        if (left[k] > 0 && col[k] % IGX_PACK8_GROUP == 0) scales[col[k] / IGX_PACK8_GROUP] = s.scale;
    }
}

// POST: there is a block output y; NEXT: there is a norm behind
template <typename T, int LANES, bool POST, bool NEXT>
__global__ __launch_bounds__(block_of(LANES)) void block_norm_kernel(NormArgs a)
{
    using Row = RowLanes<T, LANES>;
    constexpr int V = Row::V, K = Row::K;
    __shared__ float slots[32];
    const Row rl;
    int turn = 0;
    int col[K], left[K];
    float weight[K][V], scale[K][V], next_weight[K][V];
#pragma unroll
    for (int k = 0; k < K; k++) {
        col[k] = rl.col(k);
        left[k] = a.width - col[k];
        if constexpr (POST) {
            load_param<V>(a.weight, col[k], left[k], 1.0f, weight[k]);
            load_param<V>(a.scale, col[k], left[k], 1.0f, scale[k]);
        }
        if constexpr (NEXT) load_param<V>(a.next_weight, col[k], left[k], 1.0f, next_weight[k]);
    }
    for (int64_t base = (int64_t)blockIdx.x * rl.rows_per_block; base < a.rows; base += (int64_t)gridDim.x * rl.rows_per_block) {
        const int64_t row = base + rl.sub;
        const bool there = row < a.rows;
        Raw<T, V> xr[K], yr[K], gr[K];
        int have[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            have[k] = there ? left[k] : 0;
            const int64_t at = col[k] * (int64_t)sizeof(T);
            xr[k] = load_row<T, V>(a.x + row * a.x_row + at, a.x_end, have[k]);
            if constexpr (POST) {
                yr[k] = load_row<T, V>(a.y + row * a.y_row + at, a.y_end, have[k]);
                if (a.gate) gr[k] = load_row<T, V>(a.gate + row * a.gate_row + at, a.gate_end, have[k]);
            }
        }
        const int64_t at_row = row * (int64_t)a.width;
        float o[K][V];
#pragma unroll
        for (int k = 0; k < K; k++) widen_row<T, V>(xr[k], have[k], o[k]);
        if constexpr (POST) {
            float y[K][V], ss = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++) {
                widen_row<T, V>(yr[k], have[k], y[k]);
#pragma unroll
                for (int i = 0; i < V; i++) ss = fmaf(y[k][i], y[k][i], ss);
            }
            const float inv = rsqrtf(rl.sum(ss, slots, turn) / (float)a.width + a.eps);
            if (a.y_inv && there && rl.lane == 0) a.y_inv[row] = inv;
            float z[K][V];
            if (a.gate) {
#pragma unroll
                for (int k = 0; k < K; k++) widen_row<T, V>(gr[k], have[k], z[k]);
            }
            if (a.y8) checkpoint_row<V, K, LANES>(y, have, col, a.y8 + at_row, a.y8_scale + row * a.groups);
            if (a.gate && a.gate8) checkpoint_row<V, K, LANES>(z, have, col, a.gate8 + at_row, a.gate8_scale + row * a.groups);
#pragma unroll
            for (int k = 0; k < K; k++) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float f = a.gate ? activate(z[k][i], a.act) : 1.0f;
                    o[k][i] = fmaf(scale[k][i] * f, y[k][i] * inv * weight[k][i], o[k][i]);
                }
                if (have[k] > 0) store_row<T, V>(a.out + (at_row + col[k]) * sizeof(T), o[k], have[k]);
            }
        } else {
            if (a.y8) checkpoint_row<V, K, LANES>(o, have, col, a.y8 + at_row, a.y8_scale + row * a.groups);
        }
        if constexpr (NEXT) {
            float ss = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int i = 0; i < V; i++) ss = i < have[k] ? fmaf(o[k][i], o[k][i], ss) : ss;
            const float inv = rsqrtf(rl.sum(ss, slots, turn) / (float)a.width + a.eps);
            if (a.out_inv && there && rl.lane == 0) a.out_inv[row] = inv;
#pragma unroll
            for (int k = 0; k < K; k++) {
#pragma unroll
                for (int i = 0; i < V; i++) o[k][i] *= inv * next_weight[k][i];
                if (have[k] > 0) store_row<T, V>(a.next + (at_row + col[k]) * sizeof(T), o[k], have[k]);
            }
        }
    }
}

// a vector of an array that may be kept as codes
template <typename T, int V, bool CODES> struct Saved;
template <typename T, int V> struct Saved<T, V, false> {
    Raw<T, V> r;
    __device__ __forceinline__ void load(const char *p, const char *end, const int8_t *, const float *, int, int left)
    {
        r = load_row<T, V>(p, end, left);
    }
    __device__ __forceinline__ void get(float (&f)[V], int left) const { widen_row<T, V>(r, left, f); }
};
template <typename T, int V> struct Saved<T, V, true> {
    uint32_t w[V / 4];
    float scale;
    __device__ __forceinline__ void load(const char *, const char *, const int8_t *codes, const float *scales, int col, int left)
    {
        scale = 0.0f;
#pragma unroll
        for (int j = 0; j < V / 4; j++) w[j] = 0;
        if (left <= 0) return;
        scale = scales[col / IGX_PACK8_GROUP];
        if (left >= V) {
            __builtin_memcpy(w, codes + col, V);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (i < left) w[i / 4] |= (uint32_t)(uint8_t)codes[col + i] << (8 * (i % 4));
        }
    }
    __device__ __forceinline__ void get(float (&f)[V], int left) const
    {
#pragma unroll
        for (int i = 0; i < V; i++) f[i] = i < left ? (float)(int8_t)(w[i / 4] >> (8 * (i % 4))) * scale : 0.0f;
    }
};

template <typename T, int LANES, bool POST, bool NEXT, bool CODES>
__global__ __launch_bounds__(block_of(LANES)) void block_norm_backward_kernel(NormArgs a)
{
    using Row = RowLanes<T, LANES>;
    constexpr int V = Row::V, K = Row::K;
    __shared__ float slots[32];
    __shared__ float joined[LANES > 0 ? kBlock * kColumns : 1];
    const Row rl;
    int turn = 0;
    int col[K], left[K];
    float weight[K][V], scale[K][V], next_weight[K][V];
    float sw[K][V], ss[K][V], sn[K][V];
    const float per = 1.0f / (float)a.width;
#pragma unroll
    for (int k = 0; k < K; k++) {
        col[k] = rl.col(k);
        left[k] = a.width - col[k];
        if constexpr (POST) {
            load_param<V>(a.weight, col[k], left[k], 1.0f, weight[k]);
            load_param<V>(a.scale, col[k], left[k], 1.0f, scale[k]);
        }
        if constexpr (NEXT) load_param<V>(a.next_weight, col[k], left[k], 1.0f, next_weight[k]);
#pragma unroll
        for (int i = 0; i < V; i++) sw[k][i] = ss[k][i] = sn[k][i] = 0.0f;
    }
    for (int64_t base = (int64_t)blockIdx.x * rl.rows_per_block; base < a.rows; base += (int64_t)gridDim.x * rl.rows_per_block) {
        const int64_t row = base + rl.sub;
        const bool there = row < a.rows;
        const int64_t at_row = row * (int64_t)a.width;
        Raw<T, V> dor[K], dnr[K];
        Saved<T, V, CODES && !POST> xs[K];
        Saved<T, V, CODES> ys[K], gs[K];
        int have[K];
        float inv_y = 0.0f, inv_o = 0.0f;
#pragma unroll
        for (int k = 0; k < K; k++) {
            have[k] = there ? left[k] : 0;
            const int64_t at = col[k] * (int64_t)sizeof(T);
            if (a.d_out) dor[k] = load_row<T, V>(a.d_out + row * a.d_out_row + at, a.d_out_end, have[k]);
            if constexpr (NEXT) {
                if (a.d_next) dnr[k] = load_row<T, V>(a.d_next + row * a.d_next_row + at, a.d_next_end, have[k]);
                if constexpr (POST) xs[k].load(a.x + row * a.x_row + at, a.x_end, nullptr, nullptr, 0, have[k]);
                else xs[k].load(a.x + row * a.x_row + at, a.x_end, a.y8 + at_row, a.y8_scale + row * a.groups, col[k], have[k]);
            }
            if constexpr (POST) {
                ys[k].load(a.y + row * a.y_row + at, a.y_end, a.y8 + at_row, a.y8_scale + row * a.groups, col[k], have[k]);
                if (a.gate)
                    gs[k].load(a.gate + row * a.gate_row + at, a.gate_end, a.gate8 + at_row, a.gate8_scale + row * a.groups,
                               col[k], have[k]);
            }
        }
        if (there) {
            if constexpr (POST) inv_y = a.y_inv[row];
            if constexpr (NEXT) inv_o = a.out_inv[row];
        }
        float d[K][V];
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (a.d_out) {
                widen_row<T, V>(dor[k], have[k], d[k]);
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) d[k][i] = 0.0f;
            }
        }
        float unit[K][V], f[K][V], slope[K][V];  // rms(y), act(gate) and its derivative
        if constexpr (POST) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                ys[k].get(unit[k], have[k]);
                float z[V];
                if (a.gate) gs[k].get(z, have[k]);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    unit[k][i] *= inv_y;
                    f[k][i] = 1.0f;
                    slope[k][i] = 0.0f;
                    if (a.gate) activate_slope(z[i], a.act, f[k][i], slope[k][i]);
                }
            }
        }
        if constexpr (NEXT) {
            float u[K][V], t[K][V], dot = 0.0f;  // rms(out), what reaches it
#pragma unroll
            for (int k = 0; k < K; k++) {
                xs[k].get(u[k], have[k]);
                if (a.d_next) {
                    widen_row<T, V>(dnr[k], have[k], t[k]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; i++) t[k][i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < V; i++) {
                    if constexpr (POST) u[k][i] = fmaf(scale[k][i] * f[k][i], unit[k][i] * weight[k][i], u[k][i]);
                    u[k][i] *= inv_o;
                    sn[k][i] = fmaf(t[k][i], u[k][i], sn[k][i]);
                    t[k][i] *= next_weight[k][i];
                    dot = fmaf(t[k][i], u[k][i], dot);
                }
            }
            dot = rl.sum(dot, slots, turn) * per;
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int i = 0; i < V; i++) d[k][i] = fmaf(inv_o, fmaf(-u[k][i], dot, t[k][i]), d[k][i]);
        }
        if (a.d_x) {
#pragma unroll
            for (int k = 0; k < K; k++)
                if (have[k] > 0) store_row<T, V>(a.d_x + (at_row + col[k]) * sizeof(T), d[k], have[k]);
        }
        if constexpr (POST) {
            float t[K][V], dot = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++) {
                float dg[V];
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float normed = unit[k][i] * weight[k][i];
                    dg[i] = d[k][i] * scale[k][i] * normed * slope[k][i];
                    ss[k][i] = fmaf(d[k][i] * f[k][i], normed, ss[k][i]);
                    t[k][i] = d[k][i] * scale[k][i] * f[k][i];
                    sw[k][i] = fmaf(t[k][i], unit[k][i], sw[k][i]);
                    t[k][i] *= weight[k][i];
                    dot = fmaf(t[k][i], unit[k][i], dot);
                }
                if (a.d_gate && have[k] > 0) store_row<T, V>(a.d_gate + (at_row + col[k]) * sizeof(T), dg, have[k]);
            }
            dot = rl.sum(dot, slots, turn) * per;
            if (a.d_y) {
#pragma unroll
                for (int k = 0; k < K; k++) {
#pragma unroll
                    for (int i = 0; i < V; i++) t[k][i] = inv_y * fmaf(-unit[k][i], dot, t[k][i]);
                    if (have[k] > 0) store_row<T, V>(a.d_y + (at_row + col[k]) * sizeof(T), t[k], have[k]);
                }
            }
        }
    }
    // the workgroup's column sums
    int64_t at = 0;
    auto join = [&](const float (&s)[K][V], bool wanted) {
        if (!wanted) return;
        float *to = a.partial + at + (int64_t)blockIdx.x * a.width;
        at += (int64_t)gridDim.x * a.width;
        if constexpr (LANES <= 0) {
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (i < left[k]) to[col[k] + i] = s[k][i];
        } else {
            constexpr int kSpan = LANES * kColumns;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int i = 0; i < V; i++) joined[rl.sub * kSpan + col[k] + i] = s[k][i];
            __syncthreads();
            for (int c = threadIdx.x; c < a.width; c += kBlock) {
                float v = 0.0f;
                for (int r = 0; r < kBlock / LANES; r++) v += joined[r * kSpan + c];
                to[c] = v;
            }
        }
    };
    if constexpr (POST) {
        join(sw, a.sum_weight);
        join(ss, a.sum_scale);
    }
    if constexpr (NEXT) join(sn, a.sum_next);
}

struct SumArgs {
    const float *partial;
    float *to[3];
    int64_t blocks;
    int width;
};

// sums[c] = partial[0][c] + partial[1][c] + ...: 64 columns a workgroup, its 16 waves share the rows and are joined in order
__global__ __launch_bounds__(1024) void column_sum_kernel(SumArgs a)
{
    __shared__ float part[16][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int c = blockIdx.x * 64 + lane;
    const float *p = a.partial + (int64_t)blockIdx.y * a.blocks * a.width;
    float v = 0.0f;
    if (c < a.width) {
#pragma unroll 4
        for (int64_t b = wave; b < a.blocks; b += 16) v += p[b * a.width + c];
    }
    part[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && c < a.width) {
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < 16; w++) v += part[w][lane];
        a.to[blockIdx.y][c] = v;
    }
}

// lanes of a row: the fewest that hold its columns; above 64 a workgroup of that many
int lanes_for(int64_t width)
{
    int lanes = 8;
    while (lanes * kColumns < width) lanes *= 2;
    return lanes;
}

// workgroups: enough to fill every CU (16 waves each), each with at least one group of rows
int64_t blocks_for(int64_t rows, int64_t width, int64_t waves_per_cu)
{
    const int lanes = lanes_for(width);
    const int64_t threads = lanes > 64 ? lanes : kBlock, rows_per_block = lanes > 64 ? 1 : kBlock / lanes;
    const int64_t most = 256 * waves_per_cu * 64 / threads, need = ceil_div(rows, rows_per_block);
    return need < most ? need : most;
}
constexpr int64_t kForwardWaves = 32, kBackwardWaves = 16;

int check(const igx_block_norm *b, const char *who)
{
    if (!b) return fail(IGX_E_NULL, "%s: b is NULL", who);
    if (!known_dtype(b->dtype)) return fail(IGX_E_PARAM, "%s: dtype %d is not IGX_F32, IGX_F16 or IGX_BF16", who, b->dtype);
    if (b->rows < 0 || b->rows > (int64_t)1 << 40) return fail(IGX_E_SIZE, "%s: rows %lld", who, (long long)b->rows);
    if (b->width < 1 || b->width > IGX_BLOCK_NORM_MAX_WIDTH)
        return fail(IGX_E_SIZE, "%s: width %lld is outside 1 ... %d", who, (long long)b->width, IGX_BLOCK_NORM_MAX_WIDTH);
    return IGX_OK;
}

int check_parts(const igx_block_norm *b, const char *who)
{
    if (b->activation != IGX_GATE_NONE && b->activation != IGX_GATE_SIGMOID && b->activation != IGX_GATE_SILU)
        return fail(IGX_E_PARAM, "%s: activation %d is not one of IGX_GATE_*", who, b->activation);
    if (!b->y && !b->next_weight) return fail(IGX_E_NULL, "%s: neither y nor next_weight is given", who);
    if (!b->y && (b->gate || b->scale || b->gate8)) return fail(IGX_E_PARAM, "%s: gate and scale belong to y, which is NULL", who);
    if (b->y && !b->weight) return fail(IGX_E_NULL, "%s: weight is NULL", who);
    if (b->x_stride < 0 || b->y_stride < 0 || b->gate_stride < 0) return fail(IGX_E_PARAM, "%s: a row stride is negative", who);
    if ((b->y8 != nullptr) != (b->y8_scale != nullptr) || (b->gate8 != nullptr) != (b->gate8_scale != nullptr))
        return fail(IGX_E_NULL, "%s: codes without their scales, or scales without their codes", who);
    if (b->gate && (b->y8 != nullptr) != (b->gate8 != nullptr))
        return fail(IGX_E_PARAM, "%s: y and gate are checkpointed together or not at all", who);
    return IGX_OK;
}

void base_args(const igx_block_norm *b, NormArgs &a)
{
    a = NormArgs();
    const int64_t e = element_size(b->dtype);
    auto array = [&](const void *p, int64_t stride, const char *&at, const char *&end, int64_t &row) {
        at = static_cast<const char *>(p);
        row = stride * e;
        end = at ? at + ((b->rows - 1) * stride + b->width) * e : nullptr;
    };
    array(b->x, b->x_stride, a.x, a.x_end, a.x_row);
    array(b->y, b->y_stride, a.y, a.y_end, a.y_row);
    array(b->gate, b->gate_stride, a.gate, a.gate_end, a.gate_row);
    a.weight = b->weight;
    a.scale = b->scale;
    a.next_weight = b->next_weight;
    a.out = static_cast<char *>(b->out);
    a.next = static_cast<char *>(b->next);
    a.y_inv = b->y_inv_rms;
    a.out_inv = b->out_inv_rms;
    a.y8 = b->y8;
    a.gate8 = b->gate8;
    a.y8_scale = b->y8_scale;
    a.gate8_scale = b->gate8_scale;
    a.rows = b->rows;
    a.width = (int)b->width;
    a.groups = (int)ceil_div(b->width, IGX_PACK8_GROUP);
    a.act = b->activation;
    a.eps = b->eps;
}

template <typename T, int LANES> void launch_forward(const NormArgs &a, dim3 grid, dim3 block, hipStream_t s)
{
    if (a.y && a.next_weight) block_norm_kernel<T, LANES, true, true><<<grid, block, 0, s>>>(a);
    else if (a.y) block_norm_kernel<T, LANES, true, false><<<grid, block, 0, s>>>(a);
    else block_norm_kernel<T, LANES, false, true><<<grid, block, 0, s>>>(a);
}

template <typename T, int LANES, bool CODES> void launch_backward_as(const NormArgs &a, dim3 grid, dim3 block, hipStream_t s)
{
    if (a.y && a.next_weight) block_norm_backward_kernel<T, LANES, true, true, CODES><<<grid, block, 0, s>>>(a);
    else if (a.y) block_norm_backward_kernel<T, LANES, true, false, CODES><<<grid, block, 0, s>>>(a);
    else block_norm_backward_kernel<T, LANES, false, true, CODES><<<grid, block, 0, s>>>(a);
}

template <typename T, int LANES> void launch_backward(const NormArgs &a, dim3 grid, dim3 block, hipStream_t s)
{
    if (a.y8) launch_backward_as<T, LANES, true>(a, grid, block, s);
    else launch_backward_as<T, LANES, false>(a, grid, block, s);
}

template <typename T> void launch_type(const NormArgs &a, bool backward, int64_t blocks, hipStream_t s)
{
    const int lanes = lanes_for(a.width);
    const dim3 grid((unsigned)blocks), block(lanes > 64 ? lanes : kBlock);
#define IGX_NORM_GO(L)                                        \
    do {                                                      \
        if (backward) launch_backward<T, L>(a, grid, block, s); \
        else launch_forward<T, L>(a, grid, block, s);         \
    } while (0)
    if (lanes == 8) IGX_NORM_GO(8);
    else if (lanes == 16) IGX_NORM_GO(16);
    else if (lanes == 32) IGX_NORM_GO(32);
    else if (lanes == 64) IGX_NORM_GO(64);
    else if (lanes <= 512) IGX_NORM_GO(kWorkgroup);
    else IGX_NORM_GO(kLargest);
#undef IGX_NORM_GO
}

void launch(const NormArgs &a, int dtype, bool backward, int64_t blocks, hipStream_t s)
{
    if (dtype == IGX_F32) launch_type<float>(a, backward, blocks, s);
    else if (dtype == IGX_F16) launch_type<_Float16>(a, backward, blocks, s);
    else launch_type<__bf16>(a, backward, blocks, s);
}

}  // namespace
}  // namespace igx

extern "C" int igx_block_norm_forward(const igx_block_norm *b, igx_stream_t stream)
{
    int rc = igx::check(b, __func__);
    if (!rc && b->rows) rc = igx::check_parts(b, __func__);
    if (rc) return rc;
    if (b->rows == 0) return IGX_OK;
    IGX_REQUIRE_PTR(b->x, "x");
    if (b->y) IGX_REQUIRE_PTR(b->out, "out");
    if (b->next_weight) IGX_REQUIRE_PTR(b->next, "next");
    igx::NormArgs a;
    igx::base_args(b, a);
    igx::launch(a, b->dtype, false, igx::blocks_for(b->rows, b->width, igx::kForwardWaves), static_cast<hipStream_t>(stream));
    return igx::launch_status(__func__);
}

extern "C" int64_t igx_block_norm_workspace(const igx_block_norm *b)
{
    const int rc = igx::check(b, __func__);
    if (rc) return rc;
    return 3 * igx::blocks_for(b->rows, b->width, igx::kBackwardWaves) * b->width * (int64_t)sizeof(float);
}

extern "C" int igx_block_norm_backward(const igx_block_norm *b, const igx_block_norm_grad *g, igx_stream_t stream)
{
    int rc = igx::check(b, __func__);
    if (!rc && b->rows) rc = igx::check_parts(b, __func__);  // arrays without rows need not have addresses
    if (rc) return rc;
    IGX_REQUIRE_PTR(g, "g");
    if (g->d_out_stride < 0 || g->d_next_stride < 0) return igx::fail(IGX_E_PARAM, "%s: a row stride is negative", __func__);
    if (b->rows && !b->y && (g->d_y || g->d_gate || g->d_weight || g->d_scale))
        return igx::fail(IGX_E_PARAM, "%s: gradients of y's norm are wanted, but y is NULL", __func__);
    if (!b->next_weight && g->d_next_weight)
        return igx::fail(IGX_E_PARAM, "%s: d_next_weight is wanted, but next_weight is NULL", __func__);
    if (b->rows && !b->gate && g->d_gate) return igx::fail(IGX_E_PARAM, "%s: d_gate is wanted, but gate is NULL", __func__);
    float *sums[3] = {g->d_weight, g->d_scale, g->d_next_weight};
    int wanted = 0;
    for (float *p : sums) wanted += p != nullptr;
    if (wanted == 0 && !g->d_x && !g->d_y && !g->d_gate) return IGX_OK;
    const int64_t blocks = igx::blocks_for(b->rows, b->width, igx::kBackwardWaves);
    if (b->rows > 0) {
        if (b->next_weight && (b->y || !b->y8)) IGX_REQUIRE_PTR(b->x, "x");
        if (b->y) IGX_REQUIRE_PTR(b->y_inv_rms, "y_inv_rms");
        if (b->next_weight) IGX_REQUIRE_PTR(b->out_inv_rms, "out_inv_rms");
        if (wanted) {
            IGX_REQUIRE_PTR(g->workspace, "workspace");
            IGX_REQUIRE_ALIGNED(g->workspace, "workspace");
            if (g->workspace_bytes < 3 * blocks * b->width * (int64_t)sizeof(float))
                return igx::fail(IGX_E_SIZE, "%s: workspace of %lld bytes is smaller than igx_block_norm_workspace()", __func__,
                                 (long long)g->workspace_bytes);
        }
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    igx::NormArgs a;
    igx::base_args(b, a);
    const int64_t e = igx::element_size(b->dtype);
    if (b->rows > 0) {
        a.d_out = static_cast<const char *>(g->d_out);
        a.d_out_row = g->d_out_stride * e;
        if (a.d_out) a.d_out_end = a.d_out + ((b->rows - 1) * g->d_out_stride + b->width) * e;
        a.d_next = static_cast<const char *>(g->d_next);
        a.d_next_row = g->d_next_stride * e;
        if (a.d_next) a.d_next_end = a.d_next + ((b->rows - 1) * g->d_next_stride + b->width) * e;
        a.d_x = static_cast<char *>(g->d_x);
        a.d_y = static_cast<char *>(g->d_y);
        a.d_gate = static_cast<char *>(g->d_gate);
        a.partial = static_cast<float *>(g->workspace);
        a.sum_weight = g->d_weight != nullptr;
        a.sum_scale = g->d_scale != nullptr;
        a.sum_next = g->d_next_weight != nullptr;
        igx::launch(a, b->dtype, true, blocks, s);
    }
    if (wanted) {  // without rows: zeros
        igx::SumArgs sum = {static_cast<const float *>(g->workspace), {}, blocks, (int)b->width};
        int n = 0;
        for (float *p : sums)
            if (p) sum.to[n++] = p;
        igx::column_sum_kernel<<<dim3((unsigned)igx::ceil_div(b->width, 64), n), dim3(1024), 0, s>>>(sum);
    }
    return igx::launch_status(__func__);
}
