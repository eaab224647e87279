// Gradients of the block norms (block_norm.hip has the formulas): a second pass over a row's registers for each norm, and
// the column sums of the parameters in registers while the lanes walk over the rows.
#include "igx_block_norm.hpp"

namespace igx {
namespace {

// a vector of an array that may be kept as codes
template <typename T, int V, bool CODES, bool STREAM> struct Saved;
template <typename T, int V, bool STREAM> struct Saved<T, V, false, STREAM> {
    Raw<T, V> r;
    __device__ __forceinline__ void load(const char *p, const char *end, const int8_t *, const float *, int, int left)
    {
        r = load_row<T, V, STREAM>(p, end, left);
    }
    __device__ __forceinline__ void get(float (&f)[V], int left) const { widen_row<T, V>(r, left, f); }
};
template <typename T, int V, bool STREAM> struct Saved<T, V, true, STREAM> {
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

template <typename T, int LANES, bool POST, bool NEXT, bool CODES, bool STREAM>
__global__ __launch_bounds__(block_of(LANES)) void block_norm_backward_kernel(NormArgs a)
{
    using Row = RowLanes<T, LANES, false>;
    constexpr int V = Row::V, K = Row::K;
    __shared__ float slots[32];
    __shared__ float joined[LANES > 0 ? kNormBlock * Row::V : 1];
    const Row rl;
    int turn = 0;
    int col[K], left[K];
    float factor[K][V], next_weight[K][V];  // scale * weight
    float sb[K][V], sn[K][V];               // column sums of d act rms(y) and of d_next rms(out)
    const float per = 1.0f / (float)a.width;
#pragma unroll
    for (int k = 0; k < K; k++) {
        col[k] = rl.col(k);
        left[k] = a.width - col[k];
        if constexpr (POST) load_factor<V>(a, col[k], left[k], factor[k]);
        if constexpr (NEXT) load_param<V>(a.next_weight, col[k], left[k], next_weight[k]);
#pragma unroll
        for (int i = 0; i < V; i++) sb[k][i] = sn[k][i] = 0.0f;
    }
    struct Arrays {
        Raw<T, V> d_out[K], d_next[K];
        Saved<T, V, CODES && !POST, STREAM> x[K];
        Saved<T, V, CODES, STREAM> y[K], gate[K];
        float inv_y, inv_o;
    };
    auto fetch = [&](int64_t row, Arrays &r) {
        const int64_t at_row = row * (int64_t)a.width;
        r.inv_y = r.inv_o = 0.0f;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int have = row < a.rows ? left[k] : 0;
            const int64_t at = col[k] * (int64_t)sizeof(T);
            if (a.d_out) r.d_out[k] = load_row<T, V, STREAM>(a.d_out + row * a.d_out_row + at, a.d_out_end, have);
            if constexpr (NEXT) {
                if (a.d_next) r.d_next[k] = load_row<T, V, STREAM>(a.d_next + row * a.d_next_row + at, a.d_next_end, have);
                if constexpr (POST) r.x[k].load(a.x + row * a.x_row + at, a.x_end, nullptr, nullptr, 0, have);
                else r.x[k].load(a.x + row * a.x_row + at, a.x_end, a.y8 + at_row, a.y8_scale + row * a.groups, col[k], have);
            }
            if constexpr (POST) {
                r.y[k].load(a.y + row * a.y_row + at, a.y_end, a.y8 + at_row, a.y8_scale + row * a.groups, col[k], have);
                if (a.gate)
                    r.gate[k].load(a.gate + row * a.gate_row + at, a.gate_end, a.gate8 + at_row, a.gate8_scale + row * a.groups,
                                   col[k], have);
            }
        }
        if (row < a.rows) {
            if constexpr (POST) r.inv_y = a.y_inv[row];
            if constexpr (NEXT) r.inv_o = a.out_inv[row];
        }
    };
    const int64_t step = (int64_t)gridDim.x * rl.rows_per_block;
    int64_t base = (int64_t)blockIdx.x * rl.rows_per_block;
    Arrays in;
    fetch(base + rl.sub, in);
    for (; base < a.rows; base += step) {
        const int64_t row = base + rl.sub;
        const bool there = row < a.rows;
        const int64_t at_row = row * (int64_t)a.width;
        const float inv_y = in.inv_y, inv_o = in.inv_o;
        int have[K];
#pragma unroll
        for (int k = 0; k < K; k++) have[k] = there ? left[k] : 0;
        float d[K][V];
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (a.d_out) {
                widen_row<T, V>(in.d_out[k], have[k], d[k]);
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) d[k][i] = 0.0f;
            }
        }
        float unit[K][V], f[K][V], slope[K][V];  // rms(y), act(gate) and its derivative
        if constexpr (POST) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                in.y[k].get(unit[k], have[k]);
                float z[V];
                if (a.gate) in.gate[k].get(z, have[k]);
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
                in.x[k].get(u[k], have[k]);
                if (a.d_next) {
                    widen_row<T, V>(in.d_next[k], have[k], t[k]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; i++) t[k][i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < V; i++) {
                    if constexpr (POST) u[k][i] = fmaf(f[k][i] * unit[k][i], factor[k][i], u[k][i]);
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
                if (have[k] > 0) store_row<T, V, STREAM>(a.d_x + (at_row + col[k]) * sizeof(T), d[k], have[k]);
        }
        if constexpr (POST) {
            float t[K][V], dot = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++) {
                float dg[V];
#pragma unroll
                for (int i = 0; i < V; i++) {
                    sb[k][i] = fmaf(d[k][i] * f[k][i], unit[k][i], sb[k][i]);
                    const float df = d[k][i] * factor[k][i];
                    dg[i] = df * unit[k][i] * slope[k][i];
                    t[k][i] = df * f[k][i];
                    dot = fmaf(t[k][i], unit[k][i], dot);
                }
                if (a.d_gate && have[k] > 0) store_row<T, V, STREAM>(a.d_gate + (at_row + col[k]) * sizeof(T), dg, have[k]);
            }
            dot = rl.sum(dot, slots, turn) * per;
            if (a.d_y) {
#pragma unroll
                for (int k = 0; k < K; k++) {
#pragma unroll
                    for (int i = 0; i < V; i++) t[k][i] = inv_y * fmaf(-unit[k][i], dot, t[k][i]);
                    if (have[k] > 0) store_row<T, V, STREAM>(a.d_y + (at_row + col[k]) * sizeof(T), t[k], have[k]);
                }
            }
        }
        fetch(row + step, in);
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
            constexpr int kSpan = LANES * V;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int i = 0; i < V; i++) joined[rl.sub * kSpan + col[k] + i] = s[k][i];
            __syncthreads();
            for (int c = threadIdx.x; c < a.width; c += kNormBlock) {
                float v = 0.0f;
                for (int r = 0; r < kNormBlock / LANES; r++) v += joined[r * kSpan + c];
                to[c] = v;
            }
        }
    };
    if constexpr (POST) join(sb, a.sum_block);
    if constexpr (NEXT) join(sn, a.sum_next);
}

template <typename T, int LANES, bool CODES, bool STREAM> void launch_as(const NormArgs &a, dim3 grid, dim3 block, hipStream_t s)
{
    if (a.y && a.next_weight) block_norm_backward_kernel<T, LANES, true, true, CODES, STREAM><<<grid, block, 0, s>>>(a);
    else if (a.y) block_norm_backward_kernel<T, LANES, true, false, CODES, STREAM><<<grid, block, 0, s>>>(a);
    else block_norm_backward_kernel<T, LANES, false, true, CODES, STREAM><<<grid, block, 0, s>>>(a);
}

template <typename T, int LANES> void launch_lanes(const NormArgs &a, bool stream_past, dim3 grid, dim3 block, hipStream_t s)
{
    if (a.y8 && stream_past) launch_as<T, LANES, true, true>(a, grid, block, s);
    else if (a.y8) launch_as<T, LANES, true, false>(a, grid, block, s);
    else if (stream_past) launch_as<T, LANES, false, true>(a, grid, block, s);
    else launch_as<T, LANES, false, false>(a, grid, block, s);
}

template <typename T> void launch_type(const NormArgs &a, bool stream_past, int64_t blocks, hipStream_t s)
{
    const int lanes = lanes_for(a.width, sizeof(T) == 4 ? IGX_F32 : IGX_F16, false);
    const dim3 grid((unsigned)blocks), block(lanes > 64 ? lanes : kNormBlock);
    if (lanes == 8) launch_lanes<T, 8>(a, stream_past, grid, block, s);
    else if (lanes == 16) launch_lanes<T, 16>(a, stream_past, grid, block, s);
    else if (lanes == 32) launch_lanes<T, 32>(a, stream_past, grid, block, s);
    else if (lanes == 64) launch_lanes<T, 64>(a, stream_past, grid, block, s);
    else if (lanes <= 512) launch_lanes<T, kWorkgroup>(a, stream_past, grid, block, s);
    else launch_lanes<T, kLargest>(a, stream_past, grid, block, s);
}

}  // namespace

void launch_block_norm_backward(const NormArgs &a, int dtype, bool stream_past, int64_t blocks, hipStream_t s)
{
    if (dtype == IGX_F32) launch_type<float>(a, stream_past, blocks, s);
    else if (dtype == IGX_F16) launch_type<_Float16>(a, stream_past, blocks, s);
    else launch_type<__bf16>(a, stream_past, blocks, s);
}

}  // namespace igx
