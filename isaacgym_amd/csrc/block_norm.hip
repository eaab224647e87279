// The norms before and after a residual block, fused with the branch's gate and residual scale, and their gradients:
//     out = x + scale * act(gate) * (rms(y) * weight),   next = rms(out) * next_weight
//
// Row-wise and bound by HBM: forward moves up to 5 elements per (row, column), backward up to 8, a few dozen operations
// each (2^20 x 256 bf16 with gate, scale and next: 522 us forward, 5.1 TB/s, 815 backward, 5.3 TB/s; the norm alone 170 us
// forward, 6.3 TB/s, and 273 backward, 5.9 TB/s, through 8-bit codes 226 and 253).  All times here are device times of graph
// replays on one set of buffers, backward with the column sums; where the buffers lie moves them by up to 15 %.
// A row stays in the registers of the lanes that loaded it - 16 bytes a lane, 8 to 64 lanes of one wave or the waves of a
// whole workgroup, whichever the width fills - so every array is read and written once and the statistics need no second
// pass.  Groups of lanes walk over the rows, which keeps the parameter vectors in registers and lets backward add up the
// column sums there: one partial row per workgroup, joined in a fixed order by a second kernel.  STREAM variants go past
// the caches' replacement, for calls that move more than the last-level cache holds.
#include "igx_block_norm.hpp"

namespace igx {
namespace {

// Gates as their codes hold them: no further out than +-16, so that one that is shut by a very low value does not take the
// other 63 of its group their scale.  Beyond it the activations are off by less than 16 exp(-16) < 2^-19, where a code of
// such a group has steps of 16 / 127.  NaN stays.  One instruction an element, with a branch for the sigmoid's upper end (the
// whole kernel on 131 072 x 512 bf16: 177 us, 172 without limits).
template <int V, int K> __device__ __forceinline__ void limit_gates(const float (&z)[K][V], int act, float (&g)[K][V])
{
    const float most = 16.0f, lowest = act == IGX_GATE_NONE ? -__builtin_inff() : -most;
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int i = 0; i < V; i++) g[k][i] = __builtin_elementwise_maximum(z[k][i], lowest);
    if (act != IGX_GATE_SIGMOID) return;
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int i = 0; i < V; i++) g[k][i] = __builtin_elementwise_minimum(g[k][i], most);
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
                if (i < left[k]) codes[col[k] + i] = code_of(f[k][i], s.inverse);
        }
        if (left[k] > 0 && col[k] % IGX_PACK8_GROUP == 0) scales[col[k] / IGX_PACK8_GROUP] = s.scale;
    }
}

// POST: there is a block output y; NEXT: there is a norm behind
template <typename T, int LANES, bool POST, bool NEXT, bool STREAM>
__global__ __launch_bounds__(block_of(LANES)) void block_norm_kernel(NormArgs a)
{
    using Row = RowLanes<T, LANES, !POST>;
    constexpr int V = Row::V, K = Row::K;
    __shared__ float slots[32];
    const Row rl;
    int turn = 0;
    int col[K], left[K];
    float factor[K][V], next_weight[K][V];  // scale * weight
#pragma unroll
    for (int k = 0; k < K; k++) {
        col[k] = rl.col(k);
        left[k] = a.width - col[k];
        if constexpr (POST) load_factor<V>(a, col[k], left[k], factor[k]);
        if constexpr (NEXT) load_param<V>(a.next_weight, col[k], left[k], next_weight[k]);
    }
    struct Arrays {
        Raw<T, V> x[K], y[K], gate[K];
    };
    auto fetch = [&](int64_t row, Arrays &r) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int have = row < a.rows ? left[k] : 0;
            const int64_t at = col[k] * (int64_t)sizeof(T);
            r.x[k] = load_row<T, V, STREAM>(a.x + row * a.x_row + at, a.x_end, have);
            if constexpr (POST) {
                r.y[k] = load_row<T, V, STREAM>(a.y + row * a.y_row + at, a.y_end, have);
                if (a.gate) r.gate[k] = load_row<T, V, STREAM>(a.gate + row * a.gate_row + at, a.gate_end, have);
            }
        }
    };
    const int64_t step = (int64_t)gridDim.x * rl.rows_per_block;
    int64_t base = (int64_t)blockIdx.x * rl.rows_per_block;
    Arrays in;
    fetch(base + rl.sub, in);
    for (; base < a.rows; base += step) {
        const int64_t row = base + rl.sub;
        const bool there = row < a.rows;
        int have[K];
#pragma unroll
        for (int k = 0; k < K; k++) have[k] = there ? left[k] : 0;
        const int64_t at_row = row * (int64_t)a.width;
        float o[K][V];
#pragma unroll
        for (int k = 0; k < K; k++) widen_row<T, V>(in.x[k], have[k], o[k]);
        if constexpr (POST) {
            float y[K][V], ss = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++) {
                widen_row<T, V>(in.y[k], have[k], y[k]);
#pragma unroll
                for (int i = 0; i < V; i++) ss = fmaf(y[k][i], y[k][i], ss);
            }
            const float inv = rsqrtf(rl.sum(ss, slots, turn) / (float)a.width + a.eps);
            if (a.y_inv && there && rl.lane == 0) a.y_inv[row] = inv;
            float z[K][V];
            if (a.gate) {
#pragma unroll
                for (int k = 0; k < K; k++) widen_row<T, V>(in.gate[k], have[k], z[k]);
            }
            if (a.y8) checkpoint_row<V, K, LANES>(y, have, col, a.y8 + at_row, a.y8_scale + row * a.groups);
            if (a.gate && a.gate8) {
                float g[K][V];
                limit_gates(z, a.act, g);
                checkpoint_row<V, K, LANES>(g, have, col, a.gate8 + at_row, a.gate8_scale + row * a.groups);
            }
#pragma unroll
            for (int k = 0; k < K; k++) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float f = a.gate ? activate(z[k][i], a.act) : 1.0f;
                    o[k][i] = fmaf(f * (y[k][i] * inv), factor[k][i], o[k][i]);
                }
                if (have[k] > 0) store_row<T, V, STREAM>(a.out + (at_row + col[k]) * sizeof(T), o[k], have[k]);
            }
        } else {
            if (a.y8) checkpoint_row<V, K, LANES>(o, have, col, a.y8 + at_row, a.y8_scale + row * a.groups);
        }
        if constexpr (NEXT) {
            float ss = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int i = 0; i < V; i++) ss = fmaf(o[k][i], o[k][i], ss);
            const float inv = rsqrtf(rl.sum(ss, slots, turn) / (float)a.width + a.eps);
            if (a.out_inv && there && rl.lane == 0) a.out_inv[row] = inv;
#pragma unroll
            for (int k = 0; k < K; k++) {
#pragma unroll
                for (int i = 0; i < V; i++) o[k][i] *= inv * next_weight[k][i];
                if (have[k] > 0) store_row<T, V, STREAM>(a.next + (at_row + col[k]) * sizeof(T), o[k], have[k]);
            }
        }
        fetch(row + step, in);
    }
}

template <typename T, int LANES, bool STREAM> void launch_as(const NormArgs &a, dim3 grid, dim3 block, hipStream_t s)
{
    if (a.y && a.next_weight) block_norm_kernel<T, LANES, true, true, STREAM><<<grid, block, 0, s>>>(a);
    else if (a.y) block_norm_kernel<T, LANES, true, false, STREAM><<<grid, block, 0, s>>>(a);
    else block_norm_kernel<T, LANES, false, true, STREAM><<<grid, block, 0, s>>>(a);
}

template <typename T, int LANES> void launch_lanes(const NormArgs &a, bool stream_past, dim3 grid, dim3 block, hipStream_t s)
{
    if (stream_past) launch_as<T, LANES, true>(a, grid, block, s);
    else launch_as<T, LANES, false>(a, grid, block, s);
}

template <typename T> void launch_type(const NormArgs &a, bool stream_past, int64_t blocks, hipStream_t s)
{
    const int lanes = lanes_for(a.width, sizeof(T) == 4 ? IGX_F32 : IGX_F16, !a.y);
    const dim3 grid((unsigned)blocks), block(lanes > 64 ? lanes : kNormBlock);
    if (lanes == 8) launch_lanes<T, 8>(a, stream_past, grid, block, s);
    else if (lanes == 16) launch_lanes<T, 16>(a, stream_past, grid, block, s);
    else if (lanes == 32) launch_lanes<T, 32>(a, stream_past, grid, block, s);
    else if (lanes == 64) launch_lanes<T, 64>(a, stream_past, grid, block, s);
    else if (lanes <= 512) launch_lanes<T, kWorkgroup>(a, stream_past, grid, block, s);
    else launch_lanes<T, kLargest>(a, stream_past, grid, block, s);
}

}  // namespace

void launch_block_norm(const NormArgs &a, int dtype, bool stream_past, int64_t blocks, hipStream_t s)
{
    if (dtype == IGX_F32) launch_type<float>(a, stream_past, blocks, s);
    else if (dtype == IGX_F16) launch_type<_Float16>(a, stream_past, blocks, s);
    else launch_type<__bf16>(a, stream_past, blocks, s);
}

namespace {

struct SumArgs {
    const float *block, *next;    // the partial rows of each sum
    bool sum_block;               // is the block's wanted (then its workgroups come first)
    const float *weight, *scale;  // d_weight = scale * the block's sum, d_scale = weight * it
    float *d_weight, *d_scale, *d_next_weight;
    int64_t blocks;
    int width;
};

// sum[c] = partial[0][c] + partial[1][c] + ...: 64 columns a workgroup, its 16 waves share the rows and are joined in order
__global__ __launch_bounds__(1024) void column_sum_kernel(SumArgs a)
{
    __shared__ float part[16][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int c = blockIdx.x * 64 + lane;
    const bool next = !a.sum_block || blockIdx.y == 1;
    const float *p = next ? a.next : a.block;
    float v = 0.0f;
    if (c < a.width) {
#pragma unroll 16
        for (int64_t b = wave; b < a.blocks; b += 16) v += p[b * a.width + c];
    }
    part[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && c < a.width) {
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < 16; w++) v += part[w][lane];
        if (next) {
            a.d_next_weight[c] = v;
        } else {
            if (a.d_weight) a.d_weight[c] = a.scale ? v * a.scale[c] : v;
            if (a.d_scale) a.d_scale[c] = v * a.weight[c];
        }
    }
}

// Workgroups: as many as run at a time, which walk over the rows - more would start when the first are done and leave most
// of the card idle at the end (backward of 2^20 x 256 bf16: 815 us with the 12 waves a CU holds, 943 with 16).  Without a
// block (waves 0) a lane keeps only the norm's weight, and a workgroup for every group of rows is faster: 2^20 x 256 fp32
// 341 us, 378 walking.
int64_t blocks_for(int64_t rows, int64_t width, int dtype, int64_t waves_per_cu)
{
    const int lanes = lanes_for(width, dtype, waves_per_cu == 0);
    const int64_t threads = lanes > 64 ? lanes : kNormBlock, rows_per_block = lanes > 64 ? 1 : kNormBlock / lanes;
    const int64_t need = ceil_div(rows, rows_per_block);
    const int64_t most = waves_per_cu ? 256 * waves_per_cu * 64 / threads : (int64_t)1 << 21;
    return need < most ? need : most;
}
constexpr int64_t kForwardWaves = 16, kBackwardWaves = 12;

// Does the call move more than the 256 MB that the last level of cache holds?  (2^20 x 256 bf16, forward and backward: 1 340 us
// past the caches, 1 425 through them; 16 411 x 211 fp32: 48 and 45.)
bool beyond_cache(const igx_block_norm *b, int64_t arrays)
{
    return arrays * b->rows * b->width * element_size(b->dtype) > (int64_t)256 << 20;
}

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
    if (!(b->eps >= 0.0f)) return fail(IGX_E_PARAM, "%s: eps %g is negative or NaN", who, (double)b->eps);
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
    const int64_t arrays = 1 + (b->y != nullptr) * 2 + (b->gate != nullptr) + (b->next_weight != nullptr);
    igx::launch_block_norm(a, b->dtype, igx::beyond_cache(b, arrays), igx::blocks_for(b->rows, b->width, b->dtype, b->y ? igx::kForwardWaves : 0),
                           static_cast<hipStream_t>(stream));
    return igx::launch_status(__func__);
}

extern "C" int64_t igx_block_norm_workspace(const igx_block_norm *b)
{
    const int rc = igx::check(b, __func__);
    if (rc) return rc;
    return 2 * igx::blocks_for(b->rows, b->width, b->dtype, igx::kBackwardWaves) * b->width * (int64_t)sizeof(float);
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
    const bool sum_block = g->d_weight || g->d_scale, sum_next = g->d_next_weight != nullptr;
    const int wanted = sum_block + sum_next;
    if (wanted == 0 && !g->d_x && !g->d_y && !g->d_gate) return IGX_OK;
    const int64_t blocks = igx::blocks_for(b->rows, b->width, b->dtype, igx::kBackwardWaves);
    if (b->rows > 0) {
        if (b->next_weight && (b->y || !b->y8)) IGX_REQUIRE_PTR(b->x, "x");
        if (b->y) IGX_REQUIRE_PTR(b->y_inv_rms, "y_inv_rms");
        if (b->next_weight) IGX_REQUIRE_PTR(b->out_inv_rms, "out_inv_rms");
        if (wanted) {
            IGX_REQUIRE_PTR(g->workspace, "workspace");
            IGX_REQUIRE_ALIGNED(g->workspace, "workspace");
            if (g->workspace_bytes < 2 * blocks * b->width * (int64_t)sizeof(float))
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
        a.sum_block = sum_block;
        a.sum_next = sum_next;
        const int64_t arrays = (a.d_out != nullptr) + (a.d_next != nullptr) + (a.d_x != nullptr) + (a.d_y != nullptr) +
                               (a.d_gate != nullptr) + (b->y != nullptr) + (b->gate != nullptr) + (b->next_weight != nullptr);
        igx::launch_block_norm_backward(a, b->dtype, igx::beyond_cache(b, arrays), blocks, s);
    }
    if (wanted) {  // without rows: zeros
        const float *partial = static_cast<const float *>(g->workspace);
        const float *second = partial + (sum_block ? blocks * b->width : 0);
        const igx::SumArgs sum = {partial, second, sum_block, b->weight, b->scale, g->d_weight, g->d_scale,
                                  g->d_next_weight, blocks, (int)b->width};
        igx::column_sum_kernel<<<dim3((unsigned)igx::ceil_div(b->width, 64), wanted), dim3(1024), 0, s>>>(sum);
    }
    return igx::launch_status(__func__);
}
