// 8-bit checkpoints of activations: codes and one fp32 scale for every 64 elements of a row, and back.
//
// The lanes of one group take its elements 16 bytes each and agree on the largest magnitude by exchanging it within the
// wave, so the elements are read once and stay in registers: e + 1 + 4/64 bytes an element each way, bound by HBM.
#include "igx_seq.hpp"

namespace igx {
namespace {

constexpr int kBlock = 256;

template <typename T, int V>
__global__ __launch_bounds__(kBlock) void pack8_kernel(const char *x, int64_t stride, int64_t rows, int64_t width,
                                                       int64_t groups, int8_t *codes, float *scales)
{
    constexpr int LPG = IGX_PACK8_GROUP / V;  // lanes of a group
    const int64_t id = ((int64_t)blockIdx.x * kBlock + threadIdx.x) / LPG;
    const int lane = threadIdx.x % LPG;
    const int64_t row = id / groups, group = id - row * groups;
    const int64_t col = group * IGX_PACK8_GROUP + lane * V;
    const int64_t left = row < rows ? width - col : 0;
    float f[V];
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = 0.0f;
    const char *p = x + row * stride + col * (int64_t)sizeof(T);
    if (left >= V) {
        widen(load_raw<T, V>(p), f);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < left) f[i] = (float)reinterpret_cast<const T *>(p)[i];
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < V; i++) top = max(top, magnitude_bits(f[i]));
#pragma unroll
    for (int m = 1; m < LPG; m *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, m));
    const GroupScale s = group_scale(top);
    if (left <= 0) return;
    int8_t *q = codes + row * width + col;
    if (left >= V) {
        store_codes<V>(q, f, s.inverse);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < left) q[i] = (int8_t)code_of(f[i], s.inverse);
    }
    if (lane == 0) scales[row * groups + group] = s.scale;
}

template <typename T, int V>
__global__ __launch_bounds__(kBlock) void unpack8_kernel(const int8_t *codes, const float *scales, int64_t rows,
                                                         int64_t width, int64_t groups, char *x)
{
    constexpr int LPG = IGX_PACK8_GROUP / V;
    const int64_t id = ((int64_t)blockIdx.x * kBlock + threadIdx.x) / LPG;
    const int64_t row = id / groups, group = id - row * groups;
    const int64_t col = group * IGX_PACK8_GROUP + (threadIdx.x % LPG) * V;
    if (row >= rows || col >= width) return;
    const int64_t at = row * width + col;
    const float s = scales[row * groups + group];
    const int64_t left = width - col;
    float f[V];
    if (left >= V) {
        load_codes<V>(codes + at, f);
#pragma unroll
        for (int i = 0; i < V; i++) f[i] *= s;
        store_vec<T, V>(x + at * sizeof(T), f);
    } else {
        for (int i = 0; i < left; i++) reinterpret_cast<T *>(x)[at + i] = (T)((float)codes[at + i] * s);
    }
}

int check(const char *who, int32_t dtype, int64_t rows, int64_t width, int64_t &groups, int64_t &blocks)
{
    if (!known_dtype(dtype)) return fail(IGX_E_PARAM, "%s: dtype %d is not IGX_F32, IGX_F16 or IGX_BF16", who, dtype);
    if (rows < 0 || width < 0) return fail(IGX_E_SIZE, "%s: rows and width must not be negative", who);
    groups = width / IGX_PACK8_GROUP + (width % IGX_PACK8_GROUP != 0);
    const int64_t most = (int64_t)1 << 31;  // lanes of one launch stay under 2^32
    const int64_t lanes_per_group = IGX_PACK8_GROUP / (dtype == IGX_F32 ? 4 : 8);
    if (rows > most || groups > most || (groups && rows > most / lanes_per_group / groups))
        return fail(IGX_E_SIZE, "%s: %lld rows of %lld elements are more than one launch takes", who, (long long)rows,
                    (long long)width);
    blocks = ceil_div(rows * groups * lanes_per_group, kBlock);
    return IGX_OK;
}

}  // namespace
}  // namespace igx

extern "C" int igx_pack8(const void *x, int32_t dtype, int64_t rows, int64_t width, int64_t x_stride, int8_t *codes,
                         float *scales, igx_stream_t stream)
{
    int64_t groups, blocks;
    const int rc = igx::check(__func__, dtype, rows, width, groups, blocks);
    if (rc) return rc;
    if (x_stride < 0) return igx::fail(IGX_E_PARAM, "%s: x_stride must not be negative", __func__);
    if (blocks == 0) return IGX_OK;
    IGX_REQUIRE_PTR(x, "x");
    IGX_REQUIRE_PTR(codes, "codes");
    IGX_REQUIRE_PTR(scales, "scales");
    const dim3 grid((unsigned)blocks), block(igx::kBlock);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const char *p = static_cast<const char *>(x);
    const int64_t step = x_stride * igx::element_size(dtype);
    if (dtype == IGX_F32) igx::pack8_kernel<float, 4><<<grid, block, 0, s>>>(p, step, rows, width, groups, codes, scales);
    else if (dtype == IGX_F16) igx::pack8_kernel<_Float16, 8><<<grid, block, 0, s>>>(p, step, rows, width, groups, codes, scales);
    else igx::pack8_kernel<__bf16, 8><<<grid, block, 0, s>>>(p, step, rows, width, groups, codes, scales);
    return igx::launch_status(__func__);
}

extern "C" int igx_unpack8(const int8_t *codes, const float *scales, int32_t dtype, int64_t rows, int64_t width, void *x,
                           igx_stream_t stream)
{
    int64_t groups, blocks;
    const int rc = igx::check(__func__, dtype, rows, width, groups, blocks);
    if (rc) return rc;
    if (blocks == 0) return IGX_OK;
    IGX_REQUIRE_PTR(codes, "codes");
    IGX_REQUIRE_PTR(scales, "scales");
    IGX_REQUIRE_PTR(x, "x");
    const dim3 grid((unsigned)blocks), block(igx::kBlock);
    hipStream_t s = static_cast<hipStream_t>(stream);
    char *p = static_cast<char *>(x);
    if (dtype == IGX_F32) igx::unpack8_kernel<float, 4><<<grid, block, 0, s>>>(codes, scales, rows, width, groups, p);
    else if (dtype == IGX_F16) igx::unpack8_kernel<_Float16, 8><<<grid, block, 0, s>>>(codes, scales, rows, width, groups, p);
    else igx::unpack8_kernel<__bf16, 8><<<grid, block, 0, s>>>(codes, scales, rows, width, groups, p);
    return igx::launch_status(__func__);
}
