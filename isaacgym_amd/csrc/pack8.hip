// 8-bit checkpoints of activations: codes and one fp32 scale for every 64 elements of a row, and back.
//
// The lanes of one group take 32 bytes of its elements each and agree on the largest magnitude by exchanging it within the
// wave, so the elements are read once and stay in registers: e + 1 + 4/64 bytes an element each way, bound by HBM (2^20 x 256
// bf16: 146 us to pack, 5.6 TB/s, 144 to unpack, 5.7 TB/s, with 16 bytes a lane 172 and 143; 2^20 x 211 fp32: 199 and 219, with
// 16 bytes a lane 267 and 268).
#include "igx_seq.hpp"

namespace igx {
namespace {

constexpr int kBlock = 256;

// A lane's V columns of a group.  The last vector of a row that V does not divide is moved back to end with the row, where
// that keeps it in the group: the columns it shares with the lane before come out the same from both.
struct Piece {
    int64_t row, at;  // of codes and of a contiguous x
    uint32_t group, col;
    int left;         // of the V columns: V, fewer, or none
};

template <int V> __device__ __forceinline__ Piece piece_of(uint32_t rows, uint32_t width, uint32_t groups)
{
    constexpr uint32_t LPG = IGX_PACK8_GROUP / V;  // lanes of a group
    const uint32_t id = (blockIdx.x * (uint32_t)kBlock + threadIdx.x) / LPG, row = id / groups;
    Piece p;
    p.row = row;
    p.group = id - row * groups;
    p.col = p.group * IGX_PACK8_GROUP + threadIdx.x % LPG * V;
    p.left = row >= rows || p.col >= width ? 0 : width - p.col < V ? (int)(width - p.col) : V;
    if (p.left > 0 && p.left < V && width - p.group * IGX_PACK8_GROUP >= V) {
        p.col = width - V;
        p.left = V;
    }
    p.at = (int64_t)row * width + p.col;
    return p;
}

template <typename T, int V>
__global__ __launch_bounds__(kBlock) void pack8_kernel(const char *x, int64_t stride, uint32_t rows, uint32_t width,
                                                       uint32_t groups, int8_t *codes, float *scales)
{
    constexpr int LPG = IGX_PACK8_GROUP / V;
    const Piece p = piece_of<V>(rows, width, groups);
    float f[V];
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = 0.0f;
    const char *from = x + p.row * stride + (int64_t)p.col * (int64_t)sizeof(T);
    if (p.left == V) {
        widen(load_raw<T, V>(from), f);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < p.left) f[i] = (float)reinterpret_cast<const T *>(from)[i];
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < V; i++) top = max(top, magnitude_bits(f[i]));
#pragma unroll
    for (int m = 1; m < LPG; m *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, m));
    const GroupScale s = group_scale(top);
    if (p.left == V) {
        store_codes<V>(codes + p.at, f, s.inverse);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < p.left) codes[p.at + i] = code_of(f[i], s.inverse);
    }
    if (threadIdx.x % LPG == 0 && p.left > 0) scales[p.row * groups + p.group] = s.scale;
}

template <typename T, int V>
__global__ __launch_bounds__(kBlock) void unpack8_kernel(const int8_t *codes, const float *scales, uint32_t rows, uint32_t width,
                                                         uint32_t groups, char *x)
{
    const Piece p = piece_of<V>(rows, width, groups);
    if (p.left == 0) return;
    const float s = scales[p.row * groups + p.group];
    float f[V];
    if (p.left == V) {
        load_codes<V>(codes + p.at, f);
#pragma unroll
        for (int i = 0; i < V; i++) f[i] *= s;
        store_vec<T, V>(x + p.at * sizeof(T), f);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < p.left) reinterpret_cast<T *>(x)[p.at + i] = (T)((float)codes[p.at + i] * s);
    }
}

int check(const char *who, int32_t dtype, int64_t rows, int64_t width, int64_t &groups, int64_t &blocks)
{
    if (!known_dtype(dtype)) return fail(IGX_E_PARAM, "%s: dtype %d is not IGX_F32, IGX_F16 or IGX_BF16", who, dtype);
    if (rows < 0 || width < 0) return fail(IGX_E_SIZE, "%s: rows and width must not be negative", who);
    groups = width / IGX_PACK8_GROUP + (width % IGX_PACK8_GROUP != 0);
    const int64_t most = (int64_t)1 << 31;  // lanes of one launch, counted in 32 bits
    const int64_t lanes_per_group = IGX_PACK8_GROUP / (dtype == IGX_F32 ? 8 : 16);
    if (rows > most || width > most || (groups && rows > most / lanes_per_group / groups))
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
    const uint32_t n = (uint32_t)rows, w = (uint32_t)width, g = (uint32_t)groups;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const char *p = static_cast<const char *>(x);
    const int64_t step = x_stride * igx::element_size(dtype);
    if (dtype == IGX_F32) igx::pack8_kernel<float, 8><<<grid, block, 0, s>>>(p, step, n, w, g, codes, scales);
    else if (dtype == IGX_F16) igx::pack8_kernel<_Float16, 16><<<grid, block, 0, s>>>(p, step, n, w, g, codes, scales);
    else igx::pack8_kernel<__bf16, 16><<<grid, block, 0, s>>>(p, step, n, w, g, codes, scales);
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
    const uint32_t n = (uint32_t)rows, w = (uint32_t)width, g = (uint32_t)groups;
    hipStream_t s = static_cast<hipStream_t>(stream);
    char *p = static_cast<char *>(x);
    if (dtype == IGX_F32) igx::unpack8_kernel<float, 8><<<grid, block, 0, s>>>(codes, scales, n, w, g, p);
    else if (dtype == IGX_F16) igx::unpack8_kernel<_Float16, 16><<<grid, block, 0, s>>>(codes, scales, n, w, g, p);
    else igx::unpack8_kernel<__bf16, 16><<<grid, block, 0, s>>>(codes, scales, n, w, g, p);
    return igx::launch_status(__func__);
}
