// What the forward and backward kernels of the block norms share (block_norm.hip, block_norm_backward.hip).
#pragma once
#include <type_traits>

#include "igx_seq.hpp"

namespace igx {

constexpr int kNormBlock = 256;   // of the kernels whose row fits one wave

// 16-byte vectors of a row in a lane.  One, which leaves registers for enough waves (2^20 x 256 bf16 forward and backward with the
// column sums: 1 340 us, 1 545 with two; 16 411 x 211 fp32: 45, 46) - but two where the forward kernel has a single array to read
// and its norm's weight to hold (2^20 x 64 fp32: 85 us, 94 with one), and where 1024 lanes need them for the widest rows.
constexpr int vectors_of(bool alone, bool largest, int vec) { return alone || (largest && vec == 4) ? 2 : 1; }

struct NormArgs {
    const char *x, *y, *gate, *d_out, *d_next;
    const char *x_end, *y_end, *gate_end, *d_out_end, *d_next_end;  // behind each array's last element
    int64_t x_row, y_row, gate_row, d_out_row, d_next_row;          // bytes from row to row
    char *out, *next, *d_x, *d_y, *d_gate;
    const float *weight, *scale, *next_weight;
    float *y_inv, *out_inv;
    int8_t *y8, *gate8;
    float *y8_scale, *gate8_scale;
    float *partial;  // [sums][workgroups][width]: of d act rms(y), of d_next rms(out)
    int64_t rows;
    int width, groups, act;
    float eps;
    bool sum_block, sum_next;
};

// e = exp(-z) and 1 / (1 + e) from the hardware's exponential and reciprocal (1 ulp each); `rest` carries what the product
// z log2(e) loses, so that the error does not grow with |z|.  Where e leaves fp32 the result is 0 or 1 without it.
__device__ __forceinline__ float sigmoid(float z, float &e)
{
    const float log2e = 1.44269504f, ln2 = 0.693147181f, log2e_rest = 1.92596303e-8f;
    const float t = -z * log2e;
    const float rest = (fmaf(-z, log2e, -t) - z * log2e_rest) * ln2;
    e = __builtin_amdgcn_exp2f(t);
    e = fabsf(t) < 126.0f ? fmaf(e, rest, e) : e;  // not inf - inf
    return __builtin_amdgcn_rcpf(1.0f + e);
}

__device__ __forceinline__ float activate(float z, int act)
{
    if (act == IGX_GATE_NONE) return z;
    float e;
    const float p = sigmoid(z, e);
    return act == IGX_GATE_SIGMOID ? p : z * p;
}

__device__ __forceinline__ void activate_slope(float z, int act, float &f, float &slope)
{
    if (act == IGX_GATE_NONE) {
        f = z;
        slope = 1.0f;
        return;
    }
    float e;
    const float p = sigmoid(z, e), q = fminf(e, 3.0e38f) * p * p;  // p (1 - p) without the difference of near values
    f = act == IGX_GATE_SIGMOID ? p : z * p;
    slope = act == IGX_GATE_SIGMOID ? q : fmaf(z, q, p);
}

// The lanes that share a row.  LANES 8 ... 64: that many lanes of a wave, kWorkgroup: the whole workgroup of up to 512,
// kLargest: one of 1024, which leaves a lane half as many registers.
constexpr int kWorkgroup = 0, kLargest = -1;
constexpr int block_of(int lanes) { return lanes > 0 ? kNormBlock : lanes == kWorkgroup ? 512 : 1024; }

template <typename T, int LANES, bool ALONE> struct RowLanes {
    static constexpr int V = 16 / sizeof(T);
    static constexpr int K = vectors_of(ALONE, LANES == kLargest, V);
    static constexpr bool kWide = LANES <= 0;
    int lane, lanes, rows_per_block, sub;
    __device__ __forceinline__ RowLanes()
    {
        lanes = kWide ? blockDim.x : LANES;
        lane = kWide ? threadIdx.x : threadIdx.x % (kWide ? 1 : LANES);
        sub = kWide ? 0 : threadIdx.x / (kWide ? 1 : LANES);
        rows_per_block = kWide ? 1 : kNormBlock / (kWide ? 1 : LANES);
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
template <typename T, int V, bool STREAM> __device__ __forceinline__ Raw<T, V> load_row(const char *p, const char *end, int left)
{
    Raw<T, V> r = {};
    if (left <= 0) return r;
    if (p + V * sizeof(T) <= end) {
        r = load_raw<T, V, STREAM>(p);
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

template <typename T, int V, bool STREAM> __device__ __forceinline__ void store_row(char *p, const float (&f)[V], int left)
{
    if (left >= V) {
        store_vec<T, V, STREAM>(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < left) reinterpret_cast<T *>(p)[i] = (T)f[i];
    }
}

template <int V> __device__ __forceinline__ void load_param(const float *p, int col, int left, float (&f)[V])
{
    if (left >= V) {
        widen(load_raw<float, V>(p + col), f);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) f[i] = i < left ? p[col + i] : 0.0f;
    }
}

template <int V> __device__ __forceinline__ void load_factor(const NormArgs &a, int col, int left, float (&f)[V])
{
    load_param<V>(a.weight, col, left, f);
    if (!a.scale) return;
    float s[V];
    load_param<V>(a.scale, col, left, s);
#pragma unroll
    for (int i = 0; i < V; i++) f[i] *= s[i];
}

// the kernels' launches; `stream_past` picks the STREAM variants
void launch_block_norm(const NormArgs &a, int dtype, bool stream_past, int64_t blocks, hipStream_t s);
void launch_block_norm_backward(const NormArgs &a, int dtype, bool stream_past, int64_t blocks, hipStream_t s);

// Lanes of a row: the fewest that hold its columns; above 64 a workgroup of that many.
inline int lanes_for(int64_t width, int dtype, bool alone)
{
    const int vec = 16 / element_size(dtype);
    int lanes = 8;
    while (lanes < 1024 && lanes * vec * vectors_of(alone, false, vec) < width) lanes *= 2;
    return lanes;
}

}  // namespace igx
