// Element types and vector access shared by the sequence operators (recurrence.hip, block_norm.hip, pack8.hip).
//
// A lane moves 16 bytes at a time: 4 fp32 or 8 fp16 / bf16 elements.  The accesses are typed with the element's own
// alignment: global memory takes 16-byte accesses at any address here, so odd widths and shifted views use the same
// instructions as aligned ones and no second code path exists.
#pragma once
#include "igx_host.hpp"

namespace igx {

template <int DT> struct Elem;
template <> struct Elem<IGX_F32> { using type = float; static constexpr int vec = 4; };
template <> struct Elem<IGX_F16> { using type = _Float16; static constexpr int vec = 8; };
template <> struct Elem<IGX_BF16> { using type = __bf16; static constexpr int vec = 8; };

// V elements of type T at T's own alignment
template <typename T, int V> struct Pack { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };
template <typename T> struct Pack<T, 1> { typedef T type; };

template <typename T, int V> struct Raw { typename Pack<T, V>::type v; };

// STREAM: past the caches' replacement, for what is not read again soon
template <typename T, int V, bool STREAM = false> __device__ __forceinline__ Raw<T, V> load_raw(const void *p)
{
    const typename Pack<T, V>::type *q = reinterpret_cast<const typename Pack<T, V>::type *>(p);
    if constexpr (STREAM && V > 1) return {__builtin_nontemporal_load(q)};
    else return {*q};
}

template <typename T, int V> __device__ __forceinline__ float raw_at(const Raw<T, V> &r, int i)
{
    if constexpr (V == 1) return (float)r.v;
    else return (float)r.v[i];
}

template <typename T, int V> __device__ __forceinline__ void widen(const Raw<T, V> &r, float (&f)[V])
{
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = raw_at(r, i);
}

// one rounding to nearest even, the hardware's conversion
template <typename T, int V, bool STREAM = false> __device__ __forceinline__ void store_vec(void *p, const float (&f)[V])
{
    if constexpr (V == 1) {
        *reinterpret_cast<T *>(p) = (T)f[0];
    } else {
        typename Pack<T, V>::type v;
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = (T)f[i];
        if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<typename Pack<T, V>::type *>(p));
        else *reinterpret_cast<typename Pack<T, V>::type *>(p) = v;
    }
}

// ---- 8-bit codes: groups of IGX_PACK8_GROUP elements of a row share one scale ------------------------------------
constexpr float kSmallestTop = 7.52316385e-37f;  // 2^-120: 127 / top stays finite

// magnitude bits: as integers they order like the magnitudes, with inf and then NaN on top
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct GroupScale {
    float inverse, scale;  // code = rint(x * inverse), value = code * scale
};

__device__ __forceinline__ GroupScale group_scale(uint32_t top_bits)
{
    GroupScale s;
    const float top = __uint_as_float(top_bits);
    if (top_bits >= 0x7f800000u) {  // inf or NaN in the group: code 0, value NaN
        s.inverse = 0.0f;
        s.scale = __uint_as_float(0x7fc00000u);
    } else if (top < kSmallestTop) {
        s.inverse = s.scale = 0.0f;
    } else {
        s.inverse = 127.0f / top;
        s.scale = top / 127.0f;
    }
    return s;
}

// The code in the low byte.  |x| <= top, so the product lies within +-127 and the sum's last place is 1: the addition rounds
// to the nearest integer, ties to even, and its mantissa ends in the integer's two's complement.
__device__ __forceinline__ uint32_t code_bits(float x, float inverse)
{
    return __float_as_uint(x * inverse + 12582912.0f);  // 3 * 2^22
}

__device__ __forceinline__ int8_t code_of(float x, float inverse)
{
    return inverse == 0.0f ? 0 : (int8_t)code_bits(x, inverse);
}

template <int V> __device__ __forceinline__ void store_codes(int8_t *p, const float (&x)[V], float inverse)
{
    uint32_t w[V / 4];
#pragma unroll
    for (int j = 0; j < V / 4; j++) {
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; i++) c[i] = code_bits(x[4 * j + i], inverse);
        const uint32_t low = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400), high = __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400);
        w[j] = inverse == 0.0f ? 0 : __builtin_amdgcn_perm(high, low, 0x05040100);  // 0: the products may be NaN
    }
    __builtin_memcpy(p, w, V);
}

template <int V> __device__ __forceinline__ void load_codes(const int8_t *p, float (&x)[V])
{
    uint32_t w[V / 4];
    __builtin_memcpy(w, p, V);
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4)));
}

inline int element_size(int dtype) { return dtype == IGX_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == IGX_F32 || dtype == IGX_F16 || dtype == IGX_BF16; }

__host__ __device__ inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace igx
