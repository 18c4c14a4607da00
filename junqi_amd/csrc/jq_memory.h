// Element types, vector access and sums over lanes shared by the operators of a
// policy's memory (gfx950, wave64).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

#include "junqi_amd.h"

namespace jq {

typedef __bf16 bf16;

template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16 from_float<bf16>(float x) { return (bf16)x; }   // round to nearest even

// Element (b, t, h, 0) of a (batch, plies, heads, dim) tensor.
template <class T> __device__ __forceinline__ T *row_at(const jq_rows &r, int64_t b, int64_t t, int64_t h)
{
    return static_cast<T *>(r.data) + b * r.batch + t * r.ply + h * r.head;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 16 bytes of T.
template <class T> struct Vec;
template <> struct Vec<float> { typedef f32x4 type; static constexpr int N = 4; };
template <> struct Vec<bf16> { typedef bf16x8 type; static constexpr int N = 8; };

template <class T, int V> struct Pack { typedef T type __attribute__((ext_vector_type(V))); };

// V elements at any element alignment, zeros from n on (n >= 1).
template <class T, int V>
__device__ __forceinline__ typename Pack<T, V>::type load_some(const T *p, int n)
{
    typedef typename Pack<T, V>::type R;
    typedef R At __attribute__((aligned(sizeof(T))));
    if (n >= V) return *reinterpret_cast<const At *>(p);
    R r;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const T y = p[e < n ? e : n - 1];
        r[e] = e < n ? y : T(0.f);
    }
    return r;
}
template <class T, int V>
__device__ __forceinline__ void store_some(T *p, int n, typename Pack<T, V>::type r)
{
    typedef typename Pack<T, V>::type R;
    typedef R At __attribute__((aligned(sizeof(T))));
    if (n >= V) *reinterpret_cast<At *>(p) = r;
    else
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < n) p[e] = r[e];
}
template <class T, int V>
__device__ __forceinline__ void store_floats(T *p, int n, const float *x)
{
    typename Pack<T, V>::type r;
#pragma unroll
    for (int e = 0; e < V; ++e) r[e] = from_float<T>(x[e]);
    store_some<T, V>(p, n, r);
}

// x + x of the lane O lanes across (l ^ O), O a power of two, where the lanes of each
// aligned group of O hold one sum: then a mirrored row stands for O = 4 and 8, and no
// step goes through LDS.
template <int O>
__device__ __forceinline__ float plus_across(float x)
{
    static_assert(O >= 1 && O <= 32 && !(O & (O - 1)), "a power of two within the wave");
    const int i = __builtin_bit_cast(int, x);
    if constexpr (O >= 16) {   // both of a pair of rows (halves) in each: the lower's, the upper's
        const auto r = O == 16 ? __builtin_amdgcn_permlane16_swap(i, i, false, false)
                               : __builtin_amdgcn_permlane32_swap(i, i, false, false);
        const uint32_t lower = r[0], upper = r[1];   // a bit_cast of r[1] itself takes r's first bytes
        return __builtin_bit_cast(float, lower) + __builtin_bit_cast(float, upper);
    } else {
        constexpr int HOW = O == 1 ? 0xB1 : O == 2 ? 0x4E : O == 4 ? 0x141 : 0x140;   // quad_perm, half mirror, mirror
        return x + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(i, HOW, 0xF, 0xF, false));
    }
}

// The sum over each aligned group of G lanes, in every lane of it.
template <int G>
__device__ __forceinline__ float group_total(float x)
{
    if constexpr (G >= 2) x = plus_across<1>(x);
    if constexpr (G >= 4) x = plus_across<2>(x);
    if constexpr (G >= 8) x = plus_across<4>(x);
    if constexpr (G >= 16) x = plus_across<8>(x);
    if constexpr (G >= 32) x = plus_across<16>(x);
    if constexpr (G >= 64) x = plus_across<32>(x);
    return x;
}

}  // namespace jq
