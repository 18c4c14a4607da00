// Element types, vector access and wave reductions shared by the operators of a
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

// Sum over the wave, in every lane.
__device__ __forceinline__ float wave_total(float x)
{
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

}  // namespace jq
