// What the kernels of the training-loss terms (distill.hip, balance.hip) share: values of three types as floats, runs of them at any
// address, reductions over a workgroup in a fixed order.
#pragma once

#include "lpmm_common.hpp"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <math.h>

#include <type_traits>

namespace lpmm {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Types of values, one by one and in runs of 16 bytes.
struct F32 {
    using Raw = float;
    static constexpr int kRun = 4;
    static constexpr uint32_t kNoValue = 0xff800000u;  // -infinity in every place of a word
    static __device__ __forceinline__ float get(Raw v) { return v; }
    static __device__ __forceinline__ Raw put(float v) { return v; }
    static __device__ __forceinline__ void unpack(u32x4 r, float (&v)[kRun])
    {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = __uint_as_float(r[j]);
    }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[kRun])
    {
        return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    }
};
struct F16 {
    using Raw = _Float16;
    static constexpr int kRun = 8;
    static constexpr uint32_t kNoValue = 0xfc00fc00u;
    static __device__ __forceinline__ float get(Raw v) { return (float)v; }
    static __device__ __forceinline__ Raw put(float v) { return (Raw)v; }
    static __device__ __forceinline__ void unpack(u32x4 r, float (&v)[kRun])
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t word = r[j];  // a copy: the cast of an element of a vector takes the vector's first
            const f16x2 two = __builtin_bit_cast(f16x2, word);
            v[2 * j] = (float)two[0];
            v[2 * j + 1] = (float)two[1];
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[kRun])
    {
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            r[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2 * j], v[2 * j + 1]}), f16x2));
        return r;
    }
};
struct BF16 {
    using Raw = __bf16;
    static constexpr int kRun = 8;
    static constexpr uint32_t kNoValue = 0xff80ff80u;
    static __device__ __forceinline__ float get(Raw v) { return (float)v; }
    static __device__ __forceinline__ Raw put(float v) { return (Raw)v; }
    static __device__ __forceinline__ void unpack(u32x4 r, float (&v)[kRun])
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = __uint_as_float(r[j] << 16);
            v[2 * j + 1] = __uint_as_float(r[j] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&v)[kRun])
    {
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            r[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2 * j], v[2 * j + 1]}), bf16x2));
        return r;
    }
};

// 16 bytes of values at an address that only their type aligns: rows of odd lengths start anywhere, and the hardware takes a 16-byte access
// at any address of device memory.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <typename T>
__device__ __forceinline__ u32x4 load_run(const typename T::Raw *p)
{
    return *reinterpret_cast<const u32x4_any *>(p);
}

// What is read once, of an array that no cache holds.
template <typename T>
__device__ __forceinline__ u32x4 load_run_once(const typename T::Raw *p)
{
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(p));
}

template <typename T>
__device__ __forceinline__ void store_run(typename T::Raw *p, u32x4 r)
{
    *reinterpret_cast<u32x4_any *>(p) = r;
}

template <typename T>
__device__ __forceinline__ void store_run_once(typename T::Raw *p, u32x4 r)
{
    __builtin_nontemporal_store(r, reinterpret_cast<u32x4_any *>(p));
}

// 2^x, off by one unit in the last place at most; results below the smallest normal number are 0
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float wave_sum(float v)
{
    v += dpp_f32<0xB1>(v);   // quad_perm [1,0,3,2]
    v += dpp_f32<0x4E>(v);   // quad_perm [2,3,0,1]
    v += dpp_f32<0x141>(v);  // row_half_mirror
    v += dpp_f32<0x140>(v);  // row_mirror
    v += __shfl_xor(v, 16, kWave);
    v += __shfl_xor(v, 32, kWave);
    return v;
}

// Sum and maximum over N neighbouring lanes (4, 8 or 16), in all of them: what N waves left, read by lane i from place i % N.
template <int N>
__device__ __forceinline__ float lanes_sum(float v)
{
    v += dpp_f32<0xB1>(v);
    v += dpp_f32<0x4E>(v);
    if constexpr (N >= 8)
        v += dpp_f32<0x141>(v);
    if constexpr (N >= 16)
        v += dpp_f32<0x140>(v);
    return v;
}

template <int N>
__device__ __forceinline__ float lanes_max(float v)
{
    v = fmaxf(v, dpp_f32<0xB1>(v));
    v = fmaxf(v, dpp_f32<0x4E>(v));
    if constexpr (N >= 8)
        v = fmaxf(v, dpp_f32<0x141>(v));
    if constexpr (N >= 16)
        v = fmaxf(v, dpp_f32<0x140>(v));
    return v;
}

template <int THREADS>
__device__ __forceinline__ double block_sum_f64(double v, double *room)
{
    v = wave_sum_f64(v);
    if constexpr (THREADS > kWave) {
        if ((threadIdx.x & (kWave - 1)) == 0)
            room[threadIdx.x / kWave] = v;
        __syncthreads();
        v = room[0];
#pragma unroll
        for (int w = 1; w < THREADS / kWave; ++w)
            v += room[w];
        __syncthreads();
    }
    return v;
}

}  // namespace lpmm
