// What the kernels of the training-loss terms (distill.hip, balance.hip) share: values of three types as floats, runs of them at any
// address, reductions over a workgroup in a fixed order.
#pragma once

#include "lpmm_common.hpp"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <math.h>

namespace lpmm {

constexpr float kLog2e = 1.44269504088896340736f;

struct F32 {
    using Raw = float;
    static constexpr int kRun = 4;  // values in 16 bytes
    static __device__ __forceinline__ float get(Raw v) { return v; }
    static __device__ __forceinline__ Raw put(float v) { return v; }
};
struct F16 {
    using Raw = _Float16;
    static constexpr int kRun = 8;
    static __device__ __forceinline__ float get(Raw v) { return (float)v; }
    static __device__ __forceinline__ Raw put(float v) { return (Raw)v; }
};
struct BF16 {
    using Raw = __bf16;
    static constexpr int kRun = 8;
    static __device__ __forceinline__ float get(Raw v) { return (float)v; }
    static __device__ __forceinline__ Raw put(float v) { return (Raw)v; }
};

// 16 bytes of values at an address that only their type aligns: rows of odd lengths start anywhere, and the hardware takes a 16-byte access
// at any address of device memory.
template <typename T>
struct Run {
    typename T::Raw v[T::kRun];
};

template <typename T>
__device__ __forceinline__ Run<T> load_run(const typename T::Raw *p)
{
    Run<T> r;
    __builtin_memcpy(&r, p, sizeof r);
    return r;
}

template <typename T>
__device__ __forceinline__ void store_run(typename T::Raw *p, const Run<T> &r)
{
    __builtin_memcpy(p, &r, sizeof r);
}

// 2^x, off by one unit in the last place at most; results below the smallest normal number are 0
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

struct Max {
    static constexpr float kNone = -INFINITY;
    static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};
struct Sum {
    static constexpr float kNone = 0.0f;
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};

// The value of a whole workgroup in every thread; `room`: a float for each wave.  Ends with the barrier that allows the next use of `room`.
template <typename Op, int THREADS>
__device__ __forceinline__ float block_reduce(float v, float *room)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        v = Op::of(v, __shfl_xor(v, o, kWave));
    if constexpr (THREADS > kWave) {
        if ((threadIdx.x & (kWave - 1)) == 0)
            room[threadIdx.x / kWave] = v;
        __syncthreads();
        v = room[0];
#pragma unroll
        for (int w = 1; w < THREADS / kWave; ++w)
            v = Op::of(v, room[w]);
        __syncthreads();
    }
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
