// Element types of the operators that take more than fp16, and their loads of 16 bytes or element by element.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace b200 {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Two neighbours (at an even place, by whole words of memory), rounded together.
__device__ __forceinline__ float2 pair_of(const float* p) { return make_float2(p[0], p[1]); }
__device__ __forceinline__ float2 pair_of(const __half* p) { return __half22float2(*reinterpret_cast<const __half2*>(p)); }
__device__ __forceinline__ float2 pair_of(const __nv_bfloat16* p) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ void set_pair(float* p, float x, float y) { p[0] = x; p[1] = y; }
__device__ __forceinline__ void set_pair(__half* p, float x, float y) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x, y); }
__device__ __forceinline__ void set_pair(__nv_bfloat16* p, float x, float y) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x, y); }

// N elements: one access of N * sizeof(T) bytes (WHOLE), or the first `n` of them one by one.
template <typename T, int N>
struct alignas(N * sizeof(T)) Vec {
    T v[N];
};
template <bool WHOLE, typename T, int N>
__device__ __forceinline__ void load_vec(Vec<T, N>& d, const T* p, int n) {
    if (WHOLE) {
        d = *reinterpret_cast<const Vec<T, N>*>(p);
    } else {
#pragma unroll
        for (int e = 0; e < N; e++)
            if (e < n) d.v[e] = p[e];
    }
}
template <bool WHOLE, typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& d, int n) {
    if (WHOLE) {
        *reinterpret_cast<Vec<T, N>*>(p) = d;
    } else {
#pragma unroll
        for (int e = 0; e < N; e++)
            if (e < n) p[e] = d.v[e];
    }
}

inline size_t dtype_size(int dtype) { return dtype == B200_DTYPE_F32 ? 4 : (dtype == B200_DTYPE_F16 || dtype == B200_DTYPE_BF16 ? 2 : 0); }

}  // namespace b200
