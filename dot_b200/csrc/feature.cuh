// Shared device helpers of the feature operators (group norm with an
// activation, rotary positions): typed vectors of one memory access, and the
// activations with their derivatives.
//
// Both operators read and write float32, bfloat16 or float16 and compute in
// float32; a value is rounded to its type once, when it is written.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace dotb {

// N elements of T as one naturally aligned access (1 to 16 bytes).
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, N>*>(p);
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& v) {
    *reinterpret_cast<Pack<T, N>*>(p) = v;
}
template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& p, float (&f)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = to_f32(p.v[j]);
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> pack(const float (&f)[N]) {
    Pack<T, N> p;
#pragma unroll
    for (int j = 0; j < N; ++j) p.v[j] = from_f32<T>(f[j]);
    return p;
}

// Makes a register's bits opaque, so that what was computed from them is not
// kept alive across this point but computed again (a 16-bit vector costs half
// the registers of its float32 values).
template <typename T, int N>
__device__ __forceinline__ void reload(Pack<T, N>& p) {
    if constexpr (sizeof(p) >= 4) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&p);
#pragma unroll
        for (int i = 0; i < int(sizeof(p) / 4); ++i) asm volatile("" : "+r"(w[i]));
    } else {
        asm volatile("" : "+h"(*reinterpret_cast<uint16_t*>(&p)));
    }
}

// A per-channel parameter of type `dtype` (enum dot_dtype).
__device__ __forceinline__ float load_param(const void* p, int dtype, int64_t i) {
    if (dtype == 0) return static_cast<const float*>(p)[i];
    if (dtype == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, float v) {
    if (dtype == 0)
        static_cast<float*>(p)[i] = v;
    else if (dtype == 1)
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else
        static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// Activations (enum dot_activation).  The exponentials go through the SFU
// (ex2.approx, relative error 2^-22, plus |z| 2^-24 from scaling the
// argument), as does the reciprocal: 1e-6 at most where silu is not
// negligible, and below one rounding of the 16-bit types.
enum : int { kActNone = 0, kActSilu = 1, kActGelu = 2, kActRelu = 3 };

__device__ __forceinline__ float sigmoid_fast(float z) { return __fdividef(1.0f, 1.0f + ex2(-z * kLog2e)); }

// Through erfc, so that the lower tail keeps its relative accuracy.
__device__ __forceinline__ float normal_cdf(float z) { return 0.5f * erfcf(-0.70710678f * z); }

template <int ACT>
__device__ __forceinline__ float act_fwd(float z, int act_rt) {
    const int act = ACT >= 0 ? ACT : act_rt;
    if (act == kActSilu) return z * sigmoid_fast(z);
    if (act == kActGelu) return z * normal_cdf(z);
    if (act == kActRelu) return z < 0.0f ? 0.0f : z;   // a NaN stays one
    return z;
}
// d act / d z
template <int ACT>
__device__ __forceinline__ float act_slope(float z, int act_rt) {
    const int act = ACT >= 0 ? ACT : act_rt;
    if (act == kActSilu) {
        const float s = sigmoid_fast(z);
        return s * (1.0f + z * (1.0f - s));
    }
    if (act == kActGelu) {
        return normal_cdf(z) + z * 0.39894228f * ex2(-0.5f * kLog2e * z * z);
    }
    if (act == kActRelu) return z > 0.0f ? 1.0f : 0.0f;
    return 1.0f;
}

}  // namespace dotb
