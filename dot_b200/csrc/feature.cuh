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
#include <type_traits>

#include "common.cuh"
#include "pack.cuh"

namespace dotb {

// Division by a number that the host knows: n / d = (n * m) >> 32 >> s for
// n < 2^31 (Granlund and Montgomery, 1994), two instructions.
struct FastDiv {
    uint32_t d = 1, m = 0, s = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        if (d > 1) {
            while ((1ull << s) < d) ++s;                          // ceil(log2 d)
            m = uint32_t(((1ull << 31 << s) + d - 1) / d);        // ceil(2^(31+s) / d) < 2^32
            --s;
        }
    }
    __device__ __forceinline__ int div(int n) const { return d == 1 ? n : int(__umulhi(uint32_t(n), m) >> s); }
};

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
// A vector's values as pairs for the packed f32x2 arithmetic (pack.cuh), which
// halves the issue slots; a vector of one element fills half a pair.
constexpr int pairs_of(int n) { return (n + 1) / 2; }

template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& p, float2 (&f)[pairs_of(N)]) {
    if constexpr (N == 1) {
        f[0] = make_float2(to_f32(p.v[0]), 0.0f);
    } else {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            if constexpr (sizeof(T) == 4) {
                f[j] = make_float2(p.v[2 * j], p.v[2 * j + 1]);
            } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                // bfloat16 is float32's upper half
                const uint32_t w = reinterpret_cast<const uint32_t*>(&p)[j];
                f[j] = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
            } else {
                f[j] = __half22float2(reinterpret_cast<const __half2*>(&p)[j]);
            }
        }
    }
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> pack(const float2 (&f)[pairs_of(N)]) {
    Pack<T, N> p;
    if constexpr (N == 1) {
        p.v[0] = from_f32<T>(f[0].x);
    } else {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            if constexpr (sizeof(T) == 4) {
                p.v[2 * j] = f[j].x;
                p.v[2 * j + 1] = f[j].y;
            } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                reinterpret_cast<__nv_bfloat162*>(&p)[j] = __floats2bfloat162_rn(f[j].x, f[j].y);
            } else {
                reinterpret_cast<__half2*>(&p)[j] = __floats2half2_rn(f[j].x, f[j].y);
            }
        }
    }
    return p;
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> pack_zero() {
    const float2 z[pairs_of(N)] = {};
    return pack<T, N>(z);
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

// N consecutive per-channel parameters from c on, as pairs; `other` where p is NULL.
template <typename P, int N>
__device__ __forceinline__ void load_params_as(const void* p, int64_t c, float2 (&f)[pairs_of(N)]) {
    const P* at = static_cast<const P*>(p) + c;
#pragma unroll
    for (int j = 0; j < pairs_of(N); ++j) f[j] = make_float2(to_f32(at[2 * j]), N == 1 ? 0.0f : to_f32(at[2 * j + 1]));
}
template <int N>
__device__ __forceinline__ void load_params(const void* p, int dtype, int64_t c, float other, float2 (&f)[pairs_of(N)]) {
    if (p == nullptr) {
#pragma unroll
        for (int j = 0; j < pairs_of(N); ++j) f[j] = splat2(other);
    } else if (dtype == 0) {
        load_params_as<float, N>(p, c, f);
    } else if (dtype == 1) {
        load_params_as<__nv_bfloat16, N>(p, c, f);
    } else {
        load_params_as<__half, N>(p, c, f);
    }
}

// Activations (enum dot_activation), two values at a time.  The exponentials go
// through the SFU (ex2.approx, relative error 2^-22, plus |z| 2^-24 from
// scaling the argument), as does the reciprocal: 1e-6 at most where silu is not
// negligible, and below one rounding of the 16-bit types.
enum : int { kActNone = 0, kActSilu = 1, kActGelu = 2, kActRelu = 3 };

// 1/x on the SFU (rcp.approx, 1 ulp; 0 for an infinite x)
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 ex2_2(float2 x) { return make_float2(ex2(x.x), ex2(x.y)); }

__device__ __forceinline__ float2 sigmoid2(float2 z) {
    const float2 d = add2(ex2_2(mul2(z, splat2(-kLog2e))), splat2(1.0f));
    return make_float2(rcp_fast(d.x), rcp_fast(d.y));
}

// Through erfc, so that the lower tail keeps its relative accuracy.
__device__ __forceinline__ float2 normal_cdf2(float2 z) {
    return make_float2(0.5f * erfcf(-0.70710678f * z.x), 0.5f * erfcf(-0.70710678f * z.y));
}

template <int ACT>
__device__ __forceinline__ float2 act_fwd(float2 z, int act_rt) {
    const int act = ACT >= 0 ? ACT : act_rt;
    if (act == kActSilu) return mul2(z, sigmoid2(z));
    if (act == kActGelu) return mul2(z, normal_cdf2(z));
    if (act == kActRelu) return make_float2(z.x < 0.0f ? 0.0f : z.x, z.y < 0.0f ? 0.0f : z.y);   // a NaN stays one
    return z;
}
// d act / d z
template <int ACT>
__device__ __forceinline__ float2 act_slope(float2 z, int act_rt) {
    const int act = ACT >= 0 ? ACT : act_rt;
    if (act == kActSilu) {
        const float2 s = sigmoid2(z);
        return fma2(z, sub2(s, mul2(s, s)), s);   // s + z s (1 - s)
    }
    if (act == kActGelu) {
        const float2 pdf = mul2(ex2_2(mul2(mul2(z, splat2(-0.5f * kLog2e)), z)), splat2(0.39894228f));
        return fma2(z, pdf, normal_cdf2(z));
    }
    if (act == kActRelu) return make_float2(z.x > 0.0f ? 1.0f : 0.0f, z.y > 0.0f ? 1.0f : 0.0f);
    return splat2(1.0f);
}

}  // namespace dotb
