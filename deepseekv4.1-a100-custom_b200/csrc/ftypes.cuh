// Element types of the dense operators (norm.cu, dense.cu, fgemm.cu): bf16, fp16 and fp32 behind one set of conversions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace b200 {

enum : int { F_BF16 = 0, F_FP16 = 1, F_FP32 = 2 };  // the `dtype` argument of the C-ABI

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }

// two values <-> one 32-bit word of a 16-bit type
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t u);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)); }
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
}

// 8 consecutive values: one 16-byte access (16-bit types) or two (fp32)
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(u[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
// VEC consecutive values, VEC = 8 (16-byte aligned) or 1
template <typename T, int VEC> __device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
    if constexpr (VEC == 8) load8<T>(p, v);
    else v[0] = to_f32(*p);
}
template <typename T, int VEC> __device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
    if constexpr (VEC == 8) store8<T>(p, v);
    else *p = from_f32<T>(v[0]);
}

inline int f_elem_bytes(int dtype) { return dtype == F_FP32 ? 4 : 2; }

// ------------------------------------------------------------------ activations of the dense operators
enum : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4 };

// 1 / (1 + e^-z) on the special-function unit: a few fp32 ulp, far below the rounding of the 16-bit result.  e^-z overflows to +inf for
// z < -88, where the quotient is 0.
__device__ __forceinline__ float sigmoid_fast(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

// Phi(z), the normal distribution function: erfc by the rational approximation 7.1.26 of Abramowitz and Stegun, Handbook of Mathematical
// Functions, taken on the side where it is small, so that Phi of a negative z does not come out of a cancellation.  |error| of Phi <= 0.75e-7.  Its relative
// error grows down the tail: 5e-5 at z = -3, 5e-4 at -4, 1.6e-3 at -5, 1 % at -8 (0.5 (1 + erff(..)) in fp32: 8e-4 at -4, 8 % at -5, nothing left at -6).
// z Phi(z) is therefore off by half a step of fp16 more around z = -4, where it is -1.3e-4, and by more than half a step of bf16 below z = -5.5, where it
// is smaller than 1.1e-7.  A third of the instructions of 0.5 (1 + erff(..)), which made the epilogue of a large tile longer than the products under it.
__device__ __forceinline__ float normal_cdf(float z) {
    const float a = fabsf(z) * 0.70710678118654752f, t = __fdividef(1.f, 1.f + 0.3275911f * a);
    const float p = t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
    const float q = 0.5f * p * __expf(-a * a);
    return z < 0.f ? q : 1.f - q;
}

__device__ __forceinline__ float act_fwd(int act, float z) {
    switch (act) {
        case ACT_RELU: return z < 0.f ? 0.f : z;  // a NaN stays one
        case ACT_SILU: return z * sigmoid_fast(z);
        case ACT_GELU: return z * normal_cdf(z);
        // z (1 + tanh a) / 2 = z sigmoid(2 a): no cancellation for very negative z
        case ACT_GELU_TANH: return z * sigmoid_fast(1.5957691216057308f * (z + 0.044715f * z * z * z));
        default: return z;
    }
}

// act(z) and its derivative
__device__ __forceinline__ float2 act_bwd(int act, float z) {
    switch (act) {
        case ACT_RELU: return make_float2(z < 0.f ? 0.f : z, z > 0.f ? 1.f : 0.f);
        case ACT_SILU: {
            const float s = sigmoid_fast(z);
            return make_float2(z * s, s * (1.f + z * (1.f - s)));
        }
        case ACT_GELU: {
            const float p = normal_cdf(z);
            return make_float2(z * p, p + z * 0.3989422804014327f * __expf(-0.5f * z * z));
        }
        case ACT_GELU_TANH: {
            const float a2 = 1.5957691216057308f * (z + 0.044715f * z * z * z), s = sigmoid_fast(a2);
            return make_float2(z * s, s + z * s * (1.f - s) * 1.5957691216057308f * (1.f + 0.134145f * z * z));
        }
        default: return make_float2(z, 1.f);
    }
}

template <int A> struct ActCode { static constexpr int value = A; };
// n values at once, the choice of the activation outside the loop (a switch per value cost the epilogue of a 4096 x 12288 product 10 us)
template <int N>
__device__ __forceinline__ void act_fwd_n(int act, float (&z)[N]) {
    auto each = [&](auto code) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = act_fwd(decltype(code)::value, z[i]);
    };
    switch (act) {
        case ACT_RELU: each(ActCode<ACT_RELU>()); break;
        case ACT_SILU: each(ActCode<ACT_SILU>()); break;
        case ACT_GELU: each(ActCode<ACT_GELU>()); break;
        case ACT_GELU_TANH: each(ActCode<ACT_GELU_TANH>()); break;
    }
}
// act(z) into a, its derivative into d
template <int N>
__device__ __forceinline__ void act_bwd_n(int act, const float (&z)[N], float (&a)[N], float (&d)[N]) {
    auto each = [&](auto code) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float2 r = act_bwd(decltype(code)::value, z[i]);
            a[i] = r.x;
            d[i] = r.y;
        }
    };
    switch (act) {
        case ACT_NONE: each(ActCode<ACT_NONE>()); break;
        case ACT_RELU: each(ActCode<ACT_RELU>()); break;
        case ACT_SILU: each(ActCode<ACT_SILU>()); break;
        case ACT_GELU: each(ActCode<ACT_GELU>()); break;
        case ACT_GELU_TANH: each(ActCode<ACT_GELU_TANH>()); break;
    }
}

}  // namespace b200
