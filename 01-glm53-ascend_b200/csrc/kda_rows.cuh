// Element types, activations and e4m3 rounding shared by the layer's norm and
// projection kernels.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "kda_common.cuh"

namespace kda {

constexpr float kE4m3Max = 448.0f;

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(__nv_fp8_e4m3 v) { return static_cast<float>(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
// Round to nearest even, saturating at +-448; NaN stays NaN.
template <> __device__ __forceinline__ __nv_fp8_e4m3 from_f32(float v) { return __nv_fp8_e4m3(v); }

// Maxima that keep a NaN of any operand (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_abs_nan(float a, float b, float c) {   // of the magnitudes
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// fp32 arithmetic on pairs, one instruction for both.
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

// Two values in a 32-bit word, the first in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) { return make_float2(bf16_lo(v), bf16_hi(v)); }
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
// Four values in e4m3, the first in the low byte.
__device__ __forceinline__ uint32_t pack4_e4m3(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

// 1 / (1 + e^-z) of a pair by the hardware's approximate 2^x and reciprocal: 2^-22
// of itself plus 2^-24 |z| from the rounding of z log2(e), for z > -87.3. Below, where
// it is smaller than fp32's smallest normal value (2^-126), it goes to 0, and with it
// y / (1 + e^-z), by 88 * 2^-126 at most; above it goes to 1. NaN stays NaN.
__device__ __forceinline__ float exp2_approx(float z) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(z));
    return r;
}
__device__ __forceinline__ float reciprocal(float z) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(z));
    return r;
}
__device__ __forceinline__ float2 logistic2(float2 z) {
    const float2 t = mul2(z, make_float2(-1.4426950408889634f, -1.4426950408889634f));
    const float2 d = add2(make_float2(exp2_approx(t.x), exp2_approx(t.y)), make_float2(1.0f, 1.0f));
    return make_float2(reciprocal(d.x), reciprocal(d.y));
}

// The argument z for which act(y) is y / (1 + e^-z), or 1 / (1 + e^-z) for the sigmoid.
template <int ACT>
__device__ __forceinline__ float2 logistic_argument(float2 y) {
    // y/2 (1 + tanh u) = y / (1 + e^-2u): no cancellation for negative u; 2u = 2 sqrt(2/pi) (y + 0.044715 y^3)
    if constexpr (ACT == KDA_ACT_GELU_TANH)
        return mul2(y, fma2(mul2(y, y), make_float2(0.0713548163f, 0.0713548163f), make_float2(1.5957691216f, 1.5957691216f)));
    return y;
}
__device__ __forceinline__ float2 relu2(float2 y) { return make_float2(y.x < 0.0f ? 0.0f : y.x, y.y < 0.0f ? 0.0f : y.y); }
template <int ACT>
__device__ __forceinline__ float2 activate2(float2 y) {
    if constexpr (ACT == KDA_ACT_NONE) return y;
    if constexpr (ACT == KDA_ACT_RELU) return relu2(y);
    const float2 l = logistic2(logistic_argument<ACT>(y));
    return ACT == KDA_ACT_SIGMOID ? l : mul2(y, l);
}

// Programmatic dependent launch: these kernels let the next one in the stream
// start its set-up while they run, and wait for everything before them ahead
// of their first access to global memory. What they read may thus be written
// while they already run, as no memory of the read-only path may: they use
// ordinary loads (and the async proxy) throughout.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace kda
