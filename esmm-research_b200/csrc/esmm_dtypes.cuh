// Element types of the dense operators (esmm_rows.cu, esmm_linear.cu): conversions, activations.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "esmm_common.cuh"

namespace esmm {

constexpr float E4M3_MAX = 448.0f;
// Smallest amax that a row's or column's scale is made from: scales stay normal numbers whatever the row holds (a row of zeros
// has the scale 2^-100 / 448 and codes of zero), and 448 / amax does not overflow.
constexpr float E4M3_TINY = 7.88860905e-31f;   // 2^-100

inline int dtype_bytes(int dtype)
{
    return dtype == ESMM_F32 ? 4 : dtype == ESMM_F16 || dtype == ESMM_BF16 ? 2 : dtype == ESMM_E4M3 ? 1 : 0;
}

inline bool activation_known(int a) { return a >= ESMM_ACT_NONE && a <= ESMM_ACT_SILU; }

#ifdef __CUDACC__
template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two floats as one 32-bit word of two 16-bit values, `lo` in the low half
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float2 unpack_bf16(uint32_t v)
{
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}

__device__ __forceinline__ float2 unpack_f16(uint32_t v)
{
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

// two floats as two e4m3 codes, `lo` in the low byte; finite values past +-448 saturate, NaN keeps its code
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float e4m3_to_float(uint8_t code)
{
    uint32_t halves;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"((uint16_t)code));
    return unpack_f16(halves).x;
}

__device__ __forceinline__ float e4m3_scale(float amax) { return __fdiv_rn(fmaxf(amax, E4M3_TINY), E4M3_MAX); }

// y / scale from inv = 1 / scale, with the remainder's correction: as good as the division itself, so that values next to a border
// between two codes fall where the quotient does (a scale that is infinite gives what inv = 0 gives)
__device__ __forceinline__ float e4m3_quotient(float y, float scale, float inv)
{
    const float q = y * inv;
    const float c = fmaf(fmaf(-q, scale, y), inv, q);
    return inv > 0.0f ? c : q;
}

// ---- activations -------------------------------------------------------------------------------------------------
// silu(z) = z / (1 + exp(-z)).  gelu_tanh(z) = z / 2 (1 + tanh u) = z / (1 + exp(-2 u)), u = sqrt(2 / pi) (z + 0.044715 z^3): one
// exponential and one division, and no cancellation where tanh u is near -1.
constexpr float GELU_U = 0.7978845608f, GELU_CUBE = 0.044715f;

// gelu(z) = z Phi(z) = max(z, 0) - t Q(t) with t = |z| and the normal distribution's upper tail Q = 1 - Phi, so that no digit of a negative z's value cancels (from
// 1 + erf(z / sqrt 2) it was 4 % off at z = -5 and zero from -5.6 on).  Q(t) = exp(-t^2 / 2) R(t), and R as s P(s) with s = 1 / (1 + 0.3 t): P of degree 7 fitted
// to erfcx(t / sqrt 2) / 2 on 0 .. 16 for the least relative error by reweighted least squares: 2.2e-7, 6e-7 in 32-bit arithmetic.  Past 13 Q is less than 32-bit
// floats hold.  4096 x 512 x 4096 of bf16 with gelu 38.5 us by erff, 34.2 so (77 by erfcf); its gradient 2048 x 11008 of bf16 39.2, 36.6 so.
__device__ __forceinline__ float gelu_reach(float z)                    // |z|, 16 at most (NaN stays)
{
    float t;
    asm("min.NaN.f32 %0, %1, 0f41800000;" : "=f"(t) : "f"(fabsf(z)));
    return t;
}

__device__ __forceinline__ float gelu_ratio(float t)                    // R(t)
{
    const float s = __fdividef(1.0f, fmaf(0.3f, t, 1.0f));
    float r = 0.0347048553f;
    r = fmaf(r, s, -0.153187057f);
    r = fmaf(r, s, 0.199487766f);
    r = fmaf(r, s, -0.0474263256f);
    r = fmaf(r, s, 0.125291755f);
    r = fmaf(r, s, 0.100889287f);
    r = fmaf(r, s, 0.120600532f);
    r = fmaf(r, s, 0.119639078f);
    return r * s;
}

__device__ __forceinline__ float logistic(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

template <int ACT>
__device__ __forceinline__ float activate(float z)
{
    if (ACT == ESMM_ACT_RELU) return z < 0.0f ? 0.0f : z;   // (NaN stays)
    if (ACT == ESMM_ACT_GELU) {
        const float t = gelu_reach(z);
        return fmaf(-t, __expf(-0.5f * t * t) * gelu_ratio(t), z < 0.0f ? 0.0f : z);
    }
    if (ACT == ESMM_ACT_GELU_TANH) return __fdividef(z, 1.0f + __expf(-2.0f * GELU_U * z * fmaf(GELU_CUBE * z, z, 1.0f)));
    if (ACT == ESMM_ACT_SILU) return __fdividef(z, 1.0f + __expf(-z));
    return z;
}

template <int ACT>
__device__ __forceinline__ float activate_grad(float z)
{
    if (ACT == ESMM_ACT_RELU) return z > 0.0f ? 1.0f : z <= 0.0f ? 0.0f : z;
    if (ACT == ESMM_ACT_GELU) {
        const float t = gelu_reach(z), e = __expf(-0.5f * t * t), q = e * gelu_ratio(t);
        return fmaf(copysignf(t, z), e * 0.3989422804f, z < 0.0f ? q : 1.0f - q);
    }
    if (ACT == ESMM_ACT_GELU_TANH) {
        const float z2 = fminf(z * z, 1e8f);                 // (past it the logistic function is 0 or 1 and its slope 0)
        const float s = logistic(2.0f * GELU_U * z * fmaf(GELU_CUBE, z2, 1.0f));
        return s + z * s * (1.0f - s) * (2.0f * GELU_U) * fmaf(3.0f * GELU_CUBE, z2, 1.0f);
    }
    if (ACT == ESMM_ACT_SILU) {
        const float s = logistic(z);
        return s * (1.0f + z * (1.0f - s));
    }
    return 1.0f;
}

// f(std::integral_constant<int, ACT>) of the activation that `act` names
template <int V> struct ActTag { static constexpr int value = V; };
template <typename F>
__device__ __forceinline__ void with_activation(int act, F f)
{
    switch (act) {
    case ESMM_ACT_RELU: f(ActTag<ESMM_ACT_RELU>()); break;
    case ESMM_ACT_GELU: f(ActTag<ESMM_ACT_GELU>()); break;
    case ESMM_ACT_GELU_TANH: f(ActTag<ESMM_ACT_GELU_TANH>()); break;
    case ESMM_ACT_SILU: f(ActTag<ESMM_ACT_SILU>()); break;
    default: f(ActTag<ESMM_ACT_NONE>()); break;
    }
}
#endif  // __CUDACC__

}  // namespace esmm
