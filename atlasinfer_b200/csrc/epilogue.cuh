// What a quantized linear does with a finished sum before it rounds it, once, to its output's type.
//
//   y = residual + scale * act(x W^T + bias)             one weight
//   y = residual + scale * act(x W^T + bias) * (x V^T + c)     two of one shape (gate and up)
//
// in fp32.  Exponentials and reciprocals are the approximate instructions: 2^-21 relative for small arguments, and as the exponent's
// argument is rounded, up to 2^-23 more for every unit that it is away from 0 (silu(-80) is off by 2^-18.5, gelu(-12), whose
// argument is -72, by 2^-17).  That is nothing beside the rounding to 11 or 8 bits that follows.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "atlas_b200.h"

namespace atlas {

struct Epilogue {
    const uint16_t *residual = nullptr;   // [m][n], of the output's type
    int64_t ldr = 0;
    float scale = 1.0f;
    int act = 0;                          // ATLAS_ACT_*
    bool residual_by_4 = false;           // 4 neighbours of a row that begin at a multiple of 4 lie on 8 bytes
};
inline Epilogue make_epilogue(const void *residual, int64_t ldr, float scale, int act) {
    Epilogue e;
    e.residual = (const uint16_t *)residual;
    e.ldr = ldr, e.scale = scale, e.act = act;
    e.residual_by_4 = ((uintptr_t)residual & 7) == 0 && ldr % 4 == 0;
    return e;
}
inline bool is_plain(const Epilogue &e) { return !e.residual && e.scale == 1.0f && e.act == ATLAS_ACT_NONE; }

namespace {

// 1 / (1 + 2^t): 1 below, 0 above; a NaN stays one.
__device__ __forceinline__ float logistic(float t) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}
// v Phi(v) by the smaller of the normal distribution's two tails: Phi(-a) = exp(-a^2 / 2) g(t), t = 1 / (1 + 0.3 a), where g is
// smooth and a polynomial of degree 8 without a constant term is within 1.7e-7 of it, relatively, for a up to 14.5 (fitted to the
// scaled complementary error function by weighted least squares, weights raised where the error is largest: Lawson 1961).  So
// small results keep their digits, which 1 + erf(v / sqrt 2) would lose; erfcf takes three times as long (2048 tokens of
// 11008 outputs: 36 us more).
__device__ __forceinline__ float gelu(float v) {
    const float a = fabsf(v);
    float t, e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.3f, a, 1.0f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(a * (-0.72134752f * a)));
    float g = 0.035423826426f;
    g = fmaf(g, t, -0.156158789992f);
    g = fmaf(g, t, 0.204557314515f);
    g = fmaf(g, t, -0.052034448832f);
    g = fmaf(g, t, 0.127691969275f);
    g = fmaf(g, t, 0.100175894797f);
    g = fmaf(g, t, 0.120712146163f);
    g = fmaf(g, t, 0.119632005692f);
    const float tail = g * t * e;
    return v * (v < 0.0f ? tail : 1.0f - tail);
}
template <int ACT>
__device__ __forceinline__ float activated(float v) {
    if (ACT == ATLAS_ACT_RELU) {
        float r;
        asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(v));   // (NaN stays)
        return r;
    }
    if (ACT == ATLAS_ACT_SILU) return v * logistic(-1.44269504f * v);
    if (ACT == ATLAS_ACT_GELU) return gelu(v);
    if (ACT == ATLAS_ACT_GELU_TANH)   // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)), u = sqrt(2 / pi) (v + 0.044715 v^3)
        return v * logistic(v * (-2.30220821f - 0.10294324f * (v * v)));
    return v;
}
template <int ACT, int N>
__device__ __forceinline__ void activate_with(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = activated<ACT>(v[i]);
}
// (one branch for all N, so that the code of an activation stands there once)
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
    switch (act) {
        case ATLAS_ACT_RELU: activate_with<ATLAS_ACT_RELU>(v); break;
        case ATLAS_ACT_SILU: activate_with<ATLAS_ACT_SILU>(v); break;
        case ATLAS_ACT_GELU: activate_with<ATLAS_ACT_GELU>(v); break;
        case ATLAS_ACT_GELU_TANH: activate_with<ATLAS_ACT_GELU_TANH>(v); break;
    }
}
__device__ __forceinline__ float widen(uint16_t bits, bool bf16) {
    return bf16 ? __uint_as_float((uint32_t)bits << 16) : __half2float(__ushort_as_half(bits));
}
__device__ __forceinline__ uint16_t narrow(float v, bool bf16) {
    return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ float residual_at(const Epilogue &e, int64_t row, int n, bool bf16) {
    return e.residual ? widen(__ldg(e.residual + row * e.ldr + n), bf16) : 0.0f;
}
// Those of n .. n + 3 (n is a multiple of 4), of which the first `count` exist.
__device__ __forceinline__ void residual_at(const Epilogue &e, int64_t row, int n, int count, bool bf16, float (&r)[4]) {
    if (e.residual_by_4 && count >= 4) {
        const uint2 v = e.residual ? __ldg(reinterpret_cast<const uint2 *>(e.residual + row * e.ldr + n)) : make_uint2(0, 0);
        r[0] = widen((uint16_t)v.x, bf16), r[1] = widen((uint16_t)(v.x >> 16), bf16), r[2] = widen((uint16_t)v.y, bf16), r[3] = widen((uint16_t)(v.y >> 16), bf16);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = i < count ? residual_at(e, row, n + i, bf16) : 0.0f;
    }
}
// What follows the activation: `residual` is what residual_at gave.  (Without an epilogue the bits stay as they are.)
__device__ __forceinline__ float scaled(const Epilogue &e, float v, float residual) {
    v *= e.scale;
    return e.residual ? v + residual : v;
}
template <int N>
__device__ __forceinline__ void scale_and_add(const Epilogue &e, float (&v)[N], const float (&residual)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = scaled(e, v[i], residual[i]);
}

}  // namespace
}  // namespace atlas
