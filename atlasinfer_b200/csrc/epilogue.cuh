// What a quantized linear does with a finished sum before it rounds it, once, to its output's type.
//
//   y = residual + scale * act(x W^T + bias)             one weight
//   y = residual + scale * act(x W^T + bias) * (x V^T + c)     two of one shape (gate and up)
//
// in fp32.  The exponentials are the fast ones (2^-21 relative over the range where the result is not 0 or x), which is
// nothing beside the rounding to 11 or 8 bits that follows.
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
};

namespace {

template <int ACT>
__device__ __forceinline__ float activated(float v) {
    if (ACT == ATLAS_ACT_RELU) return v < 0.0f ? 0.0f : v;   // (NaN stays)
    if (ACT == ATLAS_ACT_SILU) return __fdividef(v, 1.0f + __expf(-v));
    if (ACT == ATLAS_ACT_GELU) return 0.5f * v * erfcf(-0.70710678f * v);
    if (ACT == ATLAS_ACT_GELU_TANH) {   // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
        const float u = 0.79788456f * (v + 0.044715f * v * v * v);
        return __fdividef(v, 1.0f + __expf(-2.0f * u));
    }
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
// What follows the activation: `residual` is what residual_at gave.  (Without an epilogue the bits stay as they are.)
__device__ __forceinline__ float scaled(const Epilogue &e, float v, float residual) {
    v *= e.scale;
    return e.residual ? v + residual : v;
}

}  // namespace
}  // namespace atlas
