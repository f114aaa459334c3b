// Numbers in 16 bits as fp32 and back, one, two and eight at a time.
#pragma once
#include "kv_cache.cuh"

namespace atlas {
namespace {

__device__ __forceinline__ float from16(uint16_t h, bool bf16) {
    return bf16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
}
template <bool BF16>
__device__ __forceinline__ void open16(const uint4 &v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (BF16) {
            f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            f[2 * i] = p.x, f[2 * i + 1] = p.y;
        }
    }
}
template <bool BF16>
__device__ __forceinline__ uint32_t close2(float lo, float hi) {
    if (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

}  // namespace
}  // namespace atlas
