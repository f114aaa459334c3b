// A block's output joins the stream, and the sum is normed for the next block, in one pass over the rows.
//
//   b = x, or n(x) (u + offset);   s = residual + scale * gate * b;   y = n(s) (w + offset) + bias
//   n(v) = (v - mean) * rsqrt(mean((v - mean)^2) + eps), without the mean unless it is asked for
//
// A row's numbers stay in fp32 registers from their load to the two stores, V pieces of 8 a thread, so every input is read
// once; sums go by shuffles and, where a row has several warps, through shared memory.  The mean square is taken of what is left
// after the mean, not as a difference of sums.  y is made of the sum before its rounding.
#include "rows.cuh"

namespace atlas {
namespace {

struct NormParams {
    const char *x, *residual, *gate, *weight, *bias, *post_weight;
    char *normed, *stream_out;
    int64_t x_stride, residual_stride, gate_stride;   // elements
    int64_t tokens;
    int hidden, wide;
    float scale, eps, offset, inverse_hidden;
    bool centered;
};

// 8 numbers of a row of `hidden` from `at`; in a row that allows no 16-byte loads they lie `step` apart.
template <bool BF16, bool VEC>
__device__ __forceinline__ void load8(const char *row, bool wide, int at, int step, int hidden, float (&f)[8]) {
    if (VEC) {
        if (wide) {
            const float4 a = *reinterpret_cast<const float4 *>(row + (int64_t)at * 4), b = *reinterpret_cast<const float4 *>(row + (int64_t)at * 4 + 16);
            f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
        } else {
            open16<BF16>(*reinterpret_cast<const uint4 *>(row + (int64_t)at * 2), f);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = at + i * step;
            f[i] = c >= hidden ? 0.f : wide ? reinterpret_cast<const float *>(row)[c] : from16(reinterpret_cast<const uint16_t *>(row)[c], BF16);
        }
    }
}
template <bool BF16, bool VEC>
__device__ __forceinline__ void store8(char *row, bool wide, int at, int step, int hidden, const float (&f)[8]) {
    if (VEC) {
        if (wide) {
            *reinterpret_cast<float4 *>(row + (int64_t)at * 4) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4 *>(row + (int64_t)at * 4 + 16) = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4 *>(row + (int64_t)at * 2) =
                make_uint4(close2<BF16>(f[0], f[1]), close2<BF16>(f[2], f[3]), close2<BF16>(f[4], f[5]), close2<BF16>(f[6], f[7]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = at + i * step;
            if (c >= hidden) continue;
            if (wide) reinterpret_cast<float *>(row)[c] = f[i];
            else reinterpret_cast<uint16_t *>(row)[c] = (uint16_t)close2<BF16>(f[i], 0.f);
        }
    }
}

// A row is a CTA's.  V: pieces of 8 numbers a thread.
template <int V, bool BF16, bool VEC>
__global__ void __launch_bounds__(1024) residual_norm_kernel(const NormParams p) {
    __shared__ float part[4][32];   // the sums of a row, each in a place of its own: no barrier between reading one and writing the next
    const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
    wait_for_front();
    const int64_t token = blockIdx.x;
    const char *x = p.x + token * p.x_stride * 2;
    const bool wide_stream = p.wide & ATLAS_WIDE_STREAM;
    const char *residual = p.residual ? p.residual + token * p.residual_stride * (wide_stream ? 4 : 2) : nullptr;
    const char *gate = p.gate ? p.gate + token * p.gate_stride * (p.wide & ATLAS_WIDE_GATE ? 4 : 2) : nullptr;
    // piece v of a thread: 8 neighbours, or 8 numbers `threads` apart
    auto place = [&](int v) { return VEC ? (v * threads + tid) * 8 : v * 8 * threads + tid; };
    auto there = [&](int v, int i) { return (VEC ? place(v) : place(v) + i * threads) < p.hidden; };

    auto sum_of = [&](float mine, int slot) {
#pragma unroll
        for (int k = 16; k; k /= 2) mine += __shfl_xor_sync(0xffffffffu, mine, k);
        if (warps == 1) return mine;
        if (lane == 0) part[slot][warp] = mine;
        __syncthreads();
        mine = lane < warps ? part[slot][lane] : 0.f;
#pragma unroll
        for (int k = 16; k; k /= 2) mine += __shfl_xor_sync(0xffffffffu, mine, k);
        return mine;
    };
    float f[V][8];
    auto norm = [&](int slot) {   // f becomes n(f) but for the factor that is returned
        if (p.centered) {
            float sum = 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += f[v][i];
            const float mean = sum_of(sum, slot) * p.inverse_hidden;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] = there(v, i) ? f[v][i] - mean : 0.f;
        }
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += f[v][i] * f[v][i];
        return rsqrtf(sum_of(sum, slot + 1) * p.inverse_hidden + p.eps);
    };

#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[v][i] = 0.f;
        if (there(v, 0)) load8<BF16, VEC>(x, false, place(v), threads, p.hidden, f[v]);
    }
    if (p.post_weight) {
        const float r = norm(0);
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (there(v, 0)) {
                float w[8];
                load8<BF16, VEC>(p.post_weight, p.wide & ATLAS_WIDE_POST_WEIGHT, place(v), threads, p.hidden, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] *= r * (w[i] + p.offset);
            }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (there(v, 0)) {
            float g[8];
            if (gate) {
                load8<BF16, VEC>(gate, p.wide & ATLAS_WIDE_GATE, place(v), threads, p.hidden, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] *= g[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) f[v][i] *= p.scale;
            if (residual) {
                load8<BF16, VEC>(residual, wide_stream, place(v), threads, p.hidden, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] += g[i];
            }
            if (p.stream_out) store8<BF16, VEC>(p.stream_out + token * p.hidden * (wide_stream ? 4 : 2), wide_stream, place(v), threads, p.hidden, f[v]);
        }
    const float r = norm(2);
    char *out = p.normed + token * p.hidden * 2;
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (there(v, 0)) {
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[v][i] *= r;
            if (p.weight) {
                load8<BF16, VEC>(p.weight, p.wide & ATLAS_WIDE_WEIGHT, place(v), threads, p.hidden, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] *= w[i] + p.offset;
            }
            if (p.bias) {
                load8<BF16, VEC>(p.bias, p.wide & ATLAS_WIDE_BIAS, place(v), threads, p.hidden, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] += w[i];
            }
            store8<BF16, VEC>(out, false, place(v), threads, p.hidden, f[v]);
        }
}

template <int V, bool BF16>
int launch(const NormParams &p, bool vec, int threads, cudaStream_t st, const char *what) {
    return vec ? launch_early(residual_norm_kernel<V, BF16, true>, dim3((unsigned)p.tokens), threads, 0, st, what, p)
               : launch_early(residual_norm_kernel<V, BF16, false>, dim3((unsigned)p.tokens), threads, 0, st, what, p);
}
template <bool BF16>
int by_pieces(const NormParams &p, bool vec, cudaStream_t st, const char *what) {
    const int pieces = (p.hidden + 7) / 8;
    const int v = pieces <= 1024 ? 1 : pieces <= 2048 ? 2 : 4;
    const int threads = (pieces + v * 32 - 1) / (v * 32) * 32;
    return v == 1 ? launch<1, BF16>(p, vec, threads, st, what) : v == 2 ? launch<2, BF16>(p, vec, threads, st, what) : launch<4, BF16>(p, vec, threads, st, what);
}

}  // namespace
}  // namespace atlas

extern "C" int atlas_residual_norm(const AtlasResidualNorm *q, void *stream) {
    using namespace atlas;
    clear_error();
    const char *what = "atlas_residual_norm";
    ATLAS_RETURN_IF(!q, ATLAS_ERR_BAD_ARGUMENT, "%s: no arguments", what);
    ATLAS_RETURN_IF(q->dtype != ATLAS_DTYPE_F16 && q->dtype != ATLAS_DTYPE_BF16, ATLAS_ERR_BAD_ARGUMENT, "%s: dtype %d", what, q->dtype);
    ATLAS_RETURN_IF(q->tokens < 0 || q->hidden < 1, ATLAS_ERR_BAD_ARGUMENT, "%s: %lld tokens of %lld", what, (long long)q->tokens, (long long)q->hidden);
    ATLAS_RETURN_IF(q->hidden > ATLAS_NORM_MAX_HIDDEN, ATLAS_ERR_UNSUPPORTED, "%s: hidden %lld is more than %d", what, (long long)q->hidden, ATLAS_NORM_MAX_HIDDEN);
    ATLAS_RETURN_IF(q->tokens > 0x7fffffff, ATLAS_ERR_UNSUPPORTED, "%s: %lld tokens", what, (long long)q->tokens);
    if (q->tokens == 0) return ATLAS_OK;
    ATLAS_RETURN_IF(!q->x || !q->normed, ATLAS_ERR_BAD_ARGUMENT, "%s: null pointer", what);
    const int wide = q->residual ? q->wide : q->wide & ~ATLAS_WIDE_STREAM;
    auto bytes = [&](int bit) { return wide & bit ? 4 : 2; };
    uintptr_t typed = 0, whole = q->hidden % 8 ? 1 : 0;   // addresses and strides: multiples of their types, of 16 bytes
    auto look = [&](const void *a, int size, int64_t stride) {
        if (!a) return;
        typed |= (uintptr_t)a & (uintptr_t)(size - 1);
        whole |= ((uintptr_t)a | (uintptr_t)(q->tokens > 1 ? stride * size : 0)) & 15;
    };
    look(q->x, 2, q->x_stride), look(q->normed, 2, 0), look(q->stream_out, bytes(ATLAS_WIDE_STREAM), 0);
    look(q->residual, bytes(ATLAS_WIDE_STREAM), q->residual_stride), look(q->gate, bytes(ATLAS_WIDE_GATE), q->gate_stride);
    look(q->weight, bytes(ATLAS_WIDE_WEIGHT), 0), look(q->bias, bytes(ATLAS_WIDE_BIAS), 0), look(q->post_weight, bytes(ATLAS_WIDE_POST_WEIGHT), 0);
    ATLAS_RETURN_IF(typed, ATLAS_ERR_BAD_ARGUMENT, "%s: a buffer is not aligned to its type", what);
    const int dev = check_device();
    if (dev != ATLAS_OK) return dev;
    NormParams p = {};
    p.x = (const char *)q->x, p.residual = (const char *)q->residual, p.gate = (const char *)q->gate;
    p.weight = (const char *)q->weight, p.bias = (const char *)q->bias, p.post_weight = (const char *)q->post_weight;
    p.normed = (char *)q->normed, p.stream_out = (char *)q->stream_out;
    p.x_stride = q->x_stride, p.residual_stride = q->residual_stride, p.gate_stride = q->gate_stride;
    p.tokens = q->tokens, p.hidden = (int)q->hidden, p.wide = wide;
    p.scale = q->scale, p.eps = q->eps, p.offset = q->weight_offset, p.inverse_hidden = 1.0f / (float)q->hidden;
    p.centered = q->centered != 0;
    return q->dtype == ATLAS_DTYPE_BF16 ? by_pieces<true>(p, !whole, (cudaStream_t)stream, what) : by_pieces<false>(p, !whole, (cudaStream_t)stream, what);
}
