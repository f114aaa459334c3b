// A block's output joins the stream, and the sum is normed for the next block, in one pass over the rows.
//
//   b = x, or n(x) (u + offset);   s = residual + scale * gate * b;   y = n(s) (w + offset) + bias
//   n(v) = (v - mean) * rsqrt(mean((v - mean)^2) + eps), without the mean unless it is asked for
//
// A row's numbers stay in fp32 registers from their load to the two stores, so every input is read once; sums go by shuffles and,
// where a row has several warps, through shared memory.  The mean square is taken of what is left after the mean, not as a
// difference of sums.  y is made of the sum before its rounding.
//
// Bound by HBM: 4096 x 8192 bf16 with a bf16 residual 40.9 us, 6.56 TB/s (the measured copy rate is 6.56); fp32 residual 60 us, 6.7.
// What costs: asking for the residual only after x has been used (54 us), weights kept in registers from the start (68, fewer
// rows on an SM) or asked for by prefetches (515 x 5000 with all there is 12.3 us, without 9.6).
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

// How rows are read and written.
//   WHOLE     they allow 16-byte accesses; 8 neighbours a piece
//   SHIFTED   they are not multiples of 8 numbers, but all tensors lie row behind row, so that number L of one (counted over all
//             rows) is aligned where L is a multiple of 8, whatever its type: pieces begin there.  Those at a row's ends are loaded
//             with the neighbour's numbers, which are then taken as 0, and stored number by number
//   SINGLE    neither; a piece is 8 numbers that lie `step` apart
enum Rows { WHOLE, SHIFTED, SINGLE };

template <bool WIDE>
struct Raw {
    uint32_t w[WIDE ? 8 : 4];
};
// 8 numbers of a row as they lie in memory; `hidden` is where the row ends, or, of shifted ones, the last row
template <bool WIDE, int ROWS>
__device__ __forceinline__ Raw<WIDE> load_raw(const char *row, int at, int step, int hidden) {
    Raw<WIDE> r;
    if (ROWS == WHOLE || (ROWS == SHIFTED && at + 8 <= hidden)) {
        const uint4 *from = reinterpret_cast<const uint4 *>(row + (int64_t)at * (WIDE ? 4 : 2));
#pragma unroll
        for (int i = 0; i < (WIDE ? 2 : 1); ++i) {
            const uint4 v = from[i];
            r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = at + i * step;
            const bool there = c < hidden;
            if (WIDE) {
                r.w[i] = there ? reinterpret_cast<const uint32_t *>(row)[c] : 0u;
            } else {
                const uint32_t h = there ? reinterpret_cast<const uint16_t *>(row)[c] : 0u;
                r.w[i / 2] = i & 1 ? r.w[i / 2] | h << 16 : h;
            }
        }
    }
    return r;
}
template <bool WIDE, bool BF16>
__device__ __forceinline__ void open_raw(const Raw<WIDE> &r, float (&f)[8]) {
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(r.w[i]);
    } else {
        open16<BF16>(make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]), f);
    }
}
template <bool BF16, int ROWS>
__device__ __forceinline__ void load8(const char *row, bool wide, int at, int step, int hidden, float (&f)[8]) {
    if (wide) open_raw<true, BF16>(load_raw<true, ROWS>(row, at, step, hidden), f);
    else open_raw<false, BF16>(load_raw<false, ROWS>(row, at, step, hidden), f);
}
// ... of a weight, which is one row.  A piece of a shifted row begins anywhere in it: two aligned loads of 16-bit numbers, from
// whose 16 the 8 are taken by shifts of four, two and one (by as many as for all threads of the row).
template <bool BF16, int ROWS>
__device__ __forceinline__ void load_weight(const char *row, bool wide, int at, int step, int hidden, float (&f)[8]) {
    if (ROWS != SHIFTED) return load8<BF16, ROWS>(row, wide, at, step, hidden, f);
    const int off = at & 7, from = at - off;   // (from is a multiple of 8)
    if (!wide && from >= 0 && from + 16 <= hidden) {
        const uint4 a = *reinterpret_cast<const uint4 *>(row + from * 2), b = *reinterpret_cast<const uint4 *>(row + from * 2 + 16);
        uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = off & 4 ? w[i + 2] : w[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = off & 2 ? w[i + 1] : w[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = off & 1 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
        open16<BF16>(make_uint4(w[0], w[1], w[2], w[3]), f);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = at + i;
        f[i] = c < 0 || c >= hidden ? 0.f : wide ? reinterpret_cast<const float *>(row)[c] : from16(reinterpret_cast<const uint16_t *>(row)[c], BF16);
    }
}
template <bool BF16, int ROWS>
__device__ __forceinline__ void store8(char *row, bool wide, int at, int step, int hidden, const float (&f)[8]) {
    if (ROWS == WHOLE || (ROWS == SHIFTED && at >= 0 && at + 8 <= hidden)) {
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
            if (c >= hidden || (ROWS == SHIFTED && c < 0)) continue;
            if (wide) reinterpret_cast<float *>(row)[c] = f[i];
            else reinterpret_cast<uint16_t *>(row)[c] = (uint16_t)close2<BF16>(f[i], 0.f);
        }
    }
}

enum Stream { NO_STREAM, SAME_STREAM, WIDE_STREAM };   // the residual: none, of the type of x, fp32

// V: pieces of 8 numbers a thread.  ONE: a row is a warp's, 8 rows a CTA; else a CTA's of up to MAX threads.  FULL: there may be a
// norm in front, a gate, a bias, a mean to take out; without, registers are left for more rows on an SM.
template <int V, bool BF16, int ROWS, int RESIDUAL, bool FULL, bool ONE, int MAX, int MIN>
__global__ void __launch_bounds__(MAX, MIN) residual_norm_kernel(const NormParams p) {
    constexpr bool WIDE = RESIDUAL == WIDE_STREAM;
    __shared__ float part[ONE ? 1 : 4][32];   // the sums of a row, each in a place of its own: no barrier between reading one and writing the next
    const int tid = ONE ? threadIdx.x & 31 : threadIdx.x, threads = ONE ? 32 : blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = threads >> 5;
    wait_for_front();
    const int64_t token = ONE ? (int64_t)blockIdx.x * 8 + warp : blockIdx.x;
    if (ONE && token >= p.tokens) return;
    const char *x = p.x + token * p.x_stride * 2;
    const char *residual = p.residual + token * p.residual_stride * (WIDE ? 4 : 2);
    const char *gate = FULL && p.gate ? p.gate + token * p.gate_stride * (p.wide & ATLAS_WIDE_GATE ? 4 : 2) : nullptr;
    // piece v of a thread: 8 neighbours, or 8 numbers `threads` apart
    const int step = ROWS == SINGLE ? threads : 1, shift = ROWS == SHIFTED ? (int)(token * p.hidden & 7) : 0;
    auto place = [&](int v) { return ROWS == SINGLE ? v * 8 * threads + tid : (v * threads + tid) * 8 - shift; };
    auto there = [&](int v, int i) { return place(v) + (ROWS == WHOLE ? 0 : i * step) < p.hidden && (ROWS != SHIFTED || place(v) + i >= 0); };
    auto any = [&](int v) { return place(v) < p.hidden; };
    const int end = ROWS == SHIFTED ? (int)min((p.tokens - token) * p.hidden, (int64_t)1 << 30) : p.hidden;   // of what may be loaded

    auto sum_of = [&](float mine, int slot) {
#pragma unroll
        for (int k = 16; k; k /= 2) mine += __shfl_xor_sync(0xffffffffu, mine, k);
        if (ONE || warps == 1) return mine;
        float (&to)[32] = part[ONE ? 0 : slot];
        if (lane == 0) to[warp] = mine;
        __syncthreads();
        mine = lane < warps ? to[lane] : 0.f;
#pragma unroll
        for (int k = 16; k; k /= 2) mine += __shfl_xor_sync(0xffffffffu, mine, k);
        return mine;
    };
    float f[V][8];
    auto norm = [&](int slot) {   // f becomes n(f) but for the factor that is returned
        if (FULL && p.centered) {
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

    auto only_the_row = [&](int v) {
        if (ROWS == SHIFTED && (place(v) < 0 || place(v) + 8 > p.hidden))
#pragma unroll
            for (int i = 0; i < 8; ++i) f[v][i] = there(v, i) ? f[v][i] : 0.f;
    };
    // everything that is read once is asked for before anything is used (weights come from L2 or L1)
    Raw<false> raw[V], raw_gate[V];
    Raw<WIDE> old[V];
    auto ask = [&](Raw<false> (&to)[V], const char *from) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (any(v)) to[v] = load_raw<false, ROWS>(from, place(v), step, end);
    };
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[v].w[i] = 0u;
    ask(raw, x);
    if (RESIDUAL) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (any(v)) old[v] = load_raw<WIDE, ROWS>(residual, place(v), step, end);
    }
    const bool early_gate = V <= 2 && gate && !(p.wide & ATLAS_WIDE_GATE);
    if (early_gate) ask(raw_gate, gate);
#pragma unroll
    for (int v = 0; v < V; ++v) open_raw<false, BF16>(raw[v], f[v]), only_the_row(v);
    if (FULL && p.post_weight) {
        const float r = norm(0);
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (any(v)) {
                float w[8];
                load_weight<BF16, ROWS>(p.post_weight, p.wide & ATLAS_WIDE_POST_WEIGHT, place(v), step, p.hidden, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] *= r * (w[i] + p.offset);
            }
    }
    if (gate) {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (any(v)) {
                float g[8];
                if (early_gate) open_raw<false, BF16>(raw_gate[v], g);
                else load8<BF16, ROWS>(gate, p.wide & ATLAS_WIDE_GATE, place(v), step, end, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] *= g[i];
            }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (any(v)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[v][i] *= p.scale;
            if (RESIDUAL) {
                float g[8];
                open_raw<WIDE, BF16>(old[v], g);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] += g[i];
            }
            only_the_row(v);   // (whatever the gate made of the others)
            if (p.stream_out) store8<BF16, ROWS>(p.stream_out + token * p.hidden * (WIDE ? 4 : 2), WIDE, place(v), step, p.hidden, f[v]);
        }
    const float r = norm(2);
    char *out = p.normed + token * p.hidden * 2;
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (any(v)) {
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[v][i] *= r;
            if (p.weight) {
                load_weight<BF16, ROWS>(p.weight, p.wide & ATLAS_WIDE_WEIGHT, place(v), step, p.hidden, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] *= w[i] + p.offset;
            }
            if (FULL && p.bias) {
                load_weight<BF16, ROWS>(p.bias, p.wide & ATLAS_WIDE_BIAS, place(v), step, p.hidden, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) f[v][i] += w[i];
            }
            store8<BF16, ROWS>(out, false, place(v), step, p.hidden, f[v]);
        }
}

template <int V, bool BF16, int ROWS, bool FULL, bool ONE, int MAX, int MIN>
int launch_as(const NormParams &p, int threads, cudaStream_t st, const char *what) {
    const dim3 grid((unsigned)(ONE ? ceil_div_i64(p.tokens, 8) : p.tokens));
    // (four pieces with fp32 residuals do not fit 64 registers: 4096 x 8192 65.8 us with spills, 61.6 with half as many CTAs)
    constexpr int WIDE_MIN = V == 4 && !ONE ? 1 : MIN;
    constexpr bool WIDE = !(ONE && V == 4);   // (by_pieces has no fp32 residual in four pieces of a warp)
    return !p.residual ? launch_early(residual_norm_kernel<V, BF16, ROWS, NO_STREAM, FULL, ONE, MAX, MIN>, grid, threads, 0, st, what, p)
           : WIDE && (p.wide & ATLAS_WIDE_STREAM)
               ? launch_early(residual_norm_kernel<V, BF16, ROWS, WIDE ? WIDE_STREAM : SAME_STREAM, FULL, ONE, MAX, WIDE_MIN>, grid, threads, 0, st, what, p)
               : launch_early(residual_norm_kernel<V, BF16, ROWS, SAME_STREAM, FULL, ONE, MAX, MIN>, grid, threads, 0, st, what, p);
}
bool full(const NormParams &p) { return p.post_weight || p.gate || p.bias || p.centered; }
template <int V, bool BF16, int ROWS, bool ONE, int MAX, int MIN>
int launch(const NormParams &p, int threads, cudaStream_t st, const char *what) {
    return full(p) ? launch_as<V, BF16, ROWS, true, ONE, MAX, MIN>(p, threads, st, what)
                                                           : launch_as<V, BF16, ROWS, false, ONE, MAX, MIN>(p, threads, st, what);
}
// Pieces of 8 numbers a thread, and rows a CTA.  Few rows: one piece, so that a row has the most threads (1 x 4096 1.9 us, with two
// pieces 2.1, with four 2.6).  Many: two, as soon as the CTAs no longer fit all at once (300 x 8192 4.6, 3.9, 4.7; 4096 x 8192 44.7,
// 40.9, 41.5; with fp32 residuals 60.0, 60.1, 65.8), four for wide rows without a residual (37, 26.7, 24.8).
// Many short rows: a warp each, up to 512 numbers, or up to 768 from 4096 rows on where the stream has 16 bits.  Time of a warp over
// that of a CTA (140 to 350 MB a pass; fp16; without a residual / a residual / all there is / all there is, fp32 stream):
//   20000 x 128 .27 .29 .48 .54    8192 x 256 .41 .48 .72 .86    2048 x 512 .94 .97 1.03 1.07   1184 x 512 .92 .93 1.00 1.07
//   20000 x 768 .74 .92 1.07 1.22  4096 x 768 .91 .94 .95 1.12   2048 x 768 .99 .96 1.15 1.26   1184 x 768 1.00 1.04 1.37 1.38
//   20000 x 1024 .95 1.02 1.23 1.35  4096 x 999 1.06 1.17 1.10 1.19   1184 x 999 1.25 1.26 1.59 1.64
// With gates, biases, means or norms in front, rows that do not all fit at once in CTAs of 64 registers a thread, but do in CTAs of
// 48, go there at the price of spills.  Time of the latter over that of the former (a norm in front / all, fp32 stream):
//   515 x 5001 .72 .78   592 x 5104 .79 .88   620 x 4096 .82 .90   740 x 4096 .79 .88    fewer rows: 444 x 5001 1.07 1.11
//   444 x 4096 1.07 1.23    more: 680 x 5104 1.00 1.18   900 x 4096 1.02 1.18
template <bool BF16, int ROWS>
int by_pieces(const NormParams &p, cudaStream_t st, const char *what) {
    const int pieces = (p.hidden + (ROWS == SHIFTED ? 14 : 7)) / 8;
    auto threads = [&](int v) { return (pieces + v * 32 - 1) / (v * 32) * 32; };
    if (p.tokens >= 8 * 148 && (pieces <= 64 || (pieces <= 96 && p.tokens >= 4096 && !(p.wide & ATLAS_WIDE_STREAM))))
        return pieces <= 32 ? launch<1, BF16, ROWS, true, 256, 4>(p, 256, st, what)
               : pieces <= 64 ? launch<2, BF16, ROWS, true, 256, 4>(p, 256, st, what) : launch<4, BF16, ROWS, true, 256, 4>(p, 256, st, what);
    if (p.tokens < 2 * 148 && pieces <= 1024) return launch<1, BF16, ROWS, false, 1024, 1>(p, threads(1), st, what);
    const int two = threads(2);
    if (full(p) && pieces <= 640 && p.tokens <= 5 * 148 && p.tokens > 148 * (1024 / two) && p.tokens <= 148 * (1344 / two))
        return launch_as<2, BF16, ROWS, true, false, 320, 4>(p, two, st, what);
    if (pieces <= 1024 && (p.residual || pieces <= 512)) return launch<2, BF16, ROWS, false, 512, 2>(p, threads(2), st, what);
    return pieces <= 2048 ? launch<4, BF16, ROWS, false, 512, 2>(p, threads(4), st, what) : launch<4, BF16, ROWS, false, 1024, 1>(p, threads(4), st, what);
}
template <bool BF16>
int by_rows(const NormParams &p, Rows rows, cudaStream_t st, const char *what) {
    return rows == WHOLE ? by_pieces<BF16, WHOLE>(p, st, what) : rows == SHIFTED ? by_pieces<BF16, SHIFTED>(p, st, what) : by_pieces<BF16, SINGLE>(p, st, what);
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
    uintptr_t typed = 0, apart = 0;   // addresses and strides: what they lack of multiples of their types, of 16 bytes
    bool behind = true;               // rows lie behind one another
    auto look = [&](const void *a, int size, bool rows, int64_t stride) {
        if (!a) return;
        typed |= (uintptr_t)a & (uintptr_t)(size - 1);
        apart |= (uintptr_t)a & 15;
        if (!rows || q->tokens == 1) return;
        behind = behind && stride == q->hidden;
        if (stride * size & 15) apart |= 16;
    };
    look(q->x, 2, true, q->x_stride), look(q->normed, 2, true, q->hidden), look(q->stream_out, bytes(ATLAS_WIDE_STREAM), true, q->hidden);
    look(q->residual, bytes(ATLAS_WIDE_STREAM), true, q->residual_stride), look(q->gate, bytes(ATLAS_WIDE_GATE), q->gate_stride != 0, q->gate_stride);
    look(q->weight, bytes(ATLAS_WIDE_WEIGHT), false, 0), look(q->bias, bytes(ATLAS_WIDE_BIAS), false, 0);
    look(q->post_weight, bytes(ATLAS_WIDE_POST_WEIGHT), false, 0);
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
    const bool shifted = !(apart & 15) && behind && (q->gate_stride || !q->gate) && (q->hidden + 14) / 8 <= ATLAS_NORM_MAX_HIDDEN / 8;
    const Rows rows = !apart && q->hidden % 8 == 0 ? WHOLE : shifted ? SHIFTED : SINGLE;
    return q->dtype == ATLAS_DTYPE_BF16 ? by_rows<true>(p, rows, (cudaStream_t)stream, what) : by_rows<false>(p, rows, (cudaStream_t)stream, what);
}
