// Norms and position rotation of queries and keys, and the 4-bit cache written and read token by token.
//
//   x' = x * rsqrt(mean(x^2) + eps) * (weight + offset)          over a head's D channels, if there is a weight
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t)             over the first R channels, b = a's channel + R/2, or + 1
//   keys and values, 64 channels a group: s = up7((hi - lo) / 15), z = rint(-lo / s), c = clamp(rint(x / s) + z, 0, 15)
//
// One thread holds 8 neighbouring channels of a head (16 bytes, one word of key codes, two units of value codes), D / 8
// threads a head; sums and extrema of a head or a group go by shuffles.  All of it is fp32 with products, sums and quotients
// rounded one by one, so that what is stored does not depend on how the compiler joins them; the only other roundings are
// those of the outputs, and the cache is made of the fp32 results.
//
// What bounds it: HBM in principle (4001 tokens of 72 heads of 128, 150 MB, 37 us, 4.0 TB/s, 0.62 of the measured copy rate),
// loads in flight in practice: 64 registers for 32 warps an SM with two loads each (some 100 bytes of spills); 80 registers and
// 24 warps 42 us, 48 registers and 40 warps 50, four loads ahead 43.
#include <algorithm>

#include "kv_cache.cuh"

namespace atlas {

int check_kv_shape(int64_t num_pages, int64_t kv_heads, int64_t head_dim, int64_t page_size, const char *what) {
    ATLAS_RETURN_IF(num_pages < 0 || kv_heads < 1 || kv_heads > 65535, ATLAS_ERR_BAD_ARGUMENT, "%s: %lld pages of %lld heads", what,
                    (long long)num_pages, (long long)kv_heads);
    ATLAS_RETURN_IF(head_dim != 64 && head_dim != 128 && head_dim != 256, ATLAS_ERR_UNSUPPORTED, "%s: head_dim %lld is not 64, 128 or 256", what,
                    (long long)head_dim);
    ATLAS_RETURN_IF(page_size < KV_SLAB || page_size % KV_SLAB || page_size > (1 << 20), ATLAS_ERR_UNSUPPORTED,
                    "%s: page_size %lld is not a multiple of 16 up to 2^20", what, (long long)page_size);
    return ATLAS_OK;
}

namespace {

struct Tokens {
    const char *x[3];            // q, k, v
    int64_t token_stride[3], head_stride[3];   // bytes
    char *out[2];                // q', k' (contiguous); null: not wanted
    const float *table;          // cos | sin
    const void *positions, *slots;
    const char *weight[2];
    uint8_t *cache;
    int64_t tokens, table_rows, num_slots;
    int q_heads, kv_heads, rotary, page_size;
    float eps, offset;
    bool wide_positions, wide_slots, wide_weights, interleaved;
    int steps_per_warp, parts, parts_q, parts_k;   // steps of a warp: 256 / D heads each; warps of a token, those for its queries, for its keys
};

__device__ __forceinline__ float from_bits(uint32_t v, bool high, bool bf16) {
    const uint32_t h = high ? v >> 16 : v & 0xffffu;
    return bf16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
}
template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4 &v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = from_bits(w[i / 2], i & 1, BF16);
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3]), pack2<BF16>(f[4], f[5]), pack2<BF16>(f[6], f[7]));
}
template <bool BF16>
__device__ __forceinline__ void load_weight(const char *w, bool wide, int channel, float (&f)[8]) {
    if (wide) {
        const float4 a = *reinterpret_cast<const float4 *>(w + channel * 4), b = *reinterpret_cast<const float4 *>(w + channel * 4 + 16);
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    } else {
        unpack8<BF16>(*reinterpret_cast<const uint4 *>(w + channel * 2), f);
    }
}

// x / s as fp32 rounds it, from the reciprocal as fp32 rounds it: a product, its exact remainder, a correction (Markstein 1990).
__device__ __forceinline__ float quotient(float x, float s, float inverse) {
    const float q = __fmul_rn(x, inverse);
    return __fmaf_rn(__fmaf_rn(-q, s, x), inverse, q);
}
// The integer nearest to |x| < 2^21, ties to even: it stands in the low bits of x + 1.5 * 2^23.
__device__ __forceinline__ int nearest(float x) { return __float_as_int(__fadd_rn(x, 12582912.0f)) - 0x4b400000; }

// Codes, scale and zero point of this thread's 8 channels; the 8 threads of a group hold neighbouring lanes.
__device__ __forceinline__ void quantise8(float (&x)[8], int (&code)[8], float &scale, int &zero) {
    float lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = x[i] != x[i] ? 0.0f : fminf(fmaxf(x[i], -KV_MAX_VALUE), KV_MAX_VALUE);   // (what does not fit stays finite: a
        lo = fminf(lo, x[i]);                                                            // hidden token must not spoil rows that
        hi = fmaxf(hi, x[i]);                                                            // do not see it)
    }
#pragma unroll
    for (int k = 1; k < 8; k *= 2) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, k));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, k));
    }
    const float s = quotient(__fsub_rn(hi, lo), 15.0f, 1.0f / 15.0f);
    scale = fminf(fmaxf(__int_as_float((__float_as_int(s) + 0x1ffff) & ~0x1ffff), KV_MIN_SCALE), KV_MAX_SCALE);
    const float inverse = __frcp_rn(scale);
    zero = min(nearest(quotient(-lo, scale, inverse)), 15);
#pragma unroll
    for (int i = 0; i < 8; ++i) code[i] = min(max(nearest(quotient(x[i], scale, inverse)) + zero, 0), 15);
}

template <int D>
__device__ __forceinline__ void store_key(uint8_t *slab, int token, int unit, const int (&c)[8], float scale, int zero) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= (uint32_t)c[i] << (4 * ((i & 1) * 4 + i / 2));
    *reinterpret_cast<uint32_t *>(slab + kv_key_word(D, token, unit)) = w;
    if (unit % 8 == 0)
        *reinterpret_cast<__half2 *>(slab + kv_key_params(D) + (token * (D / 64) + unit / 8) * 4) = __floats2half2_rn(scale, (float)(1024 + zero));
}
template <int D>
__device__ __forceinline__ void store_value(uint8_t *slab, int token, int unit, const int (&c)[8], float scale, int zero) {
    uint8_t *codes = slab + kv_value_codes(D);
#pragma unroll
    for (int h = 0; h < 2; ++h)
        *reinterpret_cast<uint16_t *>(codes + kv_value_unit(D, token, 2 * unit + h)) =
            (uint16_t)(c[4 * h] | c[4 * h + 1] << 4 | c[4 * h + 2] << 8 | c[4 * h + 3] << 12);
    if (unit % 8 == 0) {
        __half *p = reinterpret_cast<__half *>(slab + kv_value_params(D) + (token / 2 * (D / 64) + unit / 8) * 8) + (token & 1);
        p[0] = __float2half_rn(scale);
        p[2] = __int2half_rn(1024 + zero);
    }
}

__device__ __forceinline__ int64_t index_at(const void *p, bool wide, int64_t i) {
    return wide ? reinterpret_cast<const int64_t *>(p)[i] : reinterpret_cast<const int32_t *>(p)[i];
}

// A warp takes up to `steps_per_warp` steps over the heads of one kind (q, k or v) of one token, 256 / D heads in a step; what
// the token's heads share (angles, weights) stays in registers.
template <int D, bool BF16, bool STORE>
__global__ void __launch_bounds__(256, 4) tokens_kernel(const Tokens a) {
    constexpr int UNITS = D / 8, HEADS = 32 / UNITS;   // threads of a head, heads of a warp
    const int lane = threadIdx.x & 31, unit = lane % UNITS, sub = lane / UNITS;
    const uint32_t warp = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int token = warp / a.parts;
    int part = warp - token * a.parts;
    wait_for_front();
    if (token >= a.tokens) return;
    const int kind = part < a.parts_q ? 0 : !STORE || part < a.parts_q + a.parts_k ? 1 : 2;
    part -= kind == 0 ? 0 : kind == 1 ? a.parts_q : a.parts_q + a.parts_k;
    const int heads = kind == 0 ? a.q_heads : a.kv_heads;
    const int first = part * a.steps_per_warp * HEADS + sub, past = min(heads, (part + 1) * a.steps_per_warp * HEADS);

    const char *src = a.x[kind] + token * a.token_stride[kind] + unit * 16;
    const int64_t src_stride = a.head_stride[kind];
    char *out = kind < 2 ? a.out[kind] : nullptr;
    if (out) out += ((int64_t)token * heads * D + unit * 8) * 2;

    auto load = [&](int head) { return head < past ? *reinterpret_cast<const uint4 *>(src + head * src_stride) : make_uint4(0, 0, 0, 0); };
    constexpr int AHEAD = 2;     // loads in flight
    uint4 raw[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) raw[i] = load(first + i * HEADS);

    int64_t slot = -1;
    uint8_t *slab0 = nullptr;    // of head 0
    int in_slab = 0;
    int64_t slab_stride = 0;
    if (STORE && kind > 0) {
        slot = index_at(a.slots, a.wide_slots, token);
        if (slot >= a.num_slots) slot = -1;   // (not in the cache: not stored)
        if (slot >= 0) {
            const int64_t page = slot / a.page_size;
            const int in_page = (int)(slot - page * a.page_size), slabs = a.page_size / KV_SLAB;
            slab_stride = slabs * (int64_t)kv_slab_bytes(D);
            slab0 = a.cache + page * a.kv_heads * slab_stride + in_page / KV_SLAB * (int64_t)kv_slab_bytes(D);
            in_slab = in_page % KV_SLAB;
        }
    }

    const int half_units = a.rotary / 16;
    const bool turned = kind < 2 && a.table && unit * 8 < a.rotary;
    const bool halves = kind < 2 && a.table && !a.interleaved;
    const int mate = !turned || a.interleaved ? unit : unit < half_units ? unit + half_units : unit - half_units;
    float cs[8], sn[8];          // of the own channels; the sine with the sign that it has there
    if (turned) {
        const int64_t at = index_at(a.positions, a.wide_positions, token);
        const bool known = at >= 0 && at < a.table_rows;   // (elsewhere there is no angle: what it would turn becomes NaN)
        const float *row = a.table + (known ? at : 0) * a.rotary;
        if (a.interleaved) {
            const float4 c = *reinterpret_cast<const float4 *>(row + unit * 4), n = *reinterpret_cast<const float4 *>(row + a.rotary / 2 + unit * 4);
            cs[0] = cs[1] = c.x, cs[2] = cs[3] = c.y, cs[4] = cs[5] = c.z, cs[6] = cs[7] = c.w;
            sn[1] = n.x, sn[3] = n.y, sn[5] = n.z, sn[7] = n.w;
#pragma unroll
            for (int i = 0; i < 8; i += 2) sn[i] = -sn[i + 1];
        } else {
            const float *c = row + (unit % half_units) * 8, *n = c + a.rotary / 2;
            const float4 c0 = *reinterpret_cast<const float4 *>(c), c1 = *reinterpret_cast<const float4 *>(c + 4);
            const float4 n0 = *reinterpret_cast<const float4 *>(n), n1 = *reinterpret_cast<const float4 *>(n + 4);
            cs[0] = c0.x, cs[1] = c0.y, cs[2] = c0.z, cs[3] = c0.w, cs[4] = c1.x, cs[5] = c1.y, cs[6] = c1.z, cs[7] = c1.w;
            sn[0] = n0.x, sn[1] = n0.y, sn[2] = n0.z, sn[3] = n0.w, sn[4] = n1.x, sn[5] = n1.y, sn[6] = n1.z, sn[7] = n1.w;
            if (unit < half_units) {
#pragma unroll
                for (int i = 0; i < 8; ++i) sn[i] = -sn[i];
            }
        }
        if (!known) {
#pragma unroll
            for (int i = 0; i < 8; ++i) cs[i] = __int_as_float(0x7fc00000);
        }
    }
    const char *weight = kind < 2 ? a.weight[kind] : nullptr;
    if (weight) {                // weights go with the angles: (x norm) (w cos) + (y norm) (w' sin)
        float w[8], wm[8];       // of the own channels and of those that they turn with
        load_weight<BF16>(weight, a.wide_weights, unit * 8, w);
        load_weight<BF16>(weight, a.wide_weights, mate * 8, wm);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float own = __fadd_rn(w[i], a.offset), other = __fadd_rn(a.interleaved ? w[i ^ 1] : wm[i], a.offset);
            cs[i] = turned ? cs[i] * own : own;
            sn[i] = sn[i] * other;
        }
    }

    auto work = [&](int head, const uint4 &raw) {
        const bool live = head < past;
        float x[8];
        unpack8<BF16>(raw, x);
        if (weight) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
#pragma unroll
            for (int k = 1; k < UNITS; k *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, k);
            const float norm = rsqrtf(sum * (1.0f / D) + a.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= norm;
        }
        if (halves) {            // the numbers that these turn with, of the same head
            float y[8];
            const int from = sub * UNITS + mate;
            if (weight) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], from);
            } else {
                uint4 other;
                other.x = __shfl_sync(0xffffffffu, raw.x, from), other.y = __shfl_sync(0xffffffffu, raw.y, from);
                other.z = __shfl_sync(0xffffffffu, raw.z, from), other.w = __shfl_sync(0xffffffffu, raw.w, from);
                unpack8<BF16>(other, y);
            }
            if (turned) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = __fadd_rn(__fmul_rn(x[i], cs[i]), __fmul_rn(y[i], sn[i]));
            } else if (weight) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] *= cs[i];
            }
        } else if (turned) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float e = x[i], o = x[i + 1];
                x[i] = __fadd_rn(__fmul_rn(e, cs[i]), __fmul_rn(o, sn[i]));
                x[i + 1] = __fadd_rn(__fmul_rn(o, cs[i + 1]), __fmul_rn(e, sn[i + 1]));
            }
        } else if (weight) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= cs[i];
        }
        if (out && live) *reinterpret_cast<uint4 *>(out + (int64_t)head * (D * 2)) = pack8<BF16>(x);
        if (STORE && kind > 0) {
            int code[8], zero;
            float scale;
            quantise8(x, code, scale, zero);
            if (live && slot >= 0) {
                uint8_t *slab = slab0 + head * slab_stride;
                if (kind == 1) store_key<D>(slab, in_slab, unit, code, scale, zero);
                else store_value<D>(slab, in_slab, unit, code, scale, zero);
            }
        }
    };
    for (int head = first; head - sub < past; head += AHEAD * HEADS) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (head - sub + i * HEADS >= past) break;
            const uint4 now = raw[i];
            raw[i] = load(head + (i + AHEAD) * HEADS);
            work(head + i * HEADS, now);
        }
    }
}

// Stored keys and values as fp16 (exact) or bf16; zeros for slots that are not in the cache.  A thread makes 8 channels of both.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) load_kernel(const void *cache_bytes, const void *slots, bool wide_slots, int64_t tokens, int64_t num_slots,
                                                   int kv_heads, int page_size, void *k_to, void *v_to) {
    constexpr int UNITS = D / 8;
    const uint8_t *cache = (const uint8_t *)cache_bytes;
    char *k_out = (char *)k_to, *v_out = (char *)v_to;
    wait_for_front();
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t row = i / UNITS;
    const int unit = (int)(i % UNITS);
    if (row >= tokens * kv_heads) return;
    const int64_t token = row / kv_heads;
    const int head = (int)(row - token * kv_heads);
    const int64_t slot = index_at(slots, wide_slots, token);
    float k[8] = {}, v[8] = {};
    if (slot >= 0 && slot < num_slots) {
        const int64_t page = slot / page_size;
        const int in_page = (int)(slot - page * page_size), tok = in_page % KV_SLAB;
        const uint8_t *slab = cache + ((page * kv_heads + head) * (page_size / KV_SLAB) + in_page / KV_SLAB) * (int64_t)kv_slab_bytes(D);
        const uint32_t w = *reinterpret_cast<const uint32_t *>(slab + kv_key_word(D, tok, unit));
        const __half2 kp = *reinterpret_cast<const __half2 *>(slab + kv_key_params(D) + (tok * (D / 64) + unit / 8) * 4);
        const float ks = __low2float(kp), kz = __high2float(kp) - 1024.0f;
        const uint8_t *codes = slab + kv_value_codes(D);
        const uint32_t u = *reinterpret_cast<const uint16_t *>(codes + kv_value_unit(D, tok, 2 * unit)) |
                           (uint32_t)*reinterpret_cast<const uint16_t *>(codes + kv_value_unit(D, tok, 2 * unit + 1)) << 16;
        const __half *vp = reinterpret_cast<const __half *>(slab + kv_value_params(D) + (tok / 2 * (D / 64) + unit / 8) * 8) + (tok & 1);
        const float vs = __half2float(vp[0]), vz = __half2float(vp[2]) - 1024.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            k[c] = ks * ((float)((w >> (4 * ((c & 1) * 4 + c / 2))) & 15u) - kz);
            v[c] = vs * ((float)((u >> (4 * c)) & 15u) - vz);
        }
    }
    *reinterpret_cast<uint4 *>(k_out + (row * D + unit * 8) * 2) = pack8<BF16>(k);
    *reinterpret_cast<uint4 *>(v_out + (row * D + unit * 8) * 2) = pack8<BF16>(v);
}

template <typename F>
int by_type(int head_dim, int dtype, F &&f) {
#define ATLAS_KV_CASE(D) \
    case D: return dtype == ATLAS_DTYPE_BF16 ? f(std::integral_constant<int, D>(), std::true_type()) : f(std::integral_constant<int, D>(), std::false_type());
    switch (head_dim) {
        ATLAS_KV_CASE(64)
        ATLAS_KV_CASE(128)
        ATLAS_KV_CASE(256)
    }
#undef ATLAS_KV_CASE
    return ATLAS_ERR_UNSUPPORTED;
}

bool aligned16(const void *p, int64_t a, int64_t b) { return !((reinterpret_cast<uintptr_t>(p) | (uintptr_t)a | (uintptr_t)b) & 15); }

}  // namespace
}  // namespace atlas

extern "C" {

size_t atlas_kv_page_bytes(int head_dim, int page_size) {
    return (head_dim == 64 || head_dim == 128 || head_dim == 256) && page_size >= atlas::KV_SLAB && page_size % atlas::KV_SLAB == 0
               ? (size_t)(page_size / atlas::KV_SLAB) * atlas::kv_slab_bytes(head_dim) : 0;
}

int atlas_norm_rotate(const AtlasTokens *p, void *stream) {
    using namespace atlas;
    clear_error();
    const char *what = "atlas_norm_rotate";
    ATLAS_RETURN_IF(!p, ATLAS_ERR_BAD_ARGUMENT, "%s: no arguments", what);
    const bool store = p->cache != nullptr;
    const int shape = check_kv_shape(store ? p->num_pages : 0, p->kv_heads, p->head_dim, store ? p->page_size : KV_SLAB, what);
    if (shape != ATLAS_OK) return shape;
    ATLAS_RETURN_IF(p->dtype != ATLAS_DTYPE_F16 && p->dtype != ATLAS_DTYPE_BF16, ATLAS_ERR_BAD_ARGUMENT, "%s: dtype %d", what, p->dtype);
    ATLAS_RETURN_IF(p->tokens < 0 || p->q_heads < 0 || p->q_heads > 65535, ATLAS_ERR_BAD_ARGUMENT, "%s: %lld tokens of %d heads", what,
                    (long long)p->tokens, p->q_heads);
    if (p->tokens == 0) return ATLAS_OK;
    ATLAS_RETURN_IF((p->q_heads && (!p->q || !p->q_out)) || !p->k || (store ? !p->v || !p->slots : !p->k_out), ATLAS_ERR_BAD_ARGUMENT, "%s: null pointer", what);
    ATLAS_RETURN_IF(p->table && (!p->positions || p->table_rows < 1), ATLAS_ERR_BAD_ARGUMENT, "%s: a table needs rows and positions", what);
    ATLAS_RETURN_IF(p->table && (p->rotary_dim < 16 || p->rotary_dim % 16 || p->rotary_dim > p->head_dim), ATLAS_ERR_UNSUPPORTED,
                    "%s: rotary_dim %d is not a multiple of 16 up to head_dim", what, p->rotary_dim);
    ATLAS_RETURN_IF(p->table && p->position_bytes != 4 && p->position_bytes != 8, ATLAS_ERR_BAD_ARGUMENT, "%s: positions of %d bytes", what, p->position_bytes);
    ATLAS_RETURN_IF(store && p->slot_bytes != 4 && p->slot_bytes != 8, ATLAS_ERR_BAD_ARGUMENT, "%s: slots of %d bytes", what, p->slot_bytes);
    const bool q_fits = !p->q_heads || (aligned16(p->q, 2 * p->q_token_stride, 2 * p->q_head_stride) && aligned16(p->q_out, 0, 0));
    const bool v_fits = !store || (aligned16(p->v, 2 * p->v_token_stride, 2 * p->v_head_stride) && aligned16(p->cache, 0, 0));
    ATLAS_RETURN_IF(!q_fits || !v_fits || !aligned16(p->k, 2 * p->k_token_stride, 2 * p->k_head_stride) || !aligned16(p->k_out, 0, 0) ||
                        !aligned16(p->q_weight, 0, 0) || !aligned16(p->k_weight, 0, 0) || !aligned16(p->table, 0, 0),
                    ATLAS_ERR_BAD_ARGUMENT, "%s: pointers and strides must be multiples of 16 bytes", what);
    const int dev = check_device();
    if (dev != ATLAS_OK) return dev;

    Tokens a = {};
    a.x[0] = (const char *)p->q, a.x[1] = (const char *)p->k, a.x[2] = (const char *)p->v;
    const int64_t ts[3] = {p->q_token_stride, p->k_token_stride, p->v_token_stride}, hs[3] = {p->q_head_stride, p->k_head_stride, p->v_head_stride};
    for (int i = 0; i < 3; ++i) a.token_stride[i] = 2 * ts[i], a.head_stride[i] = 2 * hs[i];
    a.out[0] = (char *)p->q_out, a.out[1] = (char *)p->k_out;
    a.table = p->table, a.positions = p->positions, a.slots = p->slots;
    a.weight[0] = (const char *)p->q_weight, a.weight[1] = (const char *)p->k_weight;
    a.cache = (uint8_t *)p->cache;
    a.tokens = p->tokens, a.table_rows = p->table_rows, a.num_slots = store ? p->num_pages * p->page_size : 0;
    a.q_heads = p->q_heads, a.kv_heads = p->kv_heads, a.rotary = p->rotary_dim, a.page_size = store ? p->page_size : KV_SLAB;
    a.eps = p->eps, a.offset = p->weight_offset;
    a.wide_positions = p->position_bytes == 8, a.wide_slots = p->slot_bytes == 8, a.wide_weights = p->weights_f32 != 0;
    a.interleaved = p->interleaved != 0;
    // Few tokens: a step a warp, so that all loads are under way at once.  Many: up to 8 steps, which share angles and weights,
    // as long as there are 16 warps an SM (4001 tokens of 72 heads of 128: 1 step 94 us, 4 41, 8 37, 16 37).
    const int64_t at_a_time = 256 / p->head_dim, q_steps = ceil_div_i64(p->q_heads, at_a_time), kv_steps = ceil_div_i64(p->kv_heads, at_a_time);
    a.steps_per_warp = (int)std::min<int64_t>(8, std::max<int64_t>(1, p->tokens * (q_steps + (store ? 2 : 1) * kv_steps) / (148 * 16)));
    a.parts_q = (int)ceil_div_i64(q_steps, a.steps_per_warp), a.parts_k = (int)ceil_div_i64(kv_steps, a.steps_per_warp);
    a.parts = a.parts_q + (store ? 2 : 1) * a.parts_k;
    const int64_t blocks = ceil_div_i64(p->tokens * a.parts, 8);
    ATLAS_RETURN_IF(blocks > (1 << 28), ATLAS_ERR_UNSUPPORTED, "%s: %lld tokens", what, (long long)p->tokens);
    return by_type(p->head_dim, p->dtype, [&](auto d, auto bf16) {
        constexpr int D = decltype(d)::value;
        constexpr bool B = decltype(bf16)::value;
        return launch_early(store ? tokens_kernel<D, B, true> : tokens_kernel<D, B, false>, dim3((unsigned)blocks), 256, 0, (cudaStream_t)stream, what, a);
    });
}

int atlas_kv_load(const void *cache, int64_t num_pages, int kv_heads, int head_dim, int page_size, const void *slots, int slot_bytes,
                  int64_t tokens, int dtype, void *k_out, void *v_out, void *stream) {
    using namespace atlas;
    clear_error();
    const char *what = "atlas_kv_load";
    const int shape = check_kv_shape(num_pages, kv_heads, head_dim, page_size, what);
    if (shape != ATLAS_OK) return shape;
    ATLAS_RETURN_IF(dtype != ATLAS_DTYPE_F16 && dtype != ATLAS_DTYPE_BF16, ATLAS_ERR_BAD_ARGUMENT, "%s: dtype %d", what, dtype);
    ATLAS_RETURN_IF(tokens < 0 || (slot_bytes != 4 && slot_bytes != 8), ATLAS_ERR_BAD_ARGUMENT, "%s: %lld tokens, slots of %d bytes", what,
                    (long long)tokens, slot_bytes);
    if (tokens == 0) return ATLAS_OK;
    ATLAS_RETURN_IF((num_pages && !cache) || !slots || !k_out || !v_out, ATLAS_ERR_BAD_ARGUMENT, "%s: null pointer", what);
    ATLAS_RETURN_IF(!aligned16(cache, 0, 0) || !aligned16(k_out, 0, 0) || !aligned16(v_out, 0, 0), ATLAS_ERR_BAD_ARGUMENT,
                    "%s: pointers must be multiples of 16 bytes", what);
    const int dev = check_device();
    if (dev != ATLAS_OK) return dev;
    const int64_t blocks = ceil_div_i64(tokens * kv_heads * (head_dim / 8), 256);
    ATLAS_RETURN_IF(blocks > 0x7fffffff, ATLAS_ERR_UNSUPPORTED, "%s: %lld tokens", what, (long long)tokens);
    return by_type(head_dim, dtype, [&](auto d, auto bf16) {
        return launch_early(load_kernel<decltype(d)::value, decltype(bf16)::value>, dim3((unsigned)blocks), 256, 0, (cudaStream_t)stream, what, cache, slots, slot_bytes == 8,
                            tokens, num_pages * page_size, kv_heads, page_size, k_out, v_out);
    });
}

}  // extern "C"
