// What the kernels of attention over the 4-bit cache share.
#pragma once
#include "kv_cache.cuh"
#include "tensor_core.cuh"

namespace atlas {

struct Attention {
    const char *q;               // bytes
    int64_t q_token_stride, q_head_stride;
    char *out;
    const uint8_t *cache;
    const int32_t *page_table, *lengths, *query_starts;
    float *partial;
    int32_t *status;
    int64_t num_pages, table_stride, max_tokens, total_queries, uniform;
    int batch, q_heads, kv_heads, group, page_size, window, sinks, max_queries;   // group: query heads of a kv head
    float scale_log2;
    bool few_runs;               // no more sequences times kv heads than CTAs
};

// Prompts: kv_prompt.cu.  Bytes of workspace, and the launch.
bool kv_prompt_serves(const AtlasKvAttention &p);
int64_t kv_prompt_blocks(const AtlasKvAttention &p);   // row blocks of a sequence: the grid's second dimension
size_t kv_prompt_workspace_bytes(const AtlasKvAttention &p);
int kv_prompt(const Attention &a, const AtlasKvAttention &p, cudaStream_t stream);

// Dynamic shared memory above the default, set once for each device.
template <auto Kernel>
int allow_smem(int bytes, const char *what) {
    static thread_local int known = -1;
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && dev == known) return ATLAS_OK;
    const int e = check_cuda(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), what);
    if (e == ATLAS_OK) known = dev;
    return e;
}

namespace {

struct Sequence {
    int first_query;             // in q
    int length, queries;
    __device__ __forceinline__ int start() const { return length - queries; }   // position of the first query (negative if there are fewer tokens than queries)
    __device__ __forceinline__ int served(const Attention &a) const { return min(queries, a.max_queries); }
};
__device__ __forceinline__ Sequence sequence(const Attention &a, int b) {
    Sequence r;
    int64_t q0, q1;
    if (a.query_starts) {
        q0 = min(max((int64_t)a.query_starts[b], (int64_t)0), a.total_queries);
        q1 = min(max((int64_t)a.query_starts[b + 1], q0), a.total_queries);
    } else {
        q0 = b * a.uniform, q1 = q0 + a.uniform;
    }
    r.first_query = (int)q0;
    r.queries = (int)(q1 - q0);
    r.length = (int)min(max((int64_t)a.lengths[b], (int64_t)0), a.max_tokens);
    return r;
}
// Rows of q next to a sequence that are no sequence's, or beyond max_queries: in front of the first, and behind those served.
__device__ __forceinline__ int rows_in_front(const Sequence &r, int b) { return b == 0 ? r.first_query : 0; }
__device__ __forceinline__ int rows_behind(const Attention &a, const Sequence &r, int b) {
    return (b + 1 == a.batch ? (int)a.total_queries - r.first_query : r.queries) - r.served(a);
}
// Their outputs are zeros, by `threads` threads of which this one is `thread`.
__device__ __forceinline__ void zero_rows(const Attention &a, int first, int count, int d, int64_t thread, int64_t threads) {
    const int64_t pieces = (int64_t)a.q_heads * d / 8;
    uint4 *out = reinterpret_cast<uint4 *>(a.out) + first * pieces;
    for (int64_t i = thread; i < count * pieces; i += threads) out[i] = make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ void zero_rows_next_to(const Attention &a, const Sequence &r, int b, int d, int64_t thread, int64_t threads) {
    zero_rows(a, 0, rows_in_front(r, b), d, thread, threads);
    zero_rows(a, r.first_query + r.served(a), rows_behind(a, r, b), d, thread, threads);
}
// Where a row's output is, or null.
__device__ __forceinline__ char *out_row(const Attention &a, const Sequence &r, int h, int row, int d) {
    const int query = row / a.group;
    if (query >= r.served(a)) return nullptr;
    return a.out + ((int64_t)(r.first_query + query) * a.q_heads + h * a.group + row - query * a.group) * d * 2;
}

constexpr float KV_HEADROOM = 8.0f;   // log2: how far a score may pass the running maximum before sums are rescaled
constexpr float KV_SHIFT = 6.0f;      // log2: p is kept as 2^6 p, up to 2^14 in fp16; what is below 2^-31 of the maximum vanishes

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t h2(__half2 v) { return *reinterpret_cast<uint32_t *>(&v); }
__device__ __forceinline__ __half2 h2(uint32_t v) { return *reinterpret_cast<__half2 *>(&v); }

// The four pairs of a word of codes, minus the zero point: `bias` is 1024 + z, `minus16` is -(64 + z) = 960 - bias.  (Small integers
// become fp16 by the bits of 1024 in front of them, where a unit in the last place is 1: Kim et al. 2022, "Who Says Elephants Can't
// Run".)
__device__ __forceinline__ uint32_t masked_or(uint32_t w, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
    return r;
}
__device__ __forceinline__ __half2 minus16_of(__half2 bias) { return __hsub2(__float2half2_rn(960.0f), bias); }
__device__ __forceinline__ void open_word(uint32_t w, __half2 bias, __half2 minus16, __half2 (&v)[4]) {
    const __half2 sixteenth = __float2half2_rn(0.0625f);
    const uint32_t u = w >> 8;
    v[0] = __hsub2(h2(masked_or(w, 0x000f000fu, 0x64006400u)), bias);
    v[1] = __hfma2(h2(masked_or(w, 0x00f000f0u, 0x64006400u)), sixteenth, minus16);   // (1024 + 16 c) / 16 - (64 + z)
    v[2] = __hsub2(h2(masked_or(u, 0x000f000fu, 0x64006400u)), bias);
    v[3] = __hfma2(h2(masked_or(u, 0x00f000f0u, 0x64006400u)), sixteenth, minus16);
}

template <bool BF16>
__device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) {
    if (BF16) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
        return make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
    }
    const __half2 x = __floats2half2_rn(a, b), y = __floats2half2_rn(c, d);
    return make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
}

}  // namespace
}  // namespace atlas
